"""Products with weights held in 4 bits, as they are measured: packing a matrix, the product that reads it, and a routed
feed-forward whose experts' matrices are packed.

A matrix [N, K] is held in codes of 4 bits and one scale for every `group` neighbours along K. A code is a sign and one of
the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale is a number of six significant bits, so scale * code is a bfloat16
number as it stands. For a group with largest magnitude a

    scale = a / 6, rounded to six significant bits (ties to the even one);   0 for a group of zeros
    code  = the magnitude nearest to |w| / scale, ties to the one with the even code, 6 beyond 6; the sign of w

  pack     the codes and scales of a matrix, and the values they stand for
  product  out = x W^T + bias, or gated: out[:, i] = act(x W^T[:, 2 i], x W^T[:, 2 i + 1])
  experts  out[r] = sum over the row's choices (e, share) of share * Wd_e act(Wg_e x[r], Wu_e x[r])

with act(g, u) = g * sigmoid(g) * u, or bounded: g' = min(g, 7), u' = clamp(u, -7, 7), g' * sigmoid(1.702 g') * (u' + 1).
The rows are bfloat16, the sums 32-bit."""
import math

import torch

own = False
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
DEVICE = "cuda"
BOUNDED = dict(alpha=1.702, limit=7.0, shift=1.0)
SILU = dict(alpha=1.0, limit=0.0, shift=0.0)


def listed():
    return [
        # one small 32-bit matrix while a model is loaded, and the largest of a 7B model's layer
        dict(name="pack_small", op="pack", n=512, k=896, group=32, dtype="f32"),
        dict(name="pack_gate_up_7b", op="pack", n=37888, k=3584, group=128, dtype="bf16"),
        # one user of a 7B model: q||k||v with its bias, and the long sums of the down projection
        dict(name="row1_qkv_7b", op="product", rows=1, n=4608, k=3584, group=128, out="bf16", bias=True, act=""),
        dict(name="row1_down_7b", op="product", rows=1, n=3584, k=18944, group=128, out="bf16", bias=False, act=""),
        # eight users (the benchmark's batch) and a full server at the gated product, most of a step's weights
        dict(name="rows8_gate_up_7b", op="product", rows=8, n=37888, k=3584, group=128, out="bf16", bias=False, act="silu"),
        dict(name="rows64_gate_up_7b", op="product", rows=64, n=37888, k=3584, group=64, out="bf16", bias=False, act="silu"),
        # a matrix of odd sizes, for 32-bit results
        dict(name="rows17_odd", op="product", rows=17, n=1001, k=1003, group=32, out="f32", bias=True, act=""),
        # a conversation's next turn, and a prompt of the benchmark's length
        dict(name="rows203_qkv_7b", op="product", rows=203, n=4608, k=3584, group=128, out="bf16", bias=True, act=""),
        dict(name="rows2048_gate_up_7b", op="product", rows=2048, n=37888, k=3584, group=128, out="bf16", bias=False, act="silu"),
        # routed feed-forwards of the width-2048 designs: one user, a full server (some experts with few or no rows), a prompt
        dict(name="experts_row1", op="experts", rows=1, experts=16, top=4, inter=2048, hidden=2048, group=128, act="silu", skew=0.0),
        dict(name="experts_rows64", op="experts", rows=64, experts=16, top=4, inter=2048, hidden=2048, group=32, act="bounded", skew=2.0),
        dict(name="experts_rows2048", op="experts", rows=2048, experts=16, top=4, inter=2048, hidden=2048, group=128, act="silu", skew=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pack", "product", "product", "product", "experts", "experts"])
    group = rng.choice([32, 64, 128, 128])
    if op == "pack":
        n, k = _log(rng, 16, 37888), _log(rng, 64, 18944)
        return dict(op=op, n=min(n, 37888 * 3584 // k), k=k, group=group, dtype=rng.choice(["f32", "bf16", "bf16"]))
    if op == "product":
        rows, k = _log(rng, 1, 2048), _log(rng, 64, 18944)
        if rng.random() < 0.8:
            k = -(-k // 8) * 8
        n = min(_log(rng, 64, 37888), 37888 * 3584 // k)
        act = rng.choice(["", "", "silu", "bounded"])
        if act:
            n += n % 2
        return dict(op=op, rows=rows, n=n, k=k, group=group, out=rng.choice(["bf16", "bf16", "f32"]) if not act else "bf16",
                    bias=not act and rng.random() < 0.5, act=act)
    experts = rng.choice([2, 4, 7, 8, 16, 16, 32])
    inter, hidden = 8 * _log(rng, 16, 512), 8 * _log(rng, 32, 448)
    inter = min(inter, 16 * 2048 * 2048 // (experts * hidden) // 8 * 8)
    return dict(op=op, rows=_log(rng, 1, 2048), experts=experts, top=rng.randint(1, max(1, min(4, experts // 2))), inter=inter,
                hidden=hidden, group=group, act=rng.choice(["silu", "bounded"]), skew=rng.choice([0.0, 0.0, 1.0, 2.0]))


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _matrix(gen, shape, dtype=BF16):
    """Weights of std 0.02, some columns larger, as a trained matrix has them."""
    w = torch.randn(shape, generator=gen, device=DEVICE) * 0.02
    w *= 1 + 3 * (torch.rand(shape[-1], generator=gen, device=DEVICE) < 0.01)
    return w.to(dtype)


def _rows(gen, rows, k):
    """Normed activations: of unit size, a few channels far larger."""
    x = torch.randn((rows, k), generator=gen, device=DEVICE)
    return (x * (1 + 15 * (torch.rand(k, generator=gen, device=DEVICE) < 0.005))).to(BF16)


def _choices(gen, case):
    """A router's choices: logits with an offset an expert, the best `top` of them, their softmax."""
    E, rows = case["experts"], case["rows"]
    z = torch.randn((rows, E), generator=gen, device=DEVICE) + case["skew"] * torch.randn(E, generator=gen, device=DEVICE)
    best = torch.topk(z, case["top"], dim=1)
    return best.indices.to(torch.int32).contiguous(), torch.softmax(best.values, 1).contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    if case["op"] == "pack":
        return dict(w=_matrix(gen, (case["n"], case["k"]), F32 if case["dtype"] == "f32" else BF16))
    if case["op"] == "product":
        return dict(w=_matrix(gen, (case["n"], case["k"])), x=_rows(gen, case["rows"], case["k"]),
                    bias=(torch.randn(case["n"], generator=gen, device=DEVICE) * 0.1).to(BF16) if case["bias"] else None)
    E, I, D = case["experts"], case["inter"], case["hidden"]
    ids, shares = _choices(gen, case)
    # gate i of an expert in row 2 i, its up in 2 i + 1
    return dict(gate_up=_matrix(gen, (E, 2 * I, D)), down=_matrix(gen, (E, D, I)), x=_rows(gen, case["rows"], D), ids=ids,
                shares=shares)


def prepare(case, seed):
    """What a serving program holds: its matrices packed, once, and rows to multiply them with."""
    data = _inputs(case, seed)
    state = dict(data, case=case)
    if case["op"] == "pack":
        return state
    matrices = ["w"] if case["op"] == "product" else ["gate_up", "down"]
    if not own:
        for m in matrices:
            state[m] = _quantize(data[m], case["group"])
        return state
    from hector_engine_amd.kernels import fp4, ops
    for m in matrices:
        state[m] = fp4.pack(data[m], case["group"])
    if case["op"] == "product":
        state["out"] = torch.empty((case["rows"], case["n"] // 2 if case["act"] else case["n"]), device=DEVICE,
                                   dtype=F32 if case["out"] == "f32" else BF16)
        size = ops.fp4_product_workspace_bytes(case["rows"], state["w"], gated=bool(case["act"]))
    else:
        state["out"] = torch.empty((case["rows"], case["hidden"]), device=DEVICE, dtype=BF16)
        size = ops.fp4_experts_workspace_bytes(case["rows"], case["top"], state["gate_up"], state["down"])
    state["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)
    return state


# ---- the operators -----------------------------------------------------------------------------------------------------------

def _quantize(w, group):
    """(codes uint8 [..., K], scales fp32 [..., ceil(K / group)]) of a matrix."""
    k = w.shape[-1]
    groups = -(-k // group)
    f = torch.nn.functional.pad(w.float(), (0, groups * group - k)).view(*w.shape[:-1], groups, group)
    size = f.abs()
    # (in 64 bits: a sixth that is off in its last bit falls on the wrong side of a border)
    bits = (size.amax(-1).double() / 6).float().view(torch.int32)
    # six significant bits: the leading one and five of the 23 below it
    scale = ((bits + 0x1ffff + ((bits >> 18) & 1)) & ~0x3ffff).view(F32)
    s = scale.unsqueeze(-1)
    # (a border times a scale is exact; ties go to the even code)
    code = torch.zeros_like(size, dtype=torch.uint8)
    for border, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (size >= border * s) if tie_up else (size > border * s)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    code += 8 * ((f < 0) & (code > 0)).to(torch.uint8)
    return code.view(*w.shape[:-1], groups * group)[..., :k], scale


def _values(codes, scales, group):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return table[codes.int()] * scales.repeat_interleave(group, -1)[..., :codes.shape[-1]]


def _act(z, kind):
    g, u = z[..., 0::2], z[..., 1::2]
    if kind == "silu":
        return g * torch.sigmoid(g) * u
    g, u = g.clamp(max=BOUNDED["limit"]), u.clamp(-BOUNDED["limit"], BOUNDED["limit"])
    return g * torch.sigmoid(BOUNDED["alpha"] * g) * (u + BOUNDED["shift"])


def _own(state):
    from hector_engine_amd.kernels import fp4, ops
    case = state["case"]
    if case["op"] == "pack":
        return fp4.pack(state["w"], case["group"]).unpack()
    act = BOUNDED if case["act"] == "bounded" else SILU
    consts = (act["alpha"], act["limit"], act["shift"])
    if case["op"] == "product":
        ops.fp4_product(state["out"], state["x"], state["w"], state["bias"], case["rows"], gated=bool(case["act"]), act=consts,
                        workspace=state["workspace"])
    else:
        ops.fp4_experts(state["out"], state["x"], state["gate_up"], state["down"], state["ids"], state["shares"], case["rows"],
                        act=consts, workspace=state["workspace"])
    return state["out"]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "pack":
        return _values(*_quantize(state["w"], case["group"]), case["group"]).to(BF16)
    x = state["x"].float()
    if case["op"] == "product":
        y = x @ _values(*state["w"], case["group"]).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if case["act"]:
            y = _act(y, case["act"])
        return y if case["out"] == "f32" else y.to(BF16)
    out = torch.zeros((case["rows"], case["hidden"]), device=x.device)
    for e in range(case["experts"]):
        share = (state["shares"] * (state["ids"] == e)).sum(1, keepdim=True)
        codes, scales = state["gate_up"]
        h = _act(x @ _values(codes[e], scales[e], case["group"]).t(), case["act"])
        codes, scales = state["down"]
        out += share * (h @ _values(codes[e], scales[e], case["group"]).t())
    return out.to(BF16)


# ---- from the definition, in 64 bits --------------------------------------------------------------------------------------------

def _values64(w, group):
    """The values a packed matrix stands for."""
    parts = []
    for rows in w.reshape(-1, w.shape[-1]).split(4096):
        cols = []
        for part in rows.double().split(group, dim=1):
            most = part.abs().amax(1, keepdim=True)
            m, e = torch.frexp(most / torch.full_like(most, 6))      # (a quotient by a plain number may be a product)
            scale = torch.round(m * 64) / 64 * ((e.long() + 1023) << 52).view(F64)      # times 2^e, exactly
            q = part.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
            step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0)).double()
            cols.append(torch.sign(part) * torch.clamp(torch.round(q / step) * step, max=6) * scale)
        parts.append(torch.cat(cols, 1))
    return torch.cat(parts).view(w.shape)


def _act64(z, kind):
    gate, up = z.unflatten(-1, (-1, 2)).unbind(-1)
    if kind == "bounded":
        gate, up = torch.minimum(gate, torch.full_like(gate, 7.0)), torch.clamp(up, -7, 7)
        return gate / (1 + torch.exp(-1.702 * gate)) * (up + 1)
    return gate / (1 + torch.exp(-gate)) * up


def exact(case, seed):
    data = _inputs(case, seed)
    if case["op"] == "pack":
        return _values64(data["w"], case["group"])
    x = data["x"].double()
    if case["op"] == "product":
        y = torch.mm(x, _values64(data["w"], case["group"]).t().contiguous())
        if data["bias"] is not None:
            y += data["bias"].double()
        return _act64(y, case["act"]) if case["act"] else y
    out = torch.zeros((case["rows"], case["hidden"]), dtype=F64, device=DEVICE)
    for e in range(case["experts"]):
        up = _values64(data["gate_up"][e], case["group"]).t().contiguous()
        down = _values64(data["down"][e], case["group"]).t().contiguous()
        share = torch.where(data["ids"] == e, data["shares"].double(), torch.zeros((), dtype=F64, device=DEVICE)).sum(1, keepdim=True)
        out += share * torch.mm(_act64(torch.mm(x, up), case["act"]), down)
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def _packed_bytes(n, k, group):
    return n * k / 2 + 2 * n * -(-k // group)


def work(case):
    if case["op"] == "pack":
        n, k = case["n"], case["k"]
        # the matrix read; codes and scales written and read again for the values, which are written
        return {"bytes": n * k * (4 if case["dtype"] == "f32" else 2) + 2 * _packed_bytes(n, k, case["group"]) + 2 * n * k, "flops": 8 * n * k}
    rows = case["rows"]
    if case["op"] == "product":
        n, k = case["n"], case["k"]
        outputs = n // 2 if case["act"] else n
        return {"bytes": _packed_bytes(n, k, case["group"]) + 2 * rows * k + (4 if case["out"] == "f32" else 2) * rows * outputs
                + (2 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    E, I, D, top = case["experts"], case["inter"], case["hidden"], case["top"]
    used = E * (1 - (1 - top / E) ** rows)
    return {"bytes": used * (_packed_bytes(2 * I, D, case["group"]) + _packed_bytes(D, I, case["group"])) + 4 * rows * D + 8 * rows * top,
            "flops": 6 * rows * top * I * D}
