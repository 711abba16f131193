"""Parts over weights in 4 bits: what joins their sums, what is packed and what is kept."""
import pytest
import torch

from tests.plain import fp4_plain as P
from tests.test_fp4_engine_gpu import (bobevik_folders, butolorn_folders, dofipel_folders, domorax_folders, penasun_folders,  # noqa: F401
                                       volonex_folders)
from tests.test_fp4_gpu import experts_case, workspace
from tests.test_tile_routes_gpu import bound_part, context

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def routed(E, I, S, D, **more):
    """A routed feed-forward of one choice a row with a shared expert of S columns, packed, whose activations are bfloat16 numbers exactly: a gate is 96, where
    silu(96) = 96 in 32 bits, an up six times one value of x. (part, tensors)."""
    from hector_engine_amd.parts.base import BuildEnv, PartSpec, build_part
    shared = {"feed_forward": PartSpec("gated_mlp", {"hidden_size": D, "intermediate_size": S}), "name": "shared"}
    part = build_part("feed_forward", PartSpec("routed_experts", {
        "hidden_size": D, "intermediate_size": I, "experts": E, "top": 1, "correction": False, "normalize": True, "shared": shared, **more}), "m.",
        BuildEnv(torch.device("cuda:0"), BF16, True))
    gen = torch.Generator().manual_seed(E + I)
    t = {part._router: torch.randn((E, D), generator=gen).to(BF16)}
    t[part._router][:, 0] = 0
    for n, name in [(I, lambda k, e=e: part._name(e, k)) for e in range(E)] + [(S, lambda k: part.shared._names[k])]:
        gate, up = torch.zeros((n, D)), torch.zeros((n, D))
        gate[:, 0] = 6                                     # (a group's largest magnitude of 6 has the scale 1)
        up[torch.arange(n), torch.randint(1, D, (n,), generator=gen)] = 6 * torch.where(torch.rand(n, generator=gen) < 0.5, 1.0, -1.0)
        t[name("gate")], t[name("up")], t[name("down")] = gate.to(BF16), up.to(BF16), (torch.randn((D, n), generator=gen) * 0.1).to(BF16)
    part.bind({k: v.cuda() for k, v in t.items()})
    part.pack_weights(32)
    return part, t


@pytest.mark.parametrize("rows", [1, 2, 16, 40, 300])
def test_a_shared_expert_joins_the_experts_sums_in_32_bits(rows):
    """Nothing is rounded to bfloat16 between the second products and the layer's result: the sums' own bounds and half a step of the result."""
    E, I, S, D = 4, 96, 160, 200
    part, t = routed(E, I, S, D)
    assert part.shared_cols == S
    gen = torch.Generator().manual_seed(rows)
    x = torch.exp2(torch.randint(-8, -4, (rows, D), generator=gen).float()) * torch.where(torch.rand((rows, D), generator=gen) < 0.5, 1.0, -1.5)
    x[:, 0] = 16
    x = x.to(BF16)
    got = part.forward(x.cuda(), context(rows))[:rows].cpu().double()
    choice = (x.double() @ t[part._router].double().T).argmax(-1)

    def feed_forward(name, which):
        h = (x[which].double() @ t[name("gate")].double().T) * (x[which].double() @ t[name("up")].double().T)
        assert torch.equal(h.to(BF16).double(), h)
        down = P.values(t[name("down")], 32)
        return h @ down.T, P.sum_bound(h, down, 32)
    want, bound = feed_forward(lambda k: part.shared._names[k], slice(None))
    for e in range(E):
        own = choice == e
        if own.any():
            y, b = feed_forward(lambda k: part._name(e, k), own)
            want[own], bound[own] = want[own] + y, bound[own] + b
    # (an addition or two of 32 bits are within the sums' bounds, which allow a whole last place of the sum of magnitudes for each of 40 and more)
    assert ((got - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


@pytest.mark.parametrize("rows,E,top,I,D,group,act", [
    (1, 16, 4, 40, 64, 64, (1.0, 0.0, 0.0)), (1, 4, 3, 20, 35, 32, (1.0, 0.0, 0.0)), (5, 8, 3, 24, 72, 32, (1.702, 7.0, 1.0)),
    (20, 3, 3, 136, 127, 128, (1.0, 0.0, 0.0)), (40, 64, 2, 16, 48, 32, (1.0, 0.0, 0.0)), (150, 7, 2, 20, 36, 32, (1.702, 7.0, 1.0)),
    (400, 3, 2, 144, 264, 128, (1.0, 0.0, 0.0))])
def test_experts_with_rows_to_add(rows, E, top, I, D, group, act):
    from hector_engine_amd.kernels import fp4, ops
    gu, dn, x, ids, shares, exact, slack = experts_case(20, rows, E, top, I, D, group, act)
    up, down = fp4.pack(gu.cuda(), group), fp4.pack(dn.cuda(), group)
    plus = torch.randn((rows + 1, D), generator=torch.Generator().manual_seed(3))
    out = torch.full((rows + 1, D), float("nan"), dtype=BF16, device="cuda")
    for identity in (False, True):
        ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, act=act, identity=identity, plus=plus.cuda(),
                        workspace=workspace(ops.fp4_experts_workspace_bytes(rows, top, up, down)))
        got, want = out.cpu().double(), exact + plus[:rows].double()
        own = torch.zeros((rows, 1), dtype=F64)
        if identity:
            own = (shares.double() * (ids >= E)).sum(-1, keepdim=True)
            want = want + own * x.double()
        # an addition is off by half a last place of the sum so far; those of the experts' parts are in their slack
        slack1 = slack + (2 * top + 2) * 2.0 ** -24 * (plus[:rows].double().abs() + own * x.double().abs())
        assert got[rows].isnan().all()
        assert ((got[:rows] - want).abs() <= slack1 + 2.0 ** -8 * (want.abs() + slack1)).all()
        if rows > 1 and not identity:
            assert torch.equal(got[rows - 1], plus[rows - 1].to(BF16).double())      # (a row of no expert)
    with pytest.raises(TypeError, match="plus: expected torch.float32"):
        ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, plus=plus.cuda().to(BF16))
    with pytest.raises(ValueError, match="plus"):
        ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, plus=plus[:, :-1].contiguous().cuda())
    with pytest.raises(ValueError, match="plus"):
        ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, plus=plus)


@pytest.mark.parametrize("tail", [1, 16, 64])
@pytest.mark.parametrize("ordered", [False, True])
def test_the_last_rows_of_a_long_step(tail, ordered):
    """A feed-forward of more than 8192 rows runs them in turns. With stored weights a short last turn is the product and the activation, gate and up rounded between
    them; packed, it is what those rows give by themselves."""
    from hector_engine_amd.kernels import ops
    D, I, rows = 256, 512, 8192 + tail
    part = bound_part("gated_mlp", {"hidden_size": D, "intermediate_size": I}, D ** -0.5)
    part.gate_up.ordered = ordered
    x = torch.randn((rows, D), generator=torch.Generator(device="cuda").manual_seed(tail), device="cuda").to(BF16)
    last, ctx = x[8192:], context(tail)
    got = part.forward(x, context(rows))
    both, h = part.gate_up(last, tail, ctx), torch.empty((tail, I), dtype=BF16, device="cuda")
    ops.silu_mul(h, both, tail, True)
    assert torch.equal(got[8192:rows], part.down(h, tail, ctx)[:tail])
    for lin in (part.gate_up, part.down):
        lin.pack(64)
    assert torch.equal(part.forward(x, context(rows))[8192:rows], part.forward(last, context(tail))[:tail])


def test_the_first_rows_of_a_packed_matrix():
    from hector_engine_amd.kernels import fp4, ops
    w = torch.randn((100, 264), generator=torch.Generator().manual_seed(4)).cuda()
    packed = fp4.pack(w, 32)
    for rows in (16, 48, 96, 100):
        first = packed.first_rows(rows)
        assert first.pointers == packed.pointers and torch.equal(first.unpack(), packed.unpack()[:rows])
        x = torch.randn((5, 264), generator=torch.Generator().manual_seed(5)).to(BF16).cuda()
        whole, own = torch.empty((5, 100), device="cuda"), torch.full((6, rows), 7.0, device="cuda")
        ops.fp4_product(whole, x, packed, None, 5)
        ops.fp4_product(own, x, first, None, 5)
        assert torch.equal(own[:5], whole[:, :rows]) and (own[5] == 7).all()
    for rows in (0, -16, 8, 99, 112):
        with pytest.raises(ValueError, match="whole tiles of 16"):
            packed.first_rows(rows)
    with pytest.raises(ValueError, match="whole tiles of 16"):
        fp4.pack(w[None], 32).first_rows(16)


def linears(model):
    from hector_engine_amd.parts.linear import Linear
    todo = list(model.parts())
    while todo:
        p = todo.pop()
        yield from ((p, name, lin) for name, lin in vars(p).items() if isinstance(lin, Linear))
        todo += p.children()


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_packed_matrices_are_held_once(model_dirs, name):
    """What a packed engine holds of its layers' matrices is q||k||v, o, gate||up and down: q's rows alone are the first of q||k||v, as they are with stored weights."""
    import hector_engine_amd as he
    from hector_engine_amd.kernels import fp4
    eng = he.Engine(model_dirs[name], weights="fp4", weight_group=32, dtype="bfloat16", max_tokens=256, max_slots=2, max_seq_len=64)
    held, sizes = {}, 0
    for part, attr, lin in linears(eng.model):
        if lin.packed:
            for t in (lin.weight.codes, lin.weight.scales):
                held[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            if attr != "q_only":
                codes, scales = fp4.storage_shapes((lin.out_features, lin.in_features), 32)
                sizes += torch.Size(codes).numel() + 2 * torch.Size(scales).numel()
    assert sum(held.values()) == sizes > 0
    before = [lin.weight for _, _, lin in linears(eng.model)]
    eng.model.pack_weights(32)                       # (packed already: nothing changes)
    assert all(a is lin.weight for a, (_, _, lin) in zip(before, linears(eng.model)))


# What each design's layers hold as matrices of products: packed, as they are stored.
ATTENTION, LATENT = {"Attention.qkv", "Attention.q_only", "Attention.o_proj"}, {"LatentAttention.front", "LatentAttention.o_proj"}
GATED, DENSE = {"GatedMLP.gate_up", "GatedMLP.down"}, {"DenseMLP.up", "DenseMLP.down"}
PACKED = {"bobevik": (ATTENTION | GATED | {"DecayMemory.qkvg", "DecayMemory.o_proj"}, set()),
          "butolorn": (ATTENTION | DENSE | {"GatedTokenInput.gate", "GatedTokenInput.proj", "MatrixMemory.qkvg", "MatrixMemory.o_proj"}, {"MatrixMemory.gates"}),
          "dofipel": (ATTENTION | LATENT | GATED | {"LatentAttention.front_q"}, {"LatentAttention.w_keys", "LatentAttention.w_values", "RoutedExperts.router"}),
          "domorax": (ATTENTION | LATENT | GATED | DENSE | {"LatentAttention.dq", "LatentAttention.uq", "GatedDeltaRule.qkvg", "GatedDeltaRule.o_proj"},
                      {"GatedDeltaRule.gates", "LatentAttention.w_keys", "LatentAttention.w_values", "RoutedExperts.router"}),
          "penasun": (ATTENTION | {"SelectiveScanMixer.in_proj", "SelectiveScanMixer.o_proj"}, {"RoutedExperts.router"}),
          "volonex": (ATTENTION | GATED, set())}


@pytest.mark.parametrize("design", sorted(PACKED))
def test_what_is_packed(request, design):
    import hector_engine_amd as he
    from hector_engine_amd.parts.routed import RoutedExperts
    from tests.test_fp4_engine_gpu import DESIGNS, OPTS, parts_of
    folders = request.getfixturevalue(f"{design}_folders")
    packed, stored = set(), set()
    for name in sorted(DESIGNS[design]):
        eng = he.Engine(folders[name + "_calm" if name + "_calm" in folders else name], weights="fp4", weight_group=32, **OPTS)
        for part, attr, lin in linears(eng.model):
            (packed if lin.packed else stored).add(f"{type(part).__name__}.{attr}")
            assert lin.packed or isinstance(lin.weight, torch.Tensor)
        for part in parts_of(eng.model):
            if isinstance(part, RoutedExperts):
                assert part.packed is not None and part.gate_up is None and part.down is None
            for attr in ("router", "w_keys", "w_values"):
                if isinstance(getattr(part, attr, None), torch.Tensor):
                    stored.add(f"{type(part).__name__}.{attr}")
    assert (packed, stored) == (PACKED[design][0], PACKED[design][1] | {"LinearHead.linear"})
