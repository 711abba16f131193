"""Weights in 4 bits on the GPU: packing, the product and a routed feed-forward over packed experts, against their definitions in
float64 (tests/plain/fp4_plain.py). A bfloat16 result is off by half a step (2^-8 of the value at most) and the sum's own bound."""
import pytest
import torch

from tests.plain import fp4_plain as P

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def api():
    import hector_engine_amd  # noqa: F401
    from hector_engine_amd.kernels import fp4, ops
    return fp4, ops


def rnd(seed, *shape, scale=1.0, dtype=BF16):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def workspace(size):
    return torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")      # (stale memory is NaN)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 1), (16, 128), (17, 129), (5, 31), (3, 33, 200), (2, 16, 96), (40, 264), (1000, 1003)])
def test_packing_gives_the_nearest_values(api, shape, group, dtype):
    fp4, _ = api
    w = rnd(1, *shape, scale=0.02, dtype=dtype)
    packed = fp4.pack(w.cuda(), group)
    want = P.values(w, group)
    assert torch.equal(packed.unpack(F32).cpu().double(), want)
    assert torch.equal(packed.unpack().cpu().double(), want)      # exact in bfloat16 too


def test_packing_borders_zeros_and_numbers_that_are_none(api):
    fp4, _ = api
    w = torch.zeros(8, 64)
    # scale 1 (largest magnitude 6): every border between two magnitudes, both signs, and their neighbours
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    w[0, :7], w[0, 7:14], w[0, 14] = border, -border, 6.0
    w[1, :7], w[1, 7:14], w[1, 14] = torch.nextafter(border, torch.tensor(9.0)), torch.nextafter(border, torch.tensor(0.0)), -6.0
    w[2, 5] = float("nan")
    w[3, 40] = float("inf")
    w[4, 0], w[4, 1] = 3.4e38, -3.4e38             # six times the scale is still a number
    w[5, :3] = torch.tensor([1e-38, -1e-39, 1e-45])
    w[6, :] = -0.0
    w[7, 0] = 6 * (1 + 1 / 64)                     # a scale between two of six bits: the even one
    packed = fp4.pack(w.cuda(), 32)
    got = packed.unpack(F32).cpu()
    assert got[0, :15].tolist() == [0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, 6]
    assert got[1, :15].tolist() == [0.5, 1, 1.5, 2, 3, 4, 6, 0, 0.5, 1, 1.5, 2, 3, 4, -6]
    assert got[2, :32].isnan().all() and not got[2, 32:].isnan().any()
    assert got[3, 32:].isnan().all() and not got[3, :32].isnan().any()
    assert got[4].isfinite().all() and 3.3e38 < got[4, 0] <= 3.4e38 and got[4, 1] == -got[4, 0]
    assert got[5, 0] == pytest.approx(1e-38, rel=1 / 32) and got[5, 3:].abs().max() == 0
    assert got[6].abs().max() == 0 and got[7, 0] == 6.0


def test_packing_rows_that_lie_apart(api):
    fp4, _ = api
    wide = rnd(2, 50, 300, scale=0.02).cuda()
    for cut in (wide[:, :128], wide[:, 3:200], wide[::2, 8:136]):
        assert torch.equal(fp4.pack(cut, 64).unpack(), fp4.pack(cut.contiguous(), 64).unpack())


SIZES = [(1, 16, 128), (1, 1, 8), (2, 17, 40), (1, 300, 1003), (4, 64, 256), (5, 130, 2056), (16, 48, 1152), (16, 4608, 384),
         (17, 1001, 1003), (32, 96, 136), (33, 200, 520), (64, 256, 1024), (65, 80, 264), (130, 36, 640), (200, 530, 384), (300, 2050, 1160)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(api, M, N, K, group):
    fp4, ops = api
    x, w, b = rnd(3, M, K), rnd(4, N, K, scale=0.05), rnd(5, N)
    packed = fp4.pack(w.cuda(), group)
    values = P.values(w, group)
    want = x.double() @ values.T
    bound = P.sum_bound(x, values, group)
    for dtype, bias in ((F32, None), (BF16, None), (F32, b), (BF16, b.float())):
        out = torch.full((M + 1, N), float("nan"), dtype=dtype, device="cuda")
        ops.fp4_product(out, x.cuda(), packed, None if bias is None else bias.cuda(), M,
                        workspace=workspace(ops.fp4_product_workspace_bytes(M, packed)))
        exact = want if bias is None else want + bias.double()
        got = out.cpu().double()
        assert got[M].isnan().all()                  # the row behind the last is left as it was
        # (the bias's addition and the last rounding: half a step each)
        assert ((got[:M] - exact).abs() <= bound * (1 + HALF[dtype]) + (HALF[dtype] + 2.0 ** -24) * (exact.abs() + bound)).all()


@pytest.mark.parametrize("M,N,K,group", [(100, 4616, 1160, 64), (520, 4625, 1032, 128), (1100, 2052, 1003, 32), (400, 8200, 392, 32), (70, 9001, 3600, 64),
                                         (48, 12300, 904, 128), (1030, 130, 4100, 64), (155, 3630, 10112, 64), (805, 2515, 7380, 64), (141, 839, 16535, 128),
                                         (33, 2000, 6272, 32)])
def test_product_of_large_weights(api, M, N, K, group):
    """Sizes that the kernel of many rows takes, whole or in slices of K, at columns and k that end inside tiles: bias, gated, rows that lie apart."""
    fp4, ops = api
    wide, w, b = rnd(33, M, K + 16), rnd(34, N, K, scale=0.05), rnd(35, N)
    x = wide[:, 8:8 + K]
    packed = fp4.pack(w.cuda(), group)
    values = packed.unpack(F32).cpu().double()
    want, size = x.double() @ values.t(), P.sum_bound(x, values, group)
    room = wide.cuda()
    for rows, xs in ((room[:, 8:8 + K], "apart"), (x.cuda().contiguous(), "together")):
        ws = workspace(ops.fp4_product_workspace_bytes(M, packed))
        for dtype in (F32, BF16):
            out = torch.full((M + 2, N + 3), 7.0, dtype=dtype, device="cuda")
            ops.fp4_product(out[1:M + 1, 1:N + 1], rows, packed, b.cuda(), M, workspace=ws)
            full = want + b.double()
            off = (out[1:M + 1, 1:N + 1].cpu().double() - full).abs() - (size + HALF[dtype] * full.abs() + 2.0 ** -23 * full.abs())
            assert off.max() <= 0, (xs, dtype, float(off.max()))
            out[1:M + 1, 1:N + 1] = 7
            assert (out == 7).all()                  # nothing beside the results
        if N % 2 == 0:
            got = torch.empty((M, N // 2), dtype=BF16, device="cuda")
            ops.fp4_product(got, rows, packed, None, M, gated=True, workspace=ws)
            g, u, full = want[:, 0::2].abs(), want[:, 1::2].abs(), P.act(want)
            slack = 1.13 * size[:, 0::2] * (u + size[:, 1::2]) + (g + size[:, 0::2]) * size[:, 1::2] + 2.0 ** -20 * g * u * (1 + g)      # (as in test_gated_product)
            assert ((got.cpu().double() - full).abs() <= slack + HALF[BF16] * (full.abs() + slack) + 2.0 ** -120).all(), xs


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 3, 4, 6, 8, 13, 16])
@pytest.mark.parametrize("N,K", [(40, 8200), (300, 18944), (4100, 8192), (4608, 2100), (8200, 1104), (10250, 640), (21000, 512), (25000, 392)])
def test_few_rows_of_every_shape(api, N, K, M, group):
    """The numbers of weight rows and k at which few rows are cut another way, one to sixteen rows; a second call gives the same bits."""
    fp4, ops = api
    gen = torch.Generator(device="cuda").manual_seed(95)
    x, w = torch.randn((M, K), generator=gen, device="cuda").to(BF16), torch.randn((N, K), generator=gen, device="cuda") * 0.05
    # scales that differ from group to group and row to row by powers of two: a wrong one is not lost among the others
    w *= torch.exp2(torch.randint(-3, 4, (N, -(-K // 32)), generator=gen, device="cuda")).repeat_interleave(32, 1)[:, :K]
    packed = fp4.pack(w, group)
    values = packed.unpack(F32).double()
    want = x.double() @ values.T
    size = (group + -(-K // group) + 16) * 2.0 ** -23 * (x.double().abs() @ values.abs().T)      # (as sum_bound)
    out, again = torch.empty((M, N), dtype=F32, device="cuda"), torch.empty((M, N), dtype=F32, device="cuda")
    ops.fp4_product(out, x, packed, None, M)
    ops.fp4_product(again, x, packed, None, M)
    assert ((out.double() - want).abs() <= size + 2.0 ** -24 * want.abs()).all() and torch.equal(out, again)


@pytest.mark.parametrize("K", [1, 5, 7, 8, 9, 15, 121, 127, 129, 135, 255, 257])
@pytest.mark.parametrize("M", [1, 6, 16, 21])
def test_product_of_rows_that_end_anywhere(api, M, K):
    """The rows' last values inside a piece of eight, at bases of every alignment; what lies behind and between the rows is NaN."""
    fp4, ops = api
    room, w = torch.full((M, 300), float("nan"), dtype=BF16), rnd(37, 40, K, scale=0.1)
    x = rnd(36, M, K)
    packed = fp4.pack(w.cuda(), 32)
    values = P.values(w, 32)
    want, size = x.double() @ values.T, P.sum_bound(x, values, 32)
    ws = workspace(ops.fp4_product_workspace_bytes(M, packed))
    for c0 in (0, 1, 6, 300 - K):
        room[:] = float("nan")
        room[:, c0:c0 + K] = x
        out = torch.empty((M, 40), dtype=F32, device="cuda")
        ops.fp4_product(out, room.cuda()[:, c0:c0 + K], packed, None, M, workspace=ws)
        assert ((out.cpu().double() - want).abs() <= size + 2.0 ** -24 * want.abs()).all(), c0


@pytest.mark.parametrize("act", [(1.0, 0.0, 0.0), (1.702, 7.0, 1.0)])
@pytest.mark.parametrize("M,N,K", [(1, 2, 32), (3, 34, 200), (16, 512, 384), (17, 130, 136), (64, 320, 1024), (130, 258, 264), (260, 1028, 520)])
def test_gated_product(api, M, N, K, act):
    fp4, ops = api
    x, w = rnd(6, M, K), rnd(7, N, K, scale=0.1)
    packed = fp4.pack(w.cuda(), 64)
    values = P.values(w, 64)
    z, bound = x.double() @ values.T, P.sum_bound(x, values, 64)
    out = torch.full((M + 1, N // 2), float("nan"), dtype=BF16, device="cuda")
    ops.fp4_product(out, x.cuda(), packed, None, M, gated=True, act=act, workspace=workspace(ops.fp4_product_workspace_bytes(M, packed, True)))
    exact = P.act(z, *act)
    # |d act / d gate| <= 1.13 (|up| + shift), |d act / d up| <= |gate| (x * sigmoid(a x) for a >= 1 grows by at most 1.1 a step); its own
    # evaluation in 32 bits is off by a few last places, and by 2^-24 alpha |gate| where the exponential's argument is rounded
    g, u = z[:, 0::2].abs(), z[:, 1::2].abs()
    slack = 1.13 * bound[:, 0::2] * (u + bound[:, 1::2] + act[2]) + (g + bound[:, 0::2]) * bound[:, 1::2] + 2.0 ** -20 * g * (u + act[2]) * (1 + g)
    got = out.cpu().double()
    assert got[M].isnan().all()
    assert ((got[:M] - exact).abs() <= slack + HALF[BF16] * (exact.abs() + slack) + 2.0 ** -120).all()


def test_product_of_rows_that_lie_apart(api):
    """Rows at a distance, a base that is not 16-byte aligned, an output inside a wider tensor: the same bits."""
    fp4, ops = api
    w = fp4.pack(rnd(8, 100, 264, scale=0.05).cuda(), 32)
    for M in (1, 7, 40, 150):
        wide = rnd(9, M, 700).cuda()
        for c0 in (0, 8, 3):
            cut = wide[:, c0:c0 + 264]
            size = ops.fp4_product_workspace_bytes(M, w)
            want = torch.empty((M, 100), dtype=F32, device="cuda")
            ops.fp4_product(want, cut.contiguous(), w, None, M, workspace=workspace(size))
            room = torch.full((M, 170), 7.0, device="cuda")
            ops.fp4_product(room[:, 5:105], cut, w, None, M, workspace=workspace(size))
            assert torch.equal(room[:, 5:105], want)
            assert (room[:, :5] == 7).all() and (room[:, 105:] == 7).all()


def test_a_row_without_numbers_stays_alone(api):
    """NaN and infinities in a row of x, and NaN groups of a weight row, reach their own row and column and no others."""
    fp4, ops = api
    for M in (3, 16, 40, 130):
        w = rnd(10, 40, 200, scale=0.05)
        x = rnd(11, M, 200)
        clean = torch.empty((M, 40), dtype=F32, device="cuda")
        size = workspace(ops.fp4_product_workspace_bytes(M, fp4.pack(w.cuda(), 64)))
        ops.fp4_product(clean, x.cuda(), fp4.pack(w.cuda(), 64), None, M, workspace=size)
        x[1, 5], x[2, 199] = float("nan"), float("inf")
        w[7, 100] = float("nan")
        got = torch.empty_like(clean)
        ops.fp4_product(got, x.cuda(), fp4.pack(w.cuda(), 64), None, M, workspace=size)
        keep = torch.ones((M, 40), dtype=torch.bool)
        keep[1:3], keep[:, 7] = False, False
        assert torch.equal(got.cpu()[keep], clean.cpu()[keep])
        assert got[1].isnan().all() and got[:, 7].isnan().all() and not got[2].isfinite().any()
        for act in ((1.0, 0.0, 0.0), (1.702, 7.0, 1.0), (1.5957691216057308, 0.0, 0.0, 0.07135481627159956)):      # (limits do not hide a NaN)
            h = torch.empty((M, 20), dtype=BF16, device="cuda")
            ops.fp4_product(h, x.cuda(), fp4.pack(w.cuda(), 64), None, M, gated=True, act=act, workspace=size)
            assert h[1].isnan().all() and h[:, 3].isnan().all() and h.cpu()[keep[:, 0::2] & keep[:, 1::2]].isfinite().all()


def experts_case(seed, rows, E, top, I, D, group, act, holes=True):
    gu, dn, x = rnd(seed, E, 2 * I, D, scale=0.1), rnd(seed + 1, E, D, I, scale=0.1), rnd(seed + 2, rows, D)
    gen = torch.Generator().manual_seed(seed + 3)
    ids = torch.randint(0, max(1, E - 1), (rows, top), generator=gen, dtype=torch.int32)     # (the last expert has no row)
    shares = torch.rand((rows, top), generator=gen)
    if holes and rows > 1:
        ids[rows // 2, 0] = -1
        ids[rows - 1, :] = E + 3                     # a row none of whose choices is an expert
        shares[0, top - 1] = 0.0
    wu, wd = P.values(gu, group), P.values(dn, group)
    exact, slack = torch.zeros((rows, D), dtype=F64), torch.zeros((rows, D), dtype=F64)
    for r in range(rows):
        for c in range(top):
            e = int(ids[r, c])
            if not 0 <= e < E:
                continue
            s = float(shares[r, c])
            z, bound = x[r:r + 1].double() @ wu[e].T, P.sum_bound(x[r:r + 1], wu[e], group)
            h = s * P.act(z, *act)
            # as the gated product's slack; the activations times their share are rounded to bfloat16 for the second product
            g, u = z[:, 0::2].abs(), z[:, 1::2].abs()
            d = s * (1.13 * bound[:, 0::2] * (u + bound[:, 1::2] + act[2]) + (g + bound[:, 0::2]) * bound[:, 1::2]
                     + 2.0 ** -20 * g * (u + act[2]) * (1 + g))
            d = d + HALF[BF16] * (h.abs() + d)
            exact[r] += (h @ wd[e].T)[0]
            slack[r] += (d @ wd[e].abs().T + P.sum_bound(h.abs() + d, wd[e], group))[0] * (1 + top * 2.0 ** -24)
    return gu, dn, x, ids, shares, exact, slack


@pytest.mark.parametrize("rows,E,top,I,D,group,act", [
    (1, 2, 1, 8, 16, 32, (1.0, 0.0, 0.0)), (1, 16, 4, 40, 64, 64, (1.0, 0.0, 0.0)), (5, 8, 3, 24, 72, 32, (1.702, 7.0, 1.0)),
    (20, 3, 3, 136, 128, 128, (1.0, 0.0, 0.0)), (64, 4, 2, 64, 200, 32, (1.0, 0.0, 0.0)), (130, 2, 2, 48, 40, 64, (1.0, 0.0, 0.0)),
    (1, 5, 8, 136, 72, 32, (1.702, 7.0, 1.0)), (1, 4, 3, 20, 36, 64, (1.0, 0.0, 0.0)), (1, 3, 64, 24, 40, 32, (1.0, 0.0, 0.0)),
    (20, 16, 4, 72, 136, 32, (1.0, 0.0, 0.0)), (16, 2, 4, 40, 80, 64, (1.0, 0.0, 0.0)), (40, 64, 2, 16, 48, 32, (1.0, 0.0, 0.0)),
    (150, 7, 2, 20, 36, 32, (1.702, 7.0, 1.0)), (3, 200, 8, 8, 16, 32, (1.0, 0.0, 0.0)), (400, 3, 2, 144, 264, 128, (1.0, 0.0, 0.0)),
    (1, 3, 2, 3, 5, 32, (1.0, 0.0, 0.0)), (4, 4, 2, 9, 3, 64, (1.0, 0.0, 0.0)), (60, 2, 2, 3, 13, 32, (1.0, 0.0, 0.0)), (2, 2, 2, 1, 1, 32, (1.0, 0.0, 0.0)),
    (3, 4, 2, 512, 640, 128, (1.0, 0.0, 0.0)), (7, 4, 2, 512, 1280, 32, (1.0, 0.0, 0.0)), (17, 4, 2, 520, 2304, 64, (1.702, 7.0, 1.0)),
    (40, 4, 2, 512, 640, 32, (1.0, 0.0, 0.0)), (200, 4, 2, 648, 1000, 128, (1.0, 0.0, 0.0)), (600, 4, 2, 256, 900, 64, (1.0, 0.0, 0.0)),
    (1, 4, 4, 8200, 640, 128, (1.0, 0.0, 0.0)), (4, 4, 4, 8200, 320, 64, (1.0, 0.0, 0.0)), (1, 3, 2, 1032, 8200, 128, (1.0, 0.0, 0.0))])
def test_experts(api, rows, E, top, I, D, group, act):
    fp4, ops = api
    gu, dn, x, ids, shares, exact, slack = experts_case(20, rows, E, top, I, D, group, act)
    up, down = fp4.pack(gu.cuda(), group), fp4.pack(dn.cuda(), group)
    out = torch.full((rows + 1, D), float("nan"), dtype=BF16, device="cuda")
    ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, act=act,
                    workspace=workspace(ops.fp4_experts_workspace_bytes(rows, top, up, down)))
    got = out.cpu().double()
    assert got[rows].isnan().all()
    assert ((got[:rows] - exact).abs() <= slack + HALF[BF16] * (exact.abs() + slack)).all()
    if rows > 1:
        assert (got[rows - 1] == 0).all()


def test_experts_the_same_expert_twice_and_a_row_without_numbers(api):
    """A row that names one expert twice takes it twice; a NaN row reaches no other row."""
    fp4, ops = api
    E, I, D = 4, 24, 64
    up, down = fp4.pack(rnd(30, E, 2 * I, D, scale=0.1).cuda(), 32), fp4.pack(rnd(31, E, D, I, scale=0.1).cuda(), 32)
    x = rnd(32, 6, D).cuda()

    def run(x, ids, shares):
        out = torch.empty((x.shape[0], D), dtype=BF16, device="cuda")
        ops.fp4_experts(out, x, up, down, ids.cuda(), shares.cuda(), x.shape[0],
                        workspace=workspace(ops.fp4_experts_workspace_bytes(x.shape[0], ids.shape[1], up, down)))
        return out
    once = run(x, torch.full((6, 1), 2, dtype=torch.int32), torch.full((6, 1), 0.5))
    twice = run(x, torch.full((6, 2), 2, dtype=torch.int32), torch.full((6, 2), 0.25))
    assert torch.equal(once, twice)                  # 0.25 h + 0.25 h is 0.5 h exactly, in every step of the sums
    ids = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [0, 2], [1, 3]], dtype=torch.int32)
    shares = torch.full((6, 2), 0.5)
    clean = run(x, ids, shares)
    bad = x.clone()
    bad[3] = float("nan")
    got = run(bad, ids, shares)
    keep = torch.tensor([0, 1, 2, 4, 5])
    assert torch.equal(got[keep], clean[keep]) and got[3].isnan().all()


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_experts_identity_ids_that_are_none_and_weights_of_zero(api, rows):
    """An id from E on takes weight * x with identity and nothing without; below 0 nothing; a weight of 0 nothing, whatever the expert holds."""
    fp4, ops = api
    E, I, D, top = 5, 40, 72, 3
    gu, dn, x = rnd(90, E, 2 * I, D, scale=0.1), rnd(91, E, D, I, scale=0.1), rnd(92, rows, D)
    dn[4] = float("nan")                             # (the last expert is chosen with weight 0 alone)
    up, down = fp4.pack(gu.cuda(), 32), fp4.pack(dn.cuda(), 32)
    gen = torch.Generator().manual_seed(93)
    ids = torch.randint(0, 4, (rows, top), generator=gen, dtype=torch.int32)
    shares = torch.rand((rows, top), generator=gen) + 0.1
    ids[:, 1], ids[rows // 2, 0] = E + 2, -3
    ids[rows // 2, 2], shares[rows // 2, 2] = 4, 0.0
    got = {}
    for identity in (False, True):
        out = torch.empty((rows, D), dtype=BF16, device="cuda")
        ops.fp4_experts(out, x.cuda(), up, down, ids.cuda(), shares.cuda(), rows, identity=identity,
                        workspace=workspace(ops.fp4_experts_workspace_bytes(rows, top, up, down)))
        got[identity] = out.cpu().double()
    assert got[False].isfinite().all() and (got[False][rows // 2] == 0).all()
    own = shares[:, 1:2].double() * x.double()
    # each result half a step off, and the sums of 32 bits
    assert ((got[True] - got[False] - own).abs() <= HALF[BF16] * (got[True].abs() + got[False].abs()) * 1.01 + 2.0 ** -20 * own.abs()).all()


def test_a_row_does_not_depend_on_the_rows_beside_it(api):
    """Within one kernel's range of row counts a row has the same bits whatever stands beside it, and run after run."""
    fp4, ops = api
    w = fp4.pack(rnd(40, 272, 392, scale=0.05).cuda(), 64)
    for lo, hi in ((2, 16), (17, 32), (33, 64), (257, 300)):
        x = rnd(41, hi, 392).cuda()
        size = workspace(max(ops.fp4_product_workspace_bytes(lo, w), ops.fp4_product_workspace_bytes(hi, w)))
        a, b = torch.empty((hi, 272), dtype=F32, device="cuda"), torch.empty((hi, 272), dtype=F32, device="cuda")
        ops.fp4_product(a, x, w, None, hi, workspace=size)
        ops.fp4_product(b, x, w, None, hi, workspace=size)
        assert torch.equal(a, b)
        ops.fp4_product(b, x, w, None, lo, workspace=size)
        assert torch.equal(a[:lo], b[:lo])


def test_replayed_graphs_and_two_streams(api):
    """Captured calls replay, with eager work between them, on the inputs as they are then; two graphs with a workspace each, and calls on two
    streams at once, give what one alone gives."""
    fp4, ops = api
    E, I, D, rows, top = 4, 64, 128, 9, 2
    up, down = fp4.pack(rnd(50, E, 2 * I, D, scale=0.1).cuda(), 32), fp4.pack(rnd(51, E, D, I, scale=0.1).cuda(), 32)
    w = fp4.pack(rnd(52, 96, D, scale=0.1).cuda(), 32)
    ids = torch.randint(0, E, (rows, top), dtype=torch.int32, device="cuda")
    shares = torch.rand((rows, top), device="cuda")

    def make():
        st = dict(x=torch.zeros((rows, D), dtype=BF16, device="cuda"), moe=torch.empty((rows, D), dtype=BF16, device="cuda"),
                  y=torch.empty((rows, 96), dtype=F32, device="cuda"), ws=workspace(ops.fp4_experts_workspace_bytes(rows, top, up, down)),
                  ws2=workspace(ops.fp4_product_workspace_bytes(rows, w)))

        def call():
            ops.fp4_experts(st["moe"], st["x"], up, down, ids, shares, rows, workspace=st["ws"])
            ops.fp4_product(st["y"], st["moe"], w, None, rows, workspace=st["ws2"])
        return st, call

    graphs = []
    for _ in range(2):
        st, call = make()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append((st, g))
    for turn in range(4):
        for i, (st, g) in enumerate(graphs):
            st["x"].copy_(rnd(60 + 2 * turn + i, rows, D))
            g.replay()
        ref, call = make()
        for i, (st, _) in enumerate(graphs):
            ref["x"].copy_(rnd(60 + 2 * turn + i, rows, D))
            call()
            torch.cuda.synchronize()
            assert torch.equal(ref["y"], st["y"]) and torch.equal(ref["moe"], st["moe"])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = [make(), make()]
    for i, (st, _) in enumerate(runs):
        st["x"].copy_(rnd(80 + i, rows, D))
    torch.cuda.synchronize()
    for _ in range(5):
        for (st, call), s in zip(runs, streams):
            with torch.cuda.stream(s):
                call()
    torch.cuda.synchronize()
    ref, call = make()
    for i, (st, _) in enumerate(runs):
        ref["x"].copy_(rnd(80 + i, rows, D))
        call()
        torch.cuda.synchronize()
        assert torch.equal(ref["y"], st["y"])


def test_refusals(api):
    """Wrong sizes, dtypes and layouts are refused on the host, before any launch; nothing is written."""
    fp4, ops = api
    w = fp4.pack(rnd(70, 32, 64).cuda(), 32)
    stack, downs = fp4.pack(rnd(71, 2, 32, 64).cuda(), 32), fp4.pack(rnd(72, 2, 64, 16).cuda(), 32)
    x, out = rnd(73, 4, 64).cuda(), torch.full((4, 32), 7.0, device="cuda")
    with pytest.raises(ValueError, match="groups of 48"):
        fp4.pack(x, 48)
    with pytest.raises(ValueError, match="GPU tensor"):
        fp4.pack(x.cpu(), 32)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        fp4.pack(x.half(), 32)
    with pytest.raises(ValueError, match="positive sizes"):
        fp4.pack(x[:0], 32)
    with pytest.raises(ValueError, match="contiguous"):
        fp4.pack(x.t(), 32)
    with pytest.raises(TypeError, match="packed weight"):
        ops.fp4_product(out, x, x, None, 4)
    with pytest.raises(ValueError, match="2 dims"):
        ops.fp4_product(out, x, stack, None, 4)
    with pytest.raises(TypeError, match="x is torch.float32"):
        ops.fp4_product(out, x.float(), w, None, 4)
    with pytest.raises(ValueError, match=r"x\(4, 56\)"):
        ops.fp4_product(out, x[:, :56], w, None, 4)
    with pytest.raises(ValueError, match=r"is not \[5, 64\]"):
        ops.fp4_product(out, x, w, None, 5)
    with pytest.raises(ValueError, match="-1 rows"):
        ops.fp4_product(out, x, w, None, -1)
    with pytest.raises(ValueError, match="contiguous and must not overlap"):
        ops.fp4_product(out, x[:1].expand(4, 64), w, None, 4)
    with pytest.raises(TypeError, match="results in torch.float16"):
        ops.fp4_product(out.half(), x, w, None, 4)
    with pytest.raises(ValueError, match="bias"):
        ops.fp4_product(out, x, w, torch.zeros(31, device="cuda"), 4)
    with pytest.raises(ValueError, match="gated"):
        ops.fp4_product(out[:, :16].to(BF16), x, w, torch.zeros(32, device="cuda"), 4, gated=True)
    with pytest.raises(TypeError, match="results in torch.float32"):
        ops.fp4_product(out[:, :16], x, w, None, 4, gated=True)
    from hector_engine_amd.kernels.lib import KernelLibraryError
    tall, wide, many = fp4.pack(rnd(74, 4096, 1160).cuda(), 32), rnd(75, 300, 1160).cuda(), torch.full((300, 4096), 7.0, device="cuda")
    need = ops.fp4_product_workspace_bytes(300, tall)
    assert need > 0
    with pytest.raises(ValueError, match="a workspace of"):
        ops.fp4_product(many, wide, tall, None, 300)
    with pytest.raises(KernelLibraryError, match="a workspace of"):
        ops.fp4_product(many, wide, tall, None, 300, workspace=workspace(ops.fp4_product_workspace_bytes(300, tall, whole=True) - 1))
    with pytest.raises(TypeError, match="workspace"):
        ops.fp4_product(many, wide, tall, None, 300, workspace=torch.empty(need, dtype=torch.int8, device="cuda"))
    ids, shares = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    moe = torch.full((4, 64), 7.0, dtype=BF16, device="cuda")
    ws = workspace(ops.fp4_experts_workspace_bytes(4, 2, stack, downs))
    with pytest.raises(ValueError, match="a workspace of"):
        ops.fp4_experts(moe, x, stack, downs, ids, shares, 4)
    with pytest.raises(ValueError, match="a workspace of"):
        ops.fp4_experts(moe, x, stack, downs, ids, shares, 4, workspace=ws[:-1])
    with pytest.raises(ValueError, match="expected .2, 32, 64."):
        ops.fp4_experts(moe, x, downs, downs, ids, shares, 4, workspace=ws)
    with pytest.raises(TypeError, match="ids: expected torch.int32"):
        ops.fp4_experts(moe, x, stack, downs, ids.long(), shares, 4, workspace=ws)
    with pytest.raises(ValueError, match="choices"):
        ops.fp4_experts(moe, x, stack, downs, ids, shares[:, :1].contiguous(), 4, workspace=ws)
    ops.fp4_product(out, x, w, None, 0)              # no rows: nothing happens
    ops.fp4_experts(moe, x, stack, downs, ids, shares, 0, workspace=ws)
    torch.cuda.synchronize()
    assert (out == 7).all() and (moe == 7).all() and (many == 7).all()


@pytest.mark.parametrize("M,N,K,group,dtype", [(1, 64, 128, 64, BF16), (3, 100, 72, 32, F32), (8, 896, 1003, 64, BF16), (16, 3584, 512, 128, BF16), (13, 20, 9, 32, F32)])
def test_a_norm_carried_across_two_products(api, M, N, K, group, dtype):
    """The first product's results in the residual rows, r * gain and the sums of squares beside them; the second product over those,
    with a bias, gated and in 32 bits. Rows behind the last stay as they were."""
    fp4, ops = api
    x, w, b = rnd(80, M, K), fp4.pack(rnd(81, N, K, scale=0.1).cuda(), group), rnd(82, N)
    w2, b2 = fp4.pack(rnd(83, 36, N, scale=0.1).cuda(), group), rnd(84, 36)
    gain, start = rnd(85, N, dtype=dtype), rnd(86, M + 1, N, dtype=F32)
    values, values2 = w.unpack(F32).cpu().double(), w2.unpack(F32).cpu().double()
    resid = start.cuda()
    xg, squares = torch.full((M + 1, N), 7.0, dtype=BF16, device="cuda"), torch.full((M + 1, -(-N // 16)), 7.0, device="cuda")
    ops.fp4_product_carried(None, x.cuda(), w, b.cuda(), M, residual=(resid, gain.cuda(), xg, squares, 0.5))
    want = start[:M].double() + 0.5 * (x.double() @ values.T + b.double())
    size = P.sum_bound(x, values, group)
    got = resid.cpu()
    # the sum's bound, then the bias, the product with 0.5 (exact) and the addition, each within half a place of what it gives
    assert ((got[:M].double() - want).abs() <= 0.5 * size + 2.0 ** -23 * (want.abs() + (x.double() @ values.T).abs() + b.double().abs())).all()
    assert torch.equal(got[M], start[M]) and (xg[M] == 7).all() and (squares[M] == 7).all()
    r = got[:M].double()
    assert ((xg[:M].cpu().double() - r * gain.double()).abs() <= (2.0 ** -8 + 2.0 ** -23) * (r * gain.double()).abs()).all()
    parts = torch.nn.functional.pad(r ** 2, (0, -N % 16)).view(M, -1, 16).sum(-1)
    assert ((squares[:M].cpu().double() - parts).abs() <= 16 * 2.0 ** -24 * parts).all()
    eps = 1e-5
    a, scale = xg[:M].cpu().double(), 1 / (squares[:M].cpu().double().sum(-1, keepdim=True) / N + eps).sqrt()
    z, size2 = (a @ values2.T) * scale, P.sum_bound(a, values2, group) * scale
    # the scale: a sum of up to 224 squares, a division, a root and a reciprocal in 32 bits
    size2 = size2 + 16 * 2.0 ** -23 * z.abs()
    for kind in (F32, BF16):
        out = torch.full((M + 1, 36), 7.0, dtype=kind, device="cuda")
        ops.fp4_product_carried(out, xg, w2, b2.cuda(), M, row_scale=(squares, eps))
        full = z + b2.double()
        assert ((out[:M].cpu().double() - full).abs() - size2 - (HALF[kind] + 2.0 ** -23) * full.abs()).max() <= 2.0 ** -23 * b2.abs().max() and (out[M] == 7).all()
    out = torch.empty((M, 18), dtype=BF16, device="cuda")
    ops.fp4_product_carried(out, xg, w2, None, M, gated=True, row_scale=(squares, eps))
    exact, g, u = P.act(z), z[:, 0::2].abs(), z[:, 1::2].abs()
    slack = 1.13 * size2[:, 0::2] * (u + size2[:, 1::2]) + (g + size2[:, 0::2]) * size2[:, 1::2] + 2.0 ** -20 * g * u * (1 + g)      # (as in test_gated_product)
    assert ((out.cpu().double() - exact).abs() <= slack + HALF[BF16] * (exact.abs() + slack) + 2.0 ** -120).all()
    # nothing owed and nothing carried: the product
    plain, same = torch.empty((M, 36), dtype=F32, device="cuda"), torch.empty((M, 36), dtype=F32, device="cuda")
    ops.fp4_product(plain, xg, w2, b2.cuda(), M)
    ops.fp4_product_carried(same, xg, w2, b2.cuda(), M)
    assert torch.equal(plain, same)


def test_refusals_of_the_carried_product(api):
    fp4, ops = api
    w = fp4.pack(rnd(70, 32, 64).cuda(), 32)
    x, out = rnd(73, 20, 64).cuda(), torch.full((20, 32), 7.0, device="cuda")
    xg, squares, gain = torch.empty((20, 32), dtype=BF16, device="cuda"), torch.empty((20, 2), device="cuda"), torch.ones(32, device="cuda")
    for rows in (17, -1):
        with pytest.raises(ValueError, match="it takes up to 16"):
            ops.fp4_product_carried(out, x, w, None, rows)
    with pytest.raises(ValueError, match="row_scale"):
        ops.fp4_product_carried(out, x, w, None, 4, row_scale=(squares[:3].contiguous(), 1e-5))
    with pytest.raises(TypeError, match="row_scale"):
        ops.fp4_product_carried(out, x, w, None, 4, row_scale=(xg, 1e-5))
    with pytest.raises(ValueError, match="no output"):
        ops.fp4_product_carried(out, x, w, None, 4, residual=(out, gain, xg, squares))
    with pytest.raises(ValueError, match="squares"):
        ops.fp4_product_carried(None, x, w, None, 4, residual=(out, gain, xg, squares[:, :1].contiguous()))
    with pytest.raises(ValueError, match="gain"):
        ops.fp4_product_carried(None, x, w, None, 4, residual=(out, gain[:16], xg, squares))
    with pytest.raises(ValueError, match="multiple of 4"):
        ops.fp4_product_carried(None, x, fp4.pack(rnd(71, 30, 64).cuda(), 32), None, 4, residual=(out, gain, xg, squares))
    ops.fp4_product_carried(out, x, w, None, 0)
    torch.cuda.synchronize()
    assert (out == 7).all()


def test_offsets_past_32_bits(api):
    """Rows of x that span more than 4 GiB, results that do, codes that do: the same bits as at small distances."""
    fp4, ops = api
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GiB of free GPU memory")
    M, K = 70000, 128
    room = torch.empty((M, 32768), dtype=BF16, device="cuda")
    room[:, :K] = rnd(90, M, K).cuda()
    for N in (64, 2048):
        w = fp4.pack(rnd(91, N, K, scale=0.1).cuda(), 64)
        ws = workspace(ops.fp4_product_workspace_bytes(M, w))
        want, got = (torch.empty((M, N), dtype=BF16, device="cuda") for _ in range(2))
        ops.fp4_product(want, room[:, :K].contiguous(), w, None, M, workspace=ws)
        ops.fp4_product(got, room[:, :K], w, None, M, workspace=ws)
        assert torch.equal(got, want)
    x = room[:, :K].contiguous()
    ops.fp4_product(room[:, 16384:16384 + 2048], x, w, None, M, workspace=ws)
    assert torch.equal(room[:, 16384:16384 + 2048], want)
    del room, want, got
    # weight rows that repeat every 64: so do the results
    few = rnd(92, 64, 65536, scale=0.02).cuda()
    w = fp4.pack(few.repeat(2049, 1), 128)
    assert w.codes.nbytes > 1 << 32
    for M in (1, 16, 80):
        x = rnd(93, M, 65536).cuda()
        ws = workspace(ops.fp4_product_workspace_bytes(M, w))
        out = torch.empty((M, w.shape[0]), dtype=F32, device="cuda")
        ops.fp4_product(out, x, w, None, M, workspace=ws)
        exact = x.double() @ fp4.pack(few, 128).unpack(F32).double().T
        assert ((out[:, :64].double() - exact).abs().cpu() <= P.sum_bound(x, fp4.pack(few, 128).unpack(F32), 128)).all()
        assert torch.equal(out.view(M, 2049, 64), out[:, None, :64].expand(M, 2049, 64))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [1, 7, 16])
@pytest.mark.parametrize("N,K,group", [(40, 8200, 128), (300, 18944, 64), (4608, 2100, 32), (8200, 1104, 64), (10256, 640, 128), (25000, 392, 32)])
def test_a_carried_norm_at_every_shape(api, N, K, group, M):
    """The scale on the sums and the results in the residual rows, against the product without either: the same sums, so off by the roundings of
    the scale (a sum of a few hundred squares, a division, a root, a reciprocal), the product with it and the addition alone."""
    fp4, ops = api
    gen = torch.Generator(device="cuda").manual_seed(96)
    x, w = torch.randn((M, K), generator=gen, device="cuda").to(BF16), fp4.pack(torch.randn((N, K), generator=gen, device="cuda") * 0.05, group)
    plain = torch.empty((M, N), dtype=F32, device="cuda")
    ops.fp4_product(plain, x, w, None, M)
    for count in (1, 65, 224, 700):
        owed = torch.rand((M, count), generator=gen, device="cuda") * 3 * K / count
        scale = 1 / (owed.double().sum(-1, keepdim=True) / K + 1e-5).sqrt()
        out = torch.empty_like(plain)
        ops.fp4_product_carried(out, x, w, None, M, row_scale=(owed, 1e-5))
        want = plain.double() * scale
        assert ((out.double() - want).abs() <= 2.0 ** -23 * (0.5 * (count / 64 + 12) + 4) * want.abs()).all()
    start, gain = torch.randn((M, N), generator=gen, device="cuda"), torch.randn(N, generator=gen, device="cuda").to(BF16)
    resid, xg, squares = start.clone(), torch.empty((M, N), dtype=BF16, device="cuda"), torch.empty((M, -(-N // 16)), device="cuda")
    ops.fp4_product_carried(None, x, w, None, M, residual=(resid, gain, xg, squares))
    want = start.double() + plain.double()
    assert ((resid.double() - want).abs() <= 2.0 ** -23 * want.abs()).all()
    assert ((xg.double() - resid.double() * gain.double()).abs() <= (2.0 ** -8 + 2.0 ** -23) * (resid.double() * gain.double()).abs()).all()
    parts = torch.nn.functional.pad(resid.double() ** 2, (0, -N % 16)).view(M, -1, 16).sum(-1)
    assert ((squares.double() - parts).abs() <= 16 * 2.0 ** -24 * parts).all()
