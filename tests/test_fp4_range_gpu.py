"""Products with weights in 4 bits at the ends of 32-bit numbers: sums of x * code leave their range where the results do not."""
import pytest
import torch

from tests.plain import fp4_plain as P

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def large(gen, M, N, K, group):
    """x around 3e37, so that a code of 6 and some neighbours are beyond 3.4e38; weights around 1e-33, so that results are around 1e4 to 1e7. (x, packed, results, bound)."""
    from hector_engine_amd.kernels import fp4
    x = (torch.randn((M, K), generator=gen, device="cuda").clamp(-4, 4) * 3e37).to(BF16)
    w = torch.randn((N, K), generator=gen, device="cuda") * 1e-33
    packed = fp4.pack(w, group)
    values = packed.unpack(F32).double()
    size = (group + -(-K // group) + 16) * 2.0 ** -23 * (x.double().abs() @ values.abs().T)      # (as fp4_plain.sum_bound)
    return x, packed, x.double() @ values.T, size


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 3, 6, 8, 13, 16, 30])
@pytest.mark.parametrize("N,K", [(40, 264), (40, 8200), (300, 18944), (4608, 2100), (8200, 1104), (10250, 643), (25000, 392)])
def test_rows_whose_unscaled_sums_are_beyond_32_bits(N, K, M, group):
    from hector_engine_amd.kernels import ops
    gen = torch.Generator(device="cuda").manual_seed(97)
    x, packed, want, size = large(gen, M, N, K, group)
    out = torch.empty((M, N), dtype=F32, device="cuda")
    ops.fp4_product(out, x, packed, None, M, workspace=torch.empty(ops.fp4_product_workspace_bytes(M, packed), dtype=torch.uint8, device="cuda"))
    assert ((out.double() - want).abs() <= size + 2.0 ** -24 * want.abs()).all()
    if M > 1:                                        # one such row beside ordinary ones: those keep their bits or their bound
        y = x.clone()
        y[1:] = (y[1:].double() * 2.0 ** -100).to(BF16)
        ops.fp4_product(out, y, packed, None, M, workspace=torch.empty(ops.fp4_product_workspace_bytes(M, packed), dtype=torch.uint8, device="cuda"))
        assert ((out[:1].double() - want[:1]).abs() <= size[:1] + 2.0 ** -24 * want[:1].abs()).all()
        small, bound = y[1:].double() @ packed.unpack(F32).double().T, 2.0 ** -100 * size[1:]
        assert ((out[1:].double() - small).abs() <= bound + 2.0 ** -24 * small.abs()).all()


@pytest.mark.parametrize("M,N,K,group", [(1, 304, 8200, 64), (7, 4608, 2100, 32), (16, 10256, 640, 128)])
def test_a_carried_norm_over_such_rows(M, N, K, group):
    from hector_engine_amd.kernels import ops
    gen = torch.Generator(device="cuda").manual_seed(98)
    x, packed, want, size = large(gen, M, N, K, group)
    resid, xg, squares = torch.zeros((M, N), device="cuda"), torch.empty((M, N), dtype=BF16, device="cuda"), torch.empty((M, -(-N // 16)), device="cuda")
    ops.fp4_product_carried(None, x, packed, None, M, residual=(resid, torch.ones(N, device="cuda"), xg, squares))
    assert ((resid.double() - want).abs() <= size + 2.0 ** -24 * want.abs()).all()
    owed = torch.full((M, 1), 4.0 * K, device="cuda")          # a scale of a half, but for its own roundings (a division, a root, a reciprocal)
    out = torch.empty((M, N), dtype=F32, device="cuda")
    ops.fp4_product_carried(out, x, packed, None, M, row_scale=(owed, 0.0))
    assert ((out.double() - want / 2).abs() <= size / 2 + 2.0 ** -20 * want.abs()).all()


@pytest.mark.parametrize("rows", [1, 3, 20])
def test_experts_over_activations_that_large(rows):
    """Gates around 4e18, where silu(g) is g or 0: activations up to 1e38 into the second product, one row's experts in one sum among them."""
    from hector_engine_amd.kernels import fp4, ops
    E, I, D, top, group = 3, 1000, 72, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(99)
    x = torch.randn((rows, D), generator=gen, device="cuda").clamp(-3, 3).to(BF16)
    up = fp4.pack(torch.randn((E, 2 * I, D), generator=gen, device="cuda") * 4.6e17, group)
    down = fp4.pack(torch.randn((E, D, I), generator=gen, device="cuda") * 1e-33, group)
    ids = torch.stack([torch.randperm(E, generator=gen, device="cuda")[:top] for _ in range(rows)]).int()
    shares = torch.rand((rows, top), generator=gen, device="cuda") * 0.5 + 0.5
    out = torch.empty((rows, D), dtype=BF16, device="cuda")
    ops.fp4_experts(out, x, up, down, ids, shares, rows,
                    workspace=torch.empty(ops.fp4_experts_workspace_bytes(rows, top, up, down), dtype=torch.uint8, device="cuda"))
    wu, wd = up.unpack(F32).double().cpu(), down.unpack(F32).double().cpu()
    want, slack = torch.zeros((rows, D), dtype=F64), torch.zeros((rows, D), dtype=F64)
    for r in range(rows):
        for s, e in zip(shares[r].tolist(), ids[r].tolist()):
            z, b = x[r:r + 1].cpu().double() @ wu[e].T, P.sum_bound(x[r:r + 1], wu[e], group)
            g, u = z[:, 0::2].clamp(min=0), z[:, 1::2]
            h = s * g * u
            # the sums' own bounds through the product, its last places, then the rounding to bfloat16 (a gate within its bound of 0 is some 1e12: still 0 or itself)
            d = s * (b[:, 0::2] * (u.abs() + b[:, 1::2]) + g * b[:, 1::2]) + 2.0 ** -21 * h.abs()
            d = d + 2.0 ** -8 * (h.abs() + d)
            want[r] += (h @ wd[e].T)[0]
            slack[r] += (d @ wd[e].abs().T + P.sum_bound(h.abs() + d, wd[e], group))[0] * (1 + top * 2.0 ** -24)
    assert h.abs().max() > 1e36 and ((out.cpu().double() - want).abs() <= slack + 2.0 ** -8 * (want.abs() + slack)).all()
