"""Products with weights in 4 bits of more rows than a launch, or 32-bit offsets, take."""
import pytest
import torch

from tests.plain import fp4_plain as P

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("M,N,K,apart", [(1 << 21, 20, 1024, 0), ((1 << 21) + 40, 36, 1020, 0), (65535 * 16 + 17, 16, 128, 0), (1100000, 17, 40, 3), ((1 << 21) - 100, 16, 1024, 8)])
def test_more_rows_than_a_turn(M, N, K, apart):
    """Rows at both ends and around the turns' border against 64-bit sums, all of them against the same rows of another call; rows behind the last stay."""
    from hector_engine_amd.kernels import fp4, ops
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("40 GiB of free GPU memory")
    gen = torch.Generator(device="cuda").manual_seed(7)
    few = torch.randn((4096, K), generator=gen, device="cuda").to(BF16)
    room = torch.empty((M, K + apart), dtype=BF16, device="cuda")
    for r0 in range(0, M, 4096):
        n = min(4096, M - r0)
        room[r0:r0 + n, :K] = few[:n]
    x = room[:, :K]
    w = fp4.pack(torch.randn((N, K), generator=gen, device="cuda") * 0.1, 64)
    values = w.unpack(F32).cpu()
    ws = torch.full((ops.fp4_product_workspace_bytes(M, w, whole=apart == 0),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((M + 1, N), 7.0, device="cuda")
    ops.fp4_product(out, x, w, None, M, workspace=ws)
    assert (out[M] == 7).all()
    turn = min(M, ((1 << 32) - 1) // (2 * (-(-K // 128) * 128)) // 128 * 128)
    for lo, hi in ((0, 40), (turn - 40, min(turn + 40, M)), (M - 40, M)):
        want = x[lo:hi].cpu().double() @ values.double().T
        assert ((out[lo:hi].cpu().double() - want).abs() <= P.sum_bound(x[lo:hi], values, 64) + 2.0 ** -24 * want.abs()).all()
    # rows repeat every 4096, so do the results of a turn (and of all turns whose tiles are the same)
    first = out[:4096]
    for r0 in range(0, turn, 4096):
        n = min(4096, turn - r0)
        assert torch.equal(out[r0:r0 + n], first[:n])
    del room, out, ws
    torch.cuda.empty_cache()


def test_one_workspace_for_every_number_of_rows():
    """A server's: what 513 rows want serves all fewer ones, which are cut into more slices; the slices' memory is written before it is read."""
    from hector_engine_amd.kernels import fp4, ops
    gen = torch.Generator(device="cuda").manual_seed(8)
    N, K, M = 3584, 18944, 513
    x, w = torch.randn((M, K), generator=gen, device="cuda").to(BF16), fp4.pack(torch.randn((N, K), generator=gen, device="cuda") * 0.05, 128)
    values = w.unpack(F32).double()
    want, size = x.double() @ values.T, (128 + 148 + 16) * 2.0 ** -23 * (x.double().abs() @ values.abs().T)      # (as fp4_plain.sum_bound)
    ws = torch.full((ops.fp4_product_workspace_bytes(M, w, whole=True),), 0xFF, dtype=torch.uint8, device="cuda")
    assert ops.fp4_product_workspace_bytes(M, w, whole=True, alone=True) < ops.fp4_product_workspace_bytes(M - 1, w, whole=True, alone=True)
    for m in (513, 512, 65, 64, 33, 32, 17, 16, 1):
        out = torch.full((m + 1, N), 7.0, device="cuda")
        ws.fill_(0xFF)
        ops.fp4_product(out, x, w, None, m, workspace=ws)
        assert ((out[:m].double() - want[:m]).abs() <= size[:m] + 2.0 ** -24 * want[:m].abs()).all() and (out[m] == 7).all()
