"""Weights in 4 bits without a GPU: the layout's sizes, the definition, the operators' refusals and their choices by size."""
import ctypes

import pytest
import torch

from tests.plain import fp4_plain as P

F64 = torch.float64


@pytest.fixture(scope="module")
def L():
    from hector_engine_amd.kernels import lib
    return lib.load()


def refusal(L, status):
    assert status != 0
    return L.he_last_error().decode()


ROOM = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(ROOM) + 255) // 256 * 256       # (an address: no call of this file launches anything)


@pytest.mark.parametrize("shape,group,codes,scales", [
    ((16, 128), 32, (1, 1, 1024), (1, 1, 4, 16)), ((17, 129), 64, (2, 2, 1024), (2, 2, 2, 16)), ((1, 1), 128, (1, 1, 1024), (1, 1, 1, 16)),
    ((3, 40, 300), 128, (3, 3, 3, 1024), (3, 3, 3, 1, 16))])
def test_sizes_of_the_layout(shape, group, codes, scales):
    from hector_engine_amd.kernels import fp4
    assert fp4.storage_shapes(shape, group) == (codes, scales)


def test_refusals_of_packing():
    from hector_engine_amd.kernels import fp4
    for shape in ((4,), (0, 4), (4, 0), (2, 3, 4, 5)):
        with pytest.raises(ValueError, match="positive sizes"):
            fp4.storage_shapes(shape, 64)
    for group in (0, 16, 48, 256):
        with pytest.raises(ValueError, match=f"groups of {group}"):
            fp4.storage_shapes((4, 4), group)
    with pytest.raises(ValueError, match="GPU tensor"):
        fp4.pack(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="one GPU"):
        fp4.Fp4Weight(torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.zeros(1, 1, 2, 16, dtype=torch.bfloat16), (4, 64), 64)


def test_the_definition_keeps_what_it_says():
    """Values that packing gives are bfloat16 numbers; the largest of a group is off by a sixty-fourth at most, no value by more than a
    sixth of it and that; packing them again gives them again."""
    w = torch.randn(50, 300, generator=torch.Generator().manual_seed(1), dtype=F64)
    w[3, 64:128] = 0
    for group in (32, 64, 128):
        v = P.values(w, group)
        assert torch.equal(v.to(torch.bfloat16).double(), v) and (v[3, 64:96] == 0).all()
        for k0 in range(0, 300, group):
            a, b = w[:, k0:k0 + group], v[:, k0:k0 + group]
            most = a.abs().amax(-1, keepdim=True)
            at = a.abs() == most
            assert ((a - b).abs()[at] <= most.expand_as(a)[at] / 64).all()
            assert ((a - b).abs() <= most * (1 / 6 + 1 / 64)).all()
        assert torch.equal(P.values(v, group), v)


def test_refusals_of_the_product(L):
    def call(M=4, N=32, K=64, ldo=32, ldx=64, codes=AT, scales=AT, bias=None, group=32, out_dtype=0, gated=0, workspace=None, size=0):
        return refusal(L, L.he_fp4_product(AT, ldo, AT, ldx, codes, scales, bias, M, N, K, group, out_dtype, 0, gated, 1.0, 0.0, 0.0, 0.0, workspace, size, None))
    assert "groups of 48" in call(group=48)
    assert "a weight of [0, 64]" in call(N=0)
    assert "16-byte aligned" in call(codes=AT + 8) and "16-byte aligned" in call(codes=None) and "16-byte aligned" in call(scales=AT + 2)
    assert "rows of 64 at distances" in call(M=-1) and "rows of 64 at distances" in call(ldx=63) and "results of 32 at distances of 31" in call(ldo=31)
    assert "rows of 64 at distances" in call(M=(1 << 22) + 1)
    assert "dtype code 7" in call(out_dtype=7)
    assert "gated" in call(gated=1, out_dtype=0) and "gated" in call(gated=1, out_dtype=1, bias=AT) and "gated" in call(gated=1, out_dtype=1, N=33)
    need = L.he_fp4_product_workspace_bytes(3, 32, 5, 1)
    assert need > 0 and "a workspace of" in call(M=3, K=5) and "a workspace of" in call(M=3, K=5, workspace=AT, size=need - 1) \
        and "a workspace of" in call(M=3, K=5, workspace=AT + 8, size=need)


def test_refusals_of_the_carried_product(L):
    def call(out=AT, M=4, N=32, K=64, ldo=32, group=32, out_dtype=0, gated=0, bias=None, owed=None, count=2, resid=None, gain=AT, carried=AT, squares=AT):
        return refusal(L, L.he_fp4_product_carried(out, ldo, AT, K, AT, AT, bias, M, N, K, group, out_dtype, 0, gated, 1.0, 0.0, 0.0, 0.0, owed, count, 1e-5,
                                                   resid, 1.0, gain, 0, carried, squares, None))
    assert "17 rows" in call(M=17) and "rows of 7" in call(K=7) and "groups of 16" in call(group=16)
    assert "0 sums of squares" in call(owed=AT, count=0)
    for wrong in (dict(N=30), dict(gated=1), dict(out=AT, resid=AT), dict(gain=None), dict(carried=None), dict(squares=None), dict(resid=AT + 8), dict(carried=AT + 4)):
        assert "results for the residual rows" in call(**{"out": None, "resid": AT, **wrong})
    assert "dtype code 0 at distances of 31" in call(ldo=31) and "dtype code 5" in call(out_dtype=5) and "dtype code 0" in call(out=None)
    assert "gated" in call(gated=1, out_dtype=0, ldo=16)


def test_refusals_of_the_experts(L):
    def call(rows=4, top=2, experts=2, I=16, D=64, ldx=64, up=AT, down=AT, groups=(32, 32), workspace=AT, size=1 << 30):
        return refusal(L, L.he_fp4_experts(AT, AT, ldx, up, AT, down, AT, AT, AT, rows, top, experts, I, D, *groups, 0, 1.0, 0.0, 0.0, 0.0, workspace, size, None))
    assert "bad sizes" in call(rows=-1) and "bad sizes" in call(top=0) and "bad sizes" in call(I=0) and "bad sizes" in call(D=0) and "bad sizes" in call(experts=0)
    assert "too many" in call(experts=1025) and "too many" in call(rows=65536) and "too many" in call(rows=65535, top=4096)
    assert "distance of 63" in call(ldx=63)
    assert "groups of 16" in call(groups=(16, 32)) and "groups of 256" in call(groups=(32, 256))
    assert "16-byte aligned" in call(up=AT + 4) and "16-byte aligned" in call(down=None)
    need = L.he_fp4_experts_workspace_bytes(4, 2, 2, 16, 64)
    assert need > 0 and "a workspace of" in call(workspace=None) and "a workspace of" in call(size=need - 1) and "a workspace of" in call(workspace=AT + 4)


def test_no_rows_want_nothing(L):
    assert L.he_fp4_product_workspace_bytes(0, 32, 64, 1) == 0 and L.he_fp4_experts_workspace_bytes(0, 2, 2, 16, 64) == 0
    assert L.he_fp4_product(AT, 32, AT, 64, AT, AT, None, 0, 32, 64, 32, 0, 0, 0, 1.0, 0.0, 0.0, 0.0, None, 0, None) == 0
    assert L.he_fp4_experts(AT, AT, 64, AT, AT, AT, AT, AT, AT, 0, 2, 2, 16, 64, 32, 32, 0, 1.0, 0.0, 0.0, 0.0, None, 0, None) == 0


def test_which_products_want_a_workspace(L):
    """Few rows, and small weights, are read as they are wherever they lie; larger products copy rows that are not whole blocks of 128
    values or lie at odd places, and keep the sums of slices of K."""
    def wants(M, N, K, whole=1):
        return L.he_fp4_product_workspace_bytes(M, N, K, whole)
    for M in (1, 8, 16):
        assert wants(M, 37888, 3584, 0) == wants(M, 1001, 1003, 0) == 0
    assert wants(64, 1001, 1003, 0) == wants(128, 512, 896, 0) == 0
    assert wants(2048, 37888, 3584) == 0 and wants(2048, 37888, 3584, 0) == 2048 * 3584 * 2
    assert wants(2048, 37888, 3590) == wants(2048, 37888, 3590, 0) == 2048 * 3712 * 2
    slices = wants(64, 3584, 18944) / (64 * 3584 * 4)
    assert slices in (2, 4, 8, 16)


def test_the_route_of_packed_weights():
    from hector_engine_amd.kernels import routes
    import hector_engine_amd.parts.linear  # noqa: F401
    assert [r.name for r in routes.routes_of("linear", ("fp4", torch.bfloat16))] == ["fp4"]


def test_rows_that_span_4_gib_run_in_turns(L):
    """The kernel of many rows counts the bytes of its rows in 32 bits: a product of more runs in turns of whole tiles, which want one turn's workspace."""
    def wants(M, N, K, whole=1):
        return L.he_fp4_product_workspace_bytes(M, N, K, whole)
    turn = ((1 << 32) - 1) // (2 * 1024) // 128 * 128
    assert wants(turn, 2048, 1000) == wants(1 << 21, 2048, 1000) == wants(2 * turn, 2048, 1000) == wants(1 << 22, 2048, 1000) == turn * 1024 * 2
    assert wants(1 << 22, 2048, 1024) == 0 and wants(1 << 22, 2048, 1024, 0) == turn * 1024 * 2
    # a turn of a few rows of the largest K
    assert wants(64, 16, 1 << 26) == wants(16, 16, 1 << 26) == 0


def test_sixteen_rows_at_a_time_end_where_a_launch_does(L):
    """Small weights run 16 rows at a time, of which a launch has 65535; more rows go to the kernel of many rows, which copies what is not whole blocks of 128."""
    def wants(M, N, K, whole=1):
        return L.he_fp4_product_workspace_bytes(M, N, K, whole)
    assert wants(65535 * 16, 16, 100) == 0 and wants(65535 * 16 + 1, 16, 100) == (65535 * 16 + 1) * 128 * 2
    assert wants(65535 * 16, 16, 7) == 65535 * 16 * 128 * 2 and wants(1 << 22, 16, 128) == 0


@pytest.mark.parametrize("whole", [0, 1])
@pytest.mark.parametrize("N,K", [(3584, 18944), (3584, 3584), (37888, 3584), (1001, 1003), (512, 896), (130, 8200), (2048, 18944), (16, 65536), (300, 18950), (40, 5)])
def test_a_workspace_serves_fewer_rows(L, N, K, whole):
    """What is allocated for the largest batch is enough for every smaller one, and no more than the largest of their own."""
    most = 0
    for m in range(1, 1400):
        most = max(most, L.he_fp4_product_call_bytes(m, N, K, whole))
        assert L.he_fp4_product_workspace_bytes(m, N, K, whole) == most, m
    # rows beyond those that are cut along K
    for m in (5000, 20001, 200000):
        assert L.he_fp4_product_workspace_bytes(m, N, K, whole) >= max(most, *(L.he_fp4_product_call_bytes(x, N, K, whole) for x in (m // 7, m // 3, m - 1, m)))


def test_products_that_fewer_rows_cut_more_often(L):
    """The sizes at which a workspace for one number of rows was not enough for one row less."""
    for m in (32, 512):
        assert L.he_fp4_product_call_bytes(m, 3584, 18944, 1) > L.he_fp4_product_call_bytes(m + 1, 3584, 18944, 1)
        assert L.he_fp4_product_workspace_bytes(m + 1, 3584, 18944, 1) >= L.he_fp4_product_workspace_bytes(m, 3584, 18944, 1) > 0


@pytest.mark.parametrize("top,experts,I,D", [(4, 16, 2048, 2048), (2, 8, 24, 72), (8, 200, 100, 36), (1, 2, 3, 5), (3, 64, 1000, 130)])
def test_the_experts_workspace_serves_fewer_rows(L, top, experts, I, D):
    sizes = [L.he_fp4_experts_workspace_bytes(m, top, experts, I, D) for m in range(3000)]
    assert sizes == sorted(sizes)


class OfShape:
    def __init__(self, *shape):
        self.shape = shape


@pytest.mark.parametrize("top,D,I", [(4, 2048, 2048), (8, 256, 65536), (64, 100, 20000), (1, 1 << 20, 300), (2000, 64, 16)])
def test_the_most_rows_of_the_experts(L, top, D, I):
    """What the engine takes for a call's most rows is what the operator takes."""
    from hector_engine_amd.kernels import ops
    most = ops.fp4_experts_most_rows(top, OfShape(2, D, I))

    def call(rows):
        return refusal(L, L.he_fp4_experts(AT, AT, D, AT, AT, AT, AT, AT, AT, rows, top, 2, I, D, 32, 32, 0, 1.0, 0.0, 0.0, 0.0, None, 0, None))
    assert "a workspace of" in call(most) and "too many" in call(most + 1)


def test_more_experts_than_the_operator_takes_are_not_packed():
    """Refused when the model's weights are packed, not by its first step."""
    from hector_engine_amd.kernels import ops
    from hector_engine_amd.parts.base import BuildEnv, PartSpec, build_part
    from hector_engine_amd.parts.linear import Linear
    part = build_part("feed_forward", PartSpec("routed_experts", {"hidden_size": 8, "intermediate_size": 8, "experts": ops.FP4_MOST_EXPERTS + 1, "top": 2}), "m.",
                      BuildEnv(torch.device("cpu"), torch.bfloat16, True))
    part.gate_up, part.down = (Linear(torch.empty(s, dtype=torch.bfloat16, device="meta")) for s in ((16 * part.real, 8), (8, 8 * part.real)))
    with pytest.raises(ValueError, match="1025 experts cannot be packed"):
        part.pack_weights(32)
