"""Weights in 4 bits: the packed matrix, and packing one.

A matrix [N, K] (or several of one size, [E, N, K]) is kept as codes of 4 bits, a sign and one of the magnitudes
0, 0.5, 1, 1.5, 2, 3, 4, 6, and one scale for every `group` (32, 64 or 128) neighbours along K:

    scale = max |w| / 6, rounded to six significant bits          code = the nearest to w / scale, ties to the even one

so that scale * code is a bfloat16 number exactly, and a group's largest magnitude is off by at most a sixty-fourth
of it. A group of zeros has scale 0; one that holds a NaN or an infinity has a NaN scale, and every value of it is NaN.
4.125, 4.25 or 4.5 bits a value where bfloat16 has 16. (The reference's compact formats keep 4 to 5 bits a value: tools/quant_bench/README.md:305-307.)

The tiles' layout is the kernels' own (csrc/fp4.h): a packed matrix is read by ops.fp4_product, ops.fp4_experts and unpack().
"""
from __future__ import annotations

import torch

GROUPS = (32, 64, 128)
TILE_ROWS, TILE_K = 16, 128


def storage_shapes(shape: tuple, group: int) -> tuple[tuple, tuple]:
    """The shapes of the codes (uint8) and the scales (bfloat16) of a matrix [N, K], or of several [E, N, K]."""
    if len(shape) not in (2, 3) or any(s <= 0 for s in shape):
        raise ValueError(f"fp4: a matrix is [N, K] or [E, N, K] of positive sizes, not {tuple(shape)}")
    if group not in GROUPS:
        raise ValueError(f"fp4: groups of {group}, must be one of {GROUPS}")
    *lead, n, k = shape
    tiles = (*lead, -(-n // TILE_ROWS), -(-k // TILE_K))
    return (*tiles, TILE_ROWS * TILE_K // 2), (*tiles, TILE_K // group, TILE_ROWS)


class Fp4Weight:
    """A packed matrix; `shape` is the matrix's. Made by pack()."""

    dtype = "fp4"      # what a table of kernel routes looks it up by

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple, group: int):
        shape = tuple(int(s) for s in shape)
        for what, t, dtype, want in zip(("codes", "scales"), (codes, scales), (torch.uint8, torch.bfloat16), storage_shapes(shape, group)):
            if not t.is_cuda or not t.is_contiguous() or t.device != codes.device:
                raise ValueError(f"fp4: {what} must be contiguous tensors on one GPU")
            if t.dtype != dtype or tuple(t.shape) != want:
                raise ValueError(f"fp4: {what} of a matrix {shape} in groups of {group} are {dtype} {want}, not {t.dtype} {tuple(t.shape)}")
        self._hold(codes, scales, shape, group)

    def _hold(self, codes, scales, shape, group) -> None:
        self._codes, self._scales, self._shape, self._group, self._index = codes, scales, shape, group, codes.get_device()
        self.pointers = codes.data_ptr(), scales.data_ptr()

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    shape = property(lambda self: self._shape)
    group = property(lambda self: self._group)
    device_index = property(lambda self: self._index)

    @property
    def device(self) -> torch.device:
        return self._codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def dim(self) -> int:
        return len(self.shape)

    def first_rows(self, rows: int) -> "Fp4Weight":
        """The first rows of a matrix [N, K], whole tiles of 16 or all, over the same memory."""
        n, *k = self._shape
        if len(k) != 1 or not 0 < rows <= n or (rows % TILE_ROWS and rows != n):
            raise ValueError(f"fp4: the first {rows} rows of {self._shape} are not whole tiles of {TILE_ROWS}")
        tiles = -(-rows // TILE_ROWS)
        return Fp4Weight(self._codes[:tiles], self._scales[:tiles], (rows, *k), self._group)

    def unpack(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, bfloat16 (exact) or float32."""
        from . import ops
        out = self._codes.new_empty(self._shape, dtype=dtype)
        ops.fp4_unpack(out, self)
        return out


def pack(w: torch.Tensor, group: int = 64) -> Fp4Weight:
    """Packs a float32 or bfloat16 matrix on the GPU (the rows of a matrix [N, K] may lie apart)."""
    from . import ops
    shape = tuple(w.shape)
    codes, scales = storage_shapes(shape, group)
    if not w.is_cuda:
        raise ValueError("fp4.pack: expected a GPU tensor")
    packed = Fp4Weight.__new__(Fp4Weight)      # (its tensors are made here as its checks would have them)
    packed._hold(w.new_empty(codes, dtype=torch.uint8), w.new_empty(scales, dtype=torch.bfloat16), shape, group)
    ops.fp4_pack(packed, w)
    return packed
