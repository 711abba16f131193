// Weights in 4 bits. A matrix [N, K] is kept as codes of a sign and one of the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6, and a scale for
// every `group` (32, 64 or 128) neighbours along K; a scale has six significant bits, so scale * code is a bfloat16 number exactly.
//
// Layout: tiles of 16 rows x 128 k, in [matrix][N / 16][K / 128] order, rows and k filled up with zeros. A tile's codes are 1 KiB,
// 16 bytes a lane of the wavefront that reads it: lane l has row l & 15, its dword t the eight k from 32 t + 8 (l >> 4) on, the
// first in the lowest four bits - one operand of v_mfma_f32_16x16x32_bf16 after conversion. A tile's scales are bf16 [128 / group][16 rows].
// gfx950 converts such codes by pairs (v_cvt_scalef32_pk_bf16_fp4): four instructions for an operand of eight. (Integers of 4 bits
// take a shift, a mask and an or a pair, and leave an offset of 136 times the sum of x to take from the result.)
#pragma once
#include "common.h"
#include "hector_kernels.h"

#define FP4_ROWS 16
#define FP4_K 128
#define FP4_TILE_BYTES 1024

typedef __bf16 fp4_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 fp4_bf16x2 __attribute__((ext_vector_type(2)));
typedef float fp4_f32x4 __attribute__((ext_vector_type(4)));
typedef float fp4_f32x2 __attribute__((ext_vector_type(2)));

// eight codes as an operand
__device__ __forceinline__ fp4_bf16x8 fp4_operand(uint32_t codes) {
  const fp4_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 1);
  const fp4_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 3);
  return fp4_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A packed matrix, or one per group of rows (the experts of a routed feed-forward).
struct Fp4Weight {
  const uint8_t* codes;
  const uint16_t* scales;
  int N, K, group;
  int tiles, blocks;          // of a matrix: rows by 16, k by 128
};

// out = x W^T (+ bias), or gated; rows by themselves, or in groups of whole tiles of `bm` slots (group_rows)
struct Fp4Case {
  Fp4Weight w;
  const uint16_t* x;          // bf16 [rows][ldx]
  int64_t ldx;
  bool whole;                 // x may be read 16 bytes at a time
  void* out;
  int64_t ldo;
  bool out_f32, gated, clamped;
  const void* bias;           // [N] or null
  int bias_dtype;
  int M;
  GatedAct act;
  const int32_t* tile_begin;  // [groups + 1]: a group's first tile of slots; null: no groups
  int groups;
  const int32_t* rows_of;     // a slot's row of x, -1: none
  const int32_t* out_of;      // a slot's row of out, -1: none
  const float* factor;        // what a slot's results are multiplied by, or null
};
