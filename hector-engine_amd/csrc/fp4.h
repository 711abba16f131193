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

// What lanes of a wavefront have written into LDS is there for its other lanes behind this: no instruction (the unit keeps the order), but without it
// the compiler may take a lane's older read of a place for the new one where that lane has not written in between. (And what has been read may be
// written over behind it.)
__device__ __forceinline__ void fp4_written() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// eight codes as an operand
__device__ __forceinline__ fp4_bf16x8 fp4_operand(uint32_t codes) {
  const fp4_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 1);
  const fp4_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 3);
  return fp4_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight codes times their scale, as an operand (exact)
__device__ __forceinline__ fp4_bf16x8 fp4_values(uint32_t codes, float scale) {
  const fp4_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
  const fp4_f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
  const uint4 v = make_uint4(pack2_bf16(a[0] * scale, a[1] * scale), pack2_bf16(b[0] * scale, b[1] * scale),
                             pack2_bf16(c[0] * scale, c[1] * scale), pack2_bf16(d[0] * scale, d[1] * scale));
  return __builtin_bit_cast(fp4_bf16x8, v);
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
  bool out_f32, gated;
  const void* bias;           // [N] or null
  int bias_dtype;
  int M;
  GatedAct act;
  bool silu;                  // act is plain silu
  const int32_t* ids;         // [choices]: an expert each (fewer than groups, or none); a choice's row is choice / top, its results row `choice`. Or null
  const float* shares;        // [choices]: one of zero is left out
  int choices, top;
  const int32_t* tile_begin;  // [groups + 1]: a group's first tile of slots; null: no groups
  int groups;
  const int32_t* rows_of;     // a slot's row of x, -1: none
  const int32_t* out_of;      // a slot's row of out, -1: none
  const float* factor;        // what a slot's (with ids: a choice's) results are multiplied by, or null
  const float* owed;          // [M][owed_count], or null: the sums over row m times 1 / sqrt(the sum of owed[m] / owed_dim + owed_eps), x's rows being a norm's without its scale
  int owed_count, owed_dim;
  float owed_eps;
  float* resid;               // [M][N], or null: in place of out, resid += resid_scale * result, carried = bf16(resid * gain), squares[m][tile] = the
  float resid_scale;          // tile's sum of resid^2 (fp4_few.hip alone, N a multiple of 4)
  const void* gain;
  int gain_dtype;
  uint16_t* carried;
  float* squares;
  bool pairs;                 // out takes stores of four neighbouring results (gated: of two)
};

// The gated activation for results of 8 bits: the hardware's power of two and reciprocal, off by a few last places of 32-bit numbers
// (2^-22 of the value, and 2^-24 |alpha gate| where the power's argument is rounded), in a third of the instructions of the library's
// exponential and a division. NaN stays NaN behind the limits too. SILU: the constants are silu's, which takes half the instructions.
template <bool SILU>
__device__ __forceinline__ float fp4_act(float g, float u, const GatedAct& a) {
  if (SILU) return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g)) * u;
  g = g > a.limit ? a.limit : g;
  u = u > a.limit ? a.limit : u < -a.limit ? -a.limit : u;
  const float z = fmaf(a.cubic, g * g, a.alpha) * g;
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z)) * (u + a.shift);
}

// the bias of columns n to n + 3
__device__ __forceinline__ fp4_f32x4 fp4_bias(const Fp4Case& c, int n) {
  fp4_f32x4 b;
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = load_param(c.bias, min(n + e, c.w.N - 1), c.bias_dtype);
  return b;
}

// a lane's four neighbouring results, columns n to n + 3 of row `to`, whole: in one store; f: what activations are multiplied by
enum { FP4_GATED, FP4_SILU, FP4_BF16, FP4_F32 };
template <int KIND>
__device__ __forceinline__ void fp4_put(const Fp4Case& c, fp4_f32x4 v, int64_t to, int n, float f, bool whole) {
  if constexpr (KIND == FP4_GATED || KIND == FP4_SILU) {
    uint16_t* p = (uint16_t*)c.out + to * c.ldo + n / 2;
    auto act = [&](float g, float u) {
      return f == 0.f ? 0.f : fp4_act<KIND == FP4_SILU>(g, u, c.act) * f;    // (a choice without weight adds nothing, whatever its row holds)
    };
    const uint32_t pair = pack2_bf16(act(v[0], v[1]), act(v[2], v[3]));
    if (whole) {
      *reinterpret_cast<uint32_t*>(p) = pair;
    } else {
      p[0] = (uint16_t)pair;
      if (n + 2 < c.w.N) p[1] = (uint16_t)(pair >> 16);
    }
  } else if constexpr (KIND == FP4_F32) {
    float* p = (float*)c.out + to * c.ldo + n;
    if (whole) {
      *reinterpret_cast<fp4_f32x4*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < c.w.N) p[e] = v[e];
    }
  } else {
    uint16_t* p = (uint16_t*)c.out + to * c.ldo + n;
    const uint32_t a = pack2_bf16(v[0], v[1]), b = pack2_bf16(v[2], v[3]);
    if (whole) {
      *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < c.w.N) p[e] = (uint16_t)((e < 2 ? a : b) >> (16 * (e & 1)));
    }
  }
}
__device__ __forceinline__ void fp4_store(const Fp4Case& c, fp4_f32x4 v, int64_t to, int n, float f) {
  const bool whole = c.pairs && n + 4 <= c.w.N;
  if (c.gated && c.silu) return fp4_put<FP4_SILU>(c, v, to, n, f, whole);
  if (c.gated) return fp4_put<FP4_GATED>(c, v, to, n, f, whole);
  if (c.bias) v += fp4_bias(c, n);
  if (c.out_f32) fp4_put<FP4_F32>(c, v, to, n, f, whole);
  else fp4_put<FP4_BF16>(c, v, to, n, f, whole);
}

// the group of rows that tile `tile` belongs to, the last one that begins at or before it: the groups behind the first that do
// (64 are looked at in one load; a search of halves waited for each of its loads)
__device__ __forceinline__ int fp4_group_of(const int32_t* tile_begin, int groups, int tile) {
  int group = 0;
  for (int g = 1; g < groups; g += 64) {
    const int mine = g + (int)(threadIdx.x & 63);
    group += __popcll(__ballot(mine < groups && tile_begin[min(mine, groups)] <= tile));
  }
  return group;
}

// fp4_few.hip: rows in tiles of bm (4, 8 or 16); K is 8 at least
int fp4_run_few(const Fp4Case& c, int bm, int mtiles, hipStream_t s);
// one row, the sum over its choices (with ids): of expert ids[choice] with X row `choice`
int fp4_run_chain(const Fp4Case& c, hipStream_t s);
// fp4_tall.hip: rows in tiles of 16 mt, mtiles of them at most, weight rows in tiles of 64 nt, K in `parts` within a workgroup; x may be read 16 bytes at a
// time, K is a multiple of 128. slices > 1: K cut in so many (of a block at least) between workgroups too, their sums by way of sums [slices][M][N rounded up to 16].
struct Fp4Plan {
  int mt, nt, parts, slices;  // mt 0: fp4_run_few
};
int fp4_run_tall(const Fp4Case& c, Fp4Plan plan, int mtiles, float* sums, hipStream_t s);
