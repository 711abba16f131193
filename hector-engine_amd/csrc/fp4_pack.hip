// Matrices into 4 bits and back (fp4.h has the format).
#include "fp4.h"

namespace {

// Eight values times 1 / s as codes: the nearest magnitude, ties to the even code, 6 beyond 6. r is 1 / s rounded; with one step of correction
// v / s is correctly rounded, and a quotient that is not a border between two magnitudes is not rounded to one (the scale has six
// bits and the border three: the nearest other v is farther from it than half a step). So the ties are those of the exact quotient.
__device__ __forceinline__ uint32_t codes_of(const float* v, float s, float r) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float near = v[i] * r;
    q[i] = fmaf(fmaf(-near, s, v[i]), r, near);
  }
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, q[0], q[1], 1.f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[2], q[3], 1.f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[4], q[5], 1.f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[6], q[7], 1.f, 3);
  const uint32_t some = ((c & 0x77777777u) + 0x77777777u) & 0x88888888u;      // codes that are not 0: they alone keep a sign
  return c & (some | 0x77777777u);
}

// eight values from k on, zeros behind K
template <typename T>
__device__ __forceinline__ void eight(float* v, const T* row, int k, int K, bool whole) {
  if (whole && k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const uint4 p = *reinterpret_cast<const uint4*>(row + k);
      const uint32_t words[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(words[i] << 16), v[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 p = *reinterpret_cast<const float4*>(row + k + 4 * i);
        v[4 * i] = p.x, v[4 * i + 1] = p.y, v[4 * i + 2] = p.z, v[4 * i + 3] = p.w;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_float(row[k + i]) : 0.f;
}

// One wavefront a tile of 16 rows x 128 k. A group's largest magnitude is found among bit patterns, where a NaN is larger than all numbers: a
// group that holds one, or an infinity, has a NaN for its scale, and whatever is multiplied with it becomes NaN.
// Bound by its reads, which are whole lines of four rows (bf16) and take their places by way of LDS: 37888 x 3584 57 us.
// (Read in the order of the codes, half lines of 16 rows, and compared with each border in turn: 109.)
template <typename T, int GROUP, bool WHOLE>
__global__ __launch_bounds__(256) void pack_kernel(uint8_t* __restrict__ codes, uint16_t* __restrict__ scales, const T* __restrict__ w,
                                                   int64_t ldw, int N, int K, int tiles, int blocks, int64_t total) {
  constexpr int PIECES = FP4_K * sizeof(T) / 16, ROW = FP4_K * sizeof(T) + 16, AT_ONCE = 64 / PIECES;      // of a row in LDS; rows a load
  __shared__ __attribute__((aligned(16))) uint8_t lds[WHOLE ? 4 * 16 * ROW : 16];
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= total) return;
  const int lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const int64_t in_all = at / blocks;
  const int kb = (int)(at - in_all * blocks);
  const int64_t matrix = in_all / tiles;
  const int n0 = (int)(in_all - matrix * tiles) * FP4_ROWS, n = n0 + r;
  float v[4][8];
  if constexpr (WHOLE) {                                   // (a row of w is whole pieces: a piece is in it or behind it)
    uint8_t* own = lds + (threadIdx.x >> 6) * (16 * ROW);
    const int piece = lane % PIECES, k = kb * FP4_K + piece * (16 / (int)sizeof(T));
    uint4 p[16 / AT_ONCE];
#pragma unroll
    for (int i = 0; i < 16 / AT_ONCE; ++i) {
      const int row = i * AT_ONCE + lane / PIECES;
      p[i] = make_uint4(0, 0, 0, 0);
      if (n0 + row < N && k < K) p[i] = he_load16_once<uint4>(w + (matrix * N + n0 + row) * ldw + k);
    }
#pragma unroll
    for (int i = 0; i < 16 / AT_ONCE; ++i) *reinterpret_cast<uint4*>(own + (i * AT_ONCE + lane / PIECES) * ROW + piece * 16) = p[i];
    fp4_written();
#pragma unroll
    for (int t = 0; t < 4; ++t) eight(v[t], reinterpret_cast<const T*>(own + r * ROW), 32 * t + 8 * kq, FP4_K, true);
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (n < N) {
        eight(v[t], w + (matrix * N + n) * ldw, kb * FP4_K + 32 * t + 8 * kq, K, false);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[t][i] = 0.f;
      }
    }
  }
  constexpr int STEPS = GROUP / 32;
  uint32_t words[4];
#pragma unroll
  for (int g = 0; g < 4 / STEPS; ++g) {
    uint32_t most = 0;
#pragma unroll
    for (int t = g * STEPS; t < (g + 1) * STEPS; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[t][i]) & 0x7fffffffu);
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    // a sixth of it, to six significant bits (ties to even; 0x7e28 the last one whose sixfold is a number)
    const uint32_t sixth = __float_as_uint(__uint_as_float(most) / 6.f);
    const uint32_t bits = most < 0x7f800000u ? min((sixth + 0x1ffffu + ((sixth >> 18) & 1)) & ~0x3ffffu, 0x7e280000u) : 0x7fc00000u;
    if (kq == 0) scales[at * (16 * 4 / STEPS) + g * 16 + r] = (uint16_t)(bits >> 16);
    // scales whose reciprocal is out of range are multiplied by a power of two, and the values with them, exactly
    float s = __uint_as_float(bits), up = 1.f;
    if (s < 0x1p-100f) up = 0x1p100f, s *= up;
    const float inverse = 1.f / s;
#pragma unroll
    for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
      if (up != 1.f)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[t][i] *= up;
      words[t] = s > 0.f ? codes_of(v[t], s, inverse) : 0;
    }
  }
  *reinterpret_cast<uint4*>(codes + at * FP4_TILE_BYTES + lane * 16) = make_uint4(words[0], words[1], words[2], words[3]);
}

template <typename T, int GROUP>
__global__ __launch_bounds__(256) void unpack_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                                                     int N, int K, int tiles, int blocks, int64_t total, bool whole) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= total) return;
  const int lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const int64_t in_all = at / blocks;
  const int kb = (int)(at - in_all * blocks);
  const int64_t matrix = in_all / tiles;
  const int n = (int)(in_all - matrix * tiles) * FP4_ROWS + r;
  if (n >= N) return;
  constexpr int STEPS = GROUP / 32;
  const uint4 p = *reinterpret_cast<const uint4*>(codes + at * FP4_TILE_BYTES + lane * 16);
  const uint32_t words[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float s = bf16_bits_to_float(scales[at * (16 * 4 / STEPS) + t / STEPS * 16 + r]);
    const int k = kb * FP4_K + 32 * t + 8 * kq;
    float v[8];
    const fp4_bf16x8 q = fp4_operand(words[t]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)q[i] * s;
    T* to = out + (matrix * N + n) * K + k;
    if (whole && k + 8 <= K) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
      } else {
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) to[i] = from_float<T>(v[i]);
    }
  }
}

int check_sizes(const char* what, int matrices, int N, int K, int group) {
  HE_REQUIRE(matrices >= 0 && N > 0 && K > 0 && N <= (1 << 26) && K <= (1 << 26), "%s: bad sizes %d x [%d, %d]", what, matrices, N, K);
  HE_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of %d (32, 64 or 128)", what, group);
  return 0;
}

}  // namespace

// codes [matrices][N / 16][K / 128][1024 bytes], scales bf16 [matrices][N / 16][K / 128][128 / group][16] (sizes rounded up) of
// w [matrices][N][K] with rows ldw apart
extern "C" int he_fp4_pack(void* codes, void* scales, const void* w, int64_t ldw, int matrices, int N, int K, int group, int dtype, void* stream) {
  if (const int rc = check_sizes("he_fp4_pack", matrices, N, K, group)) return rc;
  HE_REQUIRE(dtype == HE_F32 || dtype == HE_BF16, "he_fp4_pack: dtype code %d", dtype);
  HE_REQUIRE(ldw >= K, "he_fp4_pack: rows of %d at a distance of %lld", K, (long long)ldw);
  HE_REQUIRE((((uintptr_t)codes) & 15) == 0, "he_fp4_pack: codes must be 16-byte aligned");
  const int tiles = (N + FP4_ROWS - 1) / FP4_ROWS, blocks = (K + FP4_K - 1) / FP4_K;
  const int64_t total = (int64_t)matrices * tiles * blocks;
  if (total == 0) return 0;
  HE_REQUIRE(total < (1ll << 26), "he_fp4_pack: %lld tiles are too many", (long long)total);
  const unsigned grid = (unsigned)((total + 3) / 4);
  const int item = dtype == HE_BF16 ? 2 : 4;
  const bool whole = ldw * item % 16 == 0 && (int64_t)K * item % 16 == 0 && ((uintptr_t)w & 15) == 0;
#define PACK(T, G)                                                                                                                       \
  (whole ? pack_kernel<T, G, true><<<grid, 256, 0, (hipStream_t)stream>>>((uint8_t*)codes, (uint16_t*)scales, (const T*)w, ldw, N, K, tiles, blocks, total) \
         : pack_kernel<T, G, false><<<grid, 256, 0, (hipStream_t)stream>>>((uint8_t*)codes, (uint16_t*)scales, (const T*)w, ldw, N, K, tiles, blocks, total))
  if (dtype == HE_BF16) {
    if (group == 32) PACK(bf16_t, 32);
    else if (group == 64) PACK(bf16_t, 64);
    else PACK(bf16_t, 128);
  } else {
    if (group == 32) PACK(float, 32);
    else if (group == 64) PACK(float, 64);
    else PACK(float, 128);
  }
#undef PACK
  return he_check_launch("he_fp4_pack");
}

// out [matrices][N][K] (contiguous) = the values
extern "C" int he_fp4_unpack(void* out, const void* codes, const void* scales, int matrices, int N, int K, int group, int dtype, void* stream) {
  if (const int rc = check_sizes("he_fp4_unpack", matrices, N, K, group)) return rc;
  HE_REQUIRE(dtype == HE_F32 || dtype == HE_BF16, "he_fp4_unpack: dtype code %d", dtype);
  HE_REQUIRE((((uintptr_t)codes) & 15) == 0, "he_fp4_unpack: codes must be 16-byte aligned");
  const int tiles = (N + FP4_ROWS - 1) / FP4_ROWS, blocks = (K + FP4_K - 1) / FP4_K;
  const int64_t total = (int64_t)matrices * tiles * blocks;
  if (total == 0) return 0;
  HE_REQUIRE(total < (1ll << 26), "he_fp4_unpack: %lld tiles are too many", (long long)total);
  const unsigned grid = (unsigned)((total + 3) / 4);
  const bool whole = K % 8 == 0 && ((uintptr_t)out & 15) == 0;
#define UNPACK(T, G) unpack_kernel<T, G><<<grid, 256, 0, (hipStream_t)stream>>>((T*)out, (const uint8_t*)codes, (const uint16_t*)scales, N, K, tiles, blocks, total, whole)
  if (dtype == HE_BF16) {
    if (group == 32) UNPACK(bf16_t, 32);
    else if (group == 64) UNPACK(bf16_t, 64);
    else UNPACK(bf16_t, 128);
  } else {
    if (group == 32) UNPACK(float, 32);
    else if (group == 64) UNPACK(float, 64);
    else UNPACK(float, 128);
  }
#undef UNPACK
  return he_check_launch("he_fp4_unpack");
}
