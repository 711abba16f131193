// Matrices into 4 bits and back (fp4.h has the format).
#include "fp4.h"

namespace {

// |v| to the nearest magnitude, ties to the even code; a border times a scale of six significant bits is exact, so no quotient is formed
__device__ __forceinline__ uint32_t code_of(float v, float s) {
  const float a = fabsf(v);
  if (!(s > 0.f)) return 0;
  uint32_t c = (a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) + (a > 2.5f * s) + (a >= 3.5f * s) + (a > 5.f * s);
  return c && v < 0.f ? c | 8 : c;
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
// Bound by its reads: a lane's 16 bytes, four of a row's neighbours a half line, the other half with the next load.
template <typename T, int GROUP>
__global__ __launch_bounds__(256) void pack_kernel(uint8_t* __restrict__ codes, uint16_t* __restrict__ scales, const T* __restrict__ w,
                                                   int64_t ldw, int N, int K, int tiles, int blocks, int64_t total, bool whole) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= total) return;
  const int lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const int64_t in_all = at / blocks;
  const int kb = (int)(at - in_all * blocks);
  const int64_t matrix = in_all / tiles;
  const int n = (int)(in_all - matrix * tiles) * FP4_ROWS + r;
  float v[4][8];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (n < N) {
      eight(v[t], w + (matrix * N + n) * ldw, kb * FP4_K + 32 * t + 8 * kq, K, whole);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[t][i] = 0.f;
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
    const float s = __uint_as_float(bits);
    if (kq == 0) scales[at * (16 * 4 / STEPS) + g * 16 + r] = (uint16_t)(bits >> 16);
#pragma unroll
    for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
      words[t] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) words[t] |= code_of(v[t][i], s) << (4 * i);
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
  HE_REQUIRE(total < (4ll << 31), "he_fp4_pack: %lld tiles are too many", (long long)total);
  const unsigned grid = (unsigned)((total + 3) / 4);
  const bool whole = (ldw * (dtype == HE_BF16 ? 2 : 4)) % 16 == 0 && ((uintptr_t)w & 15) == 0;
#define PACK(T, G) pack_kernel<T, G><<<grid, 256, 0, (hipStream_t)stream>>>((uint8_t*)codes, (uint16_t*)scales, (const T*)w, ldw, N, K, tiles, blocks, total, whole)
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
  HE_REQUIRE(total < (4ll << 31), "he_fp4_unpack: %lld tiles are too many", (long long)total);
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
