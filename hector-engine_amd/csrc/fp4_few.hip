// Products of up to 16 rows with a weight in 4 bits (fp4.h).
#include "fp4.h"

namespace {

// A workgroup has NT tiles of 16 weight rows; its W wavefronts cut K among them, and their sums meet in LDS. A wavefront's codes, scales and
// operands of X come straight from memory, D blocks of 128 k ahead, with no barrier before the end.
template <int NT, int W, int D, int GROUPS, bool WHOLE>
__global__ __launch_bounds__(64 * W) void fp4_few_kernel(Fp4Case c) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[W * NT * 1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = lane >> 4;
  const int blocks = c.w.blocks, lo = blocks * wave / W, hi = blocks * (wave + 1) / W;
  int group = 0;
  if (c.tile_begin) {
    if ((int)blockIdx.y >= c.tile_begin[c.groups]) return;
    group = fp4_group_of(c.tile_begin, c.groups, blockIdx.y);
  }
  const int m0 = blockIdx.y * 16, tile0 = blockIdx.x * NT;
  const uint8_t* codes[NT];
  const uint16_t* scales[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t at = ((int64_t)group * c.w.tiles + min(tile0 + j, c.w.tiles - 1)) * blocks;
    codes[j] = c.w.codes + at * FP4_TILE_BYTES;
    scales[j] = c.w.scales + at * (16 * GROUPS);
  }
  // (an operand's rows behind the last repeat it: each row's results are its own)
  const uint16_t* x = c.x + (c.rows_of ? (int64_t)max(c.rows_of[m0 + r16], 0) : min(m0 + r16, c.M - 1)) * c.ldx;
  const int K = c.w.K;

  uint4 q[D][NT], xs[D][4];
  uint2 s[D][NT][GROUPS];
  auto load = [&](int u, int kb) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      q[u][j] = he_load16_once<uint4>(codes[j] + (int64_t)kb * FP4_TILE_BYTES + lane * 16);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) s[u][j][g] = *reinterpret_cast<const uint2*>(scales[j] + (int64_t)kb * (16 * GROUPS) + 16 * g + 4 * kq);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int k = kb * FP4_K + 32 * t + 8 * kq;
      if (WHOLE) {
        xs[u][t] = *reinterpret_cast<const uint4*>(x + min(k, K - 8));
      } else {
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < K) words[e >> 1] |= (uint32_t)x[k + e] << (16 * (e & 1));
        xs[u][t] = make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
  };
  fp4_f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = fp4_f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int u, int kb) {
    if (WHOLE && (kb + 1) * FP4_K > K)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (kb * FP4_K + 32 * t + 8 * kq >= K) xs[u][t] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t words[4] = {q[u][j].x, q[u][j].y, q[u][j].z, q[u][j].w};
      fp4_f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const fp4_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_operand(words[t]), __builtin_bit_cast(fp4_bf16x8, xs[u][t]),
                                                       t % (4 / GROUPS) == 0 ? zero : part, 0, 0, 0);
        if ((t + 1) % (4 / GROUPS) == 0) {
          const uint2 b = s[u][j][t / (4 / GROUPS)];
          const float f[4] = {__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u)};
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(f[e], part[e], acc[j][e]);
        }
      }
    }
  };
  if (lo < hi) {
#pragma unroll
    for (int u = 0; u < D; ++u) load(u, min(lo + u, hi - 1));
    int kb = lo;
    for (; kb + D < hi; kb += D) {
#pragma unroll
      for (int u = 0; u < D; ++u) {
        multiply(u, kb + u);
        load(u, min(kb + D + u, hi - 1));
      }
    }
#pragma unroll
    for (int u = 0; u < D; ++u)
      if (kb + u < hi) multiply(u, kb + u);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) *reinterpret_cast<fp4_f32x4*>(lds + (wave * NT + j) * 1024 + lane * 16) = acc[j];
  __syncthreads();
  const int slot = m0 + r16;
  int to = slot;
  if (c.out_of) to = c.out_of[slot];
  else if (slot >= c.M) to = -1;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (j % W != wave) continue;
    fp4_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < W; ++k) v += *reinterpret_cast<const fp4_f32x4*>(lds + (k * NT + j) * 1024 + lane * 16);
    const int n = (tile0 + j) * FP4_ROWS + 4 * kq;
    if (to >= 0 && n < c.w.N) fp4_store(c, v, to, n, c.factor ? c.factor[slot] : 1.f);
  }
}

template <int NT, int W, int D, bool WHOLE>
int run_few(const Fp4Case& c, int mtiles, hipStream_t s) {
  const dim3 grid((c.w.tiles + NT - 1) / NT, mtiles);
  if (c.w.group == 128) fp4_few_kernel<NT, W, D, 1, WHOLE><<<grid, 64 * W, 0, s>>>(c);
  else if (c.w.group == 64) fp4_few_kernel<NT, W, D, 2, WHOLE><<<grid, 64 * W, 0, s>>>(c);
  else fp4_few_kernel<NT, W, D, 4, WHOLE><<<grid, 64 * W, 0, s>>>(c);
  return he_check_launch("he_fp4_product");
}

}  // namespace

int fp4_run_few(const Fp4Case& c, int mtiles, hipStream_t s) {
  HE_REQUIRE(mtiles <= 65535, "he_fp4_product: %d tiles of rows are too many for one launch", mtiles);
  if (!c.whole || c.w.K % 8) return run_few<1, 8, 2, false>(c, mtiles, s);
  // The fewest tiles a workgroup that leave enough workgroups: X is read once a workgroup. Microseconds of 1 tile of 8 wavefronts, 2 of 4, 4 of 4:
  // 1 row of 4608 x 3584 6.7, 5.7, 8.1; 3584 x 18944 14.0, 16.9, 26.9; 5120 x 27648 31.1, 23.7, 37.7; 8 rows of 37888 x 3584 31.9, 22.9, 21.5.
  const int64_t tiles = (int64_t)c.w.tiles * mtiles;
  if (tiles >= 2048) return run_few<4, 4, 2, true>(c, mtiles, s);
  if (tiles >= 256 || c.w.blocks <= 32) return run_few<2, 4, 2, true>(c, mtiles, s);
  return run_few<1, 8, 2, true>(c, mtiles, s);
}
