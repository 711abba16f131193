// Products with a weight in 4 bits (fp4.h): out[m][n] = sum_k X[m][k] W[n][k], the rows X bf16, sums 32-bit.
#include "fp4.h"

namespace {

// One workgroup: WN x WK wavefronts. The WN have NT tiles of 16 weight rows each, the WK of them share the blocks of 128 k in turn; MT tiles of
// 16 rows of X (XR of which are kept, where there are no more: the operand's other rows repeat them). X goes through LDS in stretches of CB
// blocks, in the order the operands are read; the codes come straight from memory, a lane's 16 bytes a block, two blocks a
// wavefront ahead. A group's products run into an accumulator of their own, which joins the sums times its scale.
template <int MT, int XR, int NT, int WN, int WK, int CB, int GROUPS>
__global__ __launch_bounds__(64 * WN * WK) void fp4_rows_kernel(Fp4Case c) {
  constexpr int THREADS = 64 * WN * WK, U = CB / WK;       // blocks of a wavefront in a stretch
  constexpr int STEP = MT * XR * 64, STRETCH = CB * 4 * STEP;      // bytes of 32 k, of a stretch
  static_assert(CB % WK == 0 && (MT == 1 || XR == 16), "the stretches");
  constexpr int JOIN = WK > 1 ? WK * WN * MT * NT * 1024 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STRETCH > JOIN ? 2 * STRETCH : JOIN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wk = wave / WN, r16 = lane & 15, kq = lane >> 4;
  const int blocks = c.w.blocks;
  int m0 = blockIdx.y * (16 * MT), group = 0;
  if (c.tile_begin) {
    if ((int)blockIdx.y >= c.tile_begin[c.groups]) return;
    int lo = 0, hi = c.groups;                             // the last group that begins at or before this tile
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (c.tile_begin[mid] <= (int)blockIdx.y) lo = mid;
      else hi = mid;
    }
    group = lo;
  }
  const int tile0 = (blockIdx.x * WN + wn) * NT;
  const uint8_t* codes[NT];
  const uint16_t* scales[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t at = ((int64_t)group * c.w.tiles + min(tile0 + j, c.w.tiles - 1)) * blocks;
    codes[j] = c.w.codes + at * FP4_TILE_BYTES + lane * 16;
    scales[j] = c.w.scales + at * (16 * GROUPS) + 4 * kq;
  }

  // X: pieces of eight k, the rows of a piece behind each other
  constexpr int PIECES = CB * 16 * MT * XR, EACH = (PIECES + THREADS - 1) / THREADS;
  uint4 xv[EACH];
  auto fetch = [&](int kb0) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = tid + i * THREADS, r = at % (MT * XR), k = kb0 * FP4_K + at / (MT * XR) * 8;
      xv[i] = make_uint4(0, 0, 0, 0);
      int row = m0 + r;
      if (at >= PIECES || k >= c.w.K) continue;
      if (c.rows_of) row = c.rows_of[row];
      else if (row >= c.M) row = -1;
      if (row < 0) continue;
      const uint16_t* p = c.x + row * c.ldx + k;
      if (c.whole && k + 8 <= c.w.K) {
        xv[i] = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < c.w.K) words[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
        xv[i] = make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
  };
  auto keep = [&](int at) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int p = tid + i * THREADS, r = p % (MT * XR), piece = p / (MT * XR);
      if (p >= PIECES) continue;
      // [32 k][tile of rows][eight k][row]
      *reinterpret_cast<uint4*>(lds + at + (piece >> 2) * STEP + (r / XR) * (XR * 64) + ((piece & 3) * XR + r % XR) * 16) = xv[i];
    }
  };

  fp4_f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = fp4_f32x4{0.f, 0.f, 0.f, 0.f};
  uint4 q[U][NT];
  uint2 s[U][NT][GROUPS];
  auto load = [&](int u, int kb) {
    const int at = min(kb, blocks - 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      q[u][j] = he_load16_once<uint4>(codes[j] + (int64_t)at * FP4_TILE_BYTES);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) s[u][j][g] = *reinterpret_cast<const uint2*>(scales[j] + (int64_t)at * (16 * GROUPS) + 16 * g);
    }
  };
  fetch(0);
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, wk * U + u);
  keep(0);
  int at = 0;
  for (int kb0 = 0; kb0 < blocks; kb0 += CB) {
    __syncthreads();
    const bool more = kb0 + CB < blocks;
    if (more) fetch(kb0 + CB);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + wk * U + u;
      if (kb < blocks) {
        const uint8_t* x = lds + at + (wk * U + u) * 4 * STEP + (kq * XR + r16 % XR) * 16;
        fp4_f32x4 part[MT][NT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          fp4_bf16x8 xs[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) xs[i] = *reinterpret_cast<const fp4_bf16x8*>(x + t * STEP + i * XR * 64);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint32_t words[4] = {q[u][j].x, q[u][j].y, q[u][j].z, q[u][j].w};
            const fp4_bf16x8 w = fp4_operand(words[t]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const fp4_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
              part[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xs[i], t % (4 / GROUPS) == 0 ? zero : part[i][j], 0, 0, 0);
            }
            if ((t + 1) % (4 / GROUPS) == 0) {
              const uint2 b = s[u][j][t / (4 / GROUPS)];
              const float f[4] = {__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u)};
#pragma unroll
              for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(f[e], part[i][j][e], acc[i][j][e]);
            }
          }
        }
      }
      load(u, kb + CB);
    }
    at ^= STRETCH;
    if (more) keep(at);
  }

  if (WK > 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        *reinterpret_cast<fp4_f32x4*>(lds + (((wk * WN + wn) * MT + i) * NT + j) * 1024 + lane * 16) = acc[i][j];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int slot = m0 + 16 * i + r16;
    int to = slot;
    if (c.out_of) to = c.out_of[slot];
    else if (slot >= c.M) to = -1;
    const float f = c.factor && to >= 0 ? c.factor[slot] : 1.f;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (WK > 1 && (i * NT + j) % WK != wk) continue;
      fp4_f32x4 v = acc[i][j];
      if (WK > 1) {
        v = fp4_f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < WK; ++k) v += *reinterpret_cast<const fp4_f32x4*>(lds + (((k * WN + wn) * MT + i) * NT + j) * 1024 + lane * 16);
      }
      const int n = (tile0 + j) * FP4_ROWS + 4 * kq;
      if (to < 0 || n >= c.w.N) continue;
      if (c.gated) {
        uint16_t* p = (uint16_t*)c.out + to * c.ldo + n / 2;
        auto act = [&](float g, float u) {
          const float a = c.clamped ? he_gated_act<true>(g, u, c.act) : he_gated_act<false>(g, u, c.act);
          return f == 0.f ? 0.f : a * f;
        };
        const uint32_t pair = pack2_bf16(act(v[0], v[1]), act(v[2], v[3]));
        p[0] = (uint16_t)pair;
        if (n + 2 < c.w.N) p[1] = (uint16_t)(pair >> 16);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= c.w.N) break;
        float y = v[e] * f;
        if (c.bias) y += load_param(c.bias, n + e, c.bias_dtype);
        if (c.out_f32) ((float*)c.out)[to * c.ldo + n + e] = y;
        else ((uint16_t*)c.out)[to * c.ldo + n + e] = float_to_bf16_bits(y);
      }
    }
  }
}

template <int MT, int XR, int NT, int WN, int WK, int CB>
int run_rows(const Fp4Case& c, int mtiles, hipStream_t s) {
  const dim3 grid((c.w.tiles + WN * NT - 1) / (WN * NT), mtiles);
  const int threads = 64 * WN * WK;
  if (c.w.group == 128) fp4_rows_kernel<MT, XR, NT, WN, WK, CB, 1><<<grid, threads, 0, s>>>(c);
  else if (c.w.group == 64) fp4_rows_kernel<MT, XR, NT, WN, WK, CB, 2><<<grid, threads, 0, s>>>(c);
  else fp4_rows_kernel<MT, XR, NT, WN, WK, CB, 4><<<grid, threads, 0, s>>>(c);
  return he_check_launch("he_fp4_product");
}

// rows in tiles of bm (16, 32 or 64), mtiles of them at most
int run(const Fp4Case& c, int bm, int mtiles, hipStream_t s) {
  if (mtiles == 0) return 0;
  HE_REQUIRE(mtiles <= 65535, "he_fp4_product: %d tiles of rows are too many for one launch", mtiles);
  if (bm == 16) return run_rows<1, 16, 1, 1, 8, 8>(c, mtiles, s);
  if (bm == 32) return run_rows<2, 16, 2, 4, 1, 4>(c, mtiles, s);
  return run_rows<4, 16, 2, 4, 1, 2>(c, mtiles, s);
}

int check_weight(const char* what, const Fp4Weight& w) {
  HE_REQUIRE(w.N > 0 && w.K > 0 && w.N <= (1 << 26) && w.K <= (1 << 26), "%s: a weight of [%d, %d]", what, w.N, w.K);
  HE_REQUIRE(w.group == 32 || w.group == 64 || w.group == 128, "%s: groups of %d (32, 64 or 128)", what, w.group);
  HE_REQUIRE(w.codes && w.scales && (((uintptr_t)w.codes | (uintptr_t)w.scales) & 15) == 0, "%s: codes and scales must be 16-byte aligned", what);
  return 0;
}

Fp4Weight weight(const void* codes, const void* scales, int N, int K, int group) {
  return {(const uint8_t*)codes, (const uint16_t*)scales, N, K, group, (N + FP4_ROWS - 1) / FP4_ROWS, (K + FP4_K - 1) / FP4_K};
}

bool whole_rows(const void* x, int64_t ldx) { return ((uintptr_t)x & 15) == 0 && ldx % 8 == 0; }

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The scratch of the experts of a step: the lists of he_group_rows, the activations and the results of each choice.
struct ExpertsScratch {
  int bm, mtiles;
  int64_t ints, h, partial, bytes;
};
ExpertsScratch experts_scratch(int rows, int top, int experts, int I, int D) {
  ExpertsScratch t;
  const int64_t choices = (int64_t)rows * top;
  t.bm = choices <= 16ll * experts ? 16 : choices <= 32ll * experts ? 32 : 64;
  t.mtiles = he_group_rows_most_tiles(rows, top, experts, t.bm);
  t.ints = padded(4 * he_group_rows_ints(rows, top, experts, t.bm));
  t.h = padded(choices * I * 2);
  t.partial = padded(choices * D * 4);
  t.bytes = t.ints + t.h + t.partial;
  return t;
}

// out[row] = the sum over the row's choices, in their order, of those that an expert took
__global__ __launch_bounds__(256) void add_choices_kernel(uint16_t* __restrict__ out, const float* __restrict__ partial, const int32_t* __restrict__ ids,
                                                          int top, int experts, int D) {
  const int64_t row = blockIdx.y;
  const int d = blockIdx.x * 256 + threadIdx.x;
  if (d >= D) return;
  float sum = 0.f;
  for (int k = 0; k < top; ++k) {
    const int id = ids[row * top + k];
    if (id >= 0 && id < experts) sum += partial[(row * top + k) * D + d];
  }
  out[row * D + d] = float_to_bf16_bits(sum);
}

}  // namespace

extern "C" int64_t he_fp4_product_workspace_bytes(int M, int N, int K, int gated) { return 0; }

extern "C" int he_fp4_product(void* out, int64_t ldo, const void* x, int64_t ldx, const void* codes, const void* scales, const void* bias, int M, int N,
                              int K, int group, int out_dtype, int bias_dtype, int gated, float alpha, float limit, float up_shift, float cubic,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  Fp4Case c = {};
  c.w = weight(codes, scales, N, K, group);
  if (const int rc = check_weight("he_fp4_product", c.w)) return rc;
  HE_REQUIRE(M >= 0 && ldx >= K && ldo >= (gated ? N / 2 : N), "he_fp4_product: %d rows of %d at distances %lld and %lld", M, K, (long long)ldx, (long long)ldo);
  HE_REQUIRE(out_dtype == HE_F32 || out_dtype == HE_BF16, "he_fp4_product: dtype code %d", out_dtype);
  HE_REQUIRE(!gated || (N % 2 == 0 && out_dtype == HE_BF16 && !bias), "he_fp4_product: a gated product has an even N, bfloat16 results and no bias");
  if (M == 0) return 0;
  c.x = (const uint16_t*)x, c.ldx = ldx, c.whole = whole_rows(x, ldx);
  c.out = out, c.ldo = ldo, c.out_f32 = out_dtype == HE_F32, c.gated = gated;
  c.clamped = !he_gated_act_is_silu(alpha, limit, up_shift, cubic);
  c.bias = bias, c.bias_dtype = bias_dtype, c.M = M;
  c.act = {alpha, limit > 0.f ? limit : INFINITY, up_shift, cubic};
  const int bm = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  return run(c, bm, (M + bm - 1) / bm, (hipStream_t)stream);
}

extern "C" int64_t he_fp4_experts_workspace_bytes(int rows, int top, int experts, int I, int D) {
  if (rows <= 0 || top <= 0 || experts <= 0 || I <= 0 || D <= 0) return 0;
  return experts_scratch(rows, top, experts, I, D).bytes;
}

extern "C" int he_fp4_experts(void* out, const void* x, int64_t ldx, const void* up_codes, const void* up_scales, const void* down_codes,
                              const void* down_scales, const void* ids_i32, const void* weights_f32, int rows, int top, int experts, int I, int D,
                              int group_up, int group_down, float alpha, float limit, float up_shift, float cubic, void* workspace, int64_t workspace_bytes, void* stream) {
  HE_REQUIRE(rows >= 0 && top > 0 && experts > 0 && I > 0 && D > 0 && I <= (1 << 25), "he_fp4_experts: bad sizes");
  HE_REQUIRE(experts <= HE_GROUP_ROWS_MOST && rows <= 65535 && (int64_t)rows * top < (1 << 26), "he_fp4_experts: %d experts and %d rows are too many", experts, rows);
  HE_REQUIRE(ldx >= D, "he_fp4_experts: rows of %d at a distance of %lld", D, (long long)ldx);
  Fp4Case up = {}, down = {};
  up.w = weight(up_codes, up_scales, 2 * I, D, group_up);
  down.w = weight(down_codes, down_scales, D, I, group_down);
  if (const int rc = check_weight("he_fp4_experts", up.w)) return rc;
  if (const int rc = check_weight("he_fp4_experts", down.w)) return rc;
  if (rows == 0) return 0;
  const ExpertsScratch t = experts_scratch(rows, top, experts, I, D);
  HE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= t.bytes, "he_fp4_experts: a workspace of %lld bytes, 16-byte aligned, is needed",
             (long long)t.bytes);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* p = (uint8_t*)workspace;
  GroupRows lists;
  int rc = he_group_rows(&lists, p, ids_i32, weights_f32, rows, top, experts, t.bm, stream);
  if (rc) return rc;
  uint16_t* h = (uint16_t*)(p + t.ints);
  float* partial = (float*)(p + t.ints + t.h);
  up.x = (const uint16_t*)x, up.ldx = ldx, up.whole = whole_rows(x, ldx);
  up.out = h, up.ldo = I, up.gated = true, up.clamped = !he_gated_act_is_silu(alpha, limit, up_shift, cubic);
  up.act = {alpha, limit > 0.f ? limit : INFINITY, up_shift, cubic};
  up.tile_begin = lists.tile_begin, up.groups = experts, up.rows_of = lists.rows_of, up.out_of = lists.choice_of, up.factor = lists.scale;
  if ((rc = run(up, t.bm, t.mtiles, s))) return rc;
  down.x = h, down.ldx = I, down.whole = whole_rows(h, I);
  down.out = partial, down.ldo = D, down.out_f32 = true;
  down.tile_begin = lists.tile_begin, down.groups = experts, down.rows_of = down.out_of = lists.choice_of;
  if ((rc = run(down, t.bm, t.mtiles, s))) return rc;
  add_choices_kernel<<<dim3((D + 255) / 256, rows), 256, 0, s>>>((uint16_t*)out, partial, (const int32_t*)ids_i32, top, experts, D);
  return he_check_launch("he_fp4_experts");
}
