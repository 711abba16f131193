// Products with a weight in 4 bits (fp4.h): out[m][n] = sum_k X[m][k] W[n][k], the rows X bf16, sums 32-bit.
#include <algorithm>
#include "fp4.h"

namespace {

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

bool far(int64_t rows, int64_t ld) { return rows * ld * 2 >= 1ll << 32; }

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int64_t padded_k(int K) { return ((int64_t)K + FP4_K - 1) / FP4_K * FP4_K; }

// rows of `pieces` times eight values: x's, then zeros
__global__ __launch_bounds__(256) void pad_rows_kernel(uint4* __restrict__ out, const uint16_t* __restrict__ x, int64_t ldx, int K, int pieces, int64_t total, bool whole) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  const int64_t r = at / pieces;
  const int p = (int)(at - r * pieces);
  const uint16_t* row = x + r * ldx;
  if (whole && 8 * p + 8 <= K) {
    out[at] = *reinterpret_cast<const uint4*>(row + 8 * p);
    return;
  }
  uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (8 * p + e < K) words[e >> 1] |= (uint32_t)row[8 * p + e] << (16 * (e & 1));
  out[at] = make_uint4(words[0], words[1], words[2], words[3]);
}
// X copied to `to`, its rows filled up to whole blocks
int pad_rows(Fp4Case* c, void* to, hipStream_t s) {
  const int64_t ld = padded_k(c->w.K), total = c->M * (ld / 8);
  pad_rows_kernel<<<(unsigned)((total + 255) / 256), 256, 0, s>>>((uint4*)to, c->x, c->ldx, c->w.K, (int)(ld / 8), total, c->whole);
  c->x = (const uint16_t*)to, c->ldx = ld, c->whole = true, c->w.K = (int)ld;
  return he_check_launch("he_fp4_product (rows)");
}
__global__ __launch_bounds__(256) void clear_columns_kernel(uint16_t* __restrict__ h, int64_t rows, int I, int ld) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at < rows * (ld - I)) h[at / (ld - I) * ld + I + at % (ld - I)] = 0;
}

// The rows of a turn of a product: the kernel of many rows counts the bytes of X in 32 bits.
int turn_rows(int M, int K) {
  const int64_t most = ((1ll << 32) - 1) / (2 * padded_k(K)), tile = most >= 128 ? 128 : 16;
  return (int)std::min<int64_t>(M, most / tile * tile);
}

// How a product is cut. Up to 16 rows run through the kernel that has no barriers (fp4_few.hip; 16 rows of 37888 x 3584 20.8 us, 22 in tiles of 32
// rows; 3584 x 18944 16.4 and 19.4), and so do more, 16 at a time, where the weight is small (mt 0): it reads the codes again for
// each 16, at some 4300 blocks of 128 k of 16 rows a microsecond. Tiles of more rows: a tile's time is its blocks of 128 k times the
// microseconds that a block (of each part of K) takes, alone on its unit or as its share of a unit that has several; the fewest over the shapes and the
// slices of K, whose sums cost two passes over them and a launch. (64 rows of 1024 x 3584 5.7 us in sixteens, 9.8 in tiles; of 4608 x 3584 11.1, 14; of
// 37888 x 3584 65 by the estimate, 27 to 31 in tiles. The figures are fitted to 46 products of 17 to 2048 rows, 800 to 39472 columns and K of 768 to 23040 in 40
// shapes and slices: what is chosen takes 1.02 of the time of the best in the geometric mean, 1.15 at most.)
Fp4Plan plan_of(int64_t M, int N, int K) {
  static const struct { int mt, nt, parts; double alone, shared; } shapes[] = {
      {2, 1, 2, 0.45, 0.54}, {2, 2, 2, 1.08, 0.73}, {4, 1, 1, 0.53, 0.35}, {4, 1, 2, 0.82, 0.84}, {4, 2, 2, 1.13, 1.22}, {8, 2, 1, 1.07, 0.91}, {8, 4, 1, 1.96, 1.6}};
  const int blocks = (K + FP4_K - 1) / FP4_K, cus = he_cus();
  Fp4Plan best = {0, 0, 1, 1};
  if (M <= 16) return best;
  const int64_t sixteens = (M + 15) / 16;
  double least = sixteens > 65535 ? INFINITY : 3 + 0.03 * blocks + (double)(sixteens * ((N + 15) / 16) * blocks) / 4300;      // (of a launch 65535 at most)
  for (const auto& t : shapes) {
    const int64_t tiles = (M + 16 * t.mt - 1) / (16 * t.mt) * ((N + 64 * t.nt - 1) / (64 * t.nt));
    for (int slices = 1; slices <= 16 && slices * t.parts <= blocks; slices *= 2) {
      const double load = tiles * slices > 8 * cus ? (double)tiles * slices / cus : (double)((tiles * slices + cus - 1) / cus);
      const double turn = load * t.shared > t.alone ? load * t.shared : t.alone;
      const double us = 3 + (blocks + slices * t.parts - 1) / (slices * t.parts) * turn + (slices > 1 ? 4 + 5e-6 * slices * M * N / 4 : 0) + (K % FP4_K ? 2.5 : 0);
      if (us < least) least = us, best = {t.mt, t.nt, t.parts, slices};
    }
  }
  return best;
}

// The scratch of a product's turn: the rows, where the kernel cannot read them as they are, then the slices' sums.
struct ProductScratch {
  Fp4Plan plan;
  bool copy;
  int64_t rows, bytes;
};
ProductScratch product_scratch(int M, int N, int K, bool whole) {
  ProductScratch t;
  t.plan = plan_of(M, N, K);
  t.copy = t.plan.mt ? !whole || K % FP4_K : K < 8;
  t.rows = t.copy ? padded(M * padded_k(K) * 2) : 0;
  t.bytes = t.rows + (t.plan.slices > 1 ? (int64_t)t.plan.slices * M * ((N + 15) / 16 * 16) * 4 : 0);
  return t;
}
// of all turns
int64_t product_bytes(int M, int N, int K, bool whole) {
  const int turn = turn_rows(M, K);
  return std::max(product_scratch(turn, N, K, whole).bytes, M % turn ? product_scratch(M % turn, N, K, whole).bytes : 0);
}

// Of any number of rows up to M: fewer rows may be cut into more slices (3584 x 18944: 512 rows in 4, 513 in none). Costs of slices grow evenly within sixteen rows, all
// others stay: where the first and the last of them have one plan, so have those between. Where every shape has more than eight tiles a unit none has slices.
int64_t most_product_bytes(int M, int N, int K, bool whole) {
  M = turn_rows(M, K);
  int64_t most = product_scratch(M, N, K, whole).bytes;
  for (int lo = 17; lo <= M; lo += 16) {
    if ((int64_t)(lo + 127) / 128 * ((N + 255) / 256) > 8 * he_cus()) {
      for (int hi = M; (!whole || K % FP4_K) && hi >= lo; hi = (hi - 1) / 16 * 16)      // the rows alone, of the last that are copied
        if (const ProductScratch t = product_scratch(hi, N, K, whole); t.plan.mt) return std::max(most, t.bytes);
      return most;
    }
    const ProductScratch a = product_scratch(lo, N, K, whole), b = product_scratch(std::min(lo + 15, M), N, K, whole);
    most = std::max({most, a.bytes, b.bytes});
    if (a.plan.slices == b.plan.slices && !a.plan.mt == !b.plan.mt) continue;
    for (int m = lo + 1; m < std::min(lo + 15, M); ++m) most = std::max(most, product_scratch(m, N, K, whole).bytes);
  }
  return most;
}

// The scratch of the experts of a step: the lists of he_group_rows, the activations and the results of each choice, and X where its
// rows are not whole blocks.
struct ExpertsScratch {
  int bm, mtiles;
  Fp4Plan up, down;
  int64_t ints, h, ldh, partial, x, bytes;
};
ExpertsScratch experts_scratch(int rows, int top, int experts, int I, int D) {
  ExpertsScratch t = {};
  const int64_t choices = (int64_t)rows * top;
  // A tile of rows should hold an expert's rows, of which there are more with some experts than with others. Microseconds in tiles of 4, 8, 16, 32, 64,
  // 128 rows of 16 experts of 2048 over rows of 2048, 4 chosen: 8 rows 29, 29, 36, 40; 16 rows 33, 32, 36, 44; 32 rows 47, 39, 37, 42, 49; 48 rows 59, 44, 41,
  // 46, 49; 64 rows 73, 51, 44, 45, 49; 128 rows 122, 74, 62, 50, 53; 256 rows -, -, -, 80, 68, 100; 512 rows -, -, -, 127, 94, 112; 768 rows 181, 132, 124; 1536 rows
  // 346, 233, 208. (64 rows in groups of 32: 57 in tiles of 16, 45 of 32.) Tiles of 64 rows are 128 columns wide (512 rows 94 us, 64 columns 109, whose rows
  // are read twice as often), of 32 rows 64 (64 experts of 768, 128 rows, 8 chosen: 57 us, 59 with 128).
  t.bm = choices <= 3ll * experts ? 4 : choices <= 5ll * experts ? 8 : choices <= 12ll * experts ? 16 : choices <= 32ll * experts ? 32 : choices <= 160ll * experts ? 64 : 128;
  t.mtiles = he_group_rows_most_tiles(rows, top, experts, t.bm);
  t.up = t.down = {t.bm / 16, t.bm / 32, 1, 1};
  t.ints = padded(4 * he_group_rows_ints(rows, top, experts, t.bm));
  t.ldh = t.bm <= 16 ? (I + 7) / 8 * 8 : padded_k(I);
  t.h = padded(choices * t.ldh * 2);
  t.partial = padded(choices * D * 4);
  t.x = padded(rows * padded_k(D) * 2);
  t.bytes = t.ints + t.h + t.partial + t.x;
  return t;
}

// out[row] = plus[row] (or null) + the sum over the row's choices, in their order, of those that an expert took (with a weight that is not zero), and of weight * x of those from
// `experts` on (x null: they add nothing)
__global__ __launch_bounds__(256) void add_choices_kernel(uint16_t* __restrict__ out, const float* __restrict__ partial, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ weights, const uint16_t* __restrict__ x, int64_t ldx,
                                                          const float* __restrict__ plus, int top, int experts, int D) {
  const int64_t row = blockIdx.y;
  const int d = 4 * (blockIdx.x * 256 + threadIdx.x);
  if (d >= D) return;
  const int n = min(4, D - d);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (plus)
    for (int i = 0; i < n; ++i) sum[i] = plus[row * D + d + i];
  for (int k = 0; k < top; ++k) {
    const int64_t choice = row * top + k;
    const int id = ids[choice];
    if (id < 0 || (id >= experts && !x)) continue;
    const float w = weights[choice];
    if (w == 0.f) continue;
    if (id >= experts) {
      for (int i = 0; i < n; ++i) sum[i] = fmaf(w, bf16_bits_to_float(x[row * ldx + d + i]), sum[i]);
    } else if (D % 4 == 0) {
      const float4 v = *reinterpret_cast<const float4*>(partial + choice * D + d);
      sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
    } else {
      for (int i = 0; i < n; ++i) sum[i] += partial[choice * D + d + i];
    }
  }
  for (int i = 0; i < n; ++i) out[row * D + d + i] = float_to_bf16_bits(sum[i]);
}

}  // namespace

extern "C" int64_t he_fp4_product_workspace_bytes(int M, int N, int K, int whole) {
  return M <= 0 || N <= 0 || K <= 0 ? 0 : most_product_bytes(M, N, K, whole);
}
extern "C" int64_t he_fp4_product_call_bytes(int M, int N, int K, int whole) {
  return M <= 0 || N <= 0 || K <= 0 ? 0 : product_bytes(M, N, K, whole);
}

// the case of he_fp4_product without its results
static int product_case(Fp4Case* c, const void* x, int64_t ldx, const void* codes, const void* scales, const void* bias, int M, int N, int K, int group,
                        int bias_dtype) {
  *c = {};
  c->w = weight(codes, scales, N, K, group);
  if (const int rc = check_weight("he_fp4_product", c->w)) return rc;
  HE_REQUIRE(M >= 0 && M <= (1 << 22) && ldx >= K, "he_fp4_product: %d rows of %d at distances of %lld", M, K, (long long)ldx);
  c->x = (const uint16_t*)x, c->ldx = ldx, c->whole = whole_rows(x, ldx), c->M = M, c->bias = bias, c->bias_dtype = bias_dtype;
  return 0;
}

static void results(Fp4Case* c, void* out, int64_t ldo, int out_dtype, int gated, GatedAct act) {
  c->out = out, c->ldo = ldo, c->out_f32 = out_dtype == HE_F32, c->gated = gated;
  c->silu = he_gated_act_is_silu(act.alpha, act.limit, act.shift, act.cubic);
  c->act = act;
  if (!(act.limit > 0.f)) c->act.limit = INFINITY;
  c->pairs = ldo % (gated ? 2 : 4) == 0 && ((uintptr_t)out & (out_dtype == HE_F32 ? 15 : gated ? 3 : 7)) == 0;
}

extern "C" int he_fp4_product(void* out, int64_t ldo, const void* x, int64_t ldx, const void* codes, const void* scales, const void* bias, int M, int N,
                              int K, int group, int out_dtype, int bias_dtype, int gated, float alpha, float limit, float up_shift, float cubic,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  Fp4Case c;
  if (const int rc = product_case(&c, x, ldx, codes, scales, bias, M, N, K, group, bias_dtype)) return rc;
  HE_REQUIRE(ldo >= (gated ? N / 2 : N), "he_fp4_product: results of %d at distances of %lld", gated ? N / 2 : N, (long long)ldo);
  HE_REQUIRE(out_dtype == HE_F32 || out_dtype == HE_BF16, "he_fp4_product: dtype code %d", out_dtype);
  HE_REQUIRE(!gated || (N % 2 == 0 && out_dtype == HE_BF16 && !bias), "he_fp4_product: a gated product has an even N, bfloat16 results and no bias");
  if (M == 0) return 0;
  results(&c, out, ldo, out_dtype, gated, {alpha, limit, up_shift, cubic});
  hipStream_t s = (hipStream_t)stream;
  const int turn = turn_rows(M, K);
  const bool whole = c.whole && !far(turn, ldx);
  const ProductScratch first = product_scratch(turn, N, K, whole), last = M % turn ? product_scratch(M % turn, N, K, whole) : first;
  const int64_t need = std::max(first.bytes, last.bytes);
  HE_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
             "he_fp4_product: a workspace of %lld bytes, 16-byte aligned, is needed", (long long)need);
  for (int r0 = 0; r0 < M; r0 += turn) {
    Fp4Case part = c;
    const int n = part.M = std::min(turn, M - r0);
    part.x += r0 * ldx, part.out = (uint8_t*)out + r0 * ldo * (c.out_f32 ? 4 : 2);
    const ProductScratch& t = n == turn ? first : last;
    if (t.copy)
      if (const int rc = pad_rows(&part, workspace, s)) return rc;
    const int rc = t.plan.mt == 0 ? fp4_run_few(part, n > 8 ? 16 : n > 4 ? 8 : 4, (n + 15) / 16, s)
                                  : fp4_run_tall(part, t.plan, (n + 16 * t.plan.mt - 1) / (16 * t.plan.mt), (float*)((uint8_t*)workspace + t.rows), s);
    if (rc) return rc;
  }
  return 0;
}

extern "C" int he_fp4_product_carried(void* out, int64_t ldo, const void* x, int64_t ldx, const void* codes, const void* scales, const void* bias, int M,
                                      int N, int K, int group, int out_dtype, int bias_dtype, int gated, float alpha, float limit, float up_shift, float cubic,
                                      const void* owed, int owed_count, float owed_eps, void* resid, float resid_scale, const void* gain, int gain_dtype,
                                      void* carried, void* squares, void* stream) {
  Fp4Case c;
  if (const int rc = product_case(&c, x, ldx, codes, scales, bias, M, N, K, group, bias_dtype)) return rc;
  HE_REQUIRE(M <= 16 && K >= 8, "he_fp4_product_carried: %d rows of %d (up to 16, of 8 or more)", M, K);
  HE_REQUIRE(!owed || owed_count > 0, "he_fp4_product_carried: %d sums of squares a row", owed_count);
  if (resid) {
    HE_REQUIRE(N % 4 == 0 && !gated && !out && gain && carried && squares && (((uintptr_t)resid & 15) | ((uintptr_t)carried & 7)) == 0,
               "he_fp4_product_carried: results for the residual rows are not gated, N is a multiple of 4, their buffers are there and aligned");
  } else {
    HE_REQUIRE(out && ldo >= (gated ? N / 2 : N) && (out_dtype == HE_F32 || out_dtype == HE_BF16), "he_fp4_product_carried: results of dtype code %d at distances of %lld", out_dtype, (long long)ldo);
    HE_REQUIRE(!gated || (N % 2 == 0 && out_dtype == HE_BF16 && !bias), "he_fp4_product_carried: a gated product has an even N, bfloat16 results and no bias");
  }
  if (M == 0) return 0;
  results(&c, out, ldo, out_dtype, gated, {alpha, limit, up_shift, cubic});
  c.owed = (const float*)owed, c.owed_count = owed_count, c.owed_dim = K, c.owed_eps = owed_eps;
  c.resid = (float*)resid, c.resid_scale = resid_scale, c.gain = gain, c.gain_dtype = gain_dtype, c.carried = (uint16_t*)carried, c.squares = (float*)squares;
  return fp4_run_few(c, M > 8 ? 16 : M > 4 ? 8 : 4, 1, (hipStream_t)stream);
}

extern "C" int64_t he_fp4_experts_workspace_bytes(int rows, int top, int experts, int I, int D) {
  if (rows <= 0 || top <= 0 || experts <= 0 || I <= 0 || D <= 0) return 0;
  return experts_scratch(rows, top, experts, I, D).bytes;
}

extern "C" int he_fp4_experts(void* out, const void* x, int64_t ldx, const void* up_codes, const void* up_scales, const void* down_codes,
                              const void* down_scales, const void* ids_i32, const void* weights_f32, int rows, int top, int experts, int I, int D,
                              int group_up, int group_down, int identity, float alpha, float limit, float up_shift, float cubic, void* workspace, int64_t workspace_bytes, void* stream) {
  return he_fp4_experts_plus(out, x, ldx, up_codes, up_scales, down_codes, down_scales, ids_i32, weights_f32, nullptr, rows, top, experts, I, D, group_up, group_down, identity,
                             alpha, limit, up_shift, cubic, workspace, workspace_bytes, stream);
}

extern "C" int he_fp4_experts_plus(void* out, const void* x, int64_t ldx, const void* up_codes, const void* up_scales, const void* down_codes,
                                   const void* down_scales, const void* ids_i32, const void* weights_f32, const void* plus_f32, int rows, int top, int experts, int I, int D,
                                   int group_up, int group_down, int identity, float alpha, float limit, float up_shift, float cubic, void* workspace, int64_t workspace_bytes, void* stream) {
  HE_REQUIRE(rows >= 0 && top > 0 && experts > 0 && I > 0 && D > 0 && I <= (1 << 25), "he_fp4_experts: bad sizes");
  HE_REQUIRE(experts <= HE_GROUP_ROWS_MOST && rows <= 65535 && (int64_t)rows * top < (1 << 26), "he_fp4_experts: %d experts and %d rows are too many", experts, rows);
  HE_REQUIRE(ldx >= D, "he_fp4_experts: rows of %d at a distance of %lld", D, (long long)ldx);
  Fp4Case up = {}, down = {};
  up.w = weight(up_codes, up_scales, 2 * I, D, group_up);
  down.w = weight(down_codes, down_scales, D, I, group_down);
  if (const int rc = check_weight("he_fp4_experts", up.w)) return rc;
  if (const int rc = check_weight("he_fp4_experts", down.w)) return rc;
  HE_REQUIRE(!far((int64_t)rows * top, padded_k(I)) && !far(rows, padded_k(D)), "he_fp4_experts: %d rows of %d choices are too many", rows, top);
  if (rows == 0) return 0;
  const ExpertsScratch t = experts_scratch(rows, top, experts, I, D);
  HE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= t.bytes, "he_fp4_experts: a workspace of %lld bytes, 16-byte aligned, is needed",
             (long long)t.bytes);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* p = (uint8_t*)workspace;
  const int choices = rows * top;
  // few choices are grouped by the products themselves: a launch less (16 experts of 2048 over rows of 2048, 4 chosen: 1 row 16.2 us -> 11.5, its second
  // product's sums taken over the choices too; 4 rows 24.9 -> 22.3); by many more every workgroup searches for longer than the launch takes (8 rows 28.0 -> 30.4)
  const bool by_ids = t.bm <= 16 && choices <= 16;
  GroupRows lists = {};
  int rc = 0;
  if (!by_ids && (rc = he_group_rows(&lists, p, ids_i32, weights_f32, rows, top, experts, t.bm, stream))) return rc;
  // The activations times their share are rounded to bfloat16, the second product's operands: half a step, 2^-8 of each at most. The results are 0.0023 to 0.0024 of their
  // size from 64 bits, 0.0017 with 32 bits between the products (1, 64 and 2048 rows of 16 experts of 2048). Two operands a value would take the rounding away and
  // double the second product's matrix instructions (2048 rows: 94 of 264 us).
  uint16_t* h = (uint16_t*)(p + t.ints);
  float* partial = (float*)(p + t.ints + t.h);
  up.x = (const uint16_t*)x, up.ldx = ldx, up.whole = whole_rows(x, ldx), up.M = rows;
  up.out = h, up.ldo = t.ldh, up.pairs = t.ldh % 2 == 0, up.gated = true;
  up.act = {alpha, limit > 0.f ? limit : INFINITY, up_shift, cubic}, up.silu = he_gated_act_is_silu(alpha, limit, up_shift, cubic);
  up.tile_begin = lists.tile_begin, up.groups = experts, up.rows_of = lists.rows_of, up.out_of = lists.choice_of, up.factor = lists.scale;
  down.x = h, down.ldx = t.ldh, down.whole = true;
  down.out = partial, down.ldo = D, down.out_f32 = true, down.pairs = D % 4 == 0;
  down.tile_begin = lists.tile_begin, down.groups = experts, down.rows_of = down.out_of = lists.choice_of;
  if (t.bm <= 16 ? D < 8 : D % FP4_K || !up.whole || far(rows, ldx))
    if ((rc = pad_rows(&up, p + t.ints + t.h + t.partial, s))) return rc;
  if (t.bm <= 16 ? I < 8 : I % FP4_K) {
    // (the columns behind I are multiplied with codes of zero: they have to be numbers)
    clear_columns_kernel<<<(unsigned)(((int64_t)choices * (t.ldh - I) + 255) / 256), 256, 0, s>>>(h, choices, I, (int)t.ldh);
    if ((rc = he_check_launch("he_fp4_experts (rows)"))) return rc;
    down.w.K = (int)t.ldh;
  }
  if (by_ids) {
    up.ids = down.ids = (const int32_t*)ids_i32, up.choices = down.choices = choices, up.top = top, down.top = 1;
    up.shares = down.shares = up.factor = (const float*)weights_f32;
  }
  if (by_ids && rows == 1 && !identity) {
    down.M = 1, down.out = out, down.out_f32 = false;
    down.bias = plus_f32, down.bias_dtype = HE_F32;        // (the one row of it)
    down.pairs = D % 4 == 0 && ((uintptr_t)out & 7) == 0;
    if ((rc = fp4_run_few(up, t.bm, t.mtiles, s))) return rc;
    return fp4_run_chain(down, s);
  }
  if (t.bm <= 16) {
    if ((rc = fp4_run_few(up, t.bm, t.mtiles, s)) || (rc = fp4_run_few(down, t.bm, t.mtiles, s))) return rc;
  } else {
    if ((rc = fp4_run_tall(up, t.up, t.mtiles, nullptr, s)) || (rc = fp4_run_tall(down, t.down, t.mtiles, nullptr, s))) return rc;
  }
  add_choices_kernel<<<dim3((D + 1023) / 1024, rows), 256, 0, s>>>((uint16_t*)out, partial, (const int32_t*)ids_i32, (const float*)weights_f32,
                                                                   identity ? (const uint16_t*)x : nullptr, ldx, (const float*)plus_f32, top, experts, D);
  return he_check_launch("he_fp4_experts");
}
