// Products of few rows with a weight in 4 bits (fp4.h).
#include "fp4.h"

namespace {

// eight values of X wherever they begin: the unit takes loads of sixteen bytes at any element
struct __attribute__((packed, aligned(2))) Piece {
  uint4 v;
};

// sum + a block of 128 k with the scales in the operands: a lane's codes, scales, row of X, and its first k
template <int GROUPS>
__device__ __noinline__ fp4_f32x4 scaled_block(fp4_f32x4 sum, const uint8_t* codes, const uint16_t* scales, const uint16_t* row, int k, int K) {
#pragma unroll 1
  for (int t = 0; t < 4; ++t, k += 32) {
    uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) words[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
    const fp4_bf16x8 v = __builtin_bit_cast(fp4_bf16x8, make_uint4(words[0], words[1], words[2], words[3]));
    const uint32_t scale = scales[t * GROUPS / 4 * 16];
    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_values(*reinterpret_cast<const uint32_t*>(codes + 4 * t), __uint_as_float(scale << 16)), v, sum, 0, 0, 0);
  }
  return sum;
}

enum { ROWS_ALONE, CHOICES, NORM };

// A workgroup has NT tiles of 16 weight rows; its W wavefronts cut K among them, and their sums meet in LDS. Codes, scales and X (4 XL rows of it)
// come straight into registers, D blocks of 128 k ahead, with no barrier before the end. A block of X goes from there through a
// wavefront's own part of LDS into the order of the operands: read as operands from memory, each of its rows a sixteen-byte piece a
// lane and all 16 of them whatever X has, it took a third of the time (8 rows of 37888 x 3584 19.5 us, without it 14). The scales of a block go the same
// way, in one load a wavefront (a load of 32 bytes for each tile and group: 16 rows in groups of 32 39.7 us, now 26.6).
// There the pieces of a row lie at their index xor the row, so that the rows of an operand are in different banks.
// Bound by the codes' way from memory where the weight is large: 8 rows of 37888 x 3584 14.4 us, 4.9 TB/s.
// With ids (64 choices at most) a tile's slots are found here, by every wavefront for itself: slot by slot the choices of one expert, the
// tiles in the order of their first choices. CHOICES: one row and all of its choices, a tile's sums taken over the choices' K one after the
// other (codes of expert ids[choice], X row `choice`), so that nothing is left to add up.
// NORM: a norm is carried across two products (resid, owed): the first adds its results to the residual rows and leaves r * gain and the sums of
// r^2, the second multiplies its sums by the row's scale, whose parts are read, all at once, while its first codes are on their way.
template <int NT, int W, int D, int XL, int GROUPS, int KIND>
__global__ __launch_bounds__(64 * W) void fp4_few_kernel(Fp4Case c) {
  constexpr int WORDS = NT * GROUPS * 8, EACH_S = (WORDS + 63) / 64;           // the scales of a block, two a word; of a lane
  constexpr int PLACE = XL * 1024 + WORDS * 4, OWN = 2 * PLACE > NT * 1024 ? 2 * PLACE : NT * 1024;
  __shared__ __attribute__((aligned(16))) uint8_t lds[W * OWN];
  constexpr bool CHAIN = KIND == CHOICES, CARRIED = KIND == NORM;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = lane >> 4;
  constexpr int ROWS = 4 * XL;                             // of a tile of rows
  __shared__ int32_t choice_in[W][16];                     // with ids: a slot's choice, -1: none
  __shared__ float scale_of[16];                           // with owed: a row's scale
  const int blocks = c.w.blocks, units = CHAIN ? c.choices * blocks : blocks;      // (a unit: a block of a choice)
  const int lo = units * wave / W, hi = units * (wave + 1) / W;
  int group = 0;
  int id = -1;                                             // lane i: the expert of choice i, -1: none
  if (c.ids) {
    const int choice = min(lane, c.choices - 1), given = c.ids[choice];      // (both asked for at once)
    const float share = c.shares[choice];
    if (lane < c.choices && share != 0.f && given < c.groups) id = given;
  }
  if (c.tile_begin) {
    if ((int)blockIdx.y >= c.tile_begin[c.groups]) return;
    group = fp4_group_of(c.tile_begin, c.groups, blockIdx.y);
  } else if (c.ids && !CHAIN) {
    int rank = 0;                                          // choices of the same expert in front
    for (int j = 0; j < c.choices - 1; ++j) rank += j < lane && __builtin_amdgcn_readlane(id, j) == id;
    uint64_t first = __ballot(id >= 0 && rank % ROWS == 0);
    if (__popcll(first) <= (int)blockIdx.y) return;        // (the same in all wavefronts)
    for (int i = 0; i < (int)blockIdx.y; ++i) first &= first - 1;
    const int lead = __ffsll((unsigned long long)first) - 1;
    group = __builtin_amdgcn_readlane(id, lead);
    const int base = __builtin_amdgcn_readlane(rank, lead);
    if (lane < 16) choice_in[wave][lane] = -1;
    if (id == group && rank >= base && rank < base + ROWS) choice_in[wave][rank - base] = lane;
    fp4_written();
  }
  const int m0 = blockIdx.y * ROWS, tile0 = blockIdx.x * NT;
  int64_t tile_at[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) tile_at[j] = ((int64_t)group * c.w.tiles + min(tile0 + j, c.w.tiles - 1)) * blocks;
  auto row_at = [&](int r) {                               // (rows behind the last repeat it: each row's results are its own)
    int64_t row = 0;
    if (c.ids && !CHAIN) row = max(choice_in[wave][r], 0) / c.top;
    else if (!CHAIN) row = c.rows_of ? max(c.rows_of[m0 + r], 0) : min(m0 + r, c.M - 1);
    return c.x + row * c.ldx;
  };
  // a lane's pieces of X: row 4 i + (lane >> 4), eight k from 8 (lane & 15) on
  const uint16_t* x[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) x[i] = row_at(4 * i + kq);
  const int K = c.w.K;
  uint8_t* own = lds + wave * OWN;
  const uint32_t* scales[EACH_S];
#pragma unroll
  for (int i = 0; i < EACH_S; ++i) {
    const int word = min(lane + 64 * i, WORDS - 1);
    scales[i] = (const uint32_t*)c.w.scales + ((int64_t)group * c.w.tiles + min(tile0 + word / (8 * GROUPS), c.w.tiles - 1)) * blocks * (8 * GROUPS) + word % (8 * GROUPS);
  }

  uint4 q[D][NT], xs[D][XL];
  uint32_t s[D][EACH_S];
  auto load = [&](int u, int unit) {
    int kb = unit;
    int64_t from = 0, xfrom = 0;
    if (CHAIN) {
      const int choice = unit / blocks;
      kb = unit - choice * blocks;
      from = (int64_t)max(__builtin_amdgcn_readlane(id, choice), 0) * c.w.tiles * blocks;
      xfrom = choice * c.ldx;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t at = tile_at[j] + from + kb;
      q[u][j] = he_load16_once<uint4>(c.w.codes + at * FP4_TILE_BYTES + lane * 16);
    }
#pragma unroll
    for (int i = 0; i < EACH_S; ++i) s[u][i] = scales[i][(from + kb) * (8 * GROUPS)];
    const int k = kb * FP4_K + 8 * r16;
#pragma unroll
    for (int i = 0; i < XL; ++i) xs[u][i] = reinterpret_cast<const Piece*>(x[i] + xfrom + min(k, K - 8))->v;
  };
  // X and the scales of a block into one of two places
  auto keep = [&](int u, int unit, int place) {
    const int kb = CHAIN ? unit % blocks : unit;
    const int over = kb * FP4_K + 8 * r16 + 8 - K;         // (a piece over the end of its row was loaded from the row's last eight values)
    const bool last = (kb + 1) * FP4_K > K;
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int row = 4 * i + kq;
      uint4 v = xs[u][i];
      if (last && over > 0) {
        const uint64_t a = (uint64_t)v.y << 32 | v.x, b = (uint64_t)v.w << 32 | v.z;
        const int bits = 16 * over;
        const uint64_t lo = bits < 64 ? a >> bits | b << (64 - bits) : bits < 128 ? b >> (bits - 64) : 0, hi = bits < 64 ? b >> bits : 0;
        v = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
      }
      *reinterpret_cast<uint4*>(own + place * PLACE + row * 256 + (r16 ^ row) * 16) = v;
    }
#pragma unroll
    for (int i = 0; i < EACH_S; ++i)
      if (lane + 64 * i < WORDS) *reinterpret_cast<uint32_t*>(own + place * PLACE + XL * 1024 + (lane + 64 * i) * 4) = s[u][i];
  };
  const int xrow = min(r16, 4 * XL - 1);
  fp4_f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = fp4_f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int u, int unit, int place) {
    if (CHAIN && __builtin_amdgcn_readlane(id, unit / blocks) < 0) return;      // (a choice of no expert adds nothing)
    fp4_bf16x8 v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      v[t] = *reinterpret_cast<const fp4_bf16x8*>(own + place * PLACE + xrow * 256 + ((4 * t + kq) ^ xrow) * 16);
    // (every tile's products first: a product's sums are there some 30 cycles behind it)
    fp4_f32x4 sums[NT][GROUPS];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t words[4] = {q[u][j].x, q[u][j].y, q[u][j].z, q[u][j].w};
        const fp4_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        constexpr int STEPS = 4 / GROUPS;
        sums[j][t / STEPS] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_operand(words[t]), v[t], t % STEPS == 0 ? zero : sums[j][t / STEPS], 0, 0, 0);
      }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint2 b = *reinterpret_cast<const uint2*>(own + place * PLACE + XL * 1024 + (j * GROUPS + g) * 32 + 8 * kq);
        const float f[4] = {__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u)};
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(f[e], sums[j][g][e], acc[j][e]);
      }
  };
  if (lo < hi) {
#pragma unroll
    for (int u = 0; u < D; ++u) load(u, min(lo + u, hi - 1));
  }
  if (CARRIED && c.owed) {
    constexpr int EACH = (ROWS + W - 1) / W;               // rows of a wavefront
    float sum[EACH];
#pragma unroll
    for (int r = 0; r < EACH; ++r) sum[r] = 0.f;
    for (int from = 0; from < c.owed_count; from += 256) {
      float part[EACH][4];
#pragma unroll
      for (int r = 0; r < EACH; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = min(wave + r * W, c.M - 1), at = from + 64 * i + lane;
          part[r][i] = c.owed[(int64_t)row * c.owed_count + min(at, c.owed_count - 1)];
        }
#pragma unroll
      for (int r = 0; r < EACH; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[r] += from + 64 * i + lane < c.owed_count ? part[r][i] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      const float total = wave_sum(sum[r]);
      if (lane == 0 && wave + r * W < ROWS) scale_of[wave + r * W] = 1.f / sqrtf(total / (float)c.owed_dim + c.owed_eps);
    }
  }
  if (lo < hi) {
    int kb = lo;
    for (; kb + D < hi; kb += D) {
#pragma unroll
      for (int u = 0; u < D; ++u) {
        keep(u, kb + u, u & 1);
        fp4_written();
        multiply(u, kb + u, u & 1);
        fp4_written();
        load(u, min(kb + D + u, hi - 1));
      }
    }
#pragma unroll
    for (int u = 0; u < D; ++u)
      if (kb + u < hi) {
        keep(u, kb + u, u & 1);
        fp4_written();
        multiply(u, kb + u, u & 1);
        fp4_written();
      }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j) *reinterpret_cast<fp4_f32x4*>(own + j * 1024 + lane * 16) = acc[j];
  // A group's sum of x * code can leave the range of 32 bits where its scaled one does not (128 values of x from 4.4e35 on): a wavefront that ends with infinities
  // or NaN takes those sums once more with the scales in the operands, as the kernel of many rows has them. (One block after the other in a function of its own: with the
  // loads of the loop above the kernels held so many more registers that 16 rows of 37888 x 3584 in groups of 32 took 26.3 us, 22.4 without; so 63 products of 1 to
  // 16 rows take 1.003 of the time without in the geometric mean.)
  bool off = false;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) off |= !(fabsf(acc[j][e]) < INFINITY);
  if (__any(off)) {
    const uint16_t* row = row_at(xrow);
#pragma unroll 1
    for (int j = 0; j < NT; ++j) {
      fp4_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int unit = lo; unit < hi; ++unit) {
        const int choice = CHAIN ? unit / blocks : 0, kb = unit - choice * blocks;
        const int expert = CHAIN ? __builtin_amdgcn_readlane(id, choice) : group;
        if (expert < 0) continue;
        const int64_t at = ((int64_t)expert * c.w.tiles + min(tile0 + j, c.w.tiles - 1)) * blocks + kb;
        sum = scaled_block<GROUPS>(sum, c.w.codes + at * FP4_TILE_BYTES + lane * 16, c.w.scales + at * (16 * GROUPS) + r16, row + choice * c.ldx, kb * FP4_K + 8 * kq, K);
      }
      fp4_f32x4 kept = *reinterpret_cast<const fp4_f32x4*>(own + j * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) kept[e] = fabsf(kept[e]) < INFINITY ? kept[e] : sum[e];      // (a row without numbers changes no other row's bits)
      *reinterpret_cast<fp4_f32x4*>(own + j * 1024 + lane * 16) = kept;
    }
  }
  __syncthreads();
  const int slot = m0 + r16;
  int to = slot;
  if (r16 >= ROWS) to = -1;
  else if (CHAIN) to = r16 == 0 ? 0 : -1;
  else if (c.ids) to = choice_in[wave][r16];
  else if (c.out_of) to = c.out_of[slot];
  else if (slot >= c.M) to = -1;
  static_assert(NT <= W, "a wavefront has one tile of results");
  if (wave >= NT) return;
  const int n = (tile0 + wave) * FP4_ROWS + 4 * kq;
  fp4_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < W; ++k) v += *reinterpret_cast<const fp4_f32x4*>(lds + k * OWN + wave * 1024 + lane * 16);
  if (CARRIED && c.owed && to >= 0) v *= scale_of[r16];
  if (CARRIED && c.resid) {
    // (read ahead of the products they cost every kernel that carries a norm more than they saved this one)
    float square = 0.f;
    if (to >= 0 && n < c.w.N) {
      if (c.bias) v += fp4_bias(c, n);
      fp4_f32x4* r = reinterpret_cast<fp4_f32x4*>(c.resid + (int64_t)to * c.w.N + n);
      v = *r + c.resid_scale * v;
      *r = v;
      float g[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) square = fmaf(v[e], v[e], square), g[e] = v[e] * load_param(c.gain, n + e, c.gain_dtype);
      *reinterpret_cast<uint2*>(c.carried + (int64_t)to * c.w.N + n) = make_uint2(pack2_bf16(g[0], g[1]), pack2_bf16(g[2], g[3]));
    }
    square += __shfl_xor(square, 16);
    square += __shfl_xor(square, 32);
    if (kq == 0 && to >= 0 && n < c.w.N) c.squares[(int64_t)to * c.w.tiles + tile0 + wave] = square;
    return;
  }
  if (to >= 0 && n < c.w.N) fp4_store(c, v, to, n, c.factor ? c.factor[c.ids ? to : slot] : 1.f);
}

template <int NT, int W, int D, int XL, int KIND>
int run_few(const Fp4Case& c, int mtiles, hipStream_t s) {
  const dim3 grid((c.w.tiles + NT - 1) / NT, mtiles);
  if (c.w.group == 128) fp4_few_kernel<NT, W, D, XL, 1, KIND><<<grid, 64 * W, 0, s>>>(c);
  else if (c.w.group == 64) fp4_few_kernel<NT, W, D, XL, 2, KIND><<<grid, 64 * W, 0, s>>>(c);
  else fp4_few_kernel<NT, W, D, XL, 4, KIND><<<grid, 64 * W, 0, s>>>(c);
  return he_check_launch("he_fp4_product");
}

template <int XL, int KIND>
int run_rows(const Fp4Case& c, int mtiles, hipStream_t s) {
  // Microseconds of (tiles, wavefronts, blocks ahead), weights in groups of 128 from memory: many tiles are best with many workgroups that hold
  // little, few with many wavefronts to a tile.
  //                      (1, 8, 2)  (2, 4, 2)  (2, 8, 2)  (4, 4, 2)  (4, 4, 1)
  // 16 rows, 37888 x 3584     29.6       21.4       21.8       19.9       19.7    (groups of 32: 30.7, 24.8, 30.1, 28.2, 24.8)
  // 16 rows, 10240 x 5120     15.0       13.8       14.6       11.2       13.8
  // 16 rows, 4608 x 3584       8.4        6.8        6.9        8.4       10.4
  // 8 rows, 37888 x 3584      23.3       18.4       18.5       17.8       16.8
  // 8 rows, 20480 x 5120      18.5       15.8       16.0          -       17.0
  // 1 row, 37888 x 3584       19.1       14.7       15.8       16.5       15.5
  // 1 row, 4608 x 3584         5.5        5.9        5.3        7.3        9.2
  // 1 row, 3584 x 18944       10.5       18.2       12.1       23.5       32.8    ((1, 8, 4): 9.5)
  const int64_t tiles = (int64_t)c.w.tiles * mtiles;
  if (tiles <= 256) {
    if constexpr (XL == 1) {
      if (c.w.blocks >= 64) return run_few<1, 8, 4, XL, KIND>(c, mtiles, s);
    }
    return run_few<1, 8, 2, XL, KIND>(c, mtiles, s);
  }
  if constexpr (XL == 4) {
    if (tiles >= 1280) return run_few<4, 4, 1, XL, KIND>(c, mtiles, s);
    if (tiles >= 640) return run_few<4, 4, 2, XL, KIND>(c, mtiles, s);
  }
  if constexpr (XL == 2) {
    if (tiles >= 1536) return run_few<4, 4, 1, XL, KIND>(c, mtiles, s);
  }
  return tiles <= 512 && c.w.blocks >= 16 ? run_few<2, 8, 2, XL, KIND>(c, mtiles, s) : run_few<2, 4, 2, XL, KIND>(c, mtiles, s);
}

}  // namespace

int fp4_run_chain(const Fp4Case& c, hipStream_t s) {
  HE_REQUIRE(c.w.K >= 8 && c.ids && c.choices >= 1 && c.choices <= 64 && c.M == 1, "he_fp4_experts: %d choices of a row", c.choices);
  // (two tiles a workgroup: 4 experts of 2048 over rows of 2048 12.7 us with the first product, 11.8 so; 2 of 4096 over 6144 19.5, 20.3; over 8192 the same)
  return run_few<1, 8, 2, 1, CHOICES>(c, 1, s);
}

int fp4_run_few(const Fp4Case& c, int bm, int mtiles, hipStream_t s) {
  HE_REQUIRE(c.w.K >= 8, "he_fp4_product: rows of fewer than 8 values");
  HE_REQUIRE(!c.ids || c.choices <= 64, "he_fp4_experts: %d choices to be grouped by each workgroup", c.choices);
  HE_REQUIRE(mtiles <= 65535, "he_fp4_product: %d tiles of rows are too many for one launch", mtiles);
  if (c.owed || c.resid) {
    HE_REQUIRE(mtiles == 1 && !c.ids && !c.tile_begin, "he_fp4_product: a norm is carried by one tile of rows");
    return bm > 8 ? run_rows<4, NORM>(c, 1, s) : bm > 4 ? run_rows<2, NORM>(c, 1, s) : run_rows<1, NORM>(c, 1, s);
  }
  return bm > 8 ? run_rows<4, ROWS_ALONE>(c, mtiles, s) : bm > 4 ? run_rows<2, ROWS_ALONE>(c, mtiles, s) : run_rows<1, ROWS_ALONE>(c, mtiles, s);
}
