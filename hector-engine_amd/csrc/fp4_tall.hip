// Products of 17 rows and more with a weight in 4 bits (fp4.h).
#include "fp4.h"

namespace {

typedef __attribute__((address_space(3))) void lds_void;

// one KiB, 16 bytes a lane, into LDS
__device__ __forceinline__ void load_lds(uint32_t to, uint32_t offset, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
// c += w x^T, written so that the accumulators stay where they are and the order is this file's (the compiler moves half a register
// file of them about); no result is read right behind it
__device__ __forceinline__ void product(fp4_f32x4& c, fp4_bf16x8 w, fp4_bf16x8 x) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(w), "v"(x));
}
__device__ __forceinline__ void fixed() { __builtin_amdgcn_sched_barrier(0); }

// Four wavefronts make a tile of 16 MT rows x 64 NT weight rows over a slice of K, a wavefront all of its rows and 16 NT weight rows: a code is then
// converted once for 16 MT rows. A workgroup has PARTS such fours, each with its stretch of the slice, whose sums meet in LDS at the end: a unit
// with one small tile at a time waits for loads most of it (128 rows of 4608 x 3584 in 64 x 64 17.3 us with one, 13.6 with two, 19 with four).
// X goes through LDS in blocks of 128 k, straight from memory, one block ahead; a row's sixteen-byte pieces lie at their index xor three bits of
// the row, so that the rows of an operand are in different banks. The codes come into registers one block ahead, each a value of bfloat16 before
// it is multiplied. (Scales by way of LDS too: 32 rows of 18944 x 3584 15 -> 19 us.)
// 2048 x 37888 x 3584 gated 457 us (1.22 PFLOP/s): matrix cores 0.57 of the cycles, the other vector instructions, 256 of 296 a block for the
// conversions, 0.38, and the two do not overlap. Tiles of 64 rows and fewer wait: a block takes some 1 us (64 rows of 37888 x 3584 28 of them in 27 to
// 30 us, 203 of 4608 x 3584 14 a part in 15 to 17), matrix cores 0.20 and other vector instructions 0.26 of the cycles: each block is asked for one ahead and waited for
// whole, so a unit has some 47 KB on their way at a time. (Tiles of more columns, which read the rows less often, were no faster.)
template <int MT, int NT, int PARTS, int GROUPS>
__global__ __launch_bounds__(256 * PARTS, PARTS == 1 ? 2 : 1) void fp4_tall_kernel(Fp4Case c, int mtiles, int ntiles, int slices, float* __restrict__ sums) {
  constexpr int BM = 16 * MT, BLOCK = BM * 256;            // bytes of a block of X
  constexpr int HALF = BM / 32, LOADS = 2 * HALF;          // loads of a wavefront, of 64 k and of a block
  constexpr int RING = 16 / NT < 4 * MT ? 16 / NT : 4 * MT;                // operands of X in registers: some 250 cycles of products
  constexpr int FEW = MT < 4 ? MT : 4, ROW = 64 * NT + 16, TURN = 16 * FEW * ROW;      // results: tiles of rows a turn; bytes of a row, a wavefront's turn
  __shared__ __attribute__((aligned(1024))) uint8_t lds[PARTS * (2 * BLOCK > 4 * TURN ? 2 * BLOCK : 4 * TURN)];
  __shared__ int32_t to_of[BM];                            // a slot's row of out, -1: none
  __shared__ float share_of[BM];
  const int tid = threadIdx.x, lane = tid & 63, all_wave = __builtin_amdgcn_readfirstlane(tid >> 6), wave = all_wave & 3, part = all_wave >> 2, r16 = lane & 15, kq = lane >> 4;
  // tiles of rows that read the same weights are neighbours on an XCD
  const int per_xcd = gridDim.x / HE_XCDS;
  int tile = blockIdx.x % HE_XCDS * per_xcd + blockIdx.x / HE_XCDS;
  if (tile >= mtiles * ntiles * slices) return;
  const int mt = tile % mtiles;
  tile /= mtiles;
  const int nt = tile % ntiles, slice = tile / ntiles;
  int group = 0;
  if (c.tile_begin) {
    if (mt >= c.tile_begin[c.groups]) return;
    group = fp4_group_of(c.tile_begin, c.groups, mt);
  }
  const int m0 = mt * BM, tile0 = (nt * 4 + wave) * NT, blocks = c.w.blocks;
  const int pieces = slices * PARTS, piece_no = slice * PARTS + part;
  const int lo = (int)((int64_t)blocks * piece_no / pieces), hi = (int)((int64_t)blocks * (piece_no + 1) / pieces);
  const int end = PARTS == 1 ? hi : lo + (blocks + pieces - 1) / pieces;       // (every part keeps the barriers of the longest)
  const uint8_t* codes[NT];
  const uint16_t* scales[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t at = ((int64_t)group * c.w.tiles + min(tile0 + j, c.w.tiles - 1)) * blocks;
    codes[j] = c.w.codes + at * FP4_TILE_BYTES;
    scales[j] = c.w.scales + at * (16 * GROUPS);
  }
  // X in stages of 64 k: eight rows of a stage are a KiB
  uint32_t from[HALF];
#pragma unroll
  for (int i = 0; i < HALF; ++i) {
    const int r = 8 * (wave * HALF + i) + (lane >> 3);
    const int64_t row = c.rows_of ? max(c.rows_of[m0 + r], 0) : min(m0 + r, c.M - 1);
    from[i] = (uint32_t)(row * c.ldx * 2) + ((lane & 7) ^ (r & 7)) * 16;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds + part * 2 * BLOCK + wave * HALF * 1024;
  auto fetch_x = [&](int l, int kb, uint32_t at) {
    load_lds(lds0 + at + l / HALF * (BM * 128) + l % HALF * 1024, from[l % HALF], c.x + (int64_t)kb * FP4_K + l / HALF * 64);
  };
  const uint32_t piece[2] = {(uint32_t)((kq ^ (r16 & 7)) * 16), (uint32_t)(((4 + kq) ^ (r16 & 7)) * 16)};
  uint4 q[NT], qn[NT];
  uint16_t fn[NT][GROUPS];
  uint32_t f[NT][(GROUPS + 1) / 2];                        // two to a register
  auto fetch_w = [&](int64_t kb) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      qn[j] = *reinterpret_cast<const uint4*>(codes[j] + kb * FP4_TILE_BYTES + lane * 16);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) fn[j][g] = scales[j][kb * (16 * GROUPS) + 16 * g + r16];
    }
  };
  auto take_w = [&]() {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      q[j] = qn[j];
#pragma unroll
      for (int g = 0; g < GROUPS; g += 2) f[j][g / 2] = GROUPS == 1 ? fn[j][g] : fn[j][g] | (uint32_t)fn[j][(g + 1) % GROUPS] << 16;
    }
  };
  fp4_f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = fp4_f32x4{0.f, 0.f, 0.f, 0.f};

  fetch_w(lo);
#pragma unroll
  for (int l = 0; l < LOADS; ++l) fetch_x(l, lo, 0);
  if (tid < BM) {
    const int slot = m0 + tid;
    to_of[tid] = c.out_of ? c.out_of[slot] : slot < c.M ? slot : -1;
    share_of[tid] = c.factor ? c.factor[slot] : 1.f;
  }
  uint32_t at = 0;
  for (int kb = lo; kb < end; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (PARTS > 1 && kb >= hi) continue;
    const int next = min(kb + 1, hi - 1);                  // (behind the last block the last one again, which nobody reads)
    take_w();
    fetch_w(next);
    fixed();
    // one after the other the steps of 32 k, in each the tiles of rows; beside a tile's products run the operand read of a later tile, a
    // load of the next block, and the next step's conversions
    auto convert = [&](int t, int j) {
      const uint32_t words[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
      const int g = t * GROUPS / 4;
      return fp4_values(words[t], __uint_as_float(g & 1 ? f[j][g / 2] & 0xffff0000u : f[j][g / 2] << 16));
    };
    const uint8_t* x = lds + part * 2 * BLOCK + at + r16 * 128;
    auto read = [&](int step) {
      const int t = step / MT;
      return *reinterpret_cast<const fp4_bf16x8*>(x + t / 2 * (BM * 128) + step % MT * 2048 + piece[t & 1]);
    };
    fp4_bf16x8 w[2][NT], xs[RING];
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) xs[i] = read(i);
#pragma unroll
    for (int j = 0; j < NT; ++j) w[0][j] = convert(0, j);
    fixed();
    // (a conversion's result is not read by the instructions right behind it: the compiler knows no wait states of written ones)
    asm volatile("s_nop 4");
#pragma unroll
    for (int step = 0; step < 4 * MT; ++step) {
      const int t = step / MT, i = step % MT;
      if (step + RING - 1 < 4 * MT) xs[(step + RING - 1) % RING] = read(step + RING - 1);
      if (step % 2 == 0 && step / 2 < LOADS) fetch_x(step / 2, next, at ^ BLOCK);
      if (t < 3 && i % (MT / NT) == 0) w[(t + 1) & 1][i / (MT / NT)] = convert(t + 1, i / (MT / NT));
      fixed();
#pragma unroll
      for (int j = 0; j < NT; ++j) product(acc[i][j], w[t & 1][j], xs[step % RING]);
      fixed();
    }
    at ^= BLOCK;
  }
  // the last products' results are there 18 cycles after them; nothing may be on its way into LDS that is used again
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
  fixed();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
  // some tiles of rows at a time through this wavefront's part of LDS, so that neighbouring lanes write neighbouring results
  uint8_t* own = lds + all_wave * TURN;
  static_assert(PARTS == 1 || MT == FEW, "one turn of results");
  const int n = tile0 * FP4_ROWS + lane % (4 * NT) * 4, ld_sums = c.w.tiles * FP4_ROWS;
  const bool whole = c.pairs && n + 4 <= c.w.N;
  fp4_f32x4 bias = {0.f, 0.f, 0.f, 0.f};
  if (c.bias) bias = fp4_bias(c, n);
#pragma unroll
  for (int i0 = 0; i0 < MT; i0 += FEW) {
#pragma unroll
    for (int i = i0; i < i0 + FEW; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) *reinterpret_cast<fp4_f32x4*>(own + (16 * (i - i0) + r16) * ROW + (16 * j + 4 * kq) * 4) = acc[i][j];
    if (PARTS > 1) __syncthreads();
    else fp4_written();
    // (one kind of results a loop: with the kinds told apart at each of them 128 x 256 results of K 2048 took 1.1 of the time)
    auto rows = [&](auto put) {
#pragma unroll 4
      for (int r = lane / (4 * NT) + part * (16 * FEW / PARTS); r < (part + 1) * (16 * FEW / PARTS); r += 16 / NT) {
        fp4_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < PARTS; ++k) v += *reinterpret_cast<const fp4_f32x4*>(lds + (4 * k + wave) * TURN + r * ROW + lane % (4 * NT) * 16);
        put(16 * i0 + r, v);
      }
    };
    if (slices > 1) {
      rows([&](int r, fp4_f32x4 v) {
        if (to_of[r] >= 0 && n < ld_sums) *reinterpret_cast<fp4_f32x4*>(sums + ((int64_t)slice * c.M + m0 + r) * ld_sums + n) = v;
      });
    } else if (c.gated && c.silu) {
      rows([&](int r, fp4_f32x4 v) {
        if (to_of[r] >= 0 && n < c.w.N) fp4_put<FP4_SILU>(c, v, to_of[r], n, share_of[r], whole);
      });
    } else if (c.gated) {
      rows([&](int r, fp4_f32x4 v) {
        if (to_of[r] >= 0 && n < c.w.N) fp4_put<FP4_GATED>(c, v, to_of[r], n, share_of[r], whole);
      });
    } else if (c.out_f32) {
      rows([&](int r, fp4_f32x4 v) {
        if (to_of[r] >= 0 && n < c.w.N) fp4_put<FP4_F32>(c, v + bias, to_of[r], n, 1.f, whole);
      });
    } else {
      rows([&](int r, fp4_f32x4 v) {
        if (to_of[r] >= 0 && n < c.w.N) fp4_put<FP4_BF16>(c, v + bias, to_of[r], n, 1.f, whole);
      });
    }
    fp4_written();
  }
}

// the sum of the slices, in their order
__global__ __launch_bounds__(256) void fp4_join_kernel(Fp4Case c, int slices, const float* __restrict__ sums) {
  const int quads = c.w.tiles * 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)c.M * quads) return;
  const int64_t row = at / quads;
  const int n = (int)(at - row * quads) * 4;
  if (n >= c.w.N) return;
  fp4_f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const fp4_f32x4*>(sums + (((int64_t)s * c.M + row) * quads) * 4 + n);
  fp4_store(c, v, row, n, 1.f);
}

template <int MT, int NT, int PARTS>
int run_tall(const Fp4Case& c, int mtiles, int slices, float* sums, hipStream_t s) {
  const int ntiles = (c.w.tiles + 4 * NT - 1) / (4 * NT);
  const int64_t total = (int64_t)mtiles * ntiles * slices;
  HE_REQUIRE(total < (1 << 24), "he_fp4_product: %lld tiles are too many for one launch", (long long)total);
  const unsigned grid = (unsigned)((total + HE_XCDS - 1) / HE_XCDS * HE_XCDS);
  if (c.w.group == 128) fp4_tall_kernel<MT, NT, PARTS, 1><<<grid, 256 * PARTS, 0, s>>>(c, mtiles, ntiles, slices, sums);
  else if (c.w.group == 64) fp4_tall_kernel<MT, NT, PARTS, 2><<<grid, 256 * PARTS, 0, s>>>(c, mtiles, ntiles, slices, sums);
  else fp4_tall_kernel<MT, NT, PARTS, 4><<<grid, 256 * PARTS, 0, s>>>(c, mtiles, ntiles, slices, sums);
  if (const int rc = he_check_launch("he_fp4_product")) return rc;
  if (slices == 1) return 0;
  fp4_join_kernel<<<(unsigned)(((int64_t)c.M * c.w.tiles * 4 + 255) / 256), 256, 0, s>>>(c, slices, sums);
  return he_check_launch("he_fp4_product (sum)");
}

}  // namespace

int fp4_run_tall(const Fp4Case& c, Fp4Plan plan, int mtiles, float* sums, hipStream_t s) {
  HE_REQUIRE(c.whole && c.w.K % FP4_K == 0 && plan.slices >= 1 && plan.slices <= c.w.blocks && (plan.slices == 1 || (sums && !c.tile_begin)),
             "he_fp4_product: %d slices of %d k", plan.slices, c.w.K);      // (a slice without a block would read before its first)
  switch (plan.mt * 100 + plan.nt * 10 + plan.parts) {
    case 211: return run_tall<2, 1, 1>(c, mtiles, plan.slices, sums, s);
    case 212: return run_tall<2, 1, 2>(c, mtiles, plan.slices, sums, s);
    case 222: return run_tall<2, 2, 2>(c, mtiles, plan.slices, sums, s);
    case 411: return run_tall<4, 1, 1>(c, mtiles, plan.slices, sums, s);
    case 412: return run_tall<4, 1, 2>(c, mtiles, plan.slices, sums, s);
    case 421: return run_tall<4, 2, 1>(c, mtiles, plan.slices, sums, s);
    case 422: return run_tall<4, 2, 2>(c, mtiles, plan.slices, sums, s);
    case 821: return run_tall<8, 2, 1>(c, mtiles, plan.slices, sums, s);
    case 841: return run_tall<8, 4, 1>(c, mtiles, plan.slices, sums, s);
  }
  HE_REQUIRE(false, "he_fp4_product: no tile of %d x %d in %d parts of K", 16 * plan.mt, 64 * plan.nt, plan.parts);
}
