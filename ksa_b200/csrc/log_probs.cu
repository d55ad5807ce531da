// Log probabilities of given tokens under the output head, and their gradients, without the logits in memory:
//   x_tv = h_t . w_v / tau,   y_t = x_t,label - log sum_v exp(x_tv);
//   dx_tv = dy_t ([v = label] - exp(x_tv - lse_t)) / tau,   dh = dx w,   dw = dx^T h.
//
// Bound: the products, 2 n V D operations forward and twice that backward; below some 210 rows (1376 TFLOP/s to 6550 GB/s) the weights' bytes.
//
// The backward pass needs the logits again.  Where the caller wants them kept (16 bits of each fit its limit, and the heads are wide enough that the
// product costs more than keeping it) the forward pass keeps them, as the distance below the maximum of their 128 columns in steps of 2^-10 of a power
// of two: probabilities from them are off by 2^-11.5 of themselves at most, less than the rounding of dx to bf16 (kept as bf16 a logit of 10 would be off by
// 2^-6), and what is more than 64 powers below the maximum counts as that far.  Else the product is computed again: four products in place of three.
//
// Rows without a label are left out first: the others are gathered into a dense array, and the kernels take their number from device
// memory, so that prompts and masked turns cost nothing but their labels, and what their rows hold reaches no sum.
//
// One kernel on CTA pairs (gemm2.cu describes its roles and barriers) serves four products, which differ in their epilogue:
//   kStats  h w^T: every thread has one row of the tile; it takes the maximum and the sum of exponentials of 128 columns.  A second kernel adds
//           those of a row.  Maxima and the label's logit stay as they are, not times log2(e): y is then a difference of two numbers that
//           were not rounded, where products of 20 would leave 1e-6.
//   kStatsKeep  the same, and the logits in 16 bits;  kGrad  the product again, dx in bf16 (kLpLow) from the accumulators.
//   kProducts  dx w in fp32 over the columns of one slab, and dx^T h: up to some size one launch of both, so that the many short tiles of the second fill the
//           waves of the few long ones of the first.
// dx exists for a slab of the vocabulary at a time (the caller says how wide): the slabs' dw are disjoint, and dh is added up in fp32.
#include "common.cuh"
#include "host.h"
#include "pair.cuh"
#include "vec.cuh"

#include <math.h>

namespace ksa {

constexpr int kLpBM = 128;          // rows of the tile in a CTA; a pair has 256
constexpr int kLpBN = 256;          // columns of the tile
constexpr int kLpBNh = 128;         // rows of B staged per CTA
constexpr int kLpBK = 64;
constexpr int kLpThreads = 320;     // warp 0 loads, warp 1 issues products, warps 2..5 and 6..9 epilogue: every other tile is a group's, or half of every tile
constexpr int kLpStages = 6;
constexpr int kLpGroupM = 8;
constexpr int kLpABytes = kLpBM * kLpBK * 2;
constexpr int kLpBBytes = kLpBNh * kLpBK * 2;
constexpr int kLpStageBytes = kLpABytes + kLpBBytes;
constexpr int kLpStoreBytes = 8 * 4096;                                  // a staging box of 128 bytes x 32 rows for each epilogue warp
constexpr int kLpSmem = kLpStages * kLpStageBytes + kLpStoreBytes + 256 + 1024;
static_assert(kLpSmem <= 232448, "227 KB");
static_assert(kLpSmem >= kTmemClusterAlone, "a pair holds all tensor memory: no block of another cluster beside it (host.h)");
constexpr int kLpStatCols = 128;                                        // columns that share a maximum and a sum
// Steps of kLpBK after which a logit's partial sum leaves the tensor cores.  Their accumulators cut off what does not fit, towards zero: a logit over 2560
// products came out 9e-7 of itself too small, and at a temperature of 0.6 y was off by 1.6e-6.  The epilogue adds the parts of 1024 products up:
// 5e-7, for 1 % of the time (8192 x 151936 x 2048 3830 -> 3862 us; parts of 512 2.9e-7 and 3960).  An epilogue thread then keeps 128 sums in registers, so
// that both groups of its warps share every tile; of narrower heads each takes every other tile, which costs less per tile (width 128 207 us, 235 shared).
// kGrad takes its logits whole: 9e-7 of a logit of 30 is 3e-5 of a probability, next to nothing beside dx's rounding (2^-9), and the label's 1 - p, where it
// would not be, comes from the forward pass.
constexpr int kLpChunk = 16;
constexpr float kLpCodes = 1024.f;                                      // codes of a kept logit to a power of two
// Pitches of the arrays that are made here, in elements: rows that begin on 128 bytes are loaded in whole lines.  A width of 1352 as pitch took a third
// of the loads' rate (1146 rows against 49042 tokens 150 us).
__host__ __device__ constexpr long long lp_pitch(long long n) { return (n + 63) / 64 * 64; }
constexpr int kLpRowPad = 256;                                          // rows of the gathered arrays: a multiple of this
// dx enters its products in bf16, 2^-9 of itself off.  Over many rows that is 1.4 times the error that rounding the results leaves anyway; of few rows each
// gradient is nearly one row's, whose largest elements' rounding all its values share, and was off by 2.5 times as much.  Up to so many rows
// with a label (a pair's tile has twice as many) dx is two bf16 numbers, the second of them what the rounding of the first left, in the rows
// from kLpLow on: dh is the sum of both rows' products, dw runs over both.  64 rows of 2048 against 151936 tokens 456 -> 476 us.
constexpr int kLpLow = 128;
static_assert(kLpLow == kLpBM && 2 * kLpLow <= kLpRowPad, "the second halves have rows of their own, those of the pair's other CTA");

enum LpMode : int { kStats = 0, kStatsKeep = 1, kGrad = 2, kProducts = 3 };

struct LpArgs {
  int M, N, K;                 // kStats, kGrad: rows (at most; *count says how many), columns, width.  kProducts: rows, width, columns of the slab
  const int* count;            // rows with a label
  const int* rows;             // their places among all rows
  const int* row_label;        // their labels
  float scale2;                // log2(e) / tau
  float inv_tau;
  float2* stats;               // kStats: [ceil(N / 128)][ld_stats] maximum m (times tau) and sum of exp(x - m / tau)
  float* picked;               // kStats: [rows] the label's logit, times tau
  float* tops;                 // kStatsKeep: [ceil(N / 128)][ld_stats] maxima, base 2
  long long ld_stats;
  const float* lse2;           // kGrad: [rows]
  const float* picked2;        // kGrad: [rows] the label's logit less the log-sum, base 2
  const float* dy;             // kGrad: gradient of y, by the rows' places
  int col0;                    // kGrad: first column of the slab
  int dh, dw;                  // kProducts: which are wanted
  int add_dh, add_dw;          // into fp32, added to what is there
  int planes;                  // dh: K is cut into at most so many parts, each with an output of its own
  int plane_rows;
  int* parts;                  // dh: how many parts it is
  int bf16_out;                // dw
  int* status;
};

// Steps of kLpBK that a tile's output costs besides its products: of dh, fp32 with nothing to hide behind, and of dw.
constexpr int kLpDhOutput = 10, kLpDwOutput = 4;
// All of dw, in those steps: `n` rows of the vocabulary, of `D`, over `count` rows.
__device__ __forceinline__ float lp_dw_steps(int n, int D, int count) {
  return (float)((n + 2 * kLpBM - 1) / (2 * kLpBM)) * (float)((D + kLpBN - 1) / kLpBN) * (float)((count + kLpBK - 1) / kLpBK + kLpDwOutput);
}
// Parts that K (the vocabulary) is cut into for dh.  Its tiles are few and long, 160 for 4915 rows of 2048 on 74 pairs, and the last wave of whole ones would be
// a third of the time (2594 us by itself, in parts 2300) where dw's tiles do not fill it.  Every part has an output of its own, which the
// scattering kernel adds up in order: it is told how many there are, as a rule in fp32 may come out differently in another kernel.  The rule takes the fewest steps of kLpBK on the busiest pair or, if that is more, of all pairs on average with dw's
// (`other`); a tile of a part costs 0.13 more to be read again.  By every warp, whose lanes try two numbers each.
__device__ __forceinline__ int lp_parts(int tiles, int num_kb, int n_pairs, int most, float other) {
  if (most <= 1 || num_kb <= 0 || tiles >= 64 * n_pairs) return 1;
  const int lane = threadIdx.x & 31;
  float least = INFINITY;
  int best = 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 1 + 32 * i;
    if (s > most || (s > 1 && num_kb / s < 8)) continue;
    const float each = (float)((num_kb + s - 1) / s + kLpDhOutput);
    const float steps = fmaxf((float)((tiles * s + n_pairs - 1) / n_pairs) * each, ((float)(tiles * s) * each + other) / (float)n_pairs) + 0.13f * (float)(tiles * s);
    if (steps < least) { least = steps; best = s; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float steps = __shfl_xor_sync(0xffffffffu, least, o);
    const int s = __shfl_xor_sync(0xffffffffu, best, o);
    if (steps < least || (steps == least && s < best)) { least = steps; best = s; }
  }
  const int part = (num_kb + best - 1) / best;
  return (num_kb + part - 1) / part;                                     // (rounding up may leave fewer parts than asked for; none is empty)
}

// A product's tiles, and one unit of a pair's work: a tile, one half of its columns (`side` is that half, -1 for the whole) or one part of its K.
struct LpTiles {
  int m, n, all, num_kb;
  __device__ __forceinline__ LpTiles(int M, int N, int K)
      : m((M + 2 * kLpBM - 1) / (2 * kLpBM)), n((N + kLpBN - 1) / kLpBN), all(m * n), num_kb((K + kLpBK - 1) / kLpBK) {}
  __device__ __forceinline__ void coords(int tile, int& mb, int& nb) const {
    const int per_group = kLpGroupM * n, group = tile / per_group, first_m = group * kLpGroupM;
    const int group_rows = min(m - first_m, kLpGroupM), in_group = tile - group * per_group;
    mb = first_m + in_group % group_rows;
    nb = in_group / group_rows;
  }
};
struct LpUnit {
  bool dh;
  int mb, nb, side, part, kb0, kb1;
};

// What every pair works on, in order.  dh's parts come first, all tiles of a part before the next part, so that pairs at work together read the same rows
// of both operands.  Where that leaves some pairs with one unit less, those begin with as many of the other product's tiles as make up for it.
// Of those, a last wave of at most half as many tiles as pairs is worked on as halves of 128 columns (gemm2.cu).
struct LpSchedule {
  LpTiles dh, main;
  int pair, n_pairs, parts, part_kb, dh_mine, heavy, first, first_mine, halves_from, units;

  __device__ __forceinline__ LpSchedule(const LpTiles& dh, const LpTiles& main, int pair, int n_pairs, int parts)
      : dh(dh), main(main), pair(pair), n_pairs(n_pairs), parts(parts) {
    part_kb = (dh.num_kb + parts - 1) / parts;
    const int dh_units = dh.all * parts;
    dh_mine = dh_units > pair ? (dh_units - pair + n_pairs - 1) / n_pairs : 0;
    heavy = dh_units % n_pairs;
    first = first_mine = 0;
    if (heavy > 0 && main.all > 0) {
      const int lighter = n_pairs - heavy, each = main.num_kb + kLpDwOutput;
      const int ahead = (part_kb + kLpDhOutput + each / 2) / each;       // tiles that take as long as one unit of dh
      first = ahead >= (main.all + lighter - 1) / lighter ? main.all : ahead * lighter;
      if (pair >= heavy && first > pair - heavy) first_mine = (first - (pair - heavy) + lighter - 1) / lighter;
    }
    const int left = main.all - first, last = left % n_pairs;
    halves_from = 2 * last <= n_pairs ? left - last : left;
    units = 2 * left - halves_from;
  }
  __device__ __forceinline__ bool get(int i, LpUnit& u) const {          // the i-th unit of this pair
    u.dh = i < dh_mine;
    u.side = -1;
    u.part = 0;
    if (u.dh) {
      const int unit = pair + i * n_pairs;
      u.part = unit / dh.all;
      u.kb0 = u.part * part_kb;
      u.kb1 = min(u.kb0 + part_kb, dh.num_kb);
      dh.coords(unit - u.part * dh.all, u.mb, u.nb);
      return true;
    }
    i -= dh_mine;
    int tile = pair - heavy + i * (n_pairs - heavy);
    if (i >= first_mine) {
      const int unit = pair + (i - first_mine) * n_pairs;
      if (unit >= units) return false;
      tile = unit;
      if (unit >= halves_from) {
        u.side = (unit - halves_from) & 1;
        tile = halves_from + ((unit - halves_from) >> 1);
      }
      tile += first;
    }
    u.kb0 = 0;
    u.kb1 = main.num_kb;
    main.coords(tile, u.mb, u.nb);
    return true;
  }
};

struct LpMaps {
  CUtensorMap A, B, C;
};

// A maximum with its sum of exponentials.  The sum is of 2^(x scale2 - top), top being max scale2 rounded: what the rounding took or added goes into it.
__device__ __forceinline__ float2 lp_sum(float mx, float top, float scale2, float sum) {
  return make_float2(mx, mx == -INFINITY ? sum : sum * fast_exp2(-fmaf(mx, scale2, -top)));
}

template <int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kLpThreads, 1)
log_probs_pair_kernel(const __grid_constant__ LpMaps maps, const __grid_constant__ LpMaps maps_dh, const __grid_constant__ LpArgs a) {
  constexpr bool kBMn = kMode == kProducts, kSums = kMode == kStats || kMode == kStatsKeep;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + kLpStages * kLpStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kLpStoreBytes);   // used in the leader
  uint64_t* empty = full + kLpStages;                                   // both CTAs
  uint64_t* acc_full = empty + kLpStages;                               // both CTAs, 2 buffers
  uint64_t* acc_empty = acc_full + 2;                                   // used in the leader, 2 buffers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();     // 0 = leader
  const WaitGuard guard{abort_flag, a.status};
  const int pair = (int)blockIdx.x >> 1, n_pairs = (int)gridDim.x >> 1;

  const bool split = kSums && a.K > kLpChunk * kLpBK;                     // tiles in several parts of K, shared by the epilogue's two groups

  if (threadIdx.x == 0) {
    for (int i = 0; i < kLpStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], split ? 16 : 8); }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.A);
    tma_prefetch_desc(&maps.B);
  }
  if (warp == 2) { tmem_alloc2(tmem_slot, 512); tmem_relinquish2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // both CTAs' barriers are initialised before any remote arrival
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_enter();

  const int count = *a.count;
  const int M = min(count, a.M), N = a.N;
  const bool low = (kMode == kGrad || kMode == kProducts) && M <= kLpLow;
  const int dh_rows = low && M > 0 ? kLpLow + M : M, dw_rows = low ? 2 * ((M + kLpBK - 1) / kLpBK * kLpBK) : M;
  const LpTiles dh(kMode == kProducts && a.dh ? dh_rows : 0, a.N, a.K);
  const LpTiles main_tiles(kMode != kProducts ? M : a.dw ? a.K : 0, a.N, kMode != kProducts ? a.K : dw_rows);
  const int parts = kMode == kProducts && dh.all > 0 ? lp_parts(dh.all, dh.num_kb, n_pairs, a.planes, a.dw ? lp_dw_steps(a.K, a.N, dw_rows) : 0.f) : 1;
  if (kMode == kProducts && a.dh && blockIdx.x == 0 && threadIdx.x == 0) *a.parts = dh.all > 0 ? parts : 0;
  const LpSchedule work_of(dh, main_tiles, pair, n_pairs, parts);
  const int num_kb = main_tiles.num_kb;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      LpUnit u;
      for (int i = 0; ok && work_of.get(i, u); ++i) {
        const int row0 = u.mb * 2 * kLpBM + (int)rank * kLpBM;
        const int col0 = u.side < 0 ? u.nb * kLpBN + (int)rank * kLpBNh : u.nb * kLpBN + u.side * kLpBNh + (int)rank * 64;
        const int boxes = u.side >= 0 ? 1 : 2;                           // of 64 rows
        const bool a_mn = kMode == kProducts && !u.dh;
        const CUtensorMap* mA = kMode == kProducts && u.dh ? &maps_dh.A : &maps.A;
        const CUtensorMap* mB = kMode == kProducts && u.dh ? &maps_dh.B : &maps.B;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, guard, kTimeoutStageEmpty)) { ok = false; break; }
          uint8_t* sa = smem + stage * kLpStageBytes;
          uint8_t* sb = sa + kLpABytes;
          const uint32_t bar = map_to_cta(smem_u32(&full[stage]), 0);
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * (kLpABytes + boxes * 8192));
          const bool second = low && a_mn && 2 * kb >= num_kb;           // dw: the same rows of h again, with the second halves of dx
          const int k = (second ? kb - num_kb / 2 : kb) * kLpBK;
          if (!a_mn) {
            tma_load_2d_pair(sa, mA, k, row0, bar);
          } else {
#pragma unroll
            for (int j = 0; j < kLpBM / 64; ++j) tma_load_2d_pair(sa + j * 8192, mA, row0 + j * 64, second ? kLpLow + k : k, bar);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (j >= boxes) break;
            if (!kBMn) tma_load_2d_pair(sb + j * 8192, mB, k, col0 + j * 64, bar);
            else tma_load_2d_pair(sb + j * 8192, mB, col0 + j * 64, k, bar);
          }
          if (++stage == kLpStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (rank == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      LpUnit u;
      for (int i = 0; ok && work_of.get(i, u); ++i) {
        const bool a_mn = kMode == kProducts && !u.dh;
        const uint32_t idesc = umma_idesc_bf16(2 * kLpBM, u.side < 0 ? kLpBN : kLpBNh, a_mn ? 1 : 0, kBMn ? 1 : 0);
        int from = u.kb0;
        do {                                                             // (once, of no steps at all, where nothing is multiplied)
          const int to = kSums ? min(from + kLpChunk, u.kb1) : u.kb1;
          const int buf = local & 1;
          const uint32_t acc_phase = (local >> 1) & 1;
          ++local;
          if (!mbar_wait(&acc_empty[buf], acc_phase ^ 1, guard, kTimeoutAccEmpty)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * kLpBN;
          for (int kb = from; kb < to; ++kb) {
            if (!mbar_wait(&full[stage], phase, guard, kTimeoutTmaFull)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + stage * kLpStageBytes);
            const uint32_t sb = sa + kLpABytes;
            // (advancing K by 16: 32 bytes where K is contiguous, 16 rows of 128 where it is not)
            const uint64_t da = a_mn ? smem_desc_mnmajor_sw128(sa, 8192) : smem_desc_kmajor_sw128(sa), step = a_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
            for (int k = 0; k < kLpBK / 16; ++k) {
              const uint64_t db = kBMn ? smem_desc_mnmajor_sw128(sb + k * 2048, 8192) : smem_desc_kmajor_sw128(sb + k * 32);
              umma2_ss(d_tmem, da + k * step, db, idesc, kb != from || k != 0 ? 1u : 0u);
            }
            umma2_commit_both(&empty[stage]);
            if (++stage == kLpStages) { stage = 0; phase ^= 1; }
          }
          if (ok) umma2_commit_both(&acc_full[buf]);
          from = to;
        } while (from < u.kb1 && ok);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9, both CTAs)
    const int quad = warp & 3, group = warp < 6 ? 0 : 1;
    const int dx_rows = (M + kLpBK - 1) / kLpBK * kLpBK;                 // that dx^T h reads
    int local = split ? 0 : group;
    bool ok = true;
    // One box of 128 bytes x 32 rows; `words(j)` are this lane's 16 bytes j of its row.
    auto store_box = [&](const CUtensorMap* map, auto&& words, int col, int row, bool add) {
      uint8_t* box = ring + (warp - 2) * 4096;
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the store before has read it
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) * 16)) = words(j);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if (add) tma_reduce_add_2d(map, box, col, row);
        else tma_store_2d(map, box, col, row);
        tma_store_commit();
      }
    };
    // one arrival per epilogue warp of either CTA on the leader's barrier: the accumulator buffer may be rewritten
    auto arrive = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[local & 1]), 0));
      local += split ? 1 : 2;
    };
    LpUnit u;
    for (int i = split ? 0 : group; ok && work_of.get(i, u); i += split ? 1 : 2) {
      const int nb = u.nb, side = u.side;
      const int row_w = u.mb * 2 * kLpBM + (int)rank * kLpBM + quad * 32;      // first of this warp's 32 rows
      const int second = kMode == kGrad && low && rank == 1 ? kLpLow : 0;      // the other CTA has the same rows, for the second halves of dx
      const int row = row_w - second + lane;
      const bool live = row < M;
      int label = -1;
      float lse2 = 0.f, g = 0.f, own = 0.f;
      if ((kSums || kMode == kGrad) && live) label = a.row_label[row];
      if (kMode == kGrad && live) {
        lse2 = a.lse2[row];
        g = a.dy[a.rows[row]] * a.inv_tau;
        own = g * (1.f - fast_exp2(a.picked2[row]));                     // 1 - p of the label: from the forward pass, as in log_probs_decode_kernel
        label -= a.col0;
      }
      if (!mbar_wait(&acc_full[local & 1], (local >> 1) & 1, guard, kTimeoutAccFull)) { ok = false; break; }
      tc_fence_after();
      const int part_end = split ? group + 1 : 2;
#pragma unroll 1
      for (int part = split ? group : 0; part < part_end; ++part) {           // of 128 columns
        const int col = nb * kLpBN + (side > 0 || part > 0 ? kLpStatCols : 0);
        const bool work = (side < 0 || part == 0) && col < N;
        const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + (local & 1) * kLpBN + part * kLpStatCols;
        if (kSums) {
          uint32_t r[kLpStatCols];
          if (work) {
#pragma unroll
            for (int i = 0; i < kLpStatCols / 32; ++i) tmem_ld32(t_row + i * 32, *reinterpret_cast<uint32_t(*)[32]>(r + i * 32));
            tmem_wait_ld();
          }
          if (part + 1 == part_end) arrive();
          if (split)
            for (int from = kLpChunk; from < num_kb; from += kLpChunk) {
              if (!mbar_wait(&acc_full[local & 1], (local >> 1) & 1, guard, kTimeoutAccFull)) { ok = false; break; }
              tc_fence_after();
              if (work)
#pragma unroll
                for (int i = 0; i < kLpStatCols / 32; ++i) {
                  uint32_t t[32];
                  tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + (local & 1) * kLpBN + part * kLpStatCols + i * 32, t);
                  tmem_wait_ld();
#pragma unroll
                  for (int j = 0; j < 32; ++j) r[i * 32 + j] = __float_as_uint(__uint_as_float(r[i * 32 + j]) + __uint_as_float(t[j]));
                }
              arrive();
            }
          if (!ok) break;
          if (!work) continue;
          if (col + kLpStatCols > N)
#pragma unroll
            for (int j = 0; j < kLpStatCols; ++j)
              if (col + j >= N) r[j] = 0xff800000u;                      // minus infinity
          const int at = label - col;
          if (__any_sync(0xffffffffu, at >= 0 && at < kLpStatCols)) {
            float x = 0.f;
#pragma unroll
            for (int j = 0; j < kLpStatCols; ++j) x = j == at ? __uint_as_float(r[j]) : x;
            if (at >= 0 && at < kLpStatCols) a.picked[row] = x;
          }
          float m[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) m[j] = fmaxf(__uint_as_float(r[j]), __uint_as_float(r[4 + j]));
#pragma unroll
          for (int j = 8; j < kLpStatCols; j += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = max3(m[i], __uint_as_float(r[j + 2 * i]), __uint_as_float(r[j + 2 * i + 1]));
          const float mx = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
          // (scale2 > 0.  Rounded up: no code of a kept logit may be below zero, where from 2^12 on half a step of the maximum is a quarter of a code and more)
          const float top = mx == -INFINITY ? 0.f : __fmul_ru(mx, a.scale2);
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < kLpStatCols; ++j) s[j & 3] += fast_exp2(fmaf(__uint_as_float(r[j]), a.scale2, -top));
          const long long slot = (long long)(col / kLpStatCols) * a.ld_stats + row;
          if (live) a.stats[slot] = lp_sum(mx, top, a.scale2, (s[0] + s[1]) + (s[2] + s[3]));
          if (kMode == kStatsKeep) {
            if (live) a.tops[slot] = mx == -INFINITY ? mx : top;
            const float by = -kLpCodes * a.scale2, off = top * kLpCodes;
            auto code = [&](uint32_t x) {                                // a whole number next to 2^23 has it in its low bits
              return __float_as_uint(fminf(fmaf(__uint_as_float(x), by, off), 65535.f) + 8388608.f);
            };
#pragma unroll
            for (int piece = 0; piece < 2; ++piece) {
              if (col + piece * 64 >= N) break;
              if (row_w < M) store_box(&maps.C, [&](int j) {
                const uint32_t* x = r + piece * 64 + 8 * j;
                return make_uint4(__byte_perm(code(x[0]), code(x[1]), 0x5410), __byte_perm(code(x[2]), code(x[3]), 0x5410),
                                  __byte_perm(code(x[4]), code(x[5]), 0x5410), __byte_perm(code(x[6]), code(x[7]), 0x5410));
              }, col + piece * 64, row_w, false);
            }
          }
          continue;
        }
        if (work && kMode == kGrad) {
#pragma unroll 1
          for (int piece = 0; piece < 2; ++piece) {
            const int c = col + piece * 64;
            if (c >= N) break;
            uint32_t out[32];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t r[32];
              tmem_ld32(t_row + piece * 64 + half * 32, r);
              tmem_wait_ld();
              const int at = label - c - half * 32;
              float d[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) d[j] = -g * fast_exp2(fmaf(__uint_as_float(r[j]), a.scale2, -lse2));
              if (__any_sync(0xffffffffu, at >= 0 && at < 32))
#pragma unroll
                for (int j = 0; j < 32; ++j) d[j] = j == at ? own : d[j];
              if (second)
#pragma unroll
                for (int j = 0; j < 32; ++j) d[j] -= __bfloat162float(__float2bfloat16_rn(d[j]));
#pragma unroll
              for (int j = 0; j < 16; ++j) out[half * 16 + j] = live ? pack_bf16x2(d[2 * j], d[2 * j + 1]) : 0u;
            }
            if (row_w - second < dx_rows) store_box(&maps.C, [&](int j) { return make_uint4(out[4 * j], out[4 * j + 1], out[4 * j + 2], out[4 * j + 3]); }, c, row_w, false);
          }
        } else if (work) {
          const bool bf = !u.dh && a.bf16_out;
#pragma unroll 1
          for (int piece = 0; piece < (bf ? 2 : 4); ++piece) {
            const int c = col + piece * (bf ? 64 : 32);
            if (c >= N) break;
            uint32_t out[32];
            if (bf) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                uint32_t r[32];
                tmem_ld32(t_row + piece * 64 + half * 32, r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) out[half * 16 + j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
              }
            } else {
              tmem_ld32(t_row + piece * 32, out);
              tmem_wait_ld();
            }
            if (!u.dh && num_kb == 0)                                    // no rows at all: nothing was multiplied
#pragma unroll
              for (int j = 0; j < 32; ++j) out[j] = 0u;
            if (row_w < (u.dh ? dh_rows : a.K))
              store_box(u.dh ? &maps_dh.C : &maps.C, [&](int j) { return make_uint4(out[4 * j], out[4 * j + 1], out[4 * j + 2], out[4 * j + 3]); }, c,
                        u.part * a.plane_rows + row_w, u.dh ? a.add_dh != 0 : a.add_dw != 0);
          }
        }
        if (part + 1 == part_end) arrive();
      }
    }
    if (kMode != kStats && lane == 0) tma_store_wait0();                 // its stores have written their destination
  }
  // The peer's tensor memory and barriers are written by the leader's products and commits: nobody leaves, and nothing is deallocated,
  // before both CTAs are done.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

// The log-sums of a few rows without a backward pass.  Bound: the weights' bytes.  The kernel above would multiply 256 rows, most of them padding, and the
// tensor cores' share of the power then slows the memory down (one row of 2560 against 151936 tokens 134 us by itself, 167 to 183 in a row of calls).
// Here the weights are the 128 rows of the tensor cores' product and the activations, N of them, its columns.  Every CTA has as many weight rows
// as the others, in steps of 8, in tiles of one size of at most 256, whose last rows are loaded 8 at a time: a short last tile would load
// all activations for little (1032 rows as 4 x 256 and 8: 77 rows against 151936 tokens of 2048 119.9 us).
// Epilogue: a thread has one weight row and N values; a warp adds up its 32 rows for every activation by exchanging halves, after which a
// lane has one activation's maximum (or sum), and keeps it over its tiles.  A CTA writes one maximum and sum for each activation.
constexpr int kLfThreads = 320;      // warp 0 loads, warp 1 issues products, warps 2..5 and 6..9 epilogue, each group of 128 weight rows
constexpr int kLfTile = 256;         // weight rows that share a load of the activations, at most: two products of 128 rows
constexpr int kLfMostRows = 128;
template <int N>
struct LfShape {
  static constexpr int stage_bytes = kLfTile * kLpBK * 2 + N * kLpBK * 2;
  static constexpr int stages = 200 * 1024 / stage_bytes;
  static constexpr int smem = stages * stage_bytes + 512 + N * 4 + 1024;
};

template <int N>
__global__ void __launch_bounds__(kLfThreads, 1)
log_probs_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW8, const __grid_constant__ CUtensorMap tmH, int V,
                     int D, int rows_of_cta, int tile_rows, const int* count, const int* row_label, float scale2, float2* stats, long long ld, float* picked, int* status) {
  using S = LfShape<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::stages * S::stage_bytes);
  uint64_t* empty = full + S::stages;
  uint64_t* acc_full = empty + S::stages;      // 2 buffers
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* label = reinterpret_cast<int*>(smem + S::stages * S::stage_bytes + 512);
  static_assert((2 * S::stages + 4) * 8 + 8 <= 512, "barriers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitGuard guard{abort_flag, status};
  constexpr int kCols = 4 * N <= 128 ? 128 : 4 * N <= 256 ? 256 : 512;   // two buffers of two accumulators
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 8); }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmH);
  }
  if (warp == 2) { tmem_alloc(tmem_slot, kCols); tmem_relinquish(); }
  grid_dependency_enter();
  const int n = min(*count, N);
  for (int i = threadIdx.x; i < N; i += kLfThreads) label[i] = i < n ? row_label[i] : -1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int v_lo = blockIdx.x * rows_of_cta, v_hi = min(V, v_lo + rows_of_cta);        // rows_of_cta a multiple of 8
  const int tiles = n > 0 ? (v_hi - v_lo + tile_rows - 1) / tile_rows : 0, num_kb = (D + kLpBK - 1) / kLpBK;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = 0; tile < tiles && ok; ++tile) {
        const int v0 = v_lo + tile * tile_rows, eights = (min(v_hi - v0, tile_rows) + 7) / 8;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, guard, kTimeoutStageEmpty)) { ok = false; break; }
          uint8_t* sw = smem + stage * S::stage_bytes;
          mbar_expect_tx(&full[stage], eights * 1024 + N * 128);
          int i = 0;
          for (; i + 16 <= eights; i += 16) tma_load_2d(sw + i * 1024, &tmW, kb * kLpBK, v0 + i * 8, &full[stage]);
          for (; i < eights; ++i) tma_load_2d(sw + i * 1024, &tmW8, kb * kLpBK, v0 + i * 8, &full[stage]);
          tma_load_2d(sw + kLfTile * kLpBK * 2, &tmH, kb * kLpBK, 0, &full[stage]);
          if (++stage == S::stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_bf16(128, N, 0, 0);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = 0; tile < tiles && ok; ++tile) {
        const bool both = min(v_hi - v_lo - tile * tile_rows, tile_rows) > 128;
        for (int from = 0; from < num_kb && ok; from += kLpChunk, ++local) {
          const int buf = local & 1, to = min(from + kLpChunk, num_kb);
          if (!mbar_wait(&acc_empty[buf], ((local >> 1) & 1) ^ 1, guard, kTimeoutAccEmpty)) { ok = false; break; }
          tc_fence_after();
          for (int kb = from; kb < to; ++kb) {
            if (!mbar_wait(&full[stage], phase, guard, kTimeoutTmaFull)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sw = smem_u32(smem + stage * S::stage_bytes), sh = sw + kLfTile * kLpBK * 2;
#pragma unroll
            for (int k = 0; k < kLpBK / 16; ++k) {
              const uint64_t dh = smem_desc_kmajor_sw128(sh + k * 32);
              const uint32_t add = kb != from || k != 0 ? 1u : 0u;
              umma_ss(tmem_base + buf * 2 * N, smem_desc_kmajor_sw128(sw + k * 32), dh, idesc, add);
              if (both) umma_ss(tmem_base + buf * 2 * N + N, smem_desc_kmajor_sw128(sw + 16384 + k * 32), dh, idesc, add);
            }
            umma_commit(&empty[stage]);
            if (++stage == S::stages) { stage = 0; phase ^= 1; }
          }
          if (ok) umma_commit(&acc_full[buf]);
        }
      }
    }
  } else {
    const int quad = warp & 3, half = warp < 6 ? 0 : 1;
    int local = 0;
    bool ok = true;
    float run_m[N / 32], run_s[N / 32];          // of activation 32 c + lane, over this warp's rows so far
#pragma unroll
    for (int c = 0; c < N / 32; ++c) { run_m[c] = -INFINITY; run_s[c] = 0.f; }
    for (int tile = 0; tile < tiles && ok; ++tile) {
      const int v0 = v_lo + tile * tile_rows + half * 128 + quad * 32, v = v0 + lane, v_end = min(v_hi, v_lo + (tile + 1) * tile_rows);
      float acc[N];
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.f;
      for (int from = 0; from < num_kb; from += kLpChunk, ++local) {
        if (!mbar_wait(&acc_full[local & 1], (local >> 1) & 1, guard, kTimeoutAccFull)) { ok = false; break; }
        tc_fence_after();
        if (v0 < v_end)
#pragma unroll
          for (int c = 0; c < N / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + ((local & 1) * 2 + half) * N + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c * 32 + j] += __uint_as_float(r[j]);
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[local & 1]);
      }
      if (!ok || v0 >= v_end) continue;
#pragma unroll
      for (int c = 0; c < N / 32; ++c) {
        if (c * 32 >= n) break;
        float x[32], m[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          x[j] = v < v_end ? acc[c * 32 + j] : -INFINITY;
          if (label[c * 32 + j] == v && v < v_end) picked[c * 32 + j] = x[j];
          m[j] = x[j];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)             // lanes with bit o keep the upper half of what is left
#pragma unroll
          for (int j = 0; j < o; ++j) {
            const bool up = lane & o;
            const float other = __shfl_xor_sync(0xffffffffu, up ? m[j] : m[j + o], o);
            m[j] = fmaxf(up ? m[j + o] : m[j], other);
          }
        const float now = fmaxf(run_m[c], m[0]), top = now == -INFINITY ? 0.f : now * scale2;       // of activation 32 c + lane
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = fast_exp2(fmaf(x[j], scale2, -__shfl_sync(0xffffffffu, top, j)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int j = 0; j < o; ++j) {
            const bool up = lane & o;
            const float other = __shfl_xor_sync(0xffffffffu, up ? x[j] : x[j + o], o);
            x[j] = (up ? x[j + o] : x[j]) + other;
          }
        const float2 add = lp_sum(now, top, scale2, x[0]);
        run_s[c] = run_m[c] == -INFINITY ? run_s[c] + add.y : run_s[c] * fast_exp2((run_m[c] - now) * scale2) + add.y;
        run_m[c] = now;
      }
    }
    // (the stages are free: every product has been waited for)
#pragma unroll
    for (int c = 0; c < N / 32; ++c) reinterpret_cast<float2*>(smem)[(half * 4 + quad) * N + c * 32 + lane] = make_float2(run_m[c], run_s[c]);
  }
  tc_fence_before();
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kLfThreads) {
    float m = -INFINITY, s = 0.f;
    for (int w = 0; w < 8; ++w) m = fmaxf(m, reinterpret_cast<const float2*>(smem)[w * N + i].x);
    for (int w = 0; w < 8; ++w) {
      const float2 x = reinterpret_cast<const float2*>(smem)[w * N + i];
      s += x.x == -INFINITY ? x.y : x.y * fast_exp2((x.x - m) * scale2);
    }
    stats[blockIdx.x * ld + i] = make_float2(m, s);
  }
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kCols);
  }
}

// Which rows have a label, in order: rows[i], row_label[i] and count; place[t] of every row (-1: none), and y[t] = 0 for those.  One block; a
// warp takes kLpSelectEach times 32 rows in a round, so that 8192 rows are one round of loads and one scan.
constexpr int kLpSelect = 1024;
constexpr int kLpSelectEach = 8;
__device__ __forceinline__ bool lp_has_label(long long label, int V, long long ignore) { return label != ignore && label >= 0 && label < V; }
__global__ void __launch_bounds__(kLpSelect)
log_probs_select_kernel(const long long* labels, int T, int V, long long ignore, int* rows, int* row_label, int* place, int* count, float* y) {
  __shared__ int sums[kLpSelect / 32];
  grid_dependency_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int before = 0;
  for (long long t0 = 0; t0 < T; t0 += kLpSelect * kLpSelectEach) {
    const long long t = t0 + warp * 32 * kLpSelectEach + lane;
    long long label[kLpSelectEach];
    unsigned votes[kLpSelectEach];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kLpSelectEach; ++j) label[j] = t + j * 32 < T ? labels[t + j * 32] : -1;
#pragma unroll
    for (int j = 0; j < kLpSelectEach; ++j) {
      votes[j] = __ballot_sync(0xffffffffu, t + j * 32 < T && lp_has_label(label[j], V, ignore));
      mine += __popc(votes[j]);
    }
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    int all = sums[lane];                                                // 32 warps: an inclusive sum over them in every warp
    const int own = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, all, o);
      if (lane >= o) all += v;
    }
    int at = before + __shfl_sync(0xffffffffu, all - own, warp);
#pragma unroll
    for (int j = 0; j < kLpSelectEach; ++j) {
      if (t + j * 32 < T) {
        const bool one = votes[j] >> lane & 1;
        const int i = at + __popc(votes[j] & ((1u << lane) - 1));
        place[t + j * 32] = one ? i : -1;
        if (one) { rows[i] = (int)(t + j * 32); row_label[i] = (int)label[j]; }
        else y[t + j * 32] = 0.f;
      }
      at += __popc(votes[j]);
    }
    before += __shfl_sync(0xffffffffu, all, 31);
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = before;
}

// The same and the gathering of the rows in one launch, for at most kLpFewRows rows: a block has a row, and counts the labels before it itself.
// The blocks behind the last row fill up with zeros, to `fill` rows at least.  `twice`: up to kLpLow labelled rows are there twice, which kGrad wants.
constexpr int kLpFewRows = 1024;
__global__ void __launch_bounds__(256)
log_probs_few_rows_kernel(const long long* labels, int T, int V, long long ignore, int* rows, int* row_label, int* place, int* count, float* y,
                          const bf16* h, long long ldh, bf16* dense, int D, int vec, int fill, int twice) {
  __shared__ int sums[2][8];
  grid_dependency_enter();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = 0, before = 0;
#pragma unroll
  for (int j = 0; j < kLpFewRows / 256; ++j) {
    const int i = j * 256 + threadIdx.x;
    const bool one = i < T && lp_has_label(labels[i], V, ignore);
    n += __popc(__ballot_sync(0xffffffffu, one));
    before += __popc(__ballot_sync(0xffffffffu, one && i < t));
  }
  if (lane == 0) { sums[0][warp] = n; sums[1][warp] = before; }
  __syncthreads();
  n = before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) { n += sums[0][w]; before += sums[1][w]; }
  const long long label = t < T ? labels[t] : -1;
  const bool one = t < T && lp_has_label(label, V, ignore);
  // a block without a labelled row of its own: row n + (which of those it is) of the dense array, if that is still in the last kLpBK
  const int at = one ? before : n + (t - before);
  if (threadIdx.x == 0) {
    if (t == 0) *count = n;
    if (t < T) {
      place[t] = one ? at : -1;
      if (one) { rows[at] = t; row_label[at] = (int)label; }
      else y[t] = 0.f;
    }
  }
  if (!one && at >= max((n + kLpBK - 1) / kLpBK * kLpBK, fill)) return;
  const bf16* from = h + (long long)t * ldh;
  for (int c = threadIdx.x * 8; c < D; c += 256 * 8) {
    BF8 v{{0, 0, 0, 0}};
    if (one) {
      if (vec) v = *reinterpret_cast<const BF8*>(from + c);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<bf16*>(&v)[j] = from[c + j];
    }
    *reinterpret_cast<BF8*>(dense + at * lp_pitch(D) + c) = v;
    if (twice && n <= kLpLow && one) *reinterpret_cast<BF8*>(dense + (at + kLpLow) * lp_pitch(D) + c) = v;
  }
}

// dense[i] = h[rows[i]], and zeros up to the next multiple of kLpBK: those rows are part of dw's last products.
__global__ void __launch_bounds__(256)
log_probs_gather_kernel(const bf16* h, long long ldh, const int* rows, const int* count, bf16* dense, int D, int vec, int twice) {
  grid_dependency_enter();
  const int n = *count, end = (n + kLpBK - 1) / kLpBK * kLpBK, per_row = D / 8;
  const long long all = (long long)end * per_row;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const int row = (int)(i / per_row), c = (int)(i - (long long)row * per_row) * 8;
    BF8 v{{0, 0, 0, 0}};
    if (row < n) {
      const bf16* from = h + (long long)rows[row] * ldh + c;
      if (vec) v = *reinterpret_cast<const BF8*>(from);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<bf16*>(&v)[j] = from[j];
    }
    *reinterpret_cast<BF8*>(dense + row * lp_pitch(D) + c) = v;
    if (twice && n <= kLpLow && row < n) *reinterpret_cast<BF8*>(dense + (row + kLpLow) * lp_pitch(D) + c) = v;
  }
}

// y and lse2 of a row from its columns' maxima and sums.  A block has kRows rows: 32 where that leaves enough blocks (a warp reads whole lines
// then), else 8.  A thread takes kLpSumEach at a time: their maximum, then one exponential for each.
constexpr int kLpSumEach = 8;
template <int kRows>
__global__ void __launch_bounds__(512)
log_probs_sum_kernel(const float2* stats, long long ld, int slots, const float* picked, const int* rows, const int* count, float scale2, float inv_tau, float* y,
                     float* lse2, float* picked2) {
  constexpr int kThreadsOfRow = 512 / kRows, kWarps = 16;
  __shared__ float2 part[kWarps][kRows];
  grid_dependency_enter();
  const int n = *count, r = threadIdx.x % kRows, s0 = threadIdx.x / kRows, row = blockIdx.x * kRows + r;
  if ((int)blockIdx.x * kRows >= n) return;
  float m = -INFINITY, s = 0.f;
  // (a sum without a maximum is 0, or what is no number)
  auto scaled = [&](float s, float m, float top) { return m == -INFINITY ? s : s * fast_exp2((m - top) * scale2); };
  if (row < n) {
    for (int i = s0; i < slots; i += kThreadsOfRow * kLpSumEach) {
      float2 x[kLpSumEach];
      float top = m;
#pragma unroll
      for (int j = 0; j < kLpSumEach; ++j)
        x[j] = i + j * kThreadsOfRow < slots ? stats[(long long)(i + j * kThreadsOfRow) * ld + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < kLpSumEach; ++j) top = fmaxf(top, x[j].x);
      s = scaled(s, m, top);
#pragma unroll
      for (int j = 0; j < kLpSumEach; ++j) s += scaled(x[j].y, x[j].x, top);
      m = top;
    }
  }
  auto add = [&](float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    s = scaled(s, m, top) + scaled(s2, m2, top);
    m = top;
  };
#pragma unroll
  for (int o = 16; o >= kRows; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    add(m, s, m2, s2);
  }
  if ((threadIdx.x & 31) < kRows) part[threadIdx.x >> 5][r] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < kRows && row < n) {
    m = part[0][r].x;
    s = part[0][r].y;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) add(m, s, part[w][r].x, part[w][r].y);
    const float gap = picked[row] - m;                                   // (the fast logarithm is off by 2^-22 of itself)
    const double l = log((double)s);
    y[rows[row]] = (float)((double)gap * (double)inv_tau - l);
    const float l2 = (float)(l * 1.4426950408889634);
    lse2[row] = fmaf(m, scale2, l2);
    picked2[row] = fmaf(gap, scale2, -l2);
  }
}

// dx of the rows with a label from the kept logits (both halves of it of few rows), and zeros up to the next multiple of kLpBK.  A block has 8 rows and 1024 columns, a
// warp one of the rows.
constexpr int kLpDecodeCols = 1024;
__global__ void __launch_bounds__(256)
log_probs_decode_kernel(const uint16_t* codes, long long pitch, const float* tops, long long ld, const float* lse2, const float* picked2, const float* dy,
                        const int* rows, const int* row_label, const int* count, bf16* dx, int V, float inv_tau, int col_blocks) {
  grid_dependency_enter();
  const int n = *count, lane = threadIdx.x & 31;
  const long long row = blockIdx.x / col_blocks * 8LL + (threadIdx.x >> 5);
  const int col0 = (int)(blockIdx.x % col_blocks) * kLpDecodeCols + lane * 8;
  if (row >= (n + kLpBK - 1) / kLpBK * kLpBK) return;
  const bool live = row < n;
  const float g = live ? dy[rows[row]] * inv_tau : 0.f, lse = live ? lse2[row] : 0.f;
  const int label = live ? row_label[row] : -1;
  uint4 v[4];
  float top[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = col0 + k * 256;
    v[k] = make_uint4(0, 0, 0, 0);
    top[k] = -INFINITY;
    if (live && c < V) {                                                 // (the pitch is a multiple of 8)
      v[k] = *reinterpret_cast<const uint4*>(codes + row * pitch + c);
      top[k] = tops[(long long)(c / kLpStatCols) * ld + row];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = col0 + k * 256;
    if (c >= V) break;
    const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    const float off = top[k] - lse;
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float code = __uint_as_float(0x4b000000u | (j & 1 ? u[j >> 1] >> 16 : u[j >> 1] & 0xffffu)) - 8388608.f;
      d[j] = -g * fast_exp2(fmaf(code, -1.f / kLpCodes, off));
      if (c + j == label) d[j] = g * (1.f - fast_exp2(picked2[row]));    // (of the exact logit: next to a probability of one its rounding would be all of it)
      if (!live) d[j] = 0.f;
    }
    store8(dx + row * pitch + c, d);
    if (n <= kLpLow) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] -= __bfloat162float(__float2bfloat16_rn(d[j]));
      store8(dx + (row + kLpLow) * pitch + c, d);
    }
  }
}

// dh[t] = the gathered gradient of row t in bf16, its parts added up in order, and 0 without a label.  A thread has 4 columns of a row; kSplit threads
// share them where there are few values and may be many parts (one row in 64 parts 39 us by one thread each, 6 by 8; 4915 rows in 6 parts 54 and 124).
template <int kSplit>
__global__ void __launch_bounds__(256)
log_probs_scatter_kernel(const float* dense, const int* place, const int* count, const int* parts_made, bf16* dh, int T, int D, long long plane) {
  __shared__ float4 sums[kSplit][256 / kSplit];
  grid_dependency_enter();
  const int parts = *parts_made, per_row = D / 4;
  const bool low = *count <= kLpLow;
  const int lane = threadIdx.x % (256 / kSplit), first = threadIdx.x / (256 / kSplit);
  const long long all = (long long)T * per_row;
  for (long long i0 = blockIdx.x * (256LL / kSplit); i0 < all; i0 += gridDim.x * (256LL / kSplit)) {
    const long long i = i0 + lane;
    const int t = (int)(i / per_row), c = (int)(i - (long long)t * per_row) * 4, at = i < all ? place[t] : -1;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0) {
      const float* from = dense + (long long)at * D + c;
#pragma unroll 8
      for (int p = first; p < parts; p += kSplit) {
        const float4 u = *reinterpret_cast<const float4*>(from + p * plane);
        f.x += u.x; f.y += u.y; f.z += u.z; f.w += u.w;
        if (low) {
          const float4 v = *reinterpret_cast<const float4*>(from + p * plane + (long long)kLpLow * D);
          f.x += v.x; f.y += v.y; f.z += v.z; f.w += v.w;
        }
      }
    }
    if (kSplit > 1) {
      __syncthreads();
      sums[first][lane] = f;
      __syncthreads();
      if (first != 0) continue;
#pragma unroll
      for (int p = 1; p < kSplit; ++p) {
        const float4 u = sums[p][lane];
        f.x += u.x; f.y += u.y; f.z += u.z; f.w += u.w;
      }
    }
    if (i < all) *reinterpret_cast<uint2*>(dh + i * 4) = make_uint2(pack_bf16x2(f.x, f.y), pack_bf16x2(f.z, f.w));
  }
}

static int lp_map(CUtensorMap* m, const void* base, int elem, long long cols, long long rows, long long pitch, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, str[2] = {(uint64_t)elem, (uint64_t)pitch * elem};
  const uint32_t box[2] = {(uint32_t)(128 / elem), (uint32_t)box_rows};
  return make_tmap(m, base, elem, 2, dims, str, box, true);
}

static long long lp_tiles(int M, int N) { return (long long)((M + 2 * kLpBM - 1) / (2 * kLpBM)) * ((N + kLpBN - 1) / kLpBN); }
// CTA pairs of a launch of so many units at most (where fewer rows have a label than there are, the last ones may stay idle)
static int lp_pairs(long long units, int sms) { return (int)(units < sms / 2 ? units : sms / 2); }
static long long lp_product_units(int T, int D, int n, bool dh, bool dw, int planes) { return (dh ? lp_tiles(T, D) * planes : 0) + (dw ? 2 * lp_tiles(n, D) : 0); }

// Whether both products go into one launch: up to this many steps of kLpBK on a pair (half a millisecond).  600 rows of 2048 against 20000 tokens 198 -> 160 us,
// 1000 of 512 against 50000 (half of them with a label) 145 -> 122, 3000 of 1024 against 50000 800 -> 788; 4915 of 2048 against 151936 take 8.43 ms in two
// launches and 8.63 in one, at 1.5 % fewer cycles: the clock is lower by more than that under the power limit.
constexpr long long kLpTogether = 1500;
static bool lp_together(int T, int D, int n, bool dh, bool dw, int sms) {
  const long long steps = lp_tiles(T, D) * ((n + kLpBK - 1) / kLpBK) + lp_tiles(n, D) * ((T + kLpBK - 1) / kLpBK);
  return dh && dw && steps <= kLpTogether * (sms / 2);
}

template <int kMode>
static int launch_log_probs(const LpMaps& maps, const LpMaps& maps_dh, LpArgs a, long long units, cudaStream_t st) {
  const int sms = sm_count();
  KSA_REQUIRE(sms > 1, "no device");
  KSA_REQUIRE(units > 0 && units < (1 << 28), "log_probs: %lld tiles", units);
  a.status = status_word();
  KSA_REQUIRE(a.status != nullptr, "could not allocate the status word");
  auto kern = log_probs_pair_kernel<kMode>;
  static PerDevice raised;
  KSA_CHECK_CUDA(raise_smem_limit(raised, kern, kLpSmem));
  KSA_CHECK_CUDA(launch_kernel(kern, dim3(2 * lp_pairs(units, sms)), dim3(kLpThreads), (size_t)kLpSmem, st, maps, maps_dh, a));
  return 0;
}

}  // namespace ksa

using namespace ksa;
#define ST(s) reinterpret_cast<cudaStream_t>(s)

// Weight rows of a CTA of the kernel for few rows
static int lf_rows(int V, int sms) {
  const int each = (V + sms - 1) / sms;
  return (each + 7) / 8 * 8;
}

// fp32 values of workspace for the forward pass
KSA_API long long ksa_log_probs_work(int T, int V) {
  const int sms = sm_count() > 0 ? sm_count() : 1, rows = lf_rows(V, sms);
  const long long few = T <= kLfMostRows ? (V + rows - 1) / rows : 0;
  const long long slots = (V + kLpStatCols - 1) / kLpStatCols;
  return (T + 3LL) / 4 * 4 * (2 * (few > slots ? few : slots) + 1);
}

// Forward.  h [T, D] (row pitch ldh, any alignment of its type), w [V, D] (row pitch ldw, a multiple of 8, 16-byte aligned), labels [T] int64.
// Leaves what the backward pass needs: dense [T rounded up to 256, D rounded up to 64] bf16, rows, row_label, place [T], count [1] int32, lse2 [2 T] (the log-sums
// and the labels' logits less those, base 2), and where codes is not null the logits in 16 bits, codes [T rounded up to 256, V rounded up to 64]
// with tops, fp32 [ceil(V / 128) times T rounded up to 4].  (Without codes up to 128 labelled rows are in dense twice: a backward pass without them needs that.)
// work: fp32 [ksa_log_probs_work(T, V)].  y [T] fp32.
KSA_API int ksa_log_probs(const void* h, const void* w, const void* labels, void* dense, void* rows, void* row_label, void* place, void* count,
                          void* lse2, void* work, void* y, void* codes, void* tops, int T, int V, int D, long long ldh, long long ldw, long long ignore_index, float tau,
                          void* stream) {
  KSA_ENTER(w);
  KSA_REQUIRE(T > 0 && V > 0 && D > 0, "log_probs: empty problem %d x %d x %d", T, V, D);
  KSA_REQUIRE(D % 8 == 0 && ldw % 8 == 0 && ldw >= D, "log_probs: D=%d and the weights' pitch %lld must be multiples of 8", D, ldw);
  KSA_REQUIRE(tau > 0.f && isfinite(tau), "log_probs: the temperature must be a positive number");
  KSA_REQUIRE(T <= 0x7fffffff - kLpRowPad, "log_probs: %d rows", T);
  cudaStream_t st = ST(stream);
  const int padded = (T + kLpRowPad - 1) / kLpRowPad * kLpRowPad, slots = (V + kLpStatCols - 1) / kLpStatCols;
  const long long ld = (T + 3LL) / 4 * 4;
  float2* stats = static_cast<float2*>(work);
  const float scale2 = (float)(1.4426950408889634 / (double)tau);
  float* picked = reinterpret_cast<float*>(stats + ld * slots);
  const int vec = ldh % 8 == 0 && (reinterpret_cast<uintptr_t>(h) & 15) == 0;
  const bool few = T <= kLfMostRows && codes == nullptr;
  const int columns = (T + 31) / 32 * 32;                 // of the product with few rows
  if (T <= kLpFewRows) {
    const int fill = few ? columns : 0, blocks = T + kLpBK - 1 > fill ? T + kLpBK - 1 : fill;
    KSA_CHECK_CUDA(launch_kernel(log_probs_few_rows_kernel, dim3(blocks), dim3(256), 0, st, (const long long*)labels, T, V, ignore_index, (int*)rows,
                                 (int*)row_label, (int*)place, (int*)count, (float*)y, (const bf16*)h, ldh, (bf16*)dense, D, vec, fill, (int)(codes == nullptr)));
  } else {
    KSA_CHECK_CUDA(launch_kernel(log_probs_select_kernel, dim3(1), dim3(kLpSelect), 0, st, (const long long*)labels, T, V, ignore_index, (int*)rows,
                                 (int*)row_label, (int*)place, (int*)count, (float*)y));
    const long long vectors = (T + 63LL) / 64 * 64 * (D / 8);
    const int gather_blocks = (int)(vectors < 256 * 148 * 8 ? (vectors + 255) / 256 : 148 * 8);
    KSA_CHECK_CUDA(launch_stream_kernel(4LL * T * D, log_probs_gather_kernel, dim3(gather_blocks), dim3(256), 0, st, (const bf16*)h, ldh,
                                        (const int*)rows, (const int*)count, (bf16*)dense, D, vec, (int)(codes == nullptr)));
  }
  LpMaps m;
  int rc, sums = slots;
  if (few) {
    const int sms = sm_count(), rows_of_cta = lf_rows(V, sms), ctas = (V + rows_of_cta - 1) / rows_of_cta;
    const int tiles = (rows_of_cta + kLfTile - 1) / kLfTile, tile_rows = (rows_of_cta + 8 * tiles - 1) / (8 * tiles) * 8;
    sums = ctas;
    picked = reinterpret_cast<float*>(stats + ld * sums);
    rc = lp_map(&m.A, w, 2, D, V, ldw, 128);
    if (rc == 0) rc = lp_map(&m.B, w, 2, D, V, ldw, 8);
    if (rc == 0) rc = lp_map(&m.C, dense, 2, D, padded, lp_pitch(D), columns);
    if (rc) return rc;
    int* status = status_word();
    KSA_REQUIRE(status != nullptr, "could not allocate the status word");
    auto kern = columns == 32 ? log_probs_few_kernel<32> : columns == 64 ? log_probs_few_kernel<64> : columns == 96 ? log_probs_few_kernel<96> : log_probs_few_kernel<128>;
    const int smem = columns == 32 ? LfShape<32>::smem : columns == 64 ? LfShape<64>::smem : columns == 96 ? LfShape<96>::smem : LfShape<128>::smem;
    static PerDevice raised[4];
    KSA_CHECK_CUDA(raise_smem_limit(raised[columns / 32 - 1], kern, smem));
    KSA_CHECK_CUDA(launch_kernel(kern, dim3(ctas), dim3(kLfThreads), (size_t)smem, st, m.A, m.B, m.C, V, D, rows_of_cta, tile_rows, (const int*)count, (const int*)row_label,
                                 scale2, stats, ld, picked, status));
  } else {
    rc = lp_map(&m.A, dense, 2, D, padded, lp_pitch(D), kLpBM);
    if (rc == 0) rc = lp_map(&m.B, w, 2, D, V, ldw, 64);
    if (rc == 0 && codes) rc = lp_map(&m.C, codes, 2, V, padded, lp_pitch(V), 32);
    if (rc) return rc;
    LpArgs a{};
    a.M = T; a.N = V; a.K = D;
    a.count = static_cast<const int*>(count); a.row_label = static_cast<const int*>(row_label);
    a.scale2 = scale2;
    a.stats = stats; a.picked = picked; a.ld_stats = ld; a.tops = static_cast<float*>(tops);
    const long long units = 2 * lp_tiles(T, V);
    rc = codes ? launch_log_probs<kStatsKeep>(m, m, a, units, st) : launch_log_probs<kStats>(m, m, a, units, st);
    if (rc) return rc;
  }
  const bool wide = T >= 32 * 148;
  KSA_CHECK_CUDA(launch_kernel(wide ? log_probs_sum_kernel<32> : log_probs_sum_kernel<8>, dim3(wide ? (T + 31) / 32 : (T + 7) / 8), dim3(512), 0, st,
                               (const float2*)stats, ld, sums, (const float*)picked, (const int*)rows, (const int*)count, scale2, 1.f / tau, (float*)y,
                               (float*)lse2, (float*)lse2 + T));
  return 0;
}

// Backward.  dy [T] fp32; dh [T, D] bf16 or null; dw [V, D] (row pitch lddw) or null, bf16 or (dw_fp32) fp32, there with add_dw added to.
// dx: bf16 [T rounded up to 256, slab], the vocabulary's columns being taken `slab` at a time (a multiple of 8; with codes: V rounded up to 64).
// dh32: fp32 [planes, T rounded up to 256, D] where dh is wanted, 1 to 64 planes, only one where not all columns are taken at a time; and one word
// (int32) behind the planes, how many of them were used.
KSA_API int ksa_log_probs_bwd(const void* dense, const void* w, const void* rows, const void* row_label, const void* place, const void* count,
                              const void* lse2, const void* codes, const void* tops, const void* dy, void* dx, void* dh32, void* dh, void* dw, int T, int V, int D, long long ldw,
                              long long lddw, int dw_fp32, int add_dw, int slab, int planes, float tau, void* stream) {
  KSA_ENTER(w);
  KSA_REQUIRE(T > 0 && V > 0 && D > 0 && D % 8 == 0 && ldw % 8 == 0, "log_probs: backward of %d x %d x %d", T, V, D);
  KSA_REQUIRE(!dw || lddw % (dw_fp32 ? 4 : 8) == 0, "log_probs: the pitch %lld of the weights' gradient keeps no alignment of 16 bytes", lddw);
  KSA_REQUIRE(slab > 0 && slab % 8 == 0, "log_probs: %d columns at a time (a multiple of 8)", slab);
  KSA_REQUIRE(planes >= 1 && planes <= 64 && (planes == 1 || slab >= V), "log_probs: %d planes", planes);
  KSA_REQUIRE(!codes || (tops && slab == lp_pitch(V)), "log_probs: kept logits are taken all at a time");
  KSA_REQUIRE(!(add_dw && !dw_fp32), "log_probs: only an fp32 gradient is added to");
  KSA_REQUIRE(!dh || (reinterpret_cast<uintptr_t>(dh) & 15) == 0, "log_probs: the gradient of the rows must be 16-byte aligned");
  cudaStream_t st = ST(stream);
  const int padded = (T + kLpRowPad - 1) / kLpRowPad * kLpRowPad;
  const bool together = lp_together(T, D, V < slab ? V : slab, dh != nullptr, dw != nullptr, sm_count());
  float* planes_end = dh ? static_cast<float*>(dh32) + (long long)planes * padded * D : nullptr;
  LpMaps grad, by_w, by_h;                                               // dx again; dx w; dx^T h
  int rc = lp_map(&grad.A, dense, 2, D, padded, lp_pitch(D), kLpBM);
  if (rc == 0) rc = lp_map(&by_h.B, dense, 2, D, padded, lp_pitch(D), 64);
  if (rc == 0 && dh) rc = lp_map(&by_w.C, dh32, 4, D, (long long)planes * padded, D, 32);
  for (long long v0 = 0; v0 < V && rc == 0; v0 += slab) {
    const int n = V - v0 < slab ? (int)(V - v0) : slab;
    const bf16* wv = static_cast<const bf16*>(w) + v0 * ldw;
    LpArgs a{};
    a.count = static_cast<const int*>(count); a.rows = static_cast<const int*>(rows); a.row_label = static_cast<const int*>(row_label);
    a.scale2 = (float)(1.4426950408889634 / (double)tau); a.inv_tau = 1.f / tau;
    a.lse2 = static_cast<const float*>(lse2); a.picked2 = a.lse2 + T; a.dy = static_cast<const float*>(dy); a.col0 = (int)v0;
    if (codes) {
      const int col_blocks = (V + kLpDecodeCols - 1) / kLpDecodeCols;
      const long long blocks = (T + 63LL) / 64 * 8 * col_blocks;
      KSA_REQUIRE(blocks < (1LL << 31), "log_probs: %d x %d kept logits", T, V);
      KSA_CHECK_CUDA(launch_stream_kernel(4LL * T * V, log_probs_decode_kernel, dim3((unsigned)blocks), dim3(256), 0, st, (const uint16_t*)codes,
                                          (long long)slab, (const float*)tops, (T + 3LL) / 4 * 4, a.lse2, a.picked2, a.dy, a.rows, a.row_label, a.count,
                                          (bf16*)dx, V, a.inv_tau, col_blocks));
    } else {
      a.M = T; a.N = n; a.K = D;
      rc = lp_map(&grad.B, wv, 2, D, n, ldw, 64);
      if (rc == 0) rc = lp_map(&grad.C, dx, 2, n, padded, slab, 32);
      if (rc == 0) rc = launch_log_probs<kGrad>(grad, grad, a, 2 * lp_tiles(T, n), st);
    }
    if (rc == 0 && (dh || dw)) {
      a.M = T; a.N = D; a.K = n; a.dh = a.dw = 1; a.add_dh = v0 > 0; a.add_dw = add_dw;
      a.planes = planes; a.plane_rows = padded; a.parts = reinterpret_cast<int*>(planes_end); a.bf16_out = !dw_fp32;
      if (dh) {
        rc = lp_map(&by_w.A, dx, 2, n, padded, slab, kLpBM);
        if (rc == 0) rc = lp_map(&by_w.B, wv, 2, D, n, ldw, 64);
      }
      if (rc == 0 && dw) {
        rc = lp_map(&by_h.A, dx, 2, n, padded, slab, 64);
        if (rc == 0) rc = dw_fp32 ? lp_map(&by_h.C, static_cast<float*>(dw) + v0 * lddw, 4, D, n, lddw, 32) : lp_map(&by_h.C, static_cast<bf16*>(dw) + v0 * lddw, 2, D, n, lddw, 32);
      }
      if (together) {
        if (rc == 0) rc = launch_log_probs<kProducts>(by_h, by_w, a, lp_product_units(T, D, n, true, true, planes), st);
      } else {
        a.dw = 0;
        if (rc == 0 && dh) rc = launch_log_probs<kProducts>(by_w, by_w, a, lp_product_units(T, D, n, true, false, planes), st);
        a.dh = 0; a.dw = 1;
        if (rc == 0 && dw) rc = launch_log_probs<kProducts>(by_h, by_h, a, lp_product_units(T, D, n, false, true, planes), st);
      }
    }
  }
  if (rc) return rc;
  if (dh) {
    const int split = planes > 8 && (long long)T * (D / 4) < 148 * 1024 ? 8 : 1;
    const long long blocks = ((long long)T * (D / 4) * split + 255) / 256;
    KSA_CHECK_CUDA(launch_stream_kernel(6LL * T * D, split > 1 ? log_probs_scatter_kernel<8> : log_probs_scatter_kernel<1>,
                                        dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(256), 0, st, (const float*)dh32, (const int*)place,
                                        (const int*)count, (const int*)planes_end, (bf16*)dh, T, D, (long long)padded * D));
  }
  return 0;
}
