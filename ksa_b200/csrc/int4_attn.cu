// Decode attention over a KV cache of four bits: out = softmax(q K^T * scale) V over a slice [start, start + length) of the cache for every
// (sequence, query token), the G = Hq / Hkv heads of a KV head together.
//
// What bounds it is reading the slice once, 160 bytes a slot and KV head at head dim 128 (bf16: 512).  Hence:
//   * all (slice, KV head) items in a row are one sequence of tiles of 32 slots, and every CTA takes an equal run of it, whatever the
//     slices' lengths are (they are known on the device only).  A run that covers part of an item leaves (max, sum, output) behind, and a
//     second kernel merges the parts of an item in a fixed order; an item within one run is finished there;
//   * a warp of its own keeps tiles in flight through a ring, four at a time (a tile is contiguous: 2 KB of codes and 512 bytes of scales for K and for
//     V, and up to four of one item are one bulk copy each), and four warps take one tile of every group of four;
//   * both products are mma.sync m16n8k16 with the values straight from their codes (int4.cuh) as an operand.  A lane's four words of a key
//     are values 32 t .. 32 t + 31 of it, one group with one scale; the order of the head dimension in the product is q's as well, so nothing is
//     moved.  Keys are the 16 rows of the first product and value dimensions those of the second, queries the 8 columns of both, so up to
//     eight heads waste no row; the probabilities become the second one's right operand by movmatrix.  V^T wants the same value of two
//     neighbouring keys in a register, which is a byte permutation of two words before the shift;
//   * a probability enters the second product as two bf16 terms, its rounding and what that leaves, which keeps 16 bits of it.  Up to four heads leave
//     half of the eight columns free, and these hold the same queries once more: there the second terms go along in the same instructions.  More
//     heads cost the second product twice.  Against probabilities of eight bits: one sequence of 131071 slots, 32 heads over 8, 44.6 -> 45.9 us, 64 over 8
//     49 -> 52.5; 16 of 32768, 32 over 8, 137 -> 142, 32 over 2 62 -> 69.5.
// Nothing outside a slice enters a result: slots of the slice's first and last tile that lie outside get probability 0 and scale and offset 0, so
// that a NaN there stays there.
#include <float.h>
#include <math.h>

#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4Tile = 32;        // slots of a tile, which one warp takes
constexpr int kI4Warps = 4;        // that compute, each the same tile of every group of kI4Warps tiles; one more fetches
constexpr int kI4Threads = kI4Warps * 32 + 32;
constexpr int kI4Spread = 4;       // tiles that a CTA gets at least
// CTAs of an SM (fifteen warps get 128 registers each, ten 168)
template <int NT>
constexpr int i4_ctas() { return NT == 1 ? 3 : 2; }
// Short slices: the CTAs of an item are a cluster and merge through its shared memory, in one launch and with nothing to look up but the own row's
// slice.  Full caches took, in us, by the sequence and here (32 query heads, 8 key heads of
// 128): one sequence of 256 slots 6.0 -> 4.0, 1168 8.9 -> 5.0, 4096 7.9 -> 7.7, 8192 12.2 -> 11.9, 16384 14.8 -> 19.7; six of 1168 12.1 -> 7.6, of
// 4096 17.1 -> 12.6, of 16384 37 -> 35; in two rounds of clusters twelve of 1168 14.8 -> 14.6, of 2048 17.4 -> 17.0, of 4096 24.0 -> 25.1; in
// four 24 of 1168 19.2 -> 28.4.
// Sixteen query heads a key head: two items of 2048 slots 9.1 -> 6.8, of 4096 8.3 -> 9.3, of 8192 10.8 -> 14.9; four of 4096 10.4 -> 9.7, of 8192 13.7 -> 15.1;
// eight of 8192 19.2 -> 16.5, sixteen 21.6 -> 20.4.  So more than four items go up to twice as many slots.
constexpr int kI4Cluster = 8, kI4ClusterSlots = 4096;
constexpr int kI4Align = 16;       // tiles start at multiples of this, and so does the capacity
// Probabilities are 2^(score - m), and m is the greatest score of some time ago plus kI4Above: it moves when a score is kI4Late powers of two above that
// one.  Sums of up to 2^24 probabilities so stay below 1, and those of values, which reach 2^126, within fp32; what is lost are outputs below 2^-94.
// Before the first score m is the least number, so that scores of minus infinity (products past fp32) weigh nothing.
constexpr float kI4Late = 8.f, kI4Above = 32.f;
constexpr float kI4Least = -FLT_MAX;

struct Int4Attn {
  const bf16* q;                   // [B, Tq, Hq, D], strides below, heads' rows contiguous
  long long q_sb, q_st, q_sh;
  const uint8_t *k, *v;            // [B, Hkv, cap, D / 2]
  const uint32_t *k_meta, *v_meta; // [B, Hkv, cap, D / 32]
  const int *start, *len;          // [B, Tq]
  float* part_o;                   // [CTAs + items, heads, D]
  float2* part_ml;                 // [CTAs + items, heads]: max (log2 units), sum
  int2* shared;                    // [CTAs]: the item that begins in a CTA's run and goes on behind it, and over how many CTAs (0: none does)
  bf16* out;                       // [B, Tq, Hq, D]
  int rows, Tq, Hq, Hkv, cap;      // rows = B * Tq
  int heads, blocks;               // query heads of an item; items of a KV head
  int ctas, groups;                // of the grid; of the ring, kI4Warps tiles each
  float scale;                     // its magnitude * log2(e)
  uint32_t negate;                 // the sign bits of a pair of queries where the scale is negative
};

__device__ __forceinline__ void i4_slice(const Int4Attn& a, int row, int& lo, int& hi) {
  const long long s = a.start[row], e = s + max(a.len[row], 0);
  lo = (int)max(s, 0LL);
  hi = (int)min(e, (long long)a.cap);          // whatever the device holds as slices: never past the cache
}
__device__ __forceinline__ int i4_tiles(int lo, int hi) {
  return hi > lo ? (hi - (lo & ~(kI4Align - 1)) + kI4Tile - 1) / kI4Tile : 0;
}
__device__ __forceinline__ int i4_row_tiles(const Int4Attn& a, int row) {
  if (row >= a.rows) return 0;
  int lo, hi;
  i4_slice(a, row, lo, hi);
  return i4_tiles(lo, hi);
}
// Rows' tiles, 32 rows at a time: the sum up to this lane's row.
__device__ __forceinline__ int i4_scan(int mine, int lane) {
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += x;
  }
  return sum;
}

// How the sequence of `total` tiles is shared: CTAs that take part, and their runs, the first `more` of which have one tile more than the others.
struct Int4Share {
  int ctas, per, more;
  __device__ __forceinline__ Int4Share(const Int4Attn& a, int total) {
    ctas = max(1, min(a.ctas, (total + kI4Spread - 1) / kI4Spread));
    per = total / ctas;
    more = total - per * ctas;
  }
  __device__ __forceinline__ int first(int cta) const { return per * cta + min(cta, more); }
  __device__ __forceinline__ int owner(int tile) const {
    const int wide = more * (per + 1);
    return tile < wide ? tile / (per + 1) : more + (tile - wide) / per;
  }
};

// A place in the sequence of tiles.
struct Int4Cursor {
  int row, head, tile;             // row, item of the row (KV head and block of its query heads), tile of the item
  int lo, hi, n;                   // the row's slice and tiles
  long long base;                  // where the item's first tile starts in the cache, in slots
  __device__ __forceinline__ void load(const Int4Attn& a) {
    i4_slice(a, row, lo, hi);
    n = i4_tiles(lo, hi);
  }
  __device__ __forceinline__ void enter(const Int4Attn& a) {
    base = ((long long)(a.Tq == 1 ? row : row / a.Tq) * a.Hkv + (a.blocks == 1 ? head : head / a.blocks)) * a.cap + (lo & ~(kI4Align - 1));
  }
  // The number of tiles, by a warp; `mine` and `sum` keep the last 32 rows' scan, which is all of it for up to 32 rows.
  static __device__ __forceinline__ int count(const Int4Attn& a, int& mine, int& sum, int lane) {
    const int per_row = a.Hkv * a.blocks;
    if (a.rows == 1) return (sum = mine = i4_row_tiles(a, 0)) * per_row;
    int rows = 0;
    for (int base = 0; base < a.rows; base += 32) {
      mine = i4_row_tiles(a, base + lane);
      sum = i4_scan(mine, lane);
      rows += __shfl_sync(0xffffffffu, sum, 31);
    }
    return rows * per_row;
  }
  // tile `left` of the sequence, which has to be there, by a warp
  __device__ __forceinline__ void seek(const Int4Attn& a, int left, int mine, int sum, int lane) {
    const int per_row = a.Hkv * a.blocks;
    row = 0;
    for (int base = 0; a.rows > 1 && base < a.rows; base += 32) {
      if (a.rows > 32) {
        mine = i4_row_tiles(a, base + lane);
        sum = i4_scan(mine, lane);
      }
      const int all = __shfl_sync(0xffffffffu, sum, 31) * per_row;
      if (left >= all) { left -= all; continue; }
      const int who = __ffs(__ballot_sync(0xffffffffu, left < sum * per_row)) - 1;
      left -= __shfl_sync(0xffffffffu, sum - mine, who) * per_row;
      row = base + who;
      break;
    }
    load(a);
    head = left / n;
    tile = left - head * n;
    enter(a);
  }
  // by `by` tiles, at most to the first of the next item
  __device__ __forceinline__ void advance(const Int4Attn& a, int by) {
    tile += by;
    if (tile < n) return;
    tile = 0;
    if (++head == a.Hkv * a.blocks) {
      head = 0;
      do {
        if (++row >= a.rows) return;
        load(a);
      } while (n == 0);
    }
    enter(a);
  }
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// The ring: tile i of a CTA's run lies in slot i % (groups * kI4Warps) of each of the four parts.
template <int D>
struct Int4Ring {
  uint32_t *k, *v, *k_meta, *v_meta;
  __device__ __forceinline__ Int4Ring(uint8_t* raw, int tiles) {
    k = reinterpret_cast<uint32_t*>(raw);
    v = k + tiles * (kI4Tile * D / 8);
    k_meta = v + tiles * (kI4Tile * D / 8);
    v_meta = k_meta + tiles * (kI4Tile * D / 32);
  }
};
// `tiles` tiles of the cursor's item from its own on, cut to the cache, into the ring from `slot` on.  One thread; `last`: the group is complete.
template <int D>
__device__ __forceinline__ void i4_fetch(const Int4Attn& a, const Int4Cursor& c, int tiles, const Int4Ring<D>& ring, int slot, uint64_t* bar, bool last) {
  const int first = c.tile * kI4Tile, n = min(tiles * kI4Tile, a.cap - (c.lo & ~(kI4Align - 1)) - first);
  const long long at = c.base + first;
  if (last) mbar_expect_tx(bar, n * (D + D / 4));
  else asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(n * (D + D / 4)) : "memory");
  bulk_load(ring.k + slot * (kI4Tile * D / 8), a.k + at * (D / 2), n * (D / 2), bar);
  bulk_load(ring.k_meta + slot * (kI4Tile * D / 32), a.k_meta + at * (D / 32), n * (D / 8), bar);
  bulk_load(ring.v + slot * (kI4Tile * D / 8), a.v + at * (D / 2), n * (D / 2), bar);
  bulk_load(ring.v_meta + slot * (kI4Tile * D / 32), a.v_meta + at * (D / 32), n * (D / 8), bar);
}
__device__ __forceinline__ uint32_t ld_shared1(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kI4Warps * 32) : "memory"); }

__device__ __forceinline__ float4 ld_cluster(const float4* local, uint32_t rank) {
  float4 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(local)), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster(const float2* local, uint32_t rank) {
  float2 v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
               : "=f"(v.x), "=f"(v.y) : "r"(smem_u32(local)), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Zeros for a slice without slots; one whose slots all weigh nothing is 0 / 0.
__device__ __forceinline__ void i4_store(bf16* out, const float4& o, float sum, bool empty) {
  const float inv = empty ? 0.f : __fdividef(1.f, sum);
  uint2 y;
  y.x = pack_bf16x2(o.x * inv, o.y * inv);
  y.y = pack_bf16x2(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(out) = y;
}

// A pair of probabilities without those bits of their bf16 roundings that `low` and `high` select (byte_perm): 0x1044 and 0x3244 all, 0x4444 none.
__device__ __forceinline__ uint32_t i4_rest(float x, float y, uint32_t low, uint32_t high) {
  const uint32_t r = pack_bf16x2(x, y);
  return pack_bf16x2(x - __uint_as_float(__byte_perm(r, 0, low)), y - __uint_as_float(__byte_perm(r, 0, high)));
}

// NT: query heads of an item in eights (1 or 2).  kTwin: four heads at most, columns 4 to 7 are 0 to 3 again.  kCluster: an item is shared by the kI4Cluster CTAs of a cluster, which merge through its shared memory.
template <int D, int NT, bool kTwin, bool kCluster>
__global__ void __launch_bounds__(kI4Threads, i4_ctas<NT>()) int4_attn_kernel(const Int4Attn a, int* status) {
  static_assert(!kTwin || NT == 1, "half of eight columns");
  constexpr int WK = D / 32;       // words of a key that a lane multiplies with the queries
  constexpr int WV = D / 64;       // words of a value row of which a lane holds the dimensions
  extern __shared__ __align__(128) uint8_t raw[];
  const int slots = a.groups * kI4Warps;
  const Int4Ring<D> ring(raw, slots);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring.v_meta + slots * (kI4Tile * D / 32));
  uint64_t* empty = full + a.groups;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + a.groups);
  float* s_m = reinterpret_cast<float*>(empty + a.groups + 2);                // [warps][heads]
  float* s_l = s_m + kI4Warps * a.heads;
  float* s_o = s_l + kI4Warps * a.heads;                                    // [warps][heads][D]
  float2* s_ml = reinterpret_cast<float2*>(s_o + kI4Warps * a.heads * D);   // [heads], kCluster: the CTA's

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const WaitGuard guard{abort_flag, status};
  grid_dependency_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.groups; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], kI4Warps); }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  grid_dependency_wait();

  const int per_row = a.Hkv * a.blocks, cta = blockIdx.x;
  Int4Cursor piece;                // the item that the warp is at, by its first tile of this CTA's run
  int t0, run;                     // the run: its first tile, its tiles
  Int4Share share(a, 0);
  if (kCluster) {
    const int item = cta / kI4Cluster, rank = cta % kI4Cluster;
    piece.row = item / per_row;
    piece.head = item - piece.row * per_row;
    piece.load(a);
    piece.enter(a);
    t0 = piece.tile = (int)((long long)piece.n * rank / kI4Cluster);
    run = (int)((long long)piece.n * (rank + 1) / kI4Cluster) - t0;
  } else {
    int row_tiles, row_sum;
    const int total = Int4Cursor::count(a, row_tiles, row_sum, lane);
    share = Int4Share(a, total);
    if (warp == 0) {               // rows without tiles
      for (int row = cta; row < a.rows; row += gridDim.x)
        if (i4_row_tiles(a, row) == 0)
          for (int i = lane; i < a.Hq * (D / 8); i += 32)
            reinterpret_cast<uint4*>(a.out)[(long long)row * a.Hq * (D / 8) + i] = make_uint4(0, 0, 0, 0);
    }
    if (cta >= share.ctas || total == 0) {
      if (threadIdx.x == 0) a.shared[cta] = make_int2(0, 0);
      return;
    }
    t0 = share.first(cta);
    run = share.first(cta + 1) - t0;
    piece.seek(a, t0, row_tiles, row_sum, lane);
  }

  if (warp == kI4Warps) {
    // ---------------------------------------------------------------- the warp that fetches
    int done = 0, slot = 0, group = 0;
    uint32_t phase = 1;            // a fresh barrier counts as one whose tiles have been given back
    while (done < run) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[group], phase, guard, kTimeoutStageEmpty))) break;
      const int end = min(run, done + kI4Warps);
      while (done < end) {
        const int tiles = min(end - done, piece.n - piece.tile);
        if (elect_one()) i4_fetch<D>(a, piece, tiles, ring, slot, &full[group], done + tiles == end);
        done += tiles;
        slot += tiles;
        piece.advance(a, tiles);
      }
      if (++group == a.groups) { group = slot = 0; phase ^= 1; }
    }
    // whatever the others have given up on: the last copies land before the block leaves
    const long long began = clock64();
    const int groups = (done + kI4Warps - 1) / kI4Warps;
    for (int i = max(0, groups - a.groups); i < groups; ++i)
      while (!mbar_try_wait(&full[i % a.groups], (i / a.groups) & 1) && clock64() - began < kWaitLimitCycles) {}
    if (kCluster) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // ------------------------------------------------------------------ the warps that compute
  const uint32_t k_at = smem_u32(ring.k), v_at = smem_u32(ring.v), k_meta_at = smem_u32(ring.k_meta), v_meta_at = smem_u32(ring.v_meta);
  bool ok = true;
  // A warp has a tile in every group and so waits for each: barriers know two phases, and copies of later groups may land first.
  int mine = warp, group = 0;      // this warp's tile, its group in the ring
  uint32_t phase = 0;
  int before = 0;                  // tiles of the run ahead of the item
  const uint32_t low = t < 2 ? 0x4444 : 0x1044, high = t < 2 ? 0x4444 : 0x3244;            // kTwin: columns 0 to 3 take the rounding, the others the rest
  do {
    const int here = min(run - before, piece.n - piece.tile);      // tiles of the item in the run
    const int kvh = piece.head / a.blocks, h0 = kvh * (a.Hq / a.Hkv) + piece.head % a.blocks * a.heads;
    const int heads = min(a.heads, (kvh + 1) * (a.Hq / a.Hkv) - h0);
    const int b = piece.row / a.Tq, tq = piece.row % a.Tq;
    // queries: column g of each block of eight, in the order in which a lane holds a key's values
    uint4 qv[NT][WK];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        qv[n][w] = make_uint4(0, 0, 0, 0);
        const int qe = kTwin ? g & 3 : n * 8 + g;
        if (qe < heads) qv[n][w] = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + tq * a.q_st + (h0 + qe) * a.q_sh + t * (D / 4) + w * 8);
        qv[n][w].x ^= a.negate; qv[n][w].y ^= a.negate; qv[n][w].z ^= a.negate; qv[n][w].w ^= a.negate;
      }
    float o[WV * 4][NT][4], m[NT][2], l[NT][2];      // of queries 2 t and 2 t + 1 of each block
#pragma unroll
    for (int i = 0; i < WV * 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[n][e] = kI4Least; l[n][e] = 0.f; }

    while (mine < before + here) {
      const int slot = group * kI4Warps + warp;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[group], phase, guard, kTimeoutTmaFull));
      if (!ok) break;
      const int first = (piece.lo & ~(kI4Align - 1)) + (piece.tile + mine - before) * kI4Tile;
      const uint32_t sk = k_at + slot * (kI4Tile * D / 2), sv = v_at + slot * (kI4Tile * D / 2);
      const uint32_t skm = k_meta_at + slot * (kI4Tile * D / 8), svm = v_meta_at + slot * (kI4Tile * D / 8);
#pragma unroll
      for (int u = 0; u < kI4Tile / 16; ++u) {
        const int key0 = first + u * 16;                         // the block's first slot
        if (key0 >= piece.hi || key0 + 16 <= piece.lo) continue;
        const bool whole = key0 >= piece.lo && key0 + 16 <= piece.hi;
        // ---- scores^T = K q^T: row g + 8 j is slot 8 j + 4 (g & 1) + (g / 2 ^ g & 1) of the block, for fewer conflicts of V's loads
        const int slot0 = u * 16 + (g & 1) * 4 + ((g >> 1) ^ (g & 1));
        float c[NT][4];                                          // [n][2 j + e]: key j of this lane, query 2 t + e
        {
          uint32_t words[2][WK], s2[2], o2[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int key = slot0 + j * 8;
            const uint32_t meta = ld_shared1(skm + (key * (D / 32) + t * WK / 4) * 4);
            s2[j] = i4_scale2(meta);
            o2[j] = i4_offset2(meta);
            const uint32_t at = sk + (key * (D / 8) + t * WK) * 4;
            if constexpr (D == 128) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(words[j][0]), "=r"(words[j][1]), "=r"(words[j][2 % WK]), "=r"(words[j][3 % WK]) : "r"(at) : "memory");
            else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(words[j][0]), "=r"(words[j][1]) : "r"(at) : "memory");
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[n][e] = 0.f;
#pragma unroll
          for (int w = 0; w < WK; ++w) {
            uint32_t x[4], y[4];
            i4_values(x, words[0][w], s2[0], o2[0]);
            i4_values(y, words[1][w], s2[1], o2[1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16(c[n], x[0], y[0], x[1], y[1], qv[n][w].x, qv[n][w].y);
              mma_bf16(c[n], x[2], y[2], x[3], y[3], qv[n][w].z, qv[n][w].w);
            }
          }
        }
        if (__builtin_expect(!whole, 0)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int key = first + slot0 + j * 8;
            if (key < piece.lo || key >= piece.hi) {
#pragma unroll
              for (int n = 0; n < NT; ++n) c[n][2 * j] = c[n][2 * j + 1] = -INFINITY;
            }
          }
        }
        // ---- probabilities relative to m, which moves seldom (always in a warp's first block), so that most blocks need no maximum over their rows
        // and no correction of the outputs
        float x[NT][4], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] = fmaf(c[n][e], a.scale, -m[n][e & 1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) top = max3(max3(top, x[n][0], x[n][1]), x[n][2], x[n][3]);
        if (__builtin_expect(__any_sync(0xffffffffu, top > kI4Late - kI4Above), 0)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(c[n][e], c[n][2 + e]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              mx = fmaxf(fmaf(mx, a.scale, kI4Above), m[n][e]);
              const float corr = fast_exp2(m[n][e] - mx);
              m[n][e] = mx;
              l[n][e] *= corr;
#pragma unroll
              for (int i = 0; i < WV * 4; ++i) { o[i][n][e] *= corr; o[i][n][2 + e] *= corr; }
              x[n][e] = fmaf(c[n][e], a.scale, -mx);
              x[n][2 + e] = fmaf(c[n][2 + e], a.scale, -mx);
            }
        }
        uint32_t pb[NT][2], rest[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] = fast_exp2(x[n][e]);
          l[n][0] += x[n][0] + x[n][2];
          l[n][1] += x[n][1] + x[n][3];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            pb[n][j] = transpose8(kTwin ? i4_rest(x[n][2 * j], x[n][2 * j + 1], low, high) : pack_bf16x2(x[n][2 * j], x[n][2 * j + 1]));
            if (!kTwin) rest[n][j] = transpose8(i4_rest(x[n][2 * j], x[n][2 * j + 1], 0x1044, 0x3244));
          }
        }
        // ---- out^T += V^T P^T: this lane's dimensions are D / 8 * g and on
        uint32_t rows[4][WV], meta[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = u * 16 + i * 4 + (t ^ (i & 1));
          const uint32_t at = sv + (key * (D / 8) + g * WV) * 4;
          if constexpr (D == 128) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(rows[i][0]), "=r"(rows[i][WV - 1]) : "r"(at) : "memory");
          else rows[i][0] = ld_shared1(at);
          meta[i] = ld_shared1(svm + (key * (D / 32) + g * WV / 4) * 4);
        }
        if (__builtin_expect(!whole, 0)) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + i * 4 + (t ^ (i & 1));
            if (key < piece.lo || key >= piece.hi) meta[i] = 0;
          }
        }
        uint32_t s2[2], o2[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s2[j] = __byte_perm(meta[2 * j], meta[2 * j + 1], 0x5410);
          o2[j] = __byte_perm(meta[2 * j], meta[2 * j + 1], 0x7632);
        }
#pragma unroll
        for (int w = 0; w < WV; ++w) {
          uint32_t even[2][4], odd[2][4];      // [pair of keys][value of the word / 2]
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            i4_values(even[j], __byte_perm(rows[2 * j][w], rows[2 * j + 1][w], 0x5410), s2[j], o2[j]);
            i4_values(odd[j], __byte_perm(rows[2 * j][w], rows[2 * j + 1][w], 0x7632), s2[j], o2[j]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16(o[w * 4 + i][n], even[0][i], odd[0][i], even[1][i], odd[1][i], pb[n][0], pb[n][1]);
              if (!kTwin) mma_bf16(o[w * 4 + i][n], even[0][i], odd[0][i], even[1][i], odd[1][i], rest[n][0], rest[n][1]);
            }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[group]);
      mine += kI4Warps;
      if (++group == a.groups) { group = 0; phase ^= 1; }
    }

    if (kTwin) {
#pragma unroll
      for (int i = 0; i < WV * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][0][e] += __shfl_xor_sync(0xffffffffu, o[i][0][e], 2);
    }

    // ---- the warps' parts of the item -> one
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int qe = n * 8 + t * 2 + e;
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (qe < heads) {
          if (g == 0) { s_m[warp * a.heads + qe] = m[n][e]; s_l[warp * a.heads + qe] = sum; }
          float* dst = s_o + (warp * a.heads + qe) * D + g * (D / 8);
#pragma unroll
          for (int i = 0; i < WV * 4; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[i][n][e], o[i][n][2 + e]);
        }
      }
    }
    compute_sync();
    const bool alone = !kCluster && here == piece.n;                 // the whole item is here
    const long long part = cta + (long long)piece.row * per_row + piece.head;
    bf16* out = a.out + ((long long)piece.row * a.Hq + h0) * D;
    for (int i = threadIdx.x; i < heads * (D / 4); i += kI4Warps * 32) {
      const int q = i / (D / 4), d = i % (D / 4) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kI4Warps; ++w) mx = fmaxf(mx, s_m[w * a.heads + q]);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kI4Warps; ++w) {
        const float mw = s_m[w * a.heads + q], f = mw == mx ? 1.f : fast_exp2(mw - mx);
        const float4 x = *reinterpret_cast<const float4*>(s_o + (w * a.heads + q) * D + d);
        sum = fmaf(s_l[w * a.heads + q], f, sum);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
      }
      if (kCluster) {              // in the place of the first warp's
        *reinterpret_cast<float4*>(s_o + q * D + d) = acc;
        if (d == 0) s_ml[q] = make_float2(mx, sum);
      } else if (alone) {
        i4_store(out + q * D + d, acc, sum, false);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (part * a.heads + q) * D + d) = acc;
        if (d == 0) a.part_ml[part * a.heads + q] = make_float2(mx, sum);
      }
    }
    if (kCluster) {
      cluster_sync();
      // every CTA finishes its share of the outputs
      const int n = heads * (D / 4), share_n = (n + kI4Cluster - 1) / kI4Cluster, rank = cta % kI4Cluster;
      for (int i = rank * share_n + (int)threadIdx.x; i < min((rank + 1) * share_n, n); i += kI4Warps * 32) {
        const int q = i / (D / 4), d = i % (D / 4) * 4;
        float2 ml[kI4Cluster];
        float4 x[kI4Cluster];
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int r = 0; r < kI4Cluster; ++r) {
          ml[r] = ld_cluster(s_ml + q, r);
          x[r] = ld_cluster(reinterpret_cast<const float4*>(s_o + q * D + d), r);
        }
#pragma unroll
        for (int r = 0; r < kI4Cluster; ++r) mx = fmaxf(mx, ml[r].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < kI4Cluster; ++r) {
          const float f = ml[r].x == mx ? 1.f : fast_exp2(ml[r].x - mx);
          sum = fmaf(ml[r].y, f, sum);
          acc.x = fmaf(x[r].x, f, acc.x); acc.y = fmaf(x[r].y, f, acc.y); acc.z = fmaf(x[r].z, f, acc.z); acc.w = fmaf(x[r].w, f, acc.w);
        }
        i4_store(out + q * D + d, acc, sum, piece.n == 0);
      }
      cluster_sync();              // nobody leaves while its part may still be read
      return;
    }
    compute_sync();
    before += here;
    if (before == run && threadIdx.x == 0) {
      const bool goes_on = piece.tile == 0 && here < piece.n;
      a.shared[cta] = make_int2((int)(part - cta), goes_on ? share.owner(t0 + run - here + piece.n - 1) - cta + 1 : 0);
    }
    piece.advance(a, here);
  } while (before < run);
}

// One query head of an item that begins in a CTA's run and goes on behind it.  The warps take its parts in turn, a lane D / 32 dimensions.
constexpr int kI4MergeWarps = 8;
template <int D>
__global__ void __launch_bounds__(kI4MergeWarps * 32) int4_attn_merge_kernel(const Int4Attn a) {
  constexpr int V = D / 32;
  __shared__ float s_o[kI4MergeWarps][D], s_m[kI4MergeWarps], s_l[kI4MergeWarps];
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = blockIdx.y;
  const int2 what = a.shared[blockIdx.x];
  const int item = what.x, parts = what.y, per_row = a.Hkv * a.blocks;
  if (parts == 0) return;
  const int row = item / per_row, head = item % per_row;
  const int group = a.Hq / a.Hkv, kvh = head / a.blocks, h0 = kvh * group + head % a.blocks * a.heads;
  if (h0 + q >= (kvh + 1) * group) return;
  bf16* out = a.out + ((long long)row * a.Hq + h0 + q) * D;
  const long long part0 = ((long long)blockIdx.x + item) * a.heads + q;          // in rows of part_o
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  constexpr int kAtOnce = 4;
  for (int s = warp; s < parts; s += kI4MergeWarps * kAtOnce) {
    float2 ml[kAtOnce];
    float v[kAtOnce][V];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int at = s + i * kI4MergeWarps;
      ml[i] = make_float2(-INFINITY, 0.f);
      if (at < parts) {
        const long long r = part0 + (long long)at * a.heads;
        ml[i] = a.part_ml[r];
        if (V == 4) *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(a.part_o + r * D + lane * V);
        else *reinterpret_cast<float2*>(v[i]) = *reinterpret_cast<const float2*>(a.part_o + r * D + lane * V);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (s + i * kI4MergeWarps >= parts) break;
      const float mx = fmaxf(m, ml[i].x), f0 = m == mx ? 1.f : fast_exp2(m - mx), f1 = ml[i].x == mx ? 1.f : fast_exp2(ml[i].x - mx);
      m = mx;
      l = l * f0 + ml[i].y * f1;
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = o[k] * f0 + v[i][k] * f1;
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) s_o[warp][lane * V + k] = o[k];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  if (threadIdx.x < D) {
    float mx = s_m[0], sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 1; w < kI4MergeWarps; ++w) mx = fmaxf(mx, s_m[w]);
#pragma unroll
    for (int w = 0; w < kI4MergeWarps; ++w) {
      const float f = s_m[w] == mx ? 1.f : fast_exp2(s_m[w] - mx);
      sum = fmaf(s_l[w], f, sum);
      acc = fmaf(s_o[w][threadIdx.x], f, acc);
    }
    out[threadIdx.x] = __float2bfloat16(__fdividef(acc, sum));
  }
}

constexpr int kI4SmShared = 228 * 1024;      // of which every block costs 1024 besides its own
constexpr int kI4MostGroups = 6;
struct Int4Shape {
  int heads, blocks, groups, cluster;
  long long items, tiles;          // tiles: at most
  int ctas;
  size_t smem;
};
static Int4Shape i4_shape(int rows, int Hq, int Hkv, int D, int cap) {
  Int4Shape s;
  const int group = Hq / Hkv;
  s.heads = group < 16 ? group : 16;
  s.blocks = (group + 15) / 16;
  s.items = (long long)rows * Hkv * s.blocks;
  const int per_group = kI4Warps * kI4Tile * (D + D / 4) + 16;
  const int rest = 16 + (kI4Warps * (D + 2) + 2) * s.heads * (int)sizeof(float);
  const int per_sm = s.heads <= 8 ? i4_ctas<1>() : i4_ctas<2>();
  s.groups = (kI4SmShared / per_sm - 1024 - rest) / per_group;
  if (s.groups > kI4MostGroups) s.groups = kI4MostGroups;
  s.smem = (size_t)s.groups * per_group + rest;
  s.tiles = s.items * (((long long)cap + kI4Align + kI4Tile - 1) / kI4Tile);
  const long long most = (s.tiles + kI4Spread - 1) / kI4Spread, room = (long long)sm_count() * per_sm;
  s.ctas = (int)(most < 1 ? 1 : most < room ? most : room);
  const long long rounds = (s.items * kI4Cluster + room - 1) / room;
  s.cluster = rounds <= 2 && cap <= (s.heads > 8 && s.items > 4 ? 2 * kI4ClusterSlots : kI4ClusterSlots) / rounds;
  return s;
}

template <int D, int NT, bool kTwin>
static int launch_int4_attn(const Int4Attn& a, const Int4Shape& s, cudaStream_t st) {
  constexpr int most = kI4SmShared / i4_ctas<NT>() - 1024;
  int* status = status_word();
  KSA_REQUIRE(status != nullptr, "int4_decode_attn: no status word");
  if (s.cluster) {
    static PerDevice raised;
    KSA_CHECK_CUDA(raise_smem_limit(raised, int4_attn_kernel<D, NT, kTwin, true>, most));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s.items * kI4Cluster));
    cfg.blockDim = dim3(kI4Threads);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kI4Cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = dependent_launches() ? 2 : 1;
    KSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, int4_attn_kernel<D, NT, kTwin, true>, a, status));
    return 0;
  }
  static PerDevice raised;
  KSA_CHECK_CUDA(raise_smem_limit(raised, int4_attn_kernel<D, NT, kTwin, false>, most));
  KSA_CHECK_CUDA(launch_kernel(int4_attn_kernel<D, NT, kTwin, false>, dim3(a.ctas), dim3(kI4Threads), s.smem, st, a, status));
  KSA_CHECK_CUDA(launch_kernel(int4_attn_merge_kernel<D>, dim3(a.ctas, a.heads), dim3(kI4MergeWarps * 32), 0, st, a));
  return 0;
}

}  // namespace ksa

using namespace ksa;

// Floats of the workspace of ksa_int4_decode_attn on the current device: none where clusters merge.
KSA_API long long ksa_int4_attn_workspace(int B, int Tq, int Hq, int Hkv, int D, int cap) {
  if (B <= 0 || Tq <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv != 0 || cap <= 0 || (long long)B * Tq >= (1 << 28)) return 0;
  const Int4Shape s = i4_shape(B * Tq, Hq, Hkv, D, cap);
  return s.cluster ? 0 : (s.ctas + s.items) * s.heads * (D + 2LL) + 2LL * s.ctas;
}

// q [B, Tq, Hq, D] with strides in elements (rows of a head contiguous); cache as written by ksa_int4_cache_write; start, len [B, Tq] int32;
// out [B, Tq, Hq, D].  A slice without slots gives zeros.
KSA_API int ksa_int4_decode_attn(const void* q, const void* k, const void* k_meta, const void* v, const void* v_meta, const void* start,
                                 const void* len, void* workspace, void* out, int B, int Tq, int Hq, int Hkv, int D, int cap, long long q_sb,
                                 long long q_st, long long q_sh, float scale, void* stream) {
  KSA_ENTER(q);
  KSA_REQUIRE(D == 128 || D == 64, "int4_decode_attn: head_dim %d unsupported (64 or 128)", D);
  KSA_REQUIRE(Hkv > 0 && Hq >= Hkv && Hq % Hkv == 0, "int4_decode_attn: %d query heads over %d key heads", Hq, Hkv);
  KSA_REQUIRE(cap > 0 && cap % kI4Align == 0, "int4_decode_attn: capacity %d is no multiple of %d", cap, kI4Align);
  KSA_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_meta) |
                reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(v_meta)) & 15) == 0 && q_sb % 8 == 0 && q_st % 8 == 0 && q_sh % 8 == 0,
              "int4_decode_attn: queries and cache must be 16-byte aligned");
  KSA_REQUIRE(B >= 0 && Tq >= 0 && (long long)B * Tq < (1 << 28), "int4_decode_attn: bad shape");
  KSA_REQUIRE(fabsf(scale) < INFINITY, "int4_decode_attn: the scale is not finite");
  if (B == 0 || Tq == 0) return 0;
  const Int4Shape s = i4_shape(B * Tq, Hq, Hkv, D, cap);
  KSA_REQUIRE(s.tiles < (1LL << 31) - s.ctas, "int4_decode_attn: too many queries and slots");
  KSA_REQUIRE(s.cluster || workspace != nullptr, "int4_decode_attn: no workspace");
  const long long parts = s.ctas + s.items;
  float* ws = (float*)workspace;
  Int4Attn a{(const bf16*)q, q_sb, q_st, q_sh, (const uint8_t*)k, (const uint8_t*)v, (const uint32_t*)k_meta, (const uint32_t*)v_meta,
             (const int*)start, (const int*)len, ws, (float2*)(ws + parts * s.heads * D),
             (int2*)(ws + parts * s.heads * (D + 2LL)), (bf16*)out, B * Tq, Tq, Hq, Hkv, cap, s.heads, s.blocks,
             s.ctas, s.groups, fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (D == 128)
    return s.heads <= 4 ? launch_int4_attn<128, 1, true>(a, s, st) : s.heads <= 8 ? launch_int4_attn<128, 1, false>(a, s, st) : launch_int4_attn<128, 2, false>(a, s, st);
  return s.heads <= 4 ? launch_int4_attn<64, 1, true>(a, s, st) : s.heads <= 8 ? launch_int4_attn<64, 1, false>(a, s, st) : launch_int4_attn<64, 2, false>(a, s, st);
}
