// Products of up to 32 rows with weights of four bits through tensor memory: C[M, N] = A[M, K] * W[N, K]^T, W as int4.cuh says.
//
// Reading the codes bounds it where there are many rows of the weight, unpacking them next to that, as in int4_linear.cu.  There mma.sync costs the same
// issue slots as the unpacking and twice as many from nine rows on, and every eight activation rows want registers.  Here:
//   * a lane unpacks a row of the weight, 128 columns at a time, into tensor memory, where tcgen05.mma takes it as the operand of 128 rows; the
//     activations, a TMA copy with its swizzle, are the other one, 16 or 32 of them at much the same price;
//   * three groups of four warps unpack the ring's stages in turn, each with its own slot, its own sums and a warp that issues its products.  What
//     decides is how few instructions and barriers there are to a stage: [151936, 2560] x 16 rows with all warps at one stage 79 us, with groups but
//     one issuer 72, with half a stage and two slots to a group 60, four groups with one 60, this 54 (the fetch alone 33, without the stores 40);
//   * four more warps add up the groups' sums of a pass, in their order, and write them while the next pass is being unpacked;
//   * activations that several passes want and that fit stay in shared memory, others come with each stage;
//   * few rows of the weight: the CTAs of a cluster share K, and each adds up some of the activation rows from the others' shared memory.
// Measured on 32 rows: [151936, 2560] 78 us (2.8 TB/s), [19456, 2560] 20, [6144, 2560] 11.8, [2560, 9728] 13.3 on clusters of four.
#include "int4_linear.h"

#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4WGroups = 3;                       // four warps each that unpack: a group takes every third stage
constexpr int kI4WUnpackers = 4 * kI4WGroups;
constexpr int kI4WWriters = kI4WUnpackers;          // first of the four that write results
constexpr int kI4WFetch = kI4WWriters + 4;
constexpr int kI4WIssuers = kI4WFetch + 1;          // first of those that multiply, one to a group
constexpr int kI4WThreads = (kI4WIssuers + kI4WGroups) * 32;
constexpr int kI4WStep = 256;                       // columns of a stage
constexpr int kI4WSums = kI4WGroups * 128;          // each group unpacks a stage into 128 columns; behind them its sums: two sets of 16 columns, or one of 32
constexpr int kI4WMostStages = 15;                  // a multiple of three: a stage of the ring belongs to the same groups all the time
constexpr int kI4WSmemMost = 227 * 1024;
// Activations that stay, up to so many bytes, where several passes want them: 32 rows of [40000, 2048] (128 KB) 25.0 -> 24.2 us, but of [151936, 2560]
// (160 KB, three stages left) 80 -> 85.
constexpr int kI4WKeepMost = 128 * 1024;

struct Int4Wide {
  bf16* C;
  long long ldc;
  int M, N, K, group;
  int cols;                        // activation rows in sixteens
  int parts;                       // CTAs of a cluster, which share K
  int per_cluster, per_pass;       // weight rows
  int steps;                       // of K
  int stages, stage_bytes, b_at, meta_at, meta_words;
  int keep;                        // bytes of activations that stay, 0: they come with each stage
  int early;
};

__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_address(const void* local, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
  return at;
}
__device__ __forceinline__ float ld_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive(uint64_t* bar, int rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_address(bar, rank)) : "memory");
}
// mbar_wait for arrivals of the cluster's other CTAs.
__device__ __forceinline__ bool cluster_bar_wait(uint64_t* bar, uint32_t parity, const WaitGuard& g, int code) {
  const long long began = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (done) return true;
    if (*g.abort_flag) return false;
    if (clock64() - began > kWaitLimitCycles) {
      *g.abort_flag = 1;
      atomicCAS(g.status, 0, code);
      return false;
    }
  }
}

__global__ void __launch_bounds__(kI4WThreads, 1)
int4_linear_wide_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_meta, const __grid_constant__ CUtensorMap tm_x,
                        const Int4Wide a, int* status) {
  extern __shared__ uint8_t unaligned[];
  uint8_t* ring = unaligned + (1024 - (smem_u32(unaligned) & 1023)) % 1024;
  uint8_t* kept = ring + a.stages * a.stage_bytes;                                     // [step][64-column panel][cols][128 bytes]
  float* part = reinterpret_cast<float*>(kept + a.keep);                               // [cols][128], where CTAs share K
  uint64_t* full = reinterpret_cast<uint64_t*>(part + (a.parts > 1 ? a.cols * 128 : 0));
  uint64_t* empty = full + kI4WMostStages;
  uint64_t* slot_full = empty + kI4WMostStages;
  uint64_t* slot_empty = slot_full + kI4WGroups;
  uint64_t* sums_full = slot_empty + kI4WGroups;                            // [group][set]
  uint64_t* sums_empty = sums_full + kI4WGroups * 2;
  uint64_t* x_full = sums_empty + kI4WGroups * 2;
  uint64_t* ended = x_full + 1;
  uint64_t* ready = ended + 1;                                                          // every CTA's part of a pass is there
  uint64_t* freed = ready + 1;                                                          // and has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(freed + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitGuard guard{abort_flag, status};
  const int rank = blockIdx.x % a.parts, r0 = (int)(blockIdx.x / a.parts) * a.per_cluster, mine = min(a.per_cluster, a.N - r0);
  const int passes = (mine + a.per_pass - 1) / a.per_pass;
  const int step0 = rank * a.steps / a.parts, count = (rank + 1) * a.steps / a.parts - step0, total = passes * count;
  const int groups = kI4WStep / a.group, panel = a.cols * 128, sets = a.cols == 16 ? 2 : 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], a.keep ? 4 : 1); }
    for (int i = 0; i < kI4WGroups; ++i) { mbar_init(&slot_full[i], 4); mbar_init(&slot_empty[i], 1); }
    for (int i = 0; i < kI4WGroups * 2; ++i) { mbar_init(&sums_full[i], 1); mbar_init(&sums_empty[i], 4); }
    mbar_init(x_full, 1);
    mbar_init(ended, kI4WGroups);
    mbar_init(ready, a.parts);
    mbar_init(freed, a.parts);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm);
    tma_prefetch_desc(&tm_meta);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == kI4WFetch) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (a.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");        // the barriers stand; waited for below
  grid_dependency_launch();

  if (warp == kI4WFetch) {
    // ---------------------------------------------------------------- the warp that fetches
    const uint32_t bytes = a.per_pass * 128 + groups * a.meta_words * 4 + (a.keep ? 0 : 4 * panel);      // also past the matrix's edges
    const auto weights = [&](int i) {
      const int step = step0 + i % count, row = r0 + i / count * a.per_pass;
      uint8_t* dst = ring + i % a.stages * a.stage_bytes;
      uint64_t* bar = &full[i % a.stages];
      mbar_expect_tx(bar, bytes);
      tma_load_2d(dst, &tm, step * 64, row, bar);
      tma_load_2d(dst + a.meta_at, &tm_meta, row & ~3, step * groups, bar);
    };
    const auto activations = [&](int i) {
      const int step = step0 + i % count;
      uint8_t* dst = ring + i % a.stages * a.stage_bytes + a.b_at;
      for (int j = 0; j < 4; ++j) tma_load_2d(dst + j * panel, &tm_x, step * kI4WStep + j * 64, 0, &full[i % a.stages]);
    };
    const int ahead = min(total, a.stages);
    if (!a.early) grid_dependency_wait();
    if (elect_one())
      for (int i = 0; i < ahead; ++i) weights(i);
    __syncwarp();
    if (a.early) grid_dependency_wait();
    if (elect_one()) {
      if (a.keep) {
        mbar_expect_tx(x_full, count * 4 * panel);
        for (int i = 0; i < count * 4; ++i) tma_load_2d(kept + i * panel, &tm_x, step0 * kI4WStep + i * 64, 0, x_full);
      } else {
        for (int i = 0; i < ahead; ++i) activations(i);
      }
    }
    __syncwarp();
    int done = ahead;
    for (; done < total; ++done) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[done % a.stages], done / a.stages - 1 & 1, guard, kTimeoutStageEmpty))) break;
      if (elect_one()) {
        weights(done);
        if (!a.keep) activations(done);
      }
      __syncwarp();
    }
    // whatever the others have given up on: the last copies land before the block leaves
    const long long began = clock64();
    for (int i = max(0, done - a.stages); i < done; ++i)
      while (!mbar_try_wait(&full[i % a.stages], (i / a.stages) & 1) && clock64() - began < kWaitLimitCycles) {}
    if (a.keep && total > 0)
      while (!mbar_try_wait(x_full, 0) && clock64() - began < kWaitLimitCycles) {}
  } else if (warp >= kI4WIssuers) {
    // ---------------------------------------------------------------- the warps that multiply: 128 weight rows x activation rows, 16 columns at a time
    const int group = warp - kI4WIssuers;
    const uint32_t idesc = umma_idesc_bf16(128, a.cols, 0, 0), panel16 = panel >> 4, stage16 = a.stage_bytes >> 4;
    const uint64_t x_desc = smem_desc_kmajor_sw128(smem_u32(a.keep ? kept : ring + a.b_at));
    uint64_t *my_full = slot_full + group, *my_empty = slot_empty + group;
    int stage = group, k = stage, set = 0;             // step `k` of a pass
    uint32_t phase = 0, slot_phase = 0, accumulate = 0, sums_phase = 1;
    bool ok = !a.keep || __all_sync(0xffffffffu, mbar_wait(x_full, 0, guard, kTimeoutTmaFull));
    int left = total - stage;
    for (; k >= count; k -= count) {}
    while (ok && left > 0) {
      const bool last = k + kI4WGroups >= count;                     // of this group in the pass
      const uint64_t desc = x_desc + (a.keep ? k * 4 * panel16 : stage * stage16);
      const uint32_t sums = tmem + kI4WSums + (group * sets + set) * a.cols, from = tmem + group * 128;
      if (accumulate == 0) ok = __all_sync(0xffffffffu, mbar_wait(&sums_empty[group * 2 + set], sums_phase, guard, kTimeoutAccEmpty));
      if (!a.keep) ok = ok && __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, guard, kTimeoutTmaFull));
      ok = ok && __all_sync(0xffffffffu, mbar_wait(my_full, slot_phase, guard, kTimeoutSoftmax));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int e = 0; e < 16; ++e) umma_ts(sums, from + e * 8, desc + (e >> 2) * panel16 + (e & 3) * 2, idesc, e == 0 ? accumulate : 1);
        umma_commit(my_empty);
        if (!a.keep) umma_commit(&empty[stage]);
        if (last) umma_commit(&sums_full[group * 2 + set]);
      }
      __syncwarp();
      accumulate = !last;
      if (last && ++set == sets) { set = 0; sums_phase ^= 1; }
      slot_phase ^= 1;
      left -= kI4WGroups;
      for (k += kI4WGroups; k >= count; k -= count) {}
      if ((stage += kI4WGroups) >= a.stages) { stage -= a.stages; phase ^= 1; }
    }
    if (elect_one()) umma_commit(ended);
    __syncwarp();
  } else if (warp < kI4WUnpackers) {
    // ---------------------------------------------------------------- the warps that unpack, a weight row to a lane
    const int quarter = warp & 3, group = warp >> 2;
    const int row = min(quarter * 32 + lane, a.per_pass - 1);        // lanes past the pass's rows make sums that nobody reads
    const uint32_t out = tmem + group * 128 + ((uint32_t)(quarter * 32) << 16), ring_at = smem_u32(ring);
    uint32_t chunk_at[2], meta_at[2];                                // of 64 columns; the next ones lie 32 bytes and some groups on
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      chunk_at[c] = row * 128 + (c ^ (row & 7)) * 16;
      meta_at[c] = a.meta_at + (c * 32 / a.group * a.meta_words + row) * 4;
    }
    const uint32_t meta_half = 128 / a.group * a.meta_words * 4, meta_quarter = 64 / a.group * a.meta_words * 4;
    uint32_t at = ring_at + group * a.stage_bytes, skip = r0 & 3;
    int stage = group, k = stage, left = total - k;
    uint32_t phase = 0, slot_phase = 1;
    bool ok = true;
    while (left > 0) {
      for (; k >= count; k -= count) skip = (skip + a.per_pass) & 3;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, guard, kTimeoutTmaFull));
      if (!ok) break;
#pragma unroll
      for (uint32_t half = 0; half < 2; ++half) {
        uint4 words[4];
        uint32_t m[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          words[c] = ld_shared(at + (chunk_at[c & 1] ^ (half * 64 + (c >> 1) * 32)));
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(m[c]) : "r"(at + meta_at[c & 1] + half * meta_half + (c >> 1) * meta_quarter + skip * 4) : "memory");
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          uint32_t v[32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t s2 = i4_scale2(m[s * 2 + h]), o2 = i4_offset2(m[s * 2 + h]);
            const uint32_t four[4] = {words[s * 2 + h].x, words[s * 2 + h].y, words[s * 2 + h].z, words[s * 2 + h].w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
              i4_values(w, four[q], s2, o2);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[h * 16 + q * 4 + e] = w[e];
            }
          }
          if (half == 0 && s == 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(slot_empty + group, slot_phase, guard, kTimeoutAccEmpty));
            tc_fence_after();
          }
          if (ok) tmem_st32(out + half * 64 + s * 32, v);
        }
      }
      if (!ok) break;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(slot_full + group);
        if (a.keep) mbar_arrive(&empty[stage]);                      // nothing else of the stage is wanted
      }
      slot_phase ^= 1;
      left -= kI4WGroups;
      k += kI4WGroups;
      at += kI4WGroups * a.stage_bytes;
      if ((stage += kI4WGroups) >= a.stages) { stage -= a.stages; at -= a.stages * a.stage_bytes; phase ^= 1; }
    }
  } else {
    // ---------------------------------------------------------------- the warps that write: a weight row to a thread
    grid_dependency_wait();
    const int quarter = warp & 3, r = quarter * 32 + lane;
    if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    bool ok = true;
    int taken[kI4WGroups] = {};
    for (int p = 0; p < passes; ++p) {
      const int row = r0 + p * a.per_pass, rows = min(a.per_pass, r0 + mine - row);
      bool with[kI4WGroups];                                         // a pass of one or two steps has no work for some
#pragma unroll
      for (int g = 0; g < kI4WGroups; ++g) {
        with[g] = (g + 3 - p * count % 3) % 3 < count;
        if (with[g] && ok) ok = __all_sync(0xffffffffu, mbar_wait(&sums_full[g * 2 + taken[g] % sets], taken[g] / sets & 1, guard, kTimeoutAccFull));
      }
      if (a.parts > 1 && p > 0 && ok) ok = __all_sync(0xffffffffu, cluster_bar_wait(freed, (p - 1) & 1, guard, kTimeoutPeerFlag));
      if (!ok && a.parts == 1) break;
      tc_fence_after();
      for (int c = 0; ok && c < a.cols; c += 16) {
        float y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = 0.f;
#pragma unroll
        for (int g = 0; g < kI4WGroups; ++g) {
          if (!with[g]) continue;
          uint32_t x[16];
          tmem_ld16(tmem + kI4WSums + (g * sets + taken[g] % sets) * a.cols + c + ((uint32_t)(quarter * 32) << 16), x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] += __uint_as_float(x[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (a.parts > 1) part[(c + e) * 128 + r] = y[e];
          else if (r < rows && c + e < a.M) a.C[(c + e) * a.ldc + row + r] = __float2bfloat16(y[e]);
        }
      }
      tc_fence_before();
      __syncwarp();
#pragma unroll
      for (int g = 0; g < kI4WGroups; ++g) {
        if (!with[g]) continue;
        if (lane == 0) mbar_arrive(&sums_empty[g * 2 + taken[g] % sets]);
        ++taken[g];
      }
      if (a.parts == 1) continue;
      // every CTA of the cluster adds up the parts of some activation rows, in the order of the ranks
      asm volatile("bar.sync 2, 128;" ::: "memory");
      if (warp == kI4WWriters && lane < a.parts) cluster_arrive(ready, lane);
      __syncwarp();
      if (ok) ok = __all_sync(0xffffffffu, cluster_bar_wait(ready, p & 1, guard, kTimeoutPeerFlag));
      for (int m = rank; ok && m < a.M; m += 2 * a.parts) {          // all of two rows' loads are under way at once
        float v[2][kI4WMostParts];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < kI4WMostParts; ++c)
            v[i][c] = c < a.parts && m + i * a.parts < a.M ? ld_cluster(cluster_address(part + (m + i * a.parts) * 128 + r, c)) : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y = v[i][0];
#pragma unroll
          for (int c = 1; c < kI4WMostParts; ++c) y += v[i][c];
          if (r < rows && m + i * a.parts < a.M) a.C[(m + i * a.parts) * a.ldc + row + r] = __float2bfloat16(y);
        }
      }
      asm volatile("bar.sync 2, 128;" ::: "memory");
      if (warp == kI4WWriters && lane < a.parts) cluster_arrive(freed, lane);
      __syncwarp();
    }
  }
  __syncwarp();
  if (a.parts > 1) {
    // nobody leaves while its part may still be read, or a barrier of its be arrived at
    if (warp < kI4WWriters || warp >= kI4WFetch) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kI4WFetch) {
    const long long began = clock64();                               // nothing is in flight when the tensor memory goes
    while (!mbar_try_wait(ended, 0) && clock64() - began < kWaitLimitCycles) {}
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static cudaLaunchConfig_t wide_config(cudaLaunchAttribute (&at)[2], int parts, int ctas, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kI4WThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = dependent_launches() ? 2 : 1;
  return cfg;
}

// Clusters of `parts` CTAs that fit on the device at once.
static int wide_room(int parts) {
  static std::atomic<int> known[64][kI4WMostParts + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64)
    if (const int room = known[dev][parts].load(std::memory_order_relaxed)) return room;
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg = wide_config(at, parts, parts, kI4WSmemMost, nullptr);
  cfg.numAttrs = 1;
  int room = 0;
  if (cudaOccupancyMaxActiveClusters(&room, int4_linear_wide_kernel, &cfg) != cudaSuccess) return 0;
  if (dev < 64) known[dev][parts].store(room, std::memory_order_relaxed);
  return room;
}

// How `rooms` clusters of `parts` CTAs take N rows: quarters of a stage's time (0.6 us) of a CTA, with what a pass costs besides.  Measured with 1, 2, 4 and 8
// CTAs to a cluster, 16 rows and half a stage at a time: [6144, 2560] 11.8 us, 9.8, 11.6, 16.4; [2560, 4096] 14.7, 11.4, 8.7, 10.7; [2560, 9728] 26.7, 19.1,
// 13.5, 14.6; [19456, 2560] 18.6, 22.8, 25.8, 42.9.
static int wide_cost(int N, int steps, int parts, int rooms, int* per_cluster, int* per_pass) {
  const int passes = (N + rooms * 128 - 1) / (rooms * 128);
  *per_pass = (N + rooms * passes - 1) / (rooms * passes);
  *per_cluster = *per_pass * passes;
  return passes * (4 * ((steps + parts - 1) / parts) + (parts > 1 ? 16 : 2));
}

int int4_linear_wide(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda, long long ldc,
                     cudaStream_t st) {
  int* status = status_word();
  KSA_REQUIRE(status != nullptr, "int4_linear: no status word");
  static PerDevice raised;
  KSA_CHECK_CUDA(raise_smem_limit(raised, int4_linear_wide_kernel, kI4WSmemMost));
  Int4Wide a{};
  a.C = (bf16*)C; a.ldc = ldc; a.M = M; a.N = N; a.K = K; a.group = group;
  a.cols = (M + 15) / 16 * 16;
  a.steps = (K + kI4WStep - 1) / kI4WStep;
  int best = 0;
  for (int p = 1; p <= kI4WMostParts && p <= a.steps; p *= 2) {
    const int room = p == 1 ? sm_count() : wide_room(p);
    if (room <= 0) continue;
    int per_cluster, per_pass;
    const int cost = wide_cost(N, a.steps, p, room, &per_cluster, &per_pass);
    if (a.parts == 0 || cost < best) { best = cost; a.parts = p; a.per_cluster = per_cluster; a.per_pass = per_pass; }
  }
  KSA_REQUIRE(a.parts > 0, "int4_linear: no device");
  const int passes = a.per_cluster / a.per_pass, count = (a.steps + a.parts - 1) / a.parts, step_x = 4 * a.cols * 128;
  a.keep = passes > 1 && (long long)count * step_x <= kI4WKeepMost ? count * step_x : 0;
  a.meta_words = (a.per_pass + 3 + 3) / 4 * 4;
  a.b_at = (a.per_pass * 128 + 1023) / 1024 * 1024;
  a.meta_at = a.b_at + (a.keep ? 0 : step_x);
  a.stage_bytes = (a.meta_at + kI4WStep / group * a.meta_words * 4 + 1023) / 1024 * 1024;
  a.early = weights_early();
  const int rest = 1024 + a.keep + (a.parts > 1 ? a.cols * 512 : 0) + 512;
  a.stages = (kI4WSmemMost - rest) / a.stage_bytes;
  if (a.stages > passes * count + 2) a.stages = passes * count + 2;
  if (a.stages > kI4WMostStages) a.stages = kI4WMostStages;
  a.stages = a.stages / kI4WGroups * kI4WGroups;
  KSA_REQUIRE(a.stages >= kI4WGroups, "int4_linear: no room for three stages");
  size_t smem = (size_t)a.stages * a.stage_bytes + rest;
  if (smem < (size_t)kTmemClusterAlone) smem = kTmemClusterAlone;            // all of the tensor memory: alone on its SM (host.h)
  static_assert(kI4WSmemMost >= kTmemClusterAlone, "the limit raised above covers it");
  CUtensorMap tm, tm_meta, tm_x;
  {
    uint64_t dims[2] = {(uint64_t)K / 4, (uint64_t)N}, str[2] = {2, (uint64_t)K / 2};
    uint32_t box[2] = {64, (uint32_t)a.per_pass};
    if (const int rc = make_tmap(&tm, codes, 2, 2, dims, str, box, true)) return rc;
  }
  {
    uint64_t dims[2] = {(uint64_t)pitch, (uint64_t)(K / group)}, str[2] = {4, (uint64_t)pitch * 4};
    uint32_t box[2] = {(uint32_t)a.meta_words, (uint32_t)(kI4WStep / group)};
    if (const int rc = make_tmap(&tm_meta, meta, 4, 2, dims, str, box, false)) return rc;
  }
  {
    uint64_t dims[2] = {(uint64_t)K, (uint64_t)M}, str[2] = {2, (uint64_t)(M > 1 ? lda : K) * 2};
    uint32_t box[2] = {64, (uint32_t)a.cols};
    if (const int rc = make_tmap(&tm_x, A, 2, 2, dims, str, box, true)) return rc;
  }
  const int clusters = (N + a.per_cluster - 1) / a.per_cluster;
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg = wide_config(at, a.parts, clusters * a.parts, smem, st);
  KSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, int4_linear_wide_kernel, tm, tm_meta, tm_x, a, status));
  return 0;
}

}  // namespace ksa
