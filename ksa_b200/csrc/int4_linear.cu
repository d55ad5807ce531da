// Products of a few rows with weights of four bits: C[M, N] = A[M, K] * W[N, K]^T, M <= 16, W as int4.cuh says; with kGlu W holds gate rows and then up
// rows, and C[M, N / 2] = silu(gate) * up.
//
// What bounds it is reading the codes and scales once, N * K * (1/2 + 4 / group) bytes; next to that the issue slots: a lane's eight codes cost
// twelve operations and two mma.sync.  Hence:
//   * one CTA per SM, and each owns the same number of weight rows (+-1) whatever N is; it takes them in passes of up to 128, and a pass in
//     rounds of some segments of 128 columns.  A warp fetches rounds into a ring, one box of codes and one of scales each (a box of a single segment, 4 KB,
//     cost its 0.5 us whatever its size), as far ahead as the ring reaches, in the engine's decode step ahead of the previous kernel's end;
//   * sixteen warps multiply: a round has 16 / kParts segments, and kParts warps share the rows of a segment.  They keep their sums of a pass and
//     leave them in shared memory; two more warps add the sums up and write the results while the others are at the next pass;
//   * mma.sync m16n8k16 multiplies 16 weight rows by 8 activation rows; a lane's 16 bytes of a weight row are columns 32 t .. 32 t + 31 of the segment, in
//     that order for the activations as well.  Activations that several passes want, and few of one pass, stay in shared memory, others are read as they are needed.
#include "int4_linear.h"

#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4LWarps = 16;                       // that multiply
constexpr int kI4LAdders = 2;                       // that add up and write
constexpr int kI4LThreads = (kI4LWarps + kI4LAdders + 1) * 32;
constexpr int kI4LBlocks = 2;                       // blocks of 16 weight rows of a warp
constexpr int kI4LMostStages = 12;
constexpr int kI4LMostRows = 16;
// Nine rows and more of a large weight go to int4_linear_wide.cu: from 80 weight rows a CTA and 1536 columns.  Measured on 16 rows, this kernel against
// that one: [6144, 2560] 7.7 us against 10.0, [2560, 9728] 11.5 against 12.6, [12000, 4096] 18.8 against 14.4, [19456, 2560] 16.8 against 16.4, [19456, 4096]
// 27.2 against 22.5, [151936, 2560] 71 against 54, but [40000, 1024] 15.2 against 15.7, [100000, 512] 20.3 against 20.4; on nine rows [12000, 4096] 15.8
// against 14.6, [19456, 4096] 21.8 against 22.2; on one row [151936, 2560] 52 against 53, [86978, 2368] 31 against 33.
constexpr int kI4LWideRows = 80, kI4LWideColumns = 1536;
constexpr int kI4LSmemMost = 227 * 1024;

// Optional residual add and RMSNorm ahead of the product (as in gemv.cu): the activations are bf16(rms_norm(bf16(A + delta)) * w), made by every CTA for
// itself and kept in its shared memory, while the ring fills.  Block 0 leaves A + delta in `res`.  Against two launches, one and four rows:
// [6144, 2560] 8.3 -> 6.4 us and 8.7 -> 8.2, gate and up rows of [19456, 2560] 14.8 -> 13.7 and 16.6 -> 15.5.
struct Int4Norm {
  const bf16 *delta, *w;           // rows [0, delta_rows) have a delta
  bf16* res;                       // null: nobody wants it
  long long ld_delta, ld_res;
  float eps;
  int delta_rows;
};
constexpr int kI4LNormRows = 4;

struct Int4Linear {
  const bf16* A;
  const uint32_t* meta;            // [K / group, pitch]
  bf16* C;
  long long lda, ldc;
  int M, N, K, group, pitch;       // N: rows of the weight
  int n_out, per_cta, per_pass;    // output columns: of all, of a CTA, of a pass
  int segments, stages, stage_bytes;
  int meta_words, meta_at;         // words of a group's scales in a stage, and where they begin
  int x_pitch;                     // bytes of an activation row in shared memory, 0: none are kept
  int ragged;                      // the last segment is not whole: a box for each
  int early;                       // weights are read ahead of the wait
  Int4Norm norm;
};

__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// acc[i] += rows 16 i + (g, g + 8) of the segment at `codes` times the activations' columns of it.  kShort: the last block has eight rows at most, the
// others are taken as zeros (18 rows to a CTA: [2560, 9728] 9.0 -> 8.4 us, [2560, 4096] 4.8 -> 4.4; where several warps
// share the rows nothing is gained).
template <int NB, int kCount, bool kShort>
__device__ __forceinline__ void i4l_multiply(float (&acc)[kI4LBlocks][NB][4], const uint4 (&x)[NB][4], uint32_t codes, uint32_t meta) {
  uint32_t words[kCount][2][4], s2[kCount][2], o2[kCount][2];
#pragma unroll
  for (int i = 0; i < kCount; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (kShort && i == kCount - 1 && h == 1) break;
      const uint4 four = ld_shared(codes + (i * 16 + h * 8) * 64);
      words[i][h][0] = four.x; words[i][h][1] = four.y; words[i][h][2] = four.z; words[i][h][3] = four.w;
      uint32_t m;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(m) : "r"(meta + (i * 16 + h * 8) * 4) : "memory");
      s2[i][h] = i4_scale2(m);
      o2[i][h] = i4_offset2(m);
    }
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      uint32_t v[4], w[4] = {0, 0, 0, 0};
      i4_values(v, words[i][0][q], s2[i][0], o2[i][0]);
      if (!kShort || i < kCount - 1) i4_values(w, words[i][1][q], s2[i][1], o2[i][1]);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        mma_bf16(acc[i][n], v[0], w[0], v[1], w[1], x[n][q].x, x[n][q].y);
        mma_bf16(acc[i][n], v[2], w[2], v[3], w[3], x[n][q].z, x[n][q].w);
      }
    }
}

// NB: activation rows in eights.  kParts: warps that share a segment's rows, up to 32 each (kGlu: the first half of them gate rows, the other their up rows).
// kNorm: a norm ahead.  kKept: activations stay in shared memory, which the compiler wants to know: with both ways in one kernel [2560, 9728] x 16 rows took
// 11.5 us instead of 11.1, [151936, 2560] x 1 row 51.9 instead of 50.2 (but [2560, 9728] x 5 rows, which do not stay, 8.4 instead of 8.6).
template <int NB, int kParts, bool kGlu, bool kNorm, bool kKept>
__global__ void __launch_bounds__(kI4LThreads, 1)
int4_linear_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_meta, const Int4Linear a, int* status) {
  static_assert(!kGlu || kParts >= 2, "parts for gate and up rows");
  constexpr int kTurns = kI4LWarps / kParts;                                // segments of a round
  constexpr int kRows = kI4LBlocks * 16 * kParts, kPitch = kRows + 8;        // rows of a pass; floats of a row of sums
  constexpr int kSets = kGlu ? 2 : 1, kPerSet = kParts / kSets;             // boxes of a round, warps for the rows of one
  extern __shared__ __align__(128) uint8_t raw[];
  uint8_t* ring = raw;
  float* part = reinterpret_cast<float*>(ring + a.stages * a.stage_bytes);  // [turns][NB * 8][kPitch]
  uint8_t* xs = reinterpret_cast<uint8_t*>(part + kTurns * NB * 8 * kPitch);
  uint64_t* full = reinterpret_cast<uint64_t*>(xs + a.M * a.x_pitch);
  uint64_t* empty = full + a.stages;
  uint64_t* left = empty + a.stages;                                         // the sums of a pass are there
  uint64_t* added = left + 1;                                                // and have been read
  volatile int* abort_flag = reinterpret_cast<volatile int*>(added + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const WaitGuard guard{abort_flag, status};
  const int r0 = (int)blockIdx.x * a.per_cta, mine = min(a.per_cta, a.n_out - r0);
  const int passes = (mine + a.per_pass - 1) / a.per_pass, rounds = (a.segments + kTurns - 1) / kTurns;
  const int groups = 128 / a.group;                                          // of a segment
  const int set_bytes = (kTurns * a.per_pass * 64 + 127) / 128 * 128, meta_bytes = (kTurns * groups * a.meta_words * 4 + 127) / 128 * 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], kI4LWarps); }
    mbar_init(left, kI4LWarps);
    mbar_init(added, kI4LAdders);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm);
    tma_prefetch_desc(&tm_meta);
  }
  __syncthreads();
  grid_dependency_launch();

  if (warp == kI4LWarps + kI4LAdders) {
    // ---------------------------------------------------------------- the warp that fetches
    if (!a.early) grid_dependency_wait();
    const int total = passes * rounds;
    const uint32_t bytes = kSets * kTurns * (a.per_pass * 64 + groups * a.meta_words * 4);       // also past the matrix's edges
    int stage = 0, round = 0, row = r0, done = 0;
    uint32_t phase = 1;
    for (; done < total; ++done) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase, guard, kTimeoutStageEmpty))) break;
      uint8_t* dst = ring + stage * a.stage_bytes;
      if (elect_one()) {
        mbar_expect_tx(&full[stage], bytes);
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const int from = s * a.n_out + row;
          if (!a.ragged) tma_load_3d(dst + s * set_bytes, &tm, 0, from, round * kTurns, &full[stage]);
          tma_load_2d(dst + a.meta_at + s * meta_bytes, &tm_meta, from & ~3, round * kTurns * groups, &full[stage]);
        }
      }
      __syncwarp();
      if (a.ragged && lane < kTurns) {
#pragma unroll
        for (int s = 0; s < kSets; ++s)
          tma_load_2d(dst + s * set_bytes + lane * a.per_pass * 64, &tm, (round * kTurns + lane) * 32, s * a.n_out + row, &full[stage]);
      }
      __syncwarp();
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
      if (++round == rounds) { round = 0; row += a.per_pass; }
    }
    if (a.early) grid_dependency_wait();
    // whatever the others have given up on: the last copies land before the block leaves
    const long long began = clock64();
    for (int i = max(0, done - a.stages); i < done; ++i)
      while (!mbar_try_wait(&full[i % a.stages], (i / a.stages) & 1) && clock64() - began < kWaitLimitCycles) {}
    return;
  }
  grid_dependency_wait();

  if (warp >= kI4LWarps) {
    // ---------------------------------------------------------------- the warps that add up: four columns of a row at a time
    const int me = (warp - kI4LWarps) * 32 + lane;
    for (int p = 0; p < passes; ++p) {
      const int row = r0 + p * a.per_pass, rows = min(a.per_pass, r0 + mine - row), quads = (rows + 3) / 4;
      if (!__all_sync(0xffffffffu, mbar_wait(left, p & 1, guard, kTimeoutAccFull))) break;
      for (int i = me; i < a.M * quads; i += kI4LAdders * 32) {
        const int m = i / quads, c = (i - m * quads) * 4;
        float v[kSets][4];
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[s][e] = 0.f;
#pragma unroll
          for (int w = 0; w < kTurns; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(part + (w * NB * 8 + m) * kPitch + s * (kRows / 2) + c);
            v[s][0] += x.x; v[s][1] += x.y; v[s][2] += x.z; v[s][3] += x.w;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = v[0][e];
          if (kGlu) {
            // gate and up are rounded to bf16 first, as the separate projection and activation do
            const float gt = __bfloat162float(__float2bfloat16(y)), up = __bfloat162float(__float2bfloat16(v[kSets - 1][e]));
            y = gt / (1.f + __expf(-gt)) * up;
          }
          if (c + e < rows) a.C[m * a.ldc + row + c + e] = __float2bfloat16(y);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(added);
    }
    return;
  }

  // ------------------------------------------------------------------ the warps that multiply
  if (kNorm) {
    float* s_sum = part;                                             // [warps][rows], before the first sums
    const int per = rounds * kTurns * 16;                            // pieces of 16 bytes, with zeros behind the row
    float sum[kI4LNormRows] = {0.f, 0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < per; c += kI4LWarps * 32) {
      uint4 xv[kI4LNormRows], dv[kI4LNormRows];
#pragma unroll
      for (int m = 0; m < kI4LNormRows; ++m) {
        xv[m] = dv[m] = make_uint4(0, 0, 0, 0);
        if (m < a.M && c * 8 < a.K) {
          xv[m] = *reinterpret_cast<const uint4*>(a.A + m * a.lda + c * 8);
          if (m < a.norm.delta_rows) dv[m] = *reinterpret_cast<const uint4*>(a.norm.delta + m * a.norm.ld_delta + c * 8);
        }
      }
#pragma unroll
      for (int m = 0; m < kI4LNormRows; ++m) {
        if (m >= a.M) break;
        const uint32_t x4[4] = {xv[m].x, xv[m].y, xv[m].z, xv[m].w}, d4[4] = {dv[m].x, dv[m].y, dv[m].z, dv[m].w};
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          o[q] = x4[q];
          if (m < a.norm.delta_rows) {
            const float2 x = unpack_bf16x2(x4[q]), d = unpack_bf16x2(d4[q]);
            o[q] = pack_bf16x2(x.x + d.x, x.y + d.y);
          }
          const float2 f = unpack_bf16x2(o[q]);
          sum[m] += f.x * f.x + f.y * f.y;
        }
        const uint4 r = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(xs + m * a.x_pitch + (c & ~15) * 16 + ((c & 3) * 4 + ((c >> 2) & 3)) * 16) = r;
        if (blockIdx.x == 0 && a.norm.res != nullptr && c * 8 < a.K) *reinterpret_cast<uint4*>(a.norm.res + m * a.norm.ld_res + c * 8) = r;
      }
    }
#pragma unroll
    for (int m = 0; m < kI4LNormRows; ++m) {
      sum[m] = warp_sum(sum[m]);
      if (lane == 0) s_sum[warp * kI4LNormRows + m] = sum[m];
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kI4LWarps * 32) : "memory");
    float rstd[kI4LNormRows] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kI4LWarps; ++w)
#pragma unroll
      for (int m = 0; m < kI4LNormRows; ++m) rstd[m] += s_sum[w * kI4LNormRows + m];
#pragma unroll
    for (int m = 0; m < kI4LNormRows; ++m) rstd[m] = rsqrtf(rstd[m] / (float)a.K + a.norm.eps);
    for (int c = threadIdx.x; c * 8 < a.K; c += kI4LWarps * 32) {    // a thread's own pieces again
      const uint4 wv = *reinterpret_cast<const uint4*>(a.norm.w + c * 8);
      const uint32_t w4[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
      for (int m = 0; m < kI4LNormRows; ++m) {
        if (m >= a.M) break;
        uint4* at = reinterpret_cast<uint4*>(xs + m * a.x_pitch + (c & ~15) * 16 + ((c & 3) * 4 + ((c >> 2) & 3)) * 16);
        const uint4 xv = *at;
        const uint32_t x4[4] = {xv.x, xv.y, xv.z, xv.w};
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 x = unpack_bf16x2(x4[q]), f = unpack_bf16x2(w4[q]);
          o[q] = pack_bf16x2(x.x * rstd[m] * f.x, x.y * rstd[m] * f.y);
        }
        *at = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kI4LWarps * 32) : "memory");
  } else if (kKept) {
    // an activation's 16 bytes w of the 64 that lane t wants of a segment lie at 4 w + t: four lanes read 64 bytes in a row
    const int per = rounds * kTurns * 16;
    constexpr int kAtOnce = NB * 4;
    for (int c = threadIdx.x; c < per; c += kI4LWarps * 32) {
      const int at = (c & ~15) * 16 + ((c & 3) * 4 + ((c >> 2) & 3)) * 16;
      for (int m0 = 0; m0 < a.M; m0 += kAtOnce) {
        uint4 v[kAtOnce];
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m) {
          v[m] = make_uint4(0, 0, 0, 0);
          if (m0 + m < a.M && c * 8 < a.K) v[m] = *reinterpret_cast<const uint4*>(a.A + (m0 + m) * a.lda + c * 8);         // zeros behind
        }
#pragma unroll
        for (int m = 0; m < kAtOnce; ++m)
          if (m0 + m < a.M) *reinterpret_cast<uint4*>(xs + (m0 + m) * a.x_pitch + at) = v[m];
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kI4LWarps * 32) : "memory");
  }
  const int turn = warp / kParts, set = kGlu ? warp % kParts / kPerSet : 0, which = warp % kParts % kPerSet;
  const int t_group = t * 32 / a.group;
  // this lane's activations of the warp's first segment, and those eight rows on; a row past the last is the last one again, in sums that nobody reads
  const int x_row = min(g, a.M - 1), x_next = NB == 2 ? min(g + 8, a.M - 1) - x_row : 0;
  const bf16* x_first = a.A + x_row * a.lda + turn * 128 + t * 32;
  const long long x_eight = x_next * a.lda;
  const uint32_t x_kept = smem_u32(xs) + x_row * a.x_pitch + turn * 256 + t * 16, kept_eight = x_next * a.x_pitch;
  const uint32_t ring_at = smem_u32(ring);
  bool ok = true;
  int stage = 0;
  uint32_t phase = 0;
  for (int p = 0; p < passes; ++p) {
    const int row = r0 + p * a.per_pass, blocks = (min(a.per_pass, r0 + mine - row) + 15) / 16;
    // this warp's blocks of the rows, and the first row of them
    const int each = (blocks + kPerSet - 1) / kPerSet, at = which * each * 16, count = max(0, min(each, blocks - which * each));
    const int skip = (set * a.n_out + row) & 3;
    const bool few = min(a.per_pass, r0 + mine - row) - at <= 24;            // the second block has eight rows at most
    float acc[kI4LBlocks][NB][4];
#pragma unroll
    for (int i = 0; i < kI4LBlocks; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.f;
    // where this lane reads: in a stage, and the activations of the pass's first segment
    const uint32_t codes_at = set * set_bytes + (turn * a.per_pass + at + g) * 64 + t * 16;
    const uint32_t meta_at = a.meta_at + set * meta_bytes + ((turn * groups + t_group) * a.meta_words + skip + at + g) * 4;
    const bf16* xp = x_first;
    uint32_t xk = x_kept;
    for (int round = 0, seg = turn; round < rounds; ++round, seg += kTurns, xp += kTurns * 128, xk += kTurns * 256) {
      // past K the weights are zeros, and so are the activations: an infinity there would make them NaN
      uint4 x[NB][4];
      if (kKept) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) x[n][q] = ld_shared(xk + n * kept_eight + q * 64);
      } else {
        const bool inside = seg * 128 + t * 32 < a.K;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) x[n][q] = inside ? *reinterpret_cast<const uint4*>(xp + n * x_eight + q * 8) : make_uint4(0, 0, 0, 0);
      }
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, guard, kTimeoutTmaFull));
      if (!ok) break;
      if (seg < a.segments) {                                                // what lies past K in the last one is zeros, scales and all
        const uint32_t src = ring_at + stage * a.stage_bytes, codes = src + codes_at, meta = src + meta_at;
        if (kParts == 1 && count == 2 && few) i4l_multiply<NB, 2, true>(acc, x, codes, meta);
        else if (count == 2) i4l_multiply<NB, 2, false>(acc, x, codes, meta);            // two chains of products side by side
        else if (count == 1) i4l_multiply<NB, 1, false>(acc, x, codes, meta);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
    }
    // ---- this warp's sums: acc[i][n] = (weight row g, activations 2 t and 2 t + 1), (weight row g + 8, the same)
    if (p > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(added, (p - 1) & 1, guard, kTimeoutAccEmpty));
    if (!ok) break;
#pragma unroll
    for (int i = 0; i < kI4LBlocks; ++i) {
      if (i >= count) break;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = n * 8 + t * 2 + (e & 1);
          if (m < a.M) part[(turn * NB * 8 + m) * kPitch + set * (kRows / 2) + at + i * 16 + (e >> 1) * 8 + g] = acc[i][n][e];
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(left);
  }
}

// How a CTA of `per_cta` output columns takes them with `parts` warps to a segment: rows of a pass, and the blocks of rows that a warp multiplies in all,
// with what a round costs besides (one of them) and a pass (two).
static int i4l_cost(int per_cta, int segments, int parts, int sets, int* per_pass) {
  const int most = kI4LBlocks * 16 * parts / sets, passes = (per_cta + most - 1) / most, turns = kI4LWarps / parts;
  *per_pass = (per_cta + passes - 1) / passes;
  const int each = ((*per_pass + 15) / 16 * sets + parts - 1) / parts;
  return passes * ((segments + turns - 1) / turns * (each + 1) + 2);
}

template <int NB, int kParts, bool kGlu, bool kNorm = false>
static int launch_int4_linear(Int4Linear a, const void* codes, cudaStream_t st) {
  constexpr int kTurns = kI4LWarps / kParts, kRows = kI4LBlocks * 16 * kParts, kPitch = kRows + 8, kSets = kGlu ? 2 : 1;
  int* status = status_word();
  KSA_REQUIRE(status != nullptr, "int4_linear: no status word");
  const int groups = 128 / a.group;
  a.meta_words = (a.per_pass + 3 + 3) / 4 * 4;
  a.meta_at = kSets * ((kTurns * a.per_pass * 64 + 127) / 128 * 128) + 1024;      // the last block may reach past the rows
  a.stage_bytes = a.meta_at + kSets * ((kTurns * groups * a.meta_words * 4 + 127) / 128 * 128) + 128;          // (its scales as well)
  const int part = kTurns * NB * 8 * kPitch * 4, per_stage = a.stage_bytes + 16, rest = part + 32;
  // Activations stay where a ring of 64 KB and three rounds finds room beside them: those that several passes want, and few of one pass, a piece or
  // none a thread and row, which come in while the ring fills ([6144, 2560] x 4 rows 6.2 -> 5.8 us, x 1 row 5.9 -> 5.7; more of them keep the first
  // round waiting: [2560, 9728] x 5 rows 8.5 -> 10.0, [6144, 2560] x 16 rows 7.9 -> 9.0)
  const int passes = (a.per_cta + a.per_pass - 1) / a.per_pass, x_pitch = (a.segments + kTurns - 1) / kTurns * kTurns * 256 + 64;
  const int least = 3 * per_stage > 64 * 1024 ? 3 * per_stage : 64 * 1024;
  a.x_pitch = (passes > 1 || kNorm || (a.M <= 4 && a.K <= kI4LWarps * 32 * 8)) && (long long)a.M * x_pitch + rest + least <= kI4LSmemMost ? x_pitch : 0;
  KSA_REQUIRE(!kNorm || a.x_pitch > 0, "int4_norm_linear: no room for %d rows of %d values", a.M, a.K);
  a.stages = (kI4LSmemMost - rest - a.M * a.x_pitch) / per_stage;
  const int wanted = passes * ((a.segments + kTurns - 1) / kTurns);
  if (a.stages > wanted) a.stages = wanted;
  if (a.stages > kI4LMostStages) a.stages = kI4LMostStages;
  KSA_REQUIRE(a.stages >= 1, "int4_linear: no room for a round");
  const size_t smem = (size_t)a.stages * per_stage + rest + a.M * a.x_pitch;
  CUtensorMap tm, tm_meta;
  {
    uint64_t dims[3] = {(uint64_t)(a.ragged ? a.K / 4 : 32), (uint64_t)a.N, (uint64_t)a.segments}, str[3] = {2, (uint64_t)a.K / 2, 64};
    uint32_t box[3] = {32, (uint32_t)a.per_pass, (uint32_t)kTurns};
    if (const int rc = make_tmap(&tm, codes, 2, a.ragged ? 2 : 3, dims, str, box, false)) return rc;
  }
  {
    uint64_t dims[2] = {(uint64_t)a.pitch, (uint64_t)(a.K / a.group)}, str[2] = {4, (uint64_t)a.pitch * 4};
    uint32_t box[2] = {(uint32_t)a.meta_words, (uint32_t)(kTurns * groups)};
    if (const int rc = make_tmap(&tm_meta, a.meta, 4, 2, dims, str, box, false)) return rc;
  }
  const bool kept = a.x_pitch > 0;
  auto kern = kept ? int4_linear_kernel<NB, kParts, kGlu, kNorm, true> : int4_linear_kernel<NB, kParts, kGlu, kNorm, kNorm>;
  static PerDevice raised[2];
  KSA_CHECK_CUDA(raise_smem_limit(raised[kept], kern, kI4LSmemMost));
  KSA_CHECK_CUDA(launch_kernel(kern, dim3((a.n_out + a.per_cta - 1) / a.per_cta), dim3(kI4LThreads), smem, st, tm, tm_meta, a, status));
  return 0;
}

static int int4_linear(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda, long long ldc,
                       int glu, const Int4Norm* norm, cudaStream_t st) {
  KSA_REQUIRE(M >= 0 && M <= (glu ? kI4LMostRows : kI4WMostRows), "int4_linear: %d rows (at most %d)", M, glu ? kI4LMostRows : kI4WMostRows);
  KSA_REQUIRE(group == 32 || group == 64 || group == 128, "int4_linear: groups of %d values (32, 64 or 128)", group);
  KSA_REQUIRE(K > 0 && K % group == 0 && N >= 0 && pitch >= N && pitch % 4 == 0, "int4_linear: K %d is no multiple of the group of %d", K, group);
  KSA_REQUIRE(!glu || N % 2 == 0, "int4_linear: gate and up rows must be as many, got %d together", N);
  KSA_REQUIRE(lda % 8 == 0 && ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(meta)) & 15) == 0,
              "int4_linear: rows, codes and scales must be 16-byte aligned");
  if (M == 0 || N == 0) return 0;
  const bool spread = M > 1 && lda < K;                                      // rows that lie in one another
  KSA_REQUIRE(M <= kI4LMostRows || !spread, "int4_linear: %d rows at a pitch of %lld for %d values", M, lda, K);
  const int sms = sm_count();
  KSA_REQUIRE(sms > 0, "int4_linear: no device");
  if (norm == nullptr && !glu && !spread && (M > kI4LMostRows || (M > 8 && K >= kI4LWideColumns && N >= kI4LWideRows * sms)))
    return int4_linear_wide(A, codes, meta, C, M, N, K, group, pitch, lda, ldc, st);
  Int4Linear a{};
  a.A = (const bf16*)A; a.meta = (const uint32_t*)meta; a.C = (bf16*)C;
  a.lda = lda; a.ldc = ldc; a.M = M; a.N = N; a.K = K; a.group = group; a.pitch = pitch;
  a.n_out = glu ? N / 2 : N;
  a.per_cta = (a.n_out + sms - 1) / sms;
  a.segments = (K + 127) / 128;
  a.ragged = K % 128 != 0;
  a.early = weights_early();
  int parts = 0, best = 0;
  for (int p = glu ? 2 : 1; p <= 4; p *= 2) {
    int per_pass;
    const int cost = i4l_cost(a.per_cta, a.segments, p, glu ? 2 : 1, &per_pass);
    if (parts == 0 || cost < best) { parts = p; best = cost; a.per_pass = per_pass; }
  }
  if (a.ragged) a.per_pass += a.per_pass & 1;        // a box begins on 128 bytes
  if (norm != nullptr) {
    a.norm = *norm;
    if (glu) return parts == 2 ? launch_int4_linear<1, 2, true, true>(a, codes, st) : launch_int4_linear<1, 4, true, true>(a, codes, st);
    return parts == 1 ? launch_int4_linear<1, 1, false, true>(a, codes, st) :
           parts == 2 ? launch_int4_linear<1, 2, false, true>(a, codes, st) : launch_int4_linear<1, 4, false, true>(a, codes, st);
  }
  if (glu && parts == 2) return M <= 8 ? launch_int4_linear<1, 2, true>(a, codes, st) : launch_int4_linear<2, 2, true>(a, codes, st);
  if (glu) return M <= 8 ? launch_int4_linear<1, 4, true>(a, codes, st) : launch_int4_linear<2, 4, true>(a, codes, st);
  if (parts == 1) return M <= 8 ? launch_int4_linear<1, 1, false>(a, codes, st) : launch_int4_linear<2, 1, false>(a, codes, st);
  if (parts == 2) return M <= 8 ? launch_int4_linear<1, 2, false>(a, codes, st) : launch_int4_linear<2, 2, false>(a, codes, st);
  return M <= 8 ? launch_int4_linear<1, 4, false>(a, codes, st) : launch_int4_linear<2, 4, false>(a, codes, st);
}

}  // namespace ksa

using namespace ksa;

// A [M <= 32, K] (row pitch lda; M <= 16 with glu), codes [N, K / 2], scales [K / group, pitch] words -> C [M, N] (row pitch ldc); glu: gate rows and
// then up rows, C [M, N / 2].
KSA_API int ksa_int4_linear(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda,
                            long long ldc, int glu, void* stream) {
  KSA_ENTER(A);
  return int4_linear(A, codes, meta, C, M, N, K, group, pitch, lda, ldc, glu, nullptr, reinterpret_cast<cudaStream_t>(stream));
}

// res = x + delta (rows [0, delta_rows), the others are x's; null: not wanted) and C = rms_norm(res, norm_w, eps) * W^T, M <= 4.
KSA_API int ksa_int4_norm_linear(const void* x, const void* delta, const void* norm_w, void* res, const void* codes, const void* meta, void* C, int M,
                                 int N, int K, int group, int pitch, long long ldx, long long ld_delta, long long ld_res, long long ldc, float eps,
                                 int delta_rows, int glu, void* stream) {
  KSA_ENTER(x);
  KSA_REQUIRE(M <= kI4LNormRows, "int4_norm_linear: %d rows (at most %d)", M, kI4LNormRows);
  KSA_REQUIRE(norm_w != nullptr && delta_rows >= 0 && delta_rows <= M && (delta_rows == 0 || delta != nullptr), "int4_norm_linear: incomplete arguments");
  KSA_REQUIRE(((reinterpret_cast<uintptr_t>(delta) | reinterpret_cast<uintptr_t>(norm_w) | reinterpret_cast<uintptr_t>(res)) & 15) == 0 &&
              ld_delta % 8 == 0 && ld_res % 8 == 0, "int4_norm_linear: rows must be 16-byte aligned");
  const Int4Norm norm{(const bf16*)delta, (const bf16*)norm_w, (bf16*)res, ld_delta, ld_res, eps, delta_rows};
  return int4_linear(x, codes, meta, C, M, N, K, group, pitch, ldx, ldc, glu, &norm, reinterpret_cast<cudaStream_t>(stream));
}
