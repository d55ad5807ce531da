// Losses of a post-training step over the log probabilities y of answer tokens, and their gradients.
//
// Clipped policy loss with a KL term.  d = y - y_old, r = exp(d), L = -min(r A, clip(r, 1 - low, 1 + high) A); x = y_ref - y,
// K = exp(x) - 1 - x.  The loss is the mean of L + beta K over the valid tokens, or the mean over the sequences that have one of each
// sequence's mean.  L is cut off, and has no gradient, where A > 0 and d > log(1 + high) or A < 0 and d < log(1 - low); elsewhere
// dL / dy = -A r, and dK / dy = 1 - exp(x).
// Preference loss.  D_s = sum over the valid tokens of sequence s of y - y_ref, z_i = beta (D_2i - D_2i+1); the loss is the mean over the
// pairs of (1 - smoothing) log(1 + exp(-z)) + smoothing log(1 + exp(z)), and dz = smoothing - 1 / (1 + exp(z)).
//
// Bound: memory from some hundred thousand tokens on (17 bytes of a token read by the policy loss, 9 by the preference loss), launches
// below.  The policy loss writes each token's gradient up to the normaliser in the same pass, in 32 bits, and the backward pass reads
// those: the normaliser and the incoming gradient are known only then.
//
// Work is cut into units: sequence s has pieces of kTlPiece tokens, and piece p of it is unit floor(first / kTlPiece) + s + p.  That is a
// different number for every piece, as the next sequence's first unit is at least one further than the last of this one's,
// and a block finds its sequence by bisection: no list is built first, and lengths of zero cost an empty unit.  The tokens behind the
// last sequence are one more sequence, without valid tokens.
//
// A difference of two fp32 numbers is rounded once, which exponentials bear; next to the border of the clipped range it is taken again in 64
// bits, so that a token falls on the side where it belongs.  A thread's few terms are summed in 32 bits, everything above that, and the log
// ratios of whole answers from their first token on, in 64 and in a fixed order.
#include "common.cuh"
#include "host.h"

#include <cuda_fp16.h>
#include <math.h>

namespace ksa {

constexpr int kTlThreads = 256;
// 4096 tokens to a piece: policy loss and gradient of 64 x 8192 tokens 17.3 us against 13.8 (fewer blocks than SMs), of 256 x 32768 52 against 58.
constexpr int kTlPiece = 2048;

enum TokenType : int { kTokF32 = 0, kTokBf16 = 1, kTokF16 = 2 };

struct Sequences {
  const void* cu;              // offsets [S + 1] of 32 or 64 bits, or null: rows of `length` tokens
  int wide;
  int S;
  long long n, length;

  __device__ __forceinline__ long long first(int s) const {                      // of the tokens behind the last sequence: s = S
    if (s <= 0) return 0;
    if (cu == nullptr) return min((long long)s * length, n);
    const long long v = wide ? static_cast<const long long*>(cu)[s] : (long long)static_cast<const int*>(cu)[s];
    return max(0LL, min(v, n));
  }
  __device__ __forceinline__ long long end(int s) const { return s >= S ? n : first(s + 1); }
  __device__ __forceinline__ long long unit(int s) const { return first(s) / kTlPiece + s; }
};

struct Piece {
  int s;
  long long lo, hi;            // its tokens; none where lo >= hi
};
// The last sequence whose first unit is not behind `unit`, by every warp: its lanes try 32 places at a time (two rounds of loads for 1000
// sequences, where bisection takes ten).
__device__ __forceinline__ Piece find_piece(const Sequences& q, long long unit) {
  int lo = 0, n = q.S + 1;
  while (n > 1) {
    const int step = (n + 31) / 32, at = (int)(threadIdx.x & 31) * step;
    const unsigned yes = __ballot_sync(0xffffffffu, at < n && (at == 0 || q.unit(lo + at) <= unit));
    const int found = (31 - __clz(yes)) * step;
    lo += found;
    n = min(step, n - found);
  }
  Piece p;
  p.s = lo;
  p.lo = q.first(lo) + (unit - q.unit(lo)) * kTlPiece;
  p.hi = min(q.end(lo), p.lo + kTlPiece);
  return p;
}

__device__ __forceinline__ float load_token(const void* p, int type, long long i) {
  if (type == kTokF32) return static_cast<const float*>(p)[i];
  if (type == kTokBf16) return __bfloat162float(static_cast<const bf16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void load_tokens(const void* p, int type, long long i, float (&f)[4]) {      // i a multiple of 4
  if (type == kTokF32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    return;
  }
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  const float2 a = type == kTokBf16 ? unpack_bf16x2(v.x) : __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 b = type == kTokBf16 ? unpack_bf16x2(v.y) : __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
__device__ __forceinline__ void store_token(void* p, int type, long long i, float v) {
  if (type == kTokF32) static_cast<float*>(p)[i] = v;
  else if (type == kTokBf16) static_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ void store_tokens(void* p, int type, long long i, const float (&f)[4]) {
  if (type == kTokF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    return;
  }
  uint2 v;
  if (type == kTokBf16) v = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  else {
    const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
    v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = v;
}

template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* red) {        // red: N values for every warp; the sums in all threads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  __syncthreads();
  if (lane == 0)
    for (int k = 0; k < N; ++k) red[warp * N + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    double t = lane < warps ? red[lane * N + k] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    v[k] = t;
  }
}
template <int N>
__device__ __forceinline__ void warp_sums(double (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

// exp(x) - 1 and exp(x) - 1 - x.  Within one of zero by the series, whose first terms are what the differences would lose.
struct ExpLess {
  float one, line;
};
__device__ __forceinline__ ExpLess exp_less(float x) {
  ExpLess e;
  if (!(fabsf(x) < 1.f)) {
    e.one = expf(x) - 1.f;
    e.line = e.one == INFINITY ? INFINITY : e.one - x;                            // (x itself may be infinite)
    return e;
  }
  float p = 1.f / 479001600.f;                                                    // 1 / 12!
  p = fmaf(p, x, 1.f / 39916800.f);
  p = fmaf(p, x, 1.f / 3628800.f);
  p = fmaf(p, x, 1.f / 362880.f);
  p = fmaf(p, x, 1.f / 40320.f);
  p = fmaf(p, x, 1.f / 5040.f);
  p = fmaf(p, x, 1.f / 720.f);
  p = fmaf(p, x, 1.f / 120.f);
  p = fmaf(p, x, 1.f / 24.f);
  p = fmaf(p, x, 1.f / 6.f);
  p = fmaf(p, x, 0.5f);
  e.line = x * x * p;
  e.one = fmaf(x * x, p, x);
  return e;
}

struct PolicyArgs {
  const void *y, *old, *ref, *adv;
  const uint8_t* mask;
  int ty, told, tref, tadv, adv_by_sequence, by_sequence, vec;
  double above, below;         // log(1 + high), log(1 - low)
  float above32, below32;
  float most, least;           // 1 + high, 1 - low
  float beta;
  float* grad;                 // [n] up to the normaliser, or null
  double* partial;             // [units][4]: sums of L and K, tokens that are cut off, valid tokens
  float* inv;                  // normaliser: one, or one for every sequence
  float* loss;
  float* stats;                // mean L, mean K, share that is cut off
};

struct TokenTerms {
  float L, K, g;
  int cut;
};
__device__ __forceinline__ TokenTerms policy_token(const PolicyArgs& a, float y, float old, float ref, float A) {
  TokenTerms t;
  const float d = y - old;
  t.cut = (A > 0.f && d > a.above32) || (A < 0.f && d < a.below32);
  if (fabsf(d - (A > 0.f ? a.above32 : a.below32)) < 1e-6f * fabsf(d)) {         // next to the border the difference's rounding would decide
    const double exact = (double)y - (double)old;
    t.cut = (A > 0.f && exact > a.above) || (A < 0.f && exact < a.below);
  }
  const float r = expf(d);
  const float part = A == 0.f && !isnan(d) ? 0.f : -r * A;                        // (no advantage, no loss: not even where the ratio is infinite)
  t.L = t.cut ? -(A > 0.f ? a.most : a.least) * A : part;
  t.g = t.cut ? 0.f : part;
  t.K = 0.f;
  if (a.ref) {
    const float x = ref - y;
    const ExpLess e = exp_less(x);
    t.K = e.line;
    if (a.beta != 0.f) t.g -= a.beta * e.one;
  }
  return t;
}

__global__ void __launch_bounds__(kTlThreads, 5) policy_loss_kernel(const PolicyArgs a, const Sequences q) {
  __shared__ double red[4 * kTlThreads / 32];
  grid_dependency_enter();
  const Piece p = find_piece(q, blockIdx.x);
  float sum_L = 0.f, sum_K = 0.f;
  int cut = 0, count = 0;
  const bool none = p.s >= q.S;                                                   // behind the last sequence
  const float seq_adv = a.adv_by_sequence && !none ? load_token(a.adv, a.tadv, p.s) : 0.f;
  for (long long i = (p.lo & ~3LL) + 4 * threadIdx.x; i < p.hi; i += 4 * kTlThreads) {
    const bool whole = a.vec && i >= p.lo && i + 4 <= p.hi;
    float y[4], old[4], ref[4] = {0, 0, 0, 0}, A[4], g[4];
    bool valid[4];
    if (whole && !none) {
      load_tokens(a.y, a.ty, i, y);
      load_tokens(a.old, a.told, i, old);
      if (a.ref) load_tokens(a.ref, a.tref, i, ref);
      if (!a.adv_by_sequence) load_tokens(a.adv, a.tadv, i, A);
      const uint32_t m = a.mask ? *reinterpret_cast<const uint32_t*>(a.mask + i) : 0x01010101u;
#pragma unroll
      for (int j = 0; j < 4; ++j) valid[j] = (m >> (8 * j) & 255) != 0;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        valid[j] = !none && i + j >= p.lo && i + j < p.hi && (!a.mask || a.mask[i + j] != 0);
        y[j] = old[j] = A[j] = 0.f;
        if (!valid[j]) continue;
        y[j] = load_token(a.y, a.ty, i + j);
        old[j] = load_token(a.old, a.told, i + j);
        if (a.ref) ref[j] = load_token(a.ref, a.tref, i + j);
        if (!a.adv_by_sequence) A[j] = load_token(a.adv, a.tadv, i + j);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = 0.f;
      if (!valid[j]) continue;
      const TokenTerms t = policy_token(a, y[j], old[j], ref[j], a.adv_by_sequence ? seq_adv : A[j]);
      sum_L += t.L;
      sum_K += t.K;
      cut += t.cut;
      ++count;
      g[j] = t.g;
    }
    if (a.grad) {
      if (whole) store_tokens(a.grad, kTokF32, i, g);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j >= p.lo && i + j < p.hi) a.grad[i + j] = g[j];
    }
  }
  double sums[2] = {sum_L, sum_K};
  warp_sums(sums);
  cut = __reduce_add_sync(0xffffffffu, cut);
  count = __reduce_add_sync(0xffffffffu, count);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    red[4 * warp] = sums[0];
    red[4 * warp + 1] = sums[1];
    red[4 * warp + 2] = cut;
    red[4 * warp + 3] = count;
  }
  __syncthreads();
  if (threadIdx.x < 4) {
    double v = 0;
#pragma unroll
    for (int w = 0; w < kTlThreads / 32; ++w) v += red[4 * w + threadIdx.x];
    a.partial[4 * (long long)blockIdx.x + threadIdx.x] = v;
  }
}

// The sums of a sequence's pieces, by 8 or 32 neighbouring lanes, in all of them.  Whole warps call it; `s` may lie behind the last sequence.
template <int N>
__device__ __forceinline__ void sequence_sums(const Sequences& q, int s, int lanes, const double* partial, double (&v)[N]) {
  long long unit = 0, pieces = 0;
  if (s < q.S) {
    const long long lo = q.first(s), hi = q.end(s);
    unit = q.unit(s);
    pieces = hi > lo ? (hi - lo + kTlPiece - 1) / kTlPiece : 0;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0;
  for (long long p = threadIdx.x & (lanes - 1); p < pieces; p += lanes)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += partial[N * (unit + p) + k];
#pragma unroll
  for (int k = 0; k < N; ++k)
    for (int o = lanes / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}
// A warp to a sequence while the block's warps suffice, else 8 lanes.  2 sequences of 98 pieces: 12 us by warps, 16 by 8 lanes; 2000 of one
// piece: 98 by warps, 35 by 8 lanes (policy loss with its first kernel).
__device__ __forceinline__ int sequence_lanes(const Sequences& q) { return q.S <= 32 ? 32 : 8; }

__global__ void __launch_bounds__(1024) policy_finish_kernel(const PolicyArgs a, const Sequences q, long long units) {
  __shared__ double red[4 * 32];
  grid_dependency_enter();
  double sums[4] = {0, 0, 0, 0};
  if (!a.by_sequence) {
    for (long long u = threadIdx.x; u < units; u += blockDim.x)
#pragma unroll
      for (int k = 0; k < 4; ++k) sums[k] += a.partial[4 * u + k];
    block_sums(sums, red);
  } else {
    const int lanes = sequence_lanes(q);
    for (int s0 = 0; s0 < q.S; s0 += blockDim.x / lanes) {
      const int s = s0 + threadIdx.x / lanes;
      double v[4];
      sequence_sums(q, s, lanes, a.partial, v);
      if ((threadIdx.x & (lanes - 1)) == 0 && s < q.S) {
        const double by = v[3] > 0 ? 1 / v[3] : 0;
#pragma unroll
        for (int k = 0; k < 3; ++k) sums[k] += v[k] * by;
        sums[3] += v[3] > 0;
        a.inv[s] = (float)by;
      }
    }
    block_sums(sums, red);                                                        // (a barrier: all normalisers are written)
  }
  const double by = sums[3] > 0 ? 1 / sums[3] : 0;
  if (a.by_sequence)
    for (int s = threadIdx.x; s < q.S; s += blockDim.x) a.inv[s] = (float)(a.inv[s] * by);
  if (threadIdx.x == 0) {
    if (!a.by_sequence) a.inv[0] = (float)by;
    const double L = sums[0] * by, K = sums[1] * by;
    *a.loss = (float)(a.beta != 0.f ? L + (double)a.beta * K : L);
    a.stats[0] = (float)L;
    a.stats[1] = (float)K;
    a.stats[2] = (float)(sums[2] * by);
  }
}

// dy = grad * normaliser * (incoming gradient)
__global__ void __launch_bounds__(kTlThreads)
policy_grad_kernel(const float* grad, const float* inv, const float* dloss, void* dy, int type, int by_sequence, int vec, const Sequences q) {
  grid_dependency_enter();
  const Piece p = find_piece(q, blockIdx.x);
  const float by = p.s < q.S ? *dloss * inv[by_sequence ? p.s : 0] : 0.f;
  for (long long i = (p.lo & ~3LL) + 4 * threadIdx.x; i < p.hi; i += 4 * kTlThreads) {
    float g[4];
    if (vec && i >= p.lo && i + 4 <= p.hi) {
      load_tokens(grad, kTokF32, i, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = g[j] == 0.f ? 0.f : g[j] * by;
      store_tokens(dy, type, i, g);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j >= p.lo && i + j < p.hi) store_token(dy, type, i + j, grad[i + j] == 0.f ? 0.f : grad[i + j] * by);
  }
}

struct PreferenceArgs {
  const void *y, *ref;
  const uint8_t* mask;
  int ty, tref, vec;
  float beta, smoothing;
  double* partial;             // [units]
  float* coef;                 // [S] d(loss) / dy of the valid tokens of a sequence
  float* rewards;              // [S]
  float* loss;
};

__global__ void __launch_bounds__(kTlThreads) preference_loss_kernel(const PreferenceArgs a, const Sequences q) {
  __shared__ double red[kTlThreads / 32];
  grid_dependency_enter();
  const Piece p = find_piece(q, blockIdx.x);
  double sums[1] = {0};
  if (p.s < q.S) {
    for (long long i = (p.lo & ~3LL) + 4 * threadIdx.x; i < p.hi; i += 4 * kTlThreads) {
      float y[4], ref[4] = {0, 0, 0, 0};
      if (a.vec && i >= p.lo && i + 4 <= p.hi) {
        load_tokens(a.y, a.ty, i, y);
        if (a.ref) load_tokens(a.ref, a.tref, i, ref);
        const uint32_t m = a.mask ? *reinterpret_cast<const uint32_t*>(a.mask + i) : 0x01010101u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((m >> (8 * j) & 255) != 0) sums[0] += (double)y[j] - (double)ref[j];
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j >= p.lo && i + j < p.hi && (!a.mask || a.mask[i + j] != 0))
          sums[0] += (double)load_token(a.y, a.ty, i + j) - (a.ref ? (double)load_token(a.ref, a.tref, i + j) : 0);
    }
  }
  block_sums(sums, red);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sums[0];
}

// First the sums of as many sequences as there are threads, then a pair to a thread.
__global__ void __launch_bounds__(1024) preference_finish_kernel(const PreferenceArgs a, const Sequences q) {
  __shared__ double red[32];
  __shared__ double sum_of[1024];
  grid_dependency_enter();
  const int lanes = sequence_lanes(q);
  double loss[1] = {0};
  for (int s0 = 0; s0 < q.S; s0 += 1024) {
    const int first_of_warp = (threadIdx.x & ~31) / lanes;
    for (int i0 = 0; i0 < 1024 && s0 + i0 + first_of_warp < q.S; i0 += 1024 / lanes) {               // (the same for a whole warp)
      const int i = i0 + threadIdx.x / lanes;
      double v[1];
      sequence_sums(q, s0 + i, lanes, a.partial, v);
      if ((threadIdx.x & (lanes - 1)) == 0) sum_of[i] = v[0];
    }
    __syncthreads();
    const int s = s0 + 2 * threadIdx.x;
    if (threadIdx.x < 512 && s < q.S) {
      const double better = sum_of[2 * threadIdx.x], worse = sum_of[2 * threadIdx.x + 1], z = (double)a.beta * (better - worse);
      const double even = 1 - (double)a.smoothing, one = fmax(-z, 0.0), other = fmax(z, 0.0);       // (a weight of zero takes no infinity)
      loss[0] += isnan(z) ? z : log1p(exp(-fabs(z))) + (even > 0 ? even * one : 0) + (a.smoothing > 0.f ? (double)a.smoothing * other : 0);
      const double dz = ((double)a.smoothing - 1 / (1 + exp(z))) * (double)a.beta / (q.S / 2);
      a.coef[s] = (float)dz;
      a.coef[s + 1] = (float)-dz;
      a.rewards[s] = (float)((double)a.beta * better);
      a.rewards[s + 1] = (float)((double)a.beta * worse);
    }
    __syncthreads();
  }
  block_sums(loss, red);
  if (threadIdx.x == 0) *a.loss = (float)(q.S > 0 ? loss[0] / (q.S / 2) : 0);
}

__global__ void __launch_bounds__(kTlThreads)
preference_grad_kernel(const uint8_t* mask, const float* coef, const float* dloss, void* dy, int type, int vec, const Sequences q) {
  grid_dependency_enter();
  const Piece p = find_piece(q, blockIdx.x);
  const float v = p.s < q.S ? coef[p.s] * *dloss : 0.f;
  const bool none = p.s >= q.S;
  for (long long i = (p.lo & ~3LL) + 4 * threadIdx.x; i < p.hi; i += 4 * kTlThreads) {
    if (vec && i >= p.lo && i + 4 <= p.hi) {
      const uint32_t m = none ? 0 : mask ? *reinterpret_cast<const uint32_t*>(mask + i) : 0x01010101u;
      const float g[4] = {(m & 0xff) ? v : 0.f, (m & 0xff00) ? v : 0.f, (m & 0xff0000) ? v : 0.f, (m & 0xff000000u) ? v : 0.f};
      store_tokens(dy, type, i, g);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j >= p.lo && i + j < p.hi) store_token(dy, type, i + j, !none && (!mask || mask[i + j] != 0) ? v : 0.f);
  }
}

static bool aligned_for(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type == kTokF32 ? 15 : 7)) == 0; }
static bool type_ok(int t) { return t >= kTokF32 && t <= kTokF16; }
static long long unit_count(long long n, int S) { return n / kTlPiece + S + 1; }

}  // namespace ksa

using namespace ksa;
#define ST(s) reinterpret_cast<cudaStream_t>(s)

#define KSA_SEQUENCES(name)                                                                                                    \
  KSA_REQUIRE(n >= 0 && sequences >= 0 && length >= 0, name ": %lld tokens, %d sequences", n, sequences);                         \
  KSA_REQUIRE(cu != nullptr || length * sequences <= n, name ": %d rows of %lld tokens in %lld", sequences, length, n);           \
  KSA_REQUIRE(unit_count(n, sequences) <= 0x7ffff000LL, name ": too many tokens for one call"); /* (steps of 1024 stay in 32 bits) */ \
  const Sequences q{cu, wide, sequences, n, length};                                                                             \
  const unsigned units = (unsigned)unit_count(n, sequences)

// fp64 values of workspace: 4 for each (policy), 1 for each (preference)
KSA_API long long ksa_token_loss_units(long long n, int sequences) { return unit_count(n, sequences); }

// types: of y, old, ref and adv, four bits each from the lowest.  adv: a value for every token or (adv_by_sequence) sequence.  ref, mask, cu
// and grad may be null.  bounds: four fp64 values on the host, log(1 + high), log(1 - low), 1 + high, 1 - low.  partial: fp64 [4 units];
// inv: fp32 [max(S, 1)]; loss: fp32; stats: fp32 [3], see PolicyArgs.
KSA_API int ksa_policy_loss(const void* y, const void* old, const void* ref, const void* adv, const void* mask, const void* cu, int wide, void* grad,
                            void* partial, void* inv, void* loss, void* stats, int types, long long n, int sequences, long long length, int adv_by_sequence,
                            int by_sequence, const void* bounds, float beta, void* stream) {
  KSA_ENTER(loss);
  KSA_SEQUENCES("policy_loss");
  PolicyArgs a{};
  a.y = y; a.old = old; a.ref = ref; a.adv = adv; a.mask = static_cast<const uint8_t*>(mask);
  a.ty = types & 15; a.told = types >> 4 & 15; a.tref = types >> 8 & 15; a.tadv = types >> 12 & 15;
  KSA_REQUIRE(type_ok(a.ty) && type_ok(a.told) && type_ok(a.tref) && type_ok(a.tadv), "policy_loss: types %x", types);
  a.adv_by_sequence = adv_by_sequence; a.by_sequence = by_sequence;
  a.vec = aligned_for(y, a.ty) && aligned_for(old, a.told) && (!ref || aligned_for(ref, a.tref)) && (adv_by_sequence || aligned_for(adv, a.tadv)) &&
          (reinterpret_cast<uintptr_t>(mask) & 3) == 0 && aligned_for(grad, kTokF32);
  const double* b = static_cast<const double*>(bounds);
  a.above = b[0]; a.below = b[1]; a.most = (float)b[2]; a.least = (float)b[3];
  a.above32 = (float)a.above; a.below32 = (float)a.below;
  a.beta = beta; a.grad = static_cast<float*>(grad); a.partial = static_cast<double*>(partial);
  a.inv = static_cast<float*>(inv); a.loss = static_cast<float*>(loss); a.stats = static_cast<float*>(stats);
  KSA_CHECK_CUDA(launch_stream_kernel(21LL * n, policy_loss_kernel, dim3(units), dim3(kTlThreads), 0, ST(stream), a, q));
  KSA_CHECK_CUDA(launch_kernel(policy_finish_kernel, dim3(1), dim3(1024), 0, ST(stream), a, q, (long long)units));
  return 0;
}

// dy [n] (type) from what ksa_policy_loss left in grad and inv.
KSA_API int ksa_policy_loss_bwd(const void* grad, const void* inv, const void* dloss, void* dy, int type, const void* cu, int wide, long long n,
                                int sequences, long long length, int by_sequence, void* stream) {
  KSA_ENTER(dy);
  KSA_SEQUENCES("policy_loss");
  KSA_REQUIRE(type_ok(type), "policy_loss: type %d", type);
  const int vec = aligned_for(grad, kTokF32) && aligned_for(dy, type);
  const Sequences all{nullptr, 0, 1, n, n};                                       // (one normaliser: nothing to look up)
  KSA_CHECK_CUDA(launch_stream_kernel(8LL * n, policy_grad_kernel, dim3(by_sequence ? units : (unsigned)unit_count(n, 1)), dim3(kTlThreads), 0, ST(stream),
                                      (const float*)grad, (const float*)inv, (const float*)dloss, dy, type, by_sequence, vec, by_sequence ? q : all));
  return 0;
}

// types: of y and ref.  ref, mask and cu may be null.  partial: fp64 [units]; coef and rewards: fp32 [S]; loss: fp32.
KSA_API int ksa_preference_loss(const void* y, const void* ref, const void* mask, const void* cu, int wide, void* partial, void* coef, void* rewards,
                                void* loss, int types, long long n, int sequences, long long length, float beta, float smoothing, void* stream) {
  KSA_ENTER(loss);
  KSA_SEQUENCES("preference_loss");
  KSA_REQUIRE(sequences % 2 == 0, "preference_loss: %d sequences are not pairs", sequences);
  PreferenceArgs a{};
  a.y = y; a.ref = ref; a.mask = static_cast<const uint8_t*>(mask);
  a.ty = types & 15; a.tref = types >> 4 & 15;
  KSA_REQUIRE(type_ok(a.ty) && type_ok(a.tref), "preference_loss: types %x", types);
  a.vec = aligned_for(y, a.ty) && (!ref || aligned_for(ref, a.tref)) && (reinterpret_cast<uintptr_t>(mask) & 3) == 0;
  a.beta = beta; a.smoothing = smoothing;
  a.partial = static_cast<double*>(partial); a.coef = static_cast<float*>(coef); a.rewards = static_cast<float*>(rewards);
  a.loss = static_cast<float*>(loss);
  KSA_CHECK_CUDA(launch_stream_kernel(9LL * n, preference_loss_kernel, dim3(units), dim3(kTlThreads), 0, ST(stream), a, q));
  KSA_CHECK_CUDA(launch_kernel(preference_finish_kernel, dim3(1), dim3(1024), 0, ST(stream), a, q));
  return 0;
}

KSA_API int ksa_preference_loss_bwd(const void* mask, const void* coef, const void* dloss, void* dy, int type, const void* cu, int wide, long long n,
                                    int sequences, long long length, void* stream) {
  KSA_ENTER(dy);
  KSA_SEQUENCES("preference_loss");
  KSA_REQUIRE(type_ok(type), "preference_loss: type %d", type);
  const int vec = aligned_for(dy, type) && (reinterpret_cast<uintptr_t>(mask) & 3) == 0;
  KSA_CHECK_CUDA(launch_stream_kernel(5LL * n, preference_grad_kernel, dim3(units), dim3(kTlThreads), 0, ST(stream), (const uint8_t*)mask,
                                      (const float*)coef, (const float*)dloss, dy, type, vec, q));
  return 0;
}
