// Global 2-norm of many gradient tensors, and clipping by it:  norm = scale * sqrt(sum g^2),  factor = scale * min(1, most / (norm + 1e-6)),
// clipped = g * factor.
//
// Bound: memory.  The norm reads every value once; clipping reads it again and writes it, unless the factor is one and the values stay
// where they are.  All tensors of a call are one list of chunks of 32 KB, counted from the 16-byte boundary at or below a tensor's first
// value, so that tensors of any address are read in whole 16-byte vectors but for their two ends; a table of the tensors comes with the
// launch (nothing to copy to the device, and a captured launch keeps its own).
//
// Sums: squares of a thread's part of a chunk (32 values of four bytes, 64 of two) are summed in 32 bits, everything above that in 64 and in
// a fixed order.  Where the 32-bit sum leaves 2^-80 .. 2^100 with a value that is not zero, the part is summed again in 64 bits: finite values
// give their norm wherever that is a finite fp32 number, and the sum of squares of 1e-30 is not lost.
#include "common.cuh"
#include "host.h"

#include <cuda_fp16.h>
#include <math.h>

namespace ksa {

constexpr int kGnThreads = 256;
constexpr int kGnVecs = 8;                                              // 16-byte vectors of a thread in a chunk
constexpr int kGnChunk = kGnThreads * kGnVecs * 16;
constexpr int kGnSmall = 64, kGnMost = 1000;                            // tensors of a launch: the table is a kernel parameter of at most 32764 bytes
constexpr int kGnBlocksPerSm = 6;

enum GradType : int { kGradF32 = 0, kGradBf16 = 1, kGradF16 = 2 };

template <int N>
struct GradTable {
  const void* src[N];
  void* dst[N];                                                         // clipping: where the values go
  long long n[N];                                                       // values * 4 + type
  int begin[N + 1];                                                     // first chunk of every tensor, then the number of chunks
  int tensors;
};
static_assert(sizeof(GradTable<kGnMost>) + 128 <= 32764, "kernel parameters");

struct GradChunk {
  const char* src;          // 16-byte aligned
  char* dst;                // src's counterpart, of any alignment
  long long lo, hi;         // bytes of the chunk that belong to the tensor
  int type;
};

template <int N>
__device__ __forceinline__ GradChunk grad_chunk(const GradTable<N>& t, int c) {
  int lo = 0, hi = t.tensors;                                           // the last tensor that begins at or before chunk c (empty ones begin where the next does)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.begin[mid] <= c) lo = mid; else hi = mid;
  }
  const int type = (int)(t.n[lo] & 3);
  const long long bytes = (t.n[lo] >> 2) * (type == kGradF32 ? 4 : 2), off = (long long)(c - t.begin[lo]) * kGnChunk;
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.src[lo]), skew = p & 15;
  GradChunk g;
  g.src = reinterpret_cast<const char*>(p - skew + off);
  g.dst = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(t.dst[lo]) - skew + off);
  g.lo = max((long long)skew - off, 0LL);
  g.hi = min((long long)skew + bytes - off, (long long)kGnChunk);
  g.type = type;
  return g;
}

// The 16 bytes at `at` of a chunk, with zeros outside the tensor.
__device__ __forceinline__ uint4 grad_load(const GradChunk& g, int at) {
  if (at >= g.lo && at + 16 <= g.hi) return *reinterpret_cast<const uint4*>(g.src + at);
  uint32_t w[4] = {0, 0, 0, 0};
  if (at + 16 > g.lo && at < g.hi) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int b = at + 2 * i;                                         // (tensors of four-byte values begin and end on four bytes)
      if (b >= g.lo && b + 2 <= g.hi) w[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(g.src + b) << (16 * (i & 1));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int TYPE>
__device__ __forceinline__ void grad_values(uint4 v, float (&f)[8]) {  // four values of four bytes, or eight of two
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (TYPE == kGradF32) { f[i] = __uint_as_float(u[i]); f[i + 4] = 0.f; continue; }
    const float2 t = TYPE == kGradBf16 ? unpack_bf16x2(u[i]) : __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

template <int TYPE>
__device__ __noinline__ double grad_sum_wide(const GradChunk& g) {
  double s = 0;
  for (int i = 0; i < kGnVecs; ++i) {
    float f[8];
    grad_values<TYPE>(grad_load(g, (i * kGnThreads + threadIdx.x) * 16), f);
    for (int j = 0; j < 8; ++j) s += (double)f[j] * (double)f[j];
  }
  return s;
}

// Sum of the squares of this thread's part of a chunk.
template <int TYPE>
__device__ __forceinline__ double grad_sum(const GradChunk& g) {
  uint4 v[kGnVecs];
  if (g.lo == 0 && g.hi == kGnChunk) {
#pragma unroll
    for (int i = 0; i < kGnVecs; ++i) v[i] = *reinterpret_cast<const uint4*>(g.src + (i * kGnThreads + threadIdx.x) * 16);
  } else {
#pragma unroll
    for (int i = 0; i < kGnVecs; ++i) v[i] = grad_load(g, (i * kGnThreads + threadIdx.x) * 16);
  }
  float s[2] = {0.f, 0.f};
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < kGnVecs; ++i) {
    float f[8];
    grad_values<TYPE>(v[i], f);
    any |= v[i].x | v[i].y | v[i].z | v[i].w;
#pragma unroll
    for (int j = 0; j < (TYPE == kGradF32 ? 4 : 8); ++j) s[j & 1] = fmaf(f[j], f[j], s[j & 1]);
  }
  const float sum = s[0] + s[1];
  if (sum >= 0x1p-80f && sum <= 0x1p100f) return (double)sum;
  if ((any & (TYPE == kGradF32 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0;
  return grad_sum_wide<TYPE>(g);
}

__device__ __forceinline__ double block_sum_wide(double v, double* red) {          // red: a value for every warp; the sum in all threads
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  double t = lane < warps ? red[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

template <int N>
__global__ void __launch_bounds__(kGnThreads)
grad_norm_kernel(const __grid_constant__ GradTable<N> table, double* partial) {
  __shared__ double red[32];
  grid_dependency_enter();
  double sum = 0;
  const int chunks = table.begin[table.tensors];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const GradChunk g = grad_chunk(table, c);
    sum += g.type == kGradF32 ? grad_sum<kGradF32>(g) : g.type == kGradBf16 ? grad_sum<kGradBf16>(g) : grad_sum<kGradF16>(g);
  }
  sum = block_sum_wide(sum, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

struct NormAndFactor {
  float norm, factor;
};
// Norm and factor from the blocks' sums, by a whole block.
__device__ __forceinline__ NormAndFactor grad_factor(const double* partial, int parts, float scale, float most, double* red) {
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += blockDim.x) s += partial[i];
  NormAndFactor r;
  r.norm = (float)((double)scale * sqrt(block_sum_wide(s, red)));
  const float c = most / (r.norm + 1e-6f);
  r.factor = scale * (c > 1.f ? 1.f : c);                               // (what is no number stays)
  return r;
}

__global__ void __launch_bounds__(1024) grad_factor_kernel(const double* partial, int parts, float scale, float most, float* norm, float* factor) {
  __shared__ double red[32];
  grid_dependency_enter();
  const NormAndFactor r = grad_factor(partial, parts, scale, most, red);
  if (threadIdx.x == 0) { *norm = r.norm; *factor = r.factor; }
}

template <int TYPE>
__device__ __forceinline__ void grad_clip_chunk(const GradChunk& g, float factor) {
  const bool whole = g.lo == 0 && g.hi == kGnChunk && (reinterpret_cast<uintptr_t>(g.dst) & 15) == 0;
  uint4 v[kGnVecs];
#pragma unroll
  for (int i = 0; i < kGnVecs; ++i) {
    const int at = (i * kGnThreads + threadIdx.x) * 16;
    v[i] = whole ? *reinterpret_cast<const uint4*>(g.src + at) : grad_load(g, at);
  }
#pragma unroll
  for (int i = 0; i < kGnVecs; ++i) {
    const int at = (i * kGnThreads + threadIdx.x) * 16;
    float f[8];
    grad_values<TYPE>(v[i], f);
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (TYPE == kGradF32) u[j] = __float_as_uint(f[j] * factor);
      else if (TYPE == kGradBf16) u[j] = pack_bf16x2(f[2 * j] * factor, f[2 * j + 1] * factor);
      else {
        const __half2 h = __floats2half2_rn(f[2 * j] * factor, f[2 * j + 1] * factor);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if (whole || (at >= g.lo && at + 16 <= g.hi && (reinterpret_cast<uintptr_t>(g.dst + at) & 15) == 0)) {
      *reinterpret_cast<uint4*>(g.dst + at) = make_uint4(u[0], u[1], u[2], u[3]);
    } else if (at + 16 > g.lo && at < g.hi) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int b = at + 2 * j;
        if (b >= g.lo && b + 2 <= g.hi) *reinterpret_cast<uint16_t*>(g.dst + b) = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

// The chunks from the last one on: what the norm has read last is still in the L2.
template <int N>
__global__ void __launch_bounds__(kGnThreads)
grad_clip_kernel(const __grid_constant__ GradTable<N> table, const double* partial, int parts, float scale, float most, float* norm, float* factor) {
  __shared__ double red[32];
  grid_dependency_enter();
  const NormAndFactor r = grad_factor(partial, parts, scale, most, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) { *norm = r.norm; *factor = r.factor; }
  const int chunks = table.begin[table.tensors];
  for (int c = chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const GradChunk g = grad_chunk(table, c);
    if (r.factor == 1.f && g.dst == g.src) continue;
    if (g.type == kGradF32) grad_clip_chunk<kGradF32>(g, r.factor);
    else if (g.type == kGradBf16) grad_clip_chunk<kGradBf16>(g, r.factor);
    else grad_clip_chunk<kGradF16>(g, r.factor);
  }
}

// Tensors [from, from + count) of the call into a table.  Returns the number of chunks, or -1 where there are too many.
template <int N>
static long long fill_table(GradTable<N>& t, const void* const* src, void* const* dst, const long long* meta, int count) {
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    const long long n = meta[i] >> 2, bytes = n * ((meta[i] & 3) == kGradF32 ? 4 : 2);
    t.src[i] = src[i];
    t.dst[i] = dst ? dst[i] : const_cast<void*>(src[i]);
    t.n[i] = meta[i];
    t.begin[i] = (int)chunks;
    if (n > 0) chunks += (bytes + (long long)(reinterpret_cast<uintptr_t>(src[i]) & 15) + kGnChunk - 1) / kGnChunk;
    if (chunks > (1 << 30)) return -1;
  }
  t.begin[count] = (int)chunks;
  t.tensors = count;
  return chunks;
}

template <int N>
static int grad_norm_group(const void* const* src, void* const* dst, const long long* meta, int count, double* partial, int parts, int blocks_most,
                           float scale, float most, float* norm, float* factor, int* blocks, cudaStream_t st) {
  GradTable<N> t;
  const long long chunks = fill_table(t, src, dst, meta, count);
  KSA_REQUIRE(chunks >= 0, "grad_norm: too many values for one call");
  const int grid = (int)(chunks < 1 ? 1 : chunks < blocks_most ? chunks : blocks_most);
  if (blocks) {
    *blocks = grid;
    KSA_CHECK_CUDA(launch_stream_kernel(chunks * kGnChunk, grad_norm_kernel<N>, dim3(grid), dim3(kGnThreads), 0, st, t, partial));
  } else {
    KSA_CHECK_CUDA(launch_stream_kernel(chunks * kGnChunk, grad_clip_kernel<N>, dim3(grid), dim3(kGnThreads), 0, st, t, (const double*)partial, parts,
                                        scale, most, norm, factor));
  }
  return 0;
}

}  // namespace ksa

using namespace ksa;

// Number of fp64 values of workspace that ksa_grad_norm takes for a call on `tensors` tensors.
KSA_API int ksa_grad_norm_parts(int tensors) {
  const int sms = sm_count();
  return ((tensors + kGnMost - 1) / kGnMost) * (sms > 0 ? sms : 1) * kGnBlocksPerSm;
}

// src[i]: values of tensor i (meta[i] = number * 4 + type: 0 fp32, 1 bf16, 2 fp16), each aligned to its type.  dst: null for the norm alone, else
// where the clipped values of each tensor go (src itself: in place).  norm, factor: fp32.  The arrays are host memory.
KSA_API int ksa_grad_norm(const void* src, const void* dst, const void* meta, int tensors, float scale, float most, void* partial, void* norm,
                          void* factor, void* stream) {
  KSA_ENTER(norm);
  KSA_REQUIRE(tensors >= 0, "grad_norm: %d tensors", tensors);
  KSA_REQUIRE(scale > 0.f && isfinite(scale), "grad_norm: the scale must be a positive number");
  KSA_REQUIRE(most >= 0.f, "grad_norm: the largest norm must not be negative");
  const void* const* from = static_cast<const void* const*>(src);
  void* const* to = static_cast<void* const*>(const_cast<void*>(dst));
  const long long* m = static_cast<const long long*>(meta);
  for (int i = 0; i < tensors; ++i) {
    const int type = (int)(m[i] & 3), size = type == kGradF32 ? 4 : 2;
    KSA_REQUIRE(m[i] >= 0 && type <= kGradF16, "grad_norm: tensor %d has %lld values of type %d", i, m[i] >> 2, type);
    KSA_REQUIRE((m[i] >> 2) == 0 || (reinterpret_cast<uintptr_t>(from[i]) % size == 0 && from[i] != nullptr && (!to || (to[i] != nullptr && reinterpret_cast<uintptr_t>(to[i]) % size == 0))),
                "grad_norm: tensor %d is not aligned to its type", i);
  }
  const int sms = sm_count();
  KSA_REQUIRE(sms > 0, "no device");
  const int most_blocks = sms * kGnBlocksPerSm;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  double* parts = static_cast<double*>(partial);
  int used = 0;
  for (int pass = 0; pass < (to ? 2 : 1); ++pass) {
    int i = 0;
    do {                                                                // (no tensor at all: one launch that leaves a sum of zero)
      const int count = tensors - i < kGnMost ? tensors - i : kGnMost;
      int blocks = 0;
      auto group = count <= kGnSmall ? grad_norm_group<kGnSmall> : grad_norm_group<kGnMost>;
      const int rc = group(from + i, to ? to + i : nullptr, m + i, count, pass == 0 ? parts + used : parts, used, most_blocks, scale, most,
                           static_cast<float*>(norm), static_cast<float*>(factor), pass == 0 ? &blocks : nullptr, st);
      if (rc) return rc;
      used += blocks;
      i += count;
    } while (i < tensors);
  }
  if (!to)
    KSA_CHECK_CUDA(launch_kernel(grad_factor_kernel, dim3(1), dim3(1024), 0, st, (const double*)parts, used, scale, most, static_cast<float*>(norm),
                                 static_cast<float*>(factor)));
  return 0;
}
