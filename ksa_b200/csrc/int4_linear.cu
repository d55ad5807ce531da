// Products of a few rows with weights of four bits: C[M, N] = A[M, K] * W[N, K]^T, M <= 16, W as int4.cuh says.
//
// What bounds it is reading the codes and scales once (N * K * (1/2 + 4 / group) bytes).  One CTA per SM owns the same number of weight rows
// (+-1); its warps share K in segments of 128 and keep their sums to themselves until the end of up to 64 rows, where they meet in shared memory.
// mma.sync m16n8k16 takes the activations as its 16 rows (weights in eights, so that a CTA's share of rows need not be a multiple of 16); a
// lane's 16 bytes of a weight row are values 32 t .. 32 t + 31 of the segment, in that order for the activations as well.
#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4LWarps = 16;
constexpr int kI4LThreads = kI4LWarps * 32;
constexpr int kI4LOctets = 6;      // eights of weight rows of a pass

struct Int4Linear {
  const bf16* A;
  const uint8_t* W;                // [N, K / 2]
  const uint32_t* meta;            // [K / group, pitch]
  bf16* C;
  long long lda, ldc;
  int M, N, K, group, pitch, rows; // rows of a CTA
  int early;                       // the weights are read ahead of the wait
};

// NB: activation rows in eights (1 or 2)
template <int NB>
__global__ void __launch_bounds__(kI4LThreads) int4_linear_kernel(const Int4Linear a) {
  extern __shared__ float part[];                    // [warps][NB * 8][octets * 8 + 4]
  constexpr int kPitch = kI4LOctets * 8 + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * a.rows, r1 = min(a.N, r0 + a.rows);
  const int segments = (a.K + 127) / 128;
  grid_dependency_launch();
  if (!a.early) grid_dependency_wait();
  bool waited = !a.early;
  for (int base = r0; base < r1; base += kI4LOctets * 8) {
    const int octets = min(kI4LOctets, (r1 - base + 7) / 8);
    float acc[kI4LOctets][4];
#pragma unroll
    for (int i = 0; i < kI4LOctets; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    for (int seg = warp; seg < segments; seg += kI4LWarps) {
      const int col = seg * 128 + t * 32;
      const bool in = col < a.K;
      uint4 w[kI4LOctets];
      uint32_t m[kI4LOctets];
#pragma unroll
      for (int i = 0; i < kI4LOctets; ++i) {
        w[i] = make_uint4(0, 0, 0, 0);
        m[i] = 0;
        const int row = base + i * 8 + g;
        if (i < octets && row < r1 && in) {
          w[i] = *reinterpret_cast<const uint4*>(a.W + (long long)row * (a.K / 2) + col / 2);
          m[i] = a.meta[(long long)(col / a.group) * a.pitch + row];
        }
      }
      if (!waited) { grid_dependency_wait(); waited = true; }
      uint4 x[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[n][q] = make_uint4(0, 0, 0, 0);
          if (n * 8 + g < a.M && in) x[n][q] = *reinterpret_cast<const uint4*>(a.A + (n * 8 + g) * a.lda + col + q * 8);
        }
#pragma unroll
      for (int i = 0; i < kI4LOctets; ++i) {
        if (i >= octets) break;
        const uint32_t s2 = i4_scale2(m[i]), o2 = i4_offset2(m[i]);
        const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t v[4];
          i4_values(v, words[q], s2, o2);
          const uint4 xa = x[0][q], xb = NB == 2 ? x[NB - 1][q] : make_uint4(0, 0, 0, 0);
          mma_bf16(acc[i], xa.x, xb.x, xa.y, xb.y, v[0], v[1]);
          mma_bf16(acc[i], xa.z, xb.z, xa.w, xb.w, v[2], v[3]);
        }
      }
    }
    if (!waited) { grid_dependency_wait(); waited = true; }
    // ---- the warps' sums: acc[i] = (row g, weights 2 t, 2 t + 1), (row g + 8, the same)
#pragma unroll
    for (int i = 0; i < kI4LOctets; ++i) {
      if (i >= octets) break;
      float* dst = part + (warp * NB * 8 + g) * kPitch + i * 8 + t * 2;
      *reinterpret_cast<float2*>(dst) = make_float2(acc[i][0], acc[i][1]);
      if (NB == 2) *reinterpret_cast<float2*>(dst + 8 * kPitch) = make_float2(acc[i][2], acc[i][3]);
    }
    __syncthreads();
    const int n = min(kI4LOctets * 8, r1 - base);
    for (int i = threadIdx.x; i < a.M * n; i += kI4LThreads) {
      const int row = i / n, c = i - row * n;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kI4LWarps; ++w) s += part[(w * NB * 8 + row) * kPitch + c];
      a.C[row * a.ldc + base + c] = __float2bfloat16(s);
    }
    __syncthreads();
  }
}

}  // namespace ksa

using namespace ksa;

// A [M <= 16, K] (row pitch lda), codes [N, K / 2], scales [K / group, pitch] words -> C [M, N] (row pitch ldc).
KSA_API int ksa_int4_linear(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda,
                            long long ldc, void* stream) {
  KSA_ENTER(A);
  KSA_REQUIRE(M >= 0 && M <= 16, "int4_linear: %d rows (at most 16)", M);
  KSA_REQUIRE(group == 32 || group == 64 || group == 128, "int4_linear: groups of %d values (32, 64 or 128)", group);
  KSA_REQUIRE(K > 0 && K % group == 0 && N >= 0 && pitch >= N, "int4_linear: K %d is no multiple of the group of %d", K, group);
  KSA_REQUIRE(lda % 8 == 0 && ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(codes)) & 15) == 0 &&
                  (reinterpret_cast<uintptr_t>(meta) & 3) == 0, "int4_linear: rows and codes must be 16-byte aligned");
  if (M == 0 || N == 0) return 0;
  const int sms = sm_count(), rows = (N + sms - 1) / sms;
  Int4Linear a{(const bf16*)A, (const uint8_t*)codes, (const uint32_t*)meta, (bf16*)C, lda, ldc, M, N, K, group, pitch, rows, weights_early()};
  const dim3 grid((N + rows - 1) / rows);
  const size_t smem = (size_t)kI4LWarps * (M > 8 ? 16 : 8) * (kI4LOctets * 8 + 4) * sizeof(float);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (M > 8) {
    static PerDevice raised;
    KSA_CHECK_CUDA(raise_smem_limit(raised, int4_linear_kernel<2>, smem));
    KSA_CHECK_CUDA(launch_kernel(int4_linear_kernel<2>, grid, dim3(kI4LThreads), smem, st, a));
  } else {
    static PerDevice raised;
    KSA_CHECK_CUDA(raise_smem_limit(raised, int4_linear_kernel<1>, smem));
    KSA_CHECK_CUDA(launch_kernel(int4_linear_kernel<1>, grid, dim3(kI4LThreads), smem, st, a));
  }
  return 0;
}
