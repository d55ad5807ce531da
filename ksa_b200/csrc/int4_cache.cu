// Quantising keys and values as they enter a KV cache of four bits, reading them back, and the same for weights.
//
// A thread takes eight values of a row (16 bytes), and the four threads of a group of 32 find its range with two shuffles: one read of the new
// rows, one write of codes and scales, nothing kept between.  Rows of a step are a few kilobytes and cost a launch; rows of a prompt are
// bound by the memory: 2 bytes a value read, 0.625 written.
#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4Threads = 256;
constexpr int kI4Scan = 64;      // rows of a sequence up to which a row looks through the slots behind its own

struct Int4Write {
  const bf16 *k, *v;             // [B, T, H, D], rows of a head contiguous
  uint8_t *k_codes, *v_codes;    // [B, H, cap, D / 2]
  uint32_t *k_meta, *v_meta;     // [B, H, cap, D / 32]
  const int* slots;              // [B, T]
  const int* last;               // [B, cap]: the last row of each slot, or null
  long long sb, st, sh;          // strides of k and v in elements
  int B, T, H, D, cap, scan;     // scan: look for later rows of the same slot
};

// last[b, slot] = the greatest t with that slot
__global__ void __launch_bounds__(kI4Threads) int4_last_row_kernel(const int* slots, int* last, int B, int T, int cap) {
  grid_dependency_enter();
  const long long i = (long long)blockIdx.x * kI4Threads + threadIdx.x;
  if (i >= (long long)B * T) return;
  const int slot = slots[i];
  if (slot >= 0 && slot < cap) atomicMax(last + i / T * cap + slot, (int)(i % T));
}

__global__ void __launch_bounds__(kI4Threads) int4_cache_write_kernel(Int4Write a) {
  grid_dependency_enter();
  const int per = a.D / 8;
  const long long n = (long long)a.B * a.T * a.H * per * 2, i = (long long)blockIdx.x * kI4Threads + threadIdx.x;
  // lanes of a group stay together to the end: `per` is a multiple of four
  const long long j = i < n ? i : n - 1;
  const int c = (int)(j % per), h = (int)(j / per % a.H), kv = (int)(j / per / a.H % 2);
  const long long row = j / per / a.H / 2;
  const int t = (int)(row % a.T), b = (int)(row / a.T);
  const int slot = a.slots[row];
  bool keep = i < n && slot >= 0 && slot < a.cap;
  if (keep && a.last != nullptr) keep = a.last[(long long)b * a.cap + slot] == t;
  if (keep && a.scan)
    for (int later = t + 1; later < a.T; ++later) keep &= a.slots[row - t + later] != slot;
  const uint4 raw = *reinterpret_cast<const uint4*>((kv ? a.v : a.k) + b * a.sb + t * a.st + h * a.sh + c * 8);
  uint32_t word, meta;
  i4_quantize<kI4CacheGroup / 8>(raw, word, meta);
  if (!keep) return;
  const long long at = ((long long)b * a.H + h) * a.cap + slot;
  reinterpret_cast<uint32_t*>(kv ? a.v_codes : a.k_codes)[at * per + c] = word;
  if (c % 4 == 0) (kv ? a.v_meta : a.k_meta)[at * (per / 4) + c / 4] = meta;
}

struct Int4Read {
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_meta, *v_meta;
  const int* start;              // [B]
  bf16 *k, *v;                   // [B, H, rows, D]
  int B, H, D, cap, rows;
};

__global__ void __launch_bounds__(kI4Threads) int4_cache_read_kernel(Int4Read a) {
  grid_dependency_enter();
  const int per = a.D / 8;
  const long long n = (long long)a.B * a.H * a.rows * per, i = (long long)blockIdx.x * kI4Threads + threadIdx.x;
  if (i >= 2 * n) return;
  const bool kv = i >= n;
  const long long j = kv ? i - n : i;
  const int c = (int)(j % per), r = (int)(j / per % a.rows);
  const long long bh = j / per / a.rows;
  const long long slot = (long long)a.start[bh / a.H] + r;
  uint32_t o[4] = {0, 0, 0, 0};
  if (slot >= 0 && slot < a.cap) {
    const long long at = bh * a.cap + slot;
    const uint32_t word = reinterpret_cast<const uint32_t*>(kv ? a.v_codes : a.k_codes)[at * per + c];
    const uint32_t meta = (kv ? a.v_meta : a.k_meta)[at * (per / 4) + c / 4];
    i4_values(o, word, i4_scale2(meta), i4_offset2(meta));
  }
  *reinterpret_cast<uint4*>((kv ? a.v : a.k) + j * 8) = make_uint4(o[0], o[1], o[2], o[3]);
}

// Weights: rows [N, K] (row pitch `ld`) -> codes [N, K / 2], scales [K / group, pitch] words; a row's groups of kLanes * 8 values.
template <int kLanes>
__global__ void __launch_bounds__(kI4Threads) int4_weight_kernel(const bf16* w, uint32_t* codes, uint32_t* meta, int N, int K, long long ld,
                                                                 int pitch) {
  grid_dependency_enter();
  const int per = K / 8;
  const long long n = (long long)N * per, i = (long long)blockIdx.x * kI4Threads + threadIdx.x, j = i < n ? i : n - 1;
  const int c = (int)(j % per);
  const long long row = j / per;
  const uint4 raw = *reinterpret_cast<const uint4*>(w + row * ld + c * 8);
  uint32_t word, m;
  i4_quantize<kLanes>(raw, word, m);
  if (i >= n) return;
  codes[j] = word;
  if (c % kLanes == 0) meta[(long long)(c / kLanes) * pitch + row] = m;
}

__global__ void __launch_bounds__(kI4Threads) int4_weight_values_kernel(const uint32_t* codes, const uint32_t* meta, bf16* w, int N, int K,
                                                                        int group, int pitch) {
  grid_dependency_enter();
  const int per = K / 8;
  const long long i = (long long)blockIdx.x * kI4Threads + threadIdx.x;
  if (i >= (long long)N * per) return;
  const int c = (int)(i % per);
  const uint32_t m = meta[(long long)(c * 8 / group) * pitch + i / per];
  uint32_t o[4];
  i4_values(o, codes[i], i4_scale2(m), i4_offset2(m));
  *reinterpret_cast<uint4*>(w + i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
}

static bool misaligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace ksa

using namespace ksa;

// k, v: [B, T, H, D] rows with strides (sb, st, sh) in elements.  Rows whose slot is negative or past the cache are not written; of several
// rows with one slot the last stays: `last` is a workspace [B, cap] int32 for that, or null where T is at most 64 (rows look at
// the slots behind theirs) or `distinct` says that no slot occurs twice.
KSA_API int ksa_int4_cache_write(const void* k, const void* v, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* slots,
                                 void* last, int B, int T, int H, int D, int cap, long long sb, long long st, long long sh, int distinct,
                                 void* stream) {
  KSA_ENTER(k);
  KSA_REQUIRE(D > 0 && D % kI4CacheGroup == 0, "int4_cache_write: head_dim %d is no multiple of %d", D, kI4CacheGroup);
  KSA_REQUIRE(B >= 0 && T >= 0 && H > 0 && cap > 0, "int4_cache_write: bad shape");
  KSA_REQUIRE(sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0 && !misaligned(k, 16) && !misaligned(v, 16),
              "int4_cache_write: rows must be 16-byte aligned");
  KSA_REQUIRE(!misaligned(k_codes, 4) && !misaligned(v_codes, 4) && !misaligned(k_meta, 4) && !misaligned(v_meta, 4),
              "int4_cache_write: cache tensors must be 4-byte aligned");
  KSA_REQUIRE(distinct || T <= kI4Scan || last != nullptr, "int4_cache_write: %d rows need the workspace of last rows", T);
  const long long n = (long long)B * T * H * (D / 8) * 2;
  if (n == 0) return 0;
  KSA_REQUIRE((n + kI4Threads - 1) / kI4Threads < (1LL << 31), "int4_cache_write: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool table = !distinct && T > kI4Scan;
  if (table) {
    KSA_CHECK_CUDA(cudaMemsetAsync(last, 0xFF, (size_t)B * cap * sizeof(int), s));
    KSA_CHECK_CUDA(launch_kernel(int4_last_row_kernel, dim3((unsigned)(((long long)B * T + kI4Threads - 1) / kI4Threads)), dim3(kI4Threads), 0, s,
                                 (const int*)slots, (int*)last, B, T, cap));
  }
  Int4Write a{(const bf16*)k, (const bf16*)v, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_meta, (uint32_t*)v_meta, (const int*)slots,
              table ? (const int*)last : nullptr, sb, st, sh, B, T, H, D, cap, !distinct && !table && T > 1};
  KSA_CHECK_CUDA(launch_stream_kernel(n * 21, int4_cache_write_kernel, dim3((unsigned)((n + kI4Threads - 1) / kI4Threads)), dim3(kI4Threads), 0, s, a));
  return 0;
}

// Slots [start[b], start[b] + rows) of every sequence -> k, v [B, H, rows, D] (zeros outside the cache).
KSA_API int ksa_int4_cache_read(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const void* start, void* k,
                                void* v, int B, int H, int D, int cap, int rows, void* stream) {
  KSA_ENTER(k);
  KSA_REQUIRE(D > 0 && D % kI4CacheGroup == 0, "int4_cache_read: head_dim %d is no multiple of %d", D, kI4CacheGroup);
  KSA_REQUIRE(B >= 0 && rows >= 0 && H > 0 && cap > 0, "int4_cache_read: bad shape");
  const long long n = (long long)B * H * rows * (D / 8) * 2;
  if (n == 0) return 0;
  KSA_REQUIRE((n + kI4Threads - 1) / kI4Threads < (1LL << 31), "int4_cache_read: too many rows");
  Int4Read a{(const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint32_t*)k_meta, (const uint32_t*)v_meta, (const int*)start, (bf16*)k,
             (bf16*)v, B, H, D, cap, rows};
  KSA_CHECK_CUDA(launch_stream_kernel(n * 21, int4_cache_read_kernel, dim3((unsigned)((n + kI4Threads - 1) / kI4Threads)), dim3(kI4Threads), 0,
                                      reinterpret_cast<cudaStream_t>(stream), a));
  return 0;
}

// w [N, K] bf16 (row pitch ld) -> codes [N, K / 2], scales [K / group, pitch] words.
KSA_API int ksa_int4_weight(const void* w, void* codes, void* meta, int N, int K, int group, long long ld, int pitch, void* stream) {
  KSA_ENTER(w);
  KSA_REQUIRE(group == 32 || group == 64 || group == 128, "int4_weight: groups of %d values (32, 64 or 128)", group);
  KSA_REQUIRE(K > 0 && K % group == 0 && N >= 0 && pitch >= N, "int4_weight: K %d is no multiple of the group of %d", K, group);
  KSA_REQUIRE(ld % 8 == 0 && !misaligned(w, 16), "int4_weight: rows must be 16-byte aligned");
  const long long n = (long long)N * (K / 8);
  if (n == 0) return 0;
  const dim3 grid((unsigned)((n + kI4Threads - 1) / kI4Threads));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto kern = group == 32 ? int4_weight_kernel<4> : group == 64 ? int4_weight_kernel<8> : int4_weight_kernel<16>;
  KSA_CHECK_CUDA(launch_stream_kernel(n * 21, kern, grid, dim3(kI4Threads), 0, s, (const bf16*)w, (uint32_t*)codes, (uint32_t*)meta, N, K, ld, pitch));
  return 0;
}

KSA_API int ksa_int4_weight_values(const void* codes, const void* meta, void* w, int N, int K, int group, int pitch, void* stream) {
  KSA_ENTER(codes);
  KSA_REQUIRE(group == 32 || group == 64 || group == 128, "int4_weight_values: groups of %d values (32, 64 or 128)", group);
  KSA_REQUIRE(K > 0 && K % group == 0 && N >= 0 && pitch >= N, "int4_weight_values: K %d is no multiple of the group of %d", K, group);
  const long long n = (long long)N * (K / 8);
  if (n == 0) return 0;
  KSA_CHECK_CUDA(launch_stream_kernel(n * 21, int4_weight_values_kernel, dim3((unsigned)((n + kI4Threads - 1) / kI4Threads)), dim3(kI4Threads), 0,
                                      reinterpret_cast<cudaStream_t>(stream), (const uint32_t*)codes, (const uint32_t*)meta, (bf16*)w, N, K, group,
                                      pitch));
  return 0;
}
