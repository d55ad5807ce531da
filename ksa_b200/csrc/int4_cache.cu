// Quantising keys and values as they enter a KV cache of four bits, reading them back, and the same for weights.
//
// A thread takes sixteen keys and sixteen values (32 bytes each) of a row's head, and the two threads of a group of 32 find its range with a
// shuffle: one read of the new rows, one write of codes and scales, nothing kept between.  A block takes 32 rows (at head dim 128) of
// one head, whose slots usually follow one another, and the blocks of a row's heads follow one another: whole sectors of rows that
// are open anyway.  Rows of a step are a few kilobytes and cost a launch; rows of a prompt are bound by the memory (2 bytes a value read,
// 0.625 written) and by some 15 cycles of a scheduler for every 32 values.
#include "host.h"
#include "int4.cuh"

namespace ksa {

constexpr int kI4Threads = 256;
constexpr int kI4Scan = 64;      // rows of a sequence up to which a row looks through the slots behind its own
// Up to so many rows of a sequence, slots, and rows that all blocks look at together, each block finds the last rows of its slots in shared memory; beyond
// that a kernel of its own makes a table of them in memory.  Table against this, random slots, 8 heads of 128 (and on the host 5 us less): one sequence of
// 100 rows 4.3 -> 2.7 us, 512 4.5 -> 3.1, 1024 5.3 -> 4.0, 2048 6.6 -> 6.9, 4096 8.8 -> 11.0; eight of 512 8.8 -> 8.1, of 2048 23.1 -> 30.1.
constexpr int kI4BlockRows = 2048, kI4BlockCap = 8192, kI4BlockWork = 768 << 10;

// Quotients by a size that is known at the launch, of numbers below 2^31: with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (mulhi(n, m) + n) >> l.
struct Int4Divide {
  uint32_t d, m, l;
  explicit Int4Divide(uint32_t by = 1) : d(by), l(0) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int operator()(uint32_t n) const { return (int)((__umulhi(n, m) + n) >> l); }
};

struct Int4Write {
  const bf16 *k, *v;             // [B, T, H, D], rows of a head contiguous
  uint8_t *k_codes, *v_codes;    // [B, H, cap, D / 2]
  uint32_t *k_meta, *v_meta;     // [B, H, cap, D / 32]
  const int* slots;              // [B, T]
  const int* last;               // [B, cap]: the last row of each slot, or null
  long long sb, st, sh;          // strides of k and v in elements
  int B, T, H, D, cap, scan;     // scan: look for later rows of the same slot
  int in_shared;                 // the last row of each slot is found in shared memory
  int in_block;                  // rows of a block
  Int4Divide heads_of, rows_of, chunks_of;           // by H, by T, by D / 16
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
  // lanes of a group stay together to the end: `per` is even
  const int per = a.D / 16, in_block = a.in_block, block = a.heads_of(blockIdx.x), h = blockIdx.x - block * a.H;
  const int of_block = a.chunks_of(threadIdx.x), c = threadIdx.x - of_block * per, rows = a.B * a.T;
  const int at_row = block * in_block + of_block, row = min(at_row, rows - 1);
  const int b = a.T == 1 ? row : a.rows_of(row), t = row - b * a.T;
  const int slot = a.slots[row];
  bool keep = of_block < in_block && at_row < rows && slot >= 0 && slot < a.cap;
  const long long src = b * a.sb + t * a.st + h * a.sh + c * 16;
  const uint4 k[2] = {*reinterpret_cast<const uint4*>(a.k + src), *reinterpret_cast<const uint4*>(a.k + src + 8)};
  const uint4 v[2] = {*reinterpret_cast<const uint4*>(a.v + src), *reinterpret_cast<const uint4*>(a.v + src + 8)};
  if (a.in_shared) {
    // the last of the sequence's rows from the block's first on in each of their slots; a block may hold the end of one sequence and the next ones
    extern __shared__ int last_row[];
    const int first = block * in_block, b0 = a.rows_of(first), b1 = a.rows_of(min(first + in_block, rows) - 1);
    for (int s = b0; s <= b1; ++s) {
      const int* slots = a.slots + (long long)s * a.T;
      const int from = (s == b0 ? first - b0 * a.T : 0) + threadIdx.x;
      for (int i = from; i < a.T; i += kI4Threads)
        if ((unsigned)slots[i] < (unsigned)a.cap) last_row[slots[i]] = -1;
      __syncthreads();
      for (int i = from; i < a.T; i += kI4Threads)
        if ((unsigned)slots[i] < (unsigned)a.cap) atomicMax(&last_row[slots[i]], i);
      __syncthreads();
      if (b == s && keep) keep = last_row[slot] == t;
      if (s < b1) __syncthreads();
    }
  }
  if (keep && a.last != nullptr) keep = a.last[(long long)b * a.cap + slot] == t;
  if (keep && a.scan)
    for (int later = t + 1; later < a.T; ++later) keep &= a.slots[row - t + later] != slot;
  uint2 k_words, v_words;
  uint32_t k_meta, v_meta;
  i4_quantize<kI4CacheGroup / 16>(k, k_words, k_meta);
  i4_quantize<kI4CacheGroup / 16>(v, v_words, v_meta);
  if (!keep) return;
  const long long at = (((long long)b * a.H + h) * a.cap + slot) * per + c;
  reinterpret_cast<uint2*>(a.k_codes)[at] = k_words;
  reinterpret_cast<uint2*>(a.v_codes)[at] = v_words;
  if (c % 2 == 0) {
    a.k_meta[at / 2] = k_meta;
    a.v_meta[at / 2] = v_meta;
  }
}

struct Int4Read {
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_meta, *v_meta;
  const int* start;              // [B]
  bf16 *k, *v;                   // [B, H, rows, D]
  int H, D, cap, rows, in_block;
  Int4Divide blocks_of, heads_of, chunks_of;         // by a head's blocks, by H, by D / 8
};

__global__ void __launch_bounds__(kI4Threads) int4_cache_read_kernel(Int4Read a) {
  grid_dependency_enter();
  // eight keys and eight values a thread: with sixteen a warp's stores lie 32 bytes apart (32767 rows of 8 heads 30 -> 40 us)
  const int per = a.D / 8, in_block = a.in_block, bh = a.blocks_of(blockIdx.x);
  const int of_block = a.chunks_of(threadIdx.x), c = threadIdx.x - of_block * per;
  const int r = (blockIdx.x - bh * (int)a.blocks_of.d) * in_block + of_block;
  if (of_block >= in_block || r >= a.rows) return;
  const long long slot = (long long)a.start[a.heads_of(bh)] + r;
  uint32_t k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
  if (slot >= 0 && slot < a.cap) {
    const long long at = ((long long)bh * a.cap + slot) * per + c;
    const uint32_t kw = reinterpret_cast<const uint32_t*>(a.k_codes)[at], vw = reinterpret_cast<const uint32_t*>(a.v_codes)[at];
    const uint32_t km = a.k_meta[at / 4], vm = a.v_meta[at / 4];
    i4_values(k, kw, i4_scale2(km), i4_offset2(km));
    i4_values(v, vw, i4_scale2(vm), i4_offset2(vm));
  }
  const long long to = ((long long)bh * a.rows + r) * a.D + c * 8;
  *reinterpret_cast<uint4*>(a.k + to) = make_uint4(k[0], k[1], k[2], k[3]);
  *reinterpret_cast<uint4*>(a.v + to) = make_uint4(v[0], v[1], v[2], v[3]);
}

// Slots [src[b], src[b] + rows) -> [dst[b], dst[b] + rows) of the sequences with enable[b] != 0, eight bytes a thread; slots outside the cache are left out.
struct Int4Move {
  uint8_t *k_codes, *k_meta, *v_codes, *v_meta;
  const int *src, *dst, *enable;
  int B, H, D, cap, rows;
};
__global__ void __launch_bounds__(kI4Threads) int4_cache_move_kernel(Int4Move a) {
  grid_dependency_enter();
  const int codes = a.D / 16, per = codes + a.D / 64;            // of a row: units of codes, and of codes and scales
  const long long i = (long long)blockIdx.x * kI4Threads + threadIdx.x;
  if (i >= (long long)a.B * a.H * a.rows * per * 2) return;
  const int c = (int)(i % per), kv = (int)(i / per % 2), r = (int)(i / per / 2 % a.rows);
  const long long bh = i / per / 2 / a.rows;
  const int b = (int)(bh / a.H);
  if (!a.enable[b]) return;
  const long long from = (long long)a.src[b] + r, to = (long long)a.dst[b] + r;
  if (from < 0 || to < 0 || from >= a.cap || to >= a.cap) return;
  uint8_t* base = c < codes ? (kv ? a.v_codes : a.k_codes) : (kv ? a.v_meta : a.k_meta);
  const int width = c < codes ? codes : a.D / 64, at = c < codes ? c : c - codes;
  uint2* rows = reinterpret_cast<uint2*>(base) + bh * a.cap * width + at;
  rows[to * width] = rows[from * width];
}

// Weights: rows [N, K] (row pitch `ld`) -> codes [N, K / 2], scales [K / group, pitch] words; a row's groups of kLanes * 16 values.
template <int kLanes>
__global__ void __launch_bounds__(kI4Threads) int4_weight_kernel(const bf16* w, uint2* codes, uint32_t* meta, int N, int K, long long ld, int pitch) {
  grid_dependency_enter();
  const int per = K / 16;
  const long long n = (long long)N * per, i = (long long)blockIdx.x * kI4Threads + threadIdx.x, j = i < n ? i : n - 1;
  const int c = (int)(j % per);
  const long long row = j / per;
  const bf16* src = w + row * ld + c * 16;
  const uint4 raw[2] = {*reinterpret_cast<const uint4*>(src), *reinterpret_cast<const uint4*>(src + 8)};
  uint2 words;
  uint32_t m;
  i4_quantize<kLanes>(raw, words, m);
  if (i >= n) return;
  codes[j] = words;
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

// How a write finds the last row of a slot: a look at the slots behind its own, shared memory, or a table made ahead.
enum Int4Last : int { kI4Look, kI4Shared, kI4Table };
static long long i4_blocks(int B, int T, int H, int D) {
  const int in_block = kI4Threads / (D / 16);
  return ((long long)B * T + in_block - 1) / in_block * H;
}
static Int4Last i4_last(int B, int T, int H, int D, int cap) {
  if (T <= kI4Scan) return kI4Look;
  return T <= kI4BlockRows && cap <= kI4BlockCap && i4_blocks(B, T, H, D) * T <= kI4BlockWork ? kI4Shared : kI4Table;
}

static bool misaligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace ksa

using namespace ksa;

// Whether ksa_int4_cache_write of rows whose slots may repeat wants its workspace [B, cap] int32.
KSA_API long long ksa_int4_cache_write_table(int B, int T, int H, int D, int cap) {
  return B > 0 && H > 0 && D >= 16 && D <= 16 * kI4Threads && i4_last(B, T, H, D, cap) == kI4Table;
}

// k, v: [B, T, H, D] rows with strides (sb, st, sh) in elements.  Rows whose slot is negative or past the cache are not written; of several
// rows with one slot the last stays: `last` is the workspace that ksa_int4_cache_write_table asks for, null where it does not or
// `distinct` says that no slot occurs twice.
KSA_API int ksa_int4_cache_write(const void* k, const void* v, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* slots,
                                 void* last, int B, int T, int H, int D, int cap, long long sb, long long st, long long sh, int distinct,
                                 void* stream) {
  KSA_ENTER(k);
  KSA_REQUIRE(D > 0 && D % kI4CacheGroup == 0 && D <= 8 * kI4Threads, "int4_cache_write: head_dim %d is no multiple of %d up to %d", D, kI4CacheGroup,
              8 * kI4Threads);
  KSA_REQUIRE(B >= 0 && T >= 0 && H > 0 && cap > 0, "int4_cache_write: bad shape");
  KSA_REQUIRE(sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0 && !misaligned(k, 16) && !misaligned(v, 16),
              "int4_cache_write: rows must be 16-byte aligned");
  KSA_REQUIRE(!misaligned(k_codes, 8) && !misaligned(v_codes, 8) && !misaligned(k_meta, 4) && !misaligned(v_meta, 4),
              "int4_cache_write: cache tensors must be 8-byte aligned");
  if (B == 0 || T == 0) return 0;
  const int in_block = kI4Threads / (D / 16);
  const long long rows = (long long)B * T, blocks = i4_blocks(B, T, H, D);
  KSA_REQUIRE(rows < (1LL << 31) - kI4Threads && blocks < (1LL << 31), "int4_cache_write: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Int4Last how = i4_last(B, T, H, D, cap);
  const bool in_shared = !distinct && how == kI4Shared, table = !distinct && how == kI4Table;
  KSA_REQUIRE(!table || last != nullptr, "int4_cache_write: %d rows need the workspace of last rows", T);
  if (table) {
    KSA_CHECK_CUDA(cudaMemsetAsync(last, 0xFF, (size_t)B * cap * sizeof(int), s));
    KSA_CHECK_CUDA(launch_kernel(int4_last_row_kernel, dim3((unsigned)(((long long)B * T + kI4Threads - 1) / kI4Threads)), dim3(kI4Threads), 0, s,
                                 (const int*)slots, (int*)last, B, T, cap));
  }
  Int4Write a{(const bf16*)k, (const bf16*)v, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_meta, (uint32_t*)v_meta, (const int*)slots,
              table ? (const int*)last : nullptr, sb, st, sh, B, T, H, D, cap, !distinct && T > 1 && how == kI4Look, in_shared, in_block,
              Int4Divide(H), Int4Divide(T), Int4Divide(D / 16)};
  KSA_CHECK_CUDA(launch_stream_kernel(rows * H * D * 5, int4_cache_write_kernel, dim3((unsigned)blocks), dim3(kI4Threads), in_shared ? cap * sizeof(int) : 0,
                                      s, a));
  return 0;
}

// Slots [start[b], start[b] + rows) of every sequence -> k, v [B, H, rows, D] (zeros outside the cache).
KSA_API int ksa_int4_cache_read(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const void* start, void* k,
                                void* v, int B, int H, int D, int cap, int rows, void* stream) {
  KSA_ENTER(k);
  KSA_REQUIRE(D > 0 && D % kI4CacheGroup == 0 && D <= 8 * kI4Threads, "int4_cache_read: head_dim %d is no multiple of %d up to %d", D, kI4CacheGroup,
              8 * kI4Threads);
  KSA_REQUIRE(B >= 0 && rows >= 0 && H > 0 && cap > 0, "int4_cache_read: bad shape");
  if (B == 0 || rows == 0) return 0;
  const int in_block = kI4Threads / (D / 8), of_head = (int)(((long long)rows + in_block - 1) / in_block);
  const long long blocks = (long long)B * H * of_head;
  KSA_REQUIRE(blocks < (1LL << 31), "int4_cache_read: too many rows");
  Int4Read a{(const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint32_t*)k_meta, (const uint32_t*)v_meta, (const int*)start, (bf16*)k,
             (bf16*)v, H, D, cap, rows, in_block, Int4Divide(of_head), Int4Divide(H), Int4Divide(D / 8)};
  KSA_CHECK_CUDA(launch_stream_kernel((long long)B * H * rows * D * 5, int4_cache_read_kernel, dim3((unsigned)blocks), dim3(kI4Threads), 0,
                                      reinterpret_cast<cudaStream_t>(stream), a));
  return 0;
}

// src, dst, enable: [B].  A sequence's two ranges must not overlap.
KSA_API int ksa_int4_cache_move(void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* src, const void* dst, const void* enable, int B,
                                int H, int D, int cap, int rows, void* stream) {
  KSA_ENTER(k_codes);
  KSA_REQUIRE(D > 0 && D % 64 == 0, "int4_cache_move: head_dim %d is no multiple of 64", D);
  KSA_REQUIRE(B >= 0 && rows >= 0 && H > 0 && cap > 0, "int4_cache_move: bad shape");
  const long long n = (long long)B * H * rows * (D / 16 + D / 64) * 2, blocks = (n + kI4Threads - 1) / kI4Threads;
  if (n == 0) return 0;
  KSA_REQUIRE(blocks < (1LL << 31), "int4_cache_move: too many rows");
  Int4Move a{(uint8_t*)k_codes, (uint8_t*)k_meta, (uint8_t*)v_codes, (uint8_t*)v_meta, (const int*)src, (const int*)dst, (const int*)enable, B, H, D, cap,
             rows};
  KSA_CHECK_CUDA(launch_kernel(int4_cache_move_kernel, dim3((unsigned)blocks), dim3(kI4Threads), 0, reinterpret_cast<cudaStream_t>(stream), a));
  return 0;
}

// w [N, K] bf16 (row pitch ld) -> codes [N, K / 2], scales [K / group, pitch] words.
KSA_API int ksa_int4_weight(const void* w, void* codes, void* meta, int N, int K, int group, long long ld, int pitch, void* stream) {
  KSA_ENTER(w);
  KSA_REQUIRE(group == 32 || group == 64 || group == 128, "int4_weight: groups of %d values (32, 64 or 128)", group);
  KSA_REQUIRE(K > 0 && K % group == 0 && N >= 0 && pitch >= N, "int4_weight: K %d is no multiple of the group of %d", K, group);
  KSA_REQUIRE(ld % 8 == 0 && !misaligned(w, 16), "int4_weight: rows must be 16-byte aligned");
  const long long n = (long long)N * (K / 16);
  if (n == 0) return 0;
  const dim3 grid((unsigned)((n + kI4Threads - 1) / kI4Threads));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto kern = group == 32 ? int4_weight_kernel<2> : group == 64 ? int4_weight_kernel<4> : int4_weight_kernel<8>;
  KSA_CHECK_CUDA(launch_stream_kernel(n * 42, kern, grid, dim3(kI4Threads), 0, s, (const bf16*)w, (uint2*)codes, (uint32_t*)meta, N, K, ld, pitch));
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
