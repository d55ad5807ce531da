// The ordinary calls of the operators in native code: argument checks, output tensors and launches of one operator in one call
// from Python.  The calls of a decode step or a short prompt are bound by the host (a projection through Python and ctypes took
// 17 to 19 us, of which the launch itself is 4), and so is a training step on short sequences.
//
// Every function takes plain tensors only (dense CUDA tensors of this device without conjugation, wrappers or subclasses) in the
// forms that its kernels take as they are, and returns None for anything else: the Python operator then goes its general way,
// with its own checks, errors and copies.  Nothing is kept between calls.
//
// This file knows torch, the kernel library does not: it calls the library's C entry points like any other user.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <pybind11/pybind11.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <tuple>
#include <vector>

extern "C" {
const char* ksa_last_error();
int ksa_gemm_on_pairs(int M, int N, int pair_min_tiles);
int ksa_gemm_narrow_plan(int M, int N, int K, int glu, int pair_min_tiles, int ragged);
int ksa_gemm_tall_plan(int M, int N, int K, int glu, int ragged);
int ksa_gemm_tall_bf16(const void* x, const void* w, void* c, int M, int N, int K, long long ldx, long long ldw, long long ldc, int glu,
                       int columns, int split, void* stream);
int ksa_rmsnorm_bwd_parts(int rows);
int ksa_attn_bwd_num_segments(int lq);
int ksa_gemm_bf16(const void* a, const void* b, void* c, int M, int N, int K, long long lda, long long ldb, long long ldc,
                  int a_mn_major, int b_mn_major, int out_fp32, int accumulate, float alpha, int sm_limit, void* stream);
int ksa_gemm2_bf16(const void* a, const void* b, void* c, int M, int N, int K, long long lda, long long ldb, long long ldc,
                   int a_mn_major, int b_mn_major, int out_fp32, int accumulate, float alpha, void* stream);
int ksa_gemm_narrow_bf16(const void* x, const void* w, void* c, int M, int N, int K, long long ldx, long long ldw, long long ldc,
                         int w_mn_major, int glu, int bt, int split, float alpha, void* stream);
int ksa_gemm2_swiglu_bf16(const void* a, const void* b, void* gu, void* h, int M, int F, int K, long long lda, long long ldb,
                          long long ld_gu, long long ld_h, void* stream);
int ksa_gemv_bf16(const void* a, const void* b, void* c, int M, int N, int K, long long lda, long long ldb, long long ldc,
                  void* stream);
int ksa_gemv_swiglu_bf16(const void* a, const void* b, void* c, int M, int N, int K, long long lda, long long ldb, long long ldc,
                         void* stream);
int ksa_gemv_norm_bf16(const void* x, const void* delta, const void* norm_w, void* res_out, const void* b, void* c, int M, int N,
                       int K, long long ldx, long long ld_delta, long long ld_res, long long ldb, long long ldc, float eps,
                       int delta_rows, int glu, void* stream);
int ksa_rmsnorm_fwd(const void* x, const void* delta, const void* w, void* res, void* y, void* rstd, int rows, int D, float eps,
                    int delta_rows, void* stream);
int ksa_rmsnorm_bwd(const void* dy, const void* x, const void* w, const void* rstd, const void* dres, void* dx, void* partial,
                    void* dw, int accumulate, int rows, int D, void* stream);
int ksa_qknorm_rope_fwd(const void* qkv, void* out, const void* q_w, const void* k_w, const void* pos, void* rstd,
                        long long in_stride, long long out_stride, int T, int Hq, int Hkv, int D, float theta, float eps,
                        int interleaved, int copy_v, void* stream);
int ksa_qknorm_rope_bwd(const void* qkv, const void* d_out, void* d_qkv, const void* q_w, const void* k_w, const void* pos,
                        const void* rstd, void* dqw, void* dkw, long long in_stride, long long dout_stride, int T, int Hq, int Hkv,
                        int D, float theta, float eps, int interleaved, int copy_v, void* stream);
int ksa_swiglu_fwd(const void* gu, void* out, long long rows, int F, void* stream);
int ksa_swiglu_bwd(const void* gu, const void* dout, void* dgu, long long rows, int F, void* stream);
int ksa_attn_fwd(const void* q, const void* k, const void* v, const void* ks, const void* vs, void* o, void* lse, int B, int Hq,
                 int Hkv, int HD, int Lq, int Lk, int Ns, long long q_rs, long long q_bs, long long k_rs, long long k_bs,
                 long long v_rs, long long v_bs, long long ks_rs, long long ks_bs, long long vs_rs, long long vs_bs, long long o_rs,
                 long long o_bs, int q_off, int k_off, int s_off, int chunk, int n_sum, int window, int tok_window, float scale,
                 const void* q_doc_start, const void* k_doc_end, void* stream);
int ksa_set_launch_beside(int on);
int ksa_set_dependent_launch(int mode);
int ksa_summary_attn_fwd(const void* q, const void* k, const void* v, const void* ks, const void* vs, void* o, void* lse, int B,
                         int Hq, int Hkv, int D, int Nq, int seq_len, long long q_rs, long long q_bs, long long k_rs,
                         long long k_bs, long long v_rs, long long v_bs, long long ks_rs, long long ks_bs, long long vs_rs,
                         long long vs_bs, long long o_rs, long long o_bs, int chunk, int n_sum, int chunk0, int k_off, int s_off,
                         float scale, void* stream);
int ksa_attn_bwd_fused(const void* q, const void* k, const void* v, const void* ks, const void* vs, const void* o, const void* dout,
                       const void* lse, void* stats, void* dq32, void* dq, void* dk, void* dv, void* dks, void* dvs, int B, int Hq,
                       int Hkv, int HD, int Lq, int Lk, int Ns, long long q_rs, long long q_bs, long long k_rs, long long k_bs,
                       long long v_rs, long long v_bs, long long ks_rs, long long ks_bs, long long vs_rs, long long vs_bs,
                       long long o_rs, long long o_bs, long long dq_rs, long long dq_bs, long long dk_rs, long long dk_bs,
                       long long dv_rs, long long dv_bs, long long dks_rs, long long dks_bs, long long dvs_rs, long long dvs_bs,
                       int q_off, int k_off, int s_off, int chunk, int n_sum, int window, int tok_window, float scale,
                       void* part_k, void* part_v, const void* q_doc_start, const void* k_doc_end, void* stream);
int ksa_int4_cache_write(const void* k, const void* v, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* slots, void* last,
                         int B, int T, int H, int D, int cap, long long sb, long long st, long long sh, int distinct, void* stream);
int ksa_int4_cache_read(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const void* start, void* k, void* v,
                        int B, int H, int D, int cap, int rows, void* stream);
int ksa_int4_decode_attn(const void* q, const void* k, const void* k_meta, const void* v, const void* v_meta, const void* start,
                         const void* len, void* workspace, void* out, int B, int Tq, int Hq, int Hkv, int D, int cap, long long q_sb,
                         long long q_st, long long q_sh, float scale, void* stream);
long long ksa_int4_attn_workspace(int B, int Tq, int Hq, int Hkv, int D, int cap);
long long ksa_int4_cache_write_table(int B, int T, int H, int D, int cap);
int ksa_int4_linear(const void* A, const void* codes, const void* meta, void* C, int M, int N, int K, int group, int pitch, long long lda,
                    long long ldc, int glu, void* stream);
int ksa_summary_attn_bwd(const void* q, const void* k, const void* v, const void* ks, const void* vs, const void* o,
                         const void* dout, const void* lse, void* dq, void* dk, void* dv, void* dks, void* dvs, int B, int Hq,
                         int Hkv, int D, int Nq, int seq_len, long long q_rs, long long q_bs, long long k_rs, long long k_bs,
                         long long v_rs, long long v_bs, long long ks_rs, long long ks_bs, long long vs_rs, long long vs_bs,
                         long long o_rs, long long o_bs, long long dq_rs, long long dq_bs, long long dk_rs, long long dk_bs,
                         long long dv_rs, long long dv_bs, long long dks_rs, long long dks_bs, long long dvs_rs, long long dvs_bs,
                         int chunk, int n_sum, int chunk0, int k_off, int s_off, float scale, const void* part_k,
                         const void* part_v, int n_keys, void* stream);
int ksa_grad_norm_parts(int tensors);
int ksa_grad_norm(const void* src, const void* dst, const void* meta, int tensors, float scale, float most, void* partial, void* norm,
                  void* factor, void* stream);
long long ksa_token_loss_units(long long n, int sequences);
int ksa_policy_loss(const void* y, const void* old, const void* ref, const void* adv, const void* mask, const void* cu, int wide, void* grad,
                    void* partial, void* inv, void* loss, void* stats, int types, long long n, int sequences, long long length,
                    int adv_by_sequence, int by_sequence, const void* bounds, float beta, void* stream);
int ksa_policy_loss_bwd(const void* grad, const void* inv, const void* dloss, void* dy, int type, const void* cu, int wide, long long n,
                        int sequences, long long length, int by_sequence, void* stream);
int ksa_preference_loss(const void* y, const void* ref, const void* mask, const void* cu, int wide, void* partial, void* coef, void* rewards,
                        void* loss, int types, long long n, int sequences, long long length, float beta, float smoothing, void* stream);
int ksa_preference_loss_bwd(const void* mask, const void* coef, const void* dloss, void* dy, int type, const void* cu, int wide, long long n,
                            int sequences, long long length, void* stream);
long long ksa_log_probs_work(int T, int V);
int ksa_log_probs(const void* h, const void* w, const void* labels, void* dense, void* rows, void* row_label, void* place, void* count,
                  void* lse2, void* work, void* y, void* codes, void* tops, int T, int V, int D, long long ldh, long long ldw, long long ignore_index, float tau,
                  void* stream);
int ksa_log_probs_bwd(const void* dense, const void* w, const void* rows, const void* row_label, const void* place, const void* count,
                      const void* lse2, const void* codes, const void* tops, const void* dy, void* dx, void* dh32, void* dh, void* dw, int T, int V, int D, long long ldw,
                      long long lddw, int dw_fp32, int add_dw, int slab, int planes, float tau, void* stream);
}

namespace {

using at::Tensor;
std::atomic<long long> g_launches{0};

void check(const char* name, int rc, int kernels = 1) {
  if (rc != 0) throw std::runtime_error(std::string(name) + " failed (" + std::to_string(rc) + "): " + ksa_last_error());
  g_launches.fetch_add(kernels, std::memory_order_relaxed);
}
#define LAUNCH(entry, ...) check(#entry, entry(__VA_ARGS__))
#define LAUNCH_SEVERAL(kernels, entry, ...) check(#entry, entry(__VA_ARGS__), kernels)

// The arguments of one call.  `plain` turns false at the first one that is not of the ordinary kind.
struct Args {
  PyObject* const* v;
  Py_ssize_t n, at = 0;
  bool plain = true;
  c10::DeviceIndex device = -1;      // of the first tensor; it has to be the current one

  Args(PyObject* const* v, Py_ssize_t n) : v(v), n(n) {}

  PyObject* next() {
    if (at >= n) { plain = false; return Py_None; }
    return v[at++];
  }
  bool dense(const Tensor& t) {
    static const uint64_t allowed = (c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                     c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                     c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA)).raw_repr();
    if (!t.defined() || (t.key_set().raw_repr() & ~allowed) != 0 || !t.device().is_cuda() || !t.has_storage()) return false;
    if (device < 0) {
      device = c10::cuda::current_device();
      if (device < 0) return false;
    }
    return t.device().index() == device && t.numel() > 0 && t.const_data_ptr() != nullptr;
  }
  // a tensor of the given type; `optional`: None gives nullptr
  const Tensor* tensor(at::ScalarType type = at::kBFloat16, bool optional = false) {
    PyObject* o = next();
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_CheckExact(o)) { plain = false; return nullptr; }
    const Tensor& t = THPVariable_Unpack(o);
    if (!dense(t) || t.scalar_type() != type) { plain = false; return nullptr; }
    return &t;
  }
  long long integer() {
    PyObject* o = next();
    if (!PyLong_Check(o)) { plain = false; return 0; }       // bool is one too
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) { PyErr_Clear(); plain = false; }
    if (x > INT_MAX || x < INT_MIN) plain = false;           // the entry points take sizes as int
    return x;
  }
  float real() {
    PyObject* o = next();
    const double x = PyFloat_Check(o) || PyLong_Check(o) ? PyFloat_AsDouble(o) : (plain = false, 0.0);
    if (PyErr_Occurred()) { PyErr_Clear(); plain = false; }
    return (float)x;
  }
  bool ok() { return plain && at == n; }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
  Tensor empty(at::IntArrayRef sizes, at::ScalarType type = at::kBFloat16) const {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, device)));
  }
};

bool rows2d(const Tensor* t) { return t->dim() == 2 && t->stride(1) == 1 && t->stride(0) > 0; }      // rows with any pitch
bool packed2d(const Tensor* t) { return t->dim() == 2 && t->is_contiguous(); }
bool vector(const Tensor* t, long long n) { return t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }
bool fits(long long x) { return x > 0 && x <= INT_MAX; }
const char* at_row(const Tensor& t, long long row) {
  return static_cast<const char*>(t.const_data_ptr()) + row * t.stride(0) * (long long)t.element_size();
}
char* at_row_mut(const Tensor& t, long long row) {
  return static_cast<char*>(t.mutable_data_ptr()) + row * t.stride(0) * (long long)t.element_size();
}
PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* wrap(const Tensor& a, const Tensor& b) { return Py_BuildValue("(NN)", wrap(a), wrap(b)); }
PyObject* none() { Py_RETURN_NONE; }

// While it lives, launches may run beside the kernel before them: csrc/host.h (launch_beside) says when that is sound.
struct Beside {
  explicit Beside(bool on) : before(ksa_set_launch_beside(on)) {}
  ~Beside() { ksa_set_launch_beside(before); }
  Beside(const Beside&) = delete;
  int before;
};

// While it lives, products of a thread that launches dependently read their weights early.
struct EarlyWeights {
  explicit EarlyWeights(bool on) : before(on ? ksa_set_dependent_launch(1) : 0), set(on) {
    if (set && before != 0) ksa_set_dependent_launch(before);       // ordinary launches stay ordinary
  }
  ~EarlyWeights() { if (set) ksa_set_dependent_launch(before); }
  EarlyWeights(const EarlyWeights&) = delete;
  int before;
  bool set;
};

// The kernel for C[M, N] = op(A) op(B) (+ C): the rules of `gemm` in ops/__init__.py, which explains them.
struct Product {
  const void* a;
  const void* b;
  void* c;
  long long M, N, K, lda, ldb, ldc;
  int a_mn, b_mn, fp32, accumulate;
};
void gemm(const Product& p, int pair_min, void* st) {
  const int M = (int)p.M, N = (int)p.N, K = (int)p.K;
  const bool bf16_out = !p.fp32 && !p.accumulate;
  if (M <= 16 && !p.a_mn && !p.b_mn && bf16_out && K % 8 == 0) {
    LAUNCH(ksa_gemv_bf16, p.a, p.b, p.c, M, N, K, p.lda, p.ldb, p.ldc, st);
    return;
  }
  if (!p.a_mn && !p.b_mn && bf16_out && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.ldc % 8 == 0) {
    const int plan = ksa_gemm_tall_plan(M, N, K, 0, p.lda % 64 != 0 || p.ldb % 64 != 0);
    if (plan != 0) {
      LAUNCH(ksa_gemm_tall_bf16, p.a, p.b, p.c, M, N, K, p.lda, p.ldb, p.ldc, 0, plan / 16, plan % 16, st);
      return;
    }
  }
  if (!p.a_mn && bf16_out) {
    const int plan = ksa_gemm_narrow_plan(M, N, K, 0, pair_min, (p.lda % 64 != 0) + 2 * (p.ldb % 64 != 0));
    if (plan != 0) {
      LAUNCH(ksa_gemm_narrow_bf16, p.a, p.b, p.c, M, N, K, p.lda, p.ldb, p.ldc, p.b_mn, 0, plan / 16, plan % 16, 1.f, st);
      return;
    }
  }
  if (ksa_gemm_on_pairs(M, N, pair_min))
    LAUNCH(ksa_gemm2_bf16, p.a, p.b, p.c, M, N, K, p.lda, p.ldb, p.ldc, p.a_mn, p.b_mn, p.fp32, p.accumulate, 1.f, st);
  else
    LAUNCH(ksa_gemm_bf16, p.a, p.b, p.c, M, N, K, p.lda, p.ldb, p.ldc, p.a_mn, p.b_mn, p.fp32, p.accumulate, 1.f, 0, st);
}
bool sizes_ok(const Product& p) { return fits(p.M) && fits(p.N) && fits(p.K); }

// gemm(a, b, out | None, fp32 output, a_mn, b_mn, accumulate, pair_min) -> out
PyObject* py_gemm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *w = a.tensor();
  PyObject* o = a.next();
  const bool fp32 = a.integer() != 0;
  const Tensor* out = nullptr;
  if (o != Py_None) {
    if (!THPVariable_CheckExact(o)) return none();
    out = &THPVariable_Unpack(o);
    if (!a.dense(*out) || out->scalar_type() != (fp32 ? at::kFloat : at::kBFloat16)) return none();
  }
  const int a_mn = a.integer() != 0, b_mn = a.integer() != 0, acc = a.integer() != 0, pair_min = (int)a.integer();
  if (!a.ok() || !rows2d(x) || !rows2d(w) || (acc && !out)) return none();
  Product p{x->const_data_ptr(), w->const_data_ptr(), nullptr, x->size(a_mn), w->size(b_mn), x->size(!a_mn), x->stride(0),
            w->stride(0), 0, a_mn, b_mn, fp32, acc};
  if (p.K != w->size(!b_mn) || !sizes_ok(p)) return none();
  if (out && !(rows2d(out) && out->size(0) == p.M && out->size(1) == p.N)) return none();
  Tensor made;
  {
    pybind11::gil_scoped_release no_gil;
    if (!out) made = a.empty({p.M, p.N}, fp32 ? at::kFloat : at::kBFloat16);
    const Tensor& c = out ? *out : made;
    p.c = c.mutable_data_ptr();
    p.ldc = c.stride(0);
    gemm(p, pair_min, a.stream());
  }
  if (out) { Py_INCREF(o); return o; }
  return wrap(made);
  END_HANDLE_TH_ERRORS
}

// linear(x, w, pair_min, weights_ready) -> y [..., N], for any x with contiguous rows.  weights_ready: no kernel that may still run when
// the one before this product has begun its work writes w (csrc/host.h, kLaunchEarlyWeights)
PyObject* py_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *w = a.tensor();
  const int pair_min = (int)a.integer();
  const bool ready = a.integer() != 0;
  if (!a.ok() || !rows2d(w) || !(rows2d(x) || (x->dim() > 0 && x->is_contiguous())) || x->size(-1) != w->size(1)) return none();
  if (c10::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad())) return none();
  const long long K = w->size(1), M = x->numel() / K;
  Product p{x->const_data_ptr(), w->const_data_ptr(), nullptr, M, w->size(0), K, x->dim() == 2 ? x->stride(0) : K, w->stride(0),
            w->size(0), 0, 0, 0, 0};
  if (!sizes_ok(p)) return none();
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    auto sizes = x->sizes().vec();
    sizes.back() = p.N;
    y = a.empty(sizes);
    p.c = y.mutable_data_ptr();
    const EarlyWeights early(ready);
    gemm(p, pair_min, a.stream());
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// linear_dw(dy, x, lo, hi, out | None, accumulate, pair_min, beside) -> dy[lo:hi]^T x[lo:hi], into an fp32 buffer or as bf16.
// beside: the caller launched another product of the same tensors just before (csrc/host.h, launch_beside)
PyObject* py_linear_dw(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *dy = a.tensor(), *x = a.tensor();
  const long long lo = a.integer(), hi = a.integer();
  const Tensor* out = a.tensor(at::kFloat, true);
  const int acc = a.integer() != 0, pair_min = (int)a.integer();
  const bool on = a.integer() != 0;
  if (!a.ok() || !rows2d(dy) || !rows2d(x) || dy->size(0) != x->size(0) || lo < 0 || hi <= lo || hi > x->size(0)) return none();
  Product p{at_row(*dy, lo), at_row(*x, lo), nullptr, dy->size(1), x->size(1), hi - lo, dy->stride(0), x->stride(0), 0, 1, 1,
            out != nullptr, out != nullptr && acc};
  if (!sizes_ok(p) || (out && !(rows2d(out) && out->size(0) == p.M && out->size(1) == p.N))) return none();
  Tensor made;
  {
    pybind11::gil_scoped_release no_gil;
    if (!out) made = a.empty({p.M, p.N});
    const Tensor& c = out ? *out : made;
    p.c = c.mutable_data_ptr();
    p.ldc = c.stride(0);
    const Beside beside(on && out);      // memory allocated here might be what the kernel before has just let go
    gemm(p, pair_min, a.stream());
  }
  return wrap(out ? *out : made);
  END_HANDLE_TH_ERRORS
}

// dual_linear(x, w_a, w_b, n_a, b_mn, pair_min): rows [:n_a] of x times w_a, the others times w_b.  b_mn: the weights as they lie,
// [K, N] (the gradient of x from that of y)
PyObject* py_dual_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *wa = a.tensor(), *wb = a.tensor();
  const long long n_a = a.integer();
  const int b_mn = a.integer() != 0, pair_min = (int)a.integer();
  if (!a.ok() || !packed2d(x) || !rows2d(wa) || !rows2d(wb) || wa->sizes() != wb->sizes() || n_a < 0 || n_a > x->size(0)) return none();
  const long long R = x->size(0), N = wa->size(b_mn), K = wa->size(!b_mn);
  if (K != x->size(1) || !fits(R) || !fits(N) || !fits(K)) return none();
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = a.empty({R, N});
    void* st = a.stream();
    if (n_a > 0)
      gemm({x->const_data_ptr(), wa->const_data_ptr(), y.mutable_data_ptr(), n_a, N, K, K, wa->stride(0), N, 0, b_mn, 0, 0}, pair_min, st);
    const Beside beside(n_a > 16);     // at most 16 text rows take a product that lets its successors start before it waits
    if (R > n_a)
      gemm({at_row(*x, n_a), wb->const_data_ptr(), at_row_mut(y, n_a), R - n_a, N, K, K, wb->stride(0), N, 0, b_mn, 0, 0}, pair_min, st);
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// rms_norm(x, delta | None, w, eps) -> (x + delta, norm, 1 / rms), or (norm, 1 / rms) without delta
PyObject* py_rms_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *d = a.tensor(at::kBFloat16, true), *w = a.tensor();
  const float eps = a.real();
  if (!a.ok() || !packed2d(x) || !vector(w, x->size(1)) || !fits(x->size(0)) || !fits(x->size(1))) return none();
  if (d && !(packed2d(d) && d->size(1) == x->size(1) && d->size(0) <= x->size(0))) return none();
  const int rows = (int)x->size(0), D = (int)x->size(1);
  Tensor res, y, rstd;
  {
    pybind11::gil_scoped_release no_gil;
    y = a.empty({rows, D});
    if (d) res = a.empty({rows, D});
    rstd = a.empty({rows}, at::kFloat);
    LAUNCH(ksa_rmsnorm_fwd, x->const_data_ptr(), d ? d->const_data_ptr() : nullptr, w->const_data_ptr(),
           d ? res.mutable_data_ptr() : nullptr, y.mutable_data_ptr(), rstd.mutable_data_ptr(), rows, D, eps, d ? (int)d->size(0) : 0,
           a.stream());
  }
  if (!d) return wrap(y, rstd);
  return Py_BuildValue("(NNN)", wrap(res), wrap(y), wrap(rstd));
  END_HANDLE_TH_ERRORS
}

// rms_norm_bwd(dy, x, w, rstd, dres | None, dw (fp32), accumulate) -> dx
PyObject* py_rms_norm_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *dy = a.tensor(), *x = a.tensor(), *w = a.tensor(), *rstd = a.tensor(at::kFloat), *dres = a.tensor(at::kBFloat16, true),
               *dw = a.tensor(at::kFloat);
  const int acc = a.integer() != 0;
  if (!a.ok() || !packed2d(x) || !packed2d(dy) || dy->sizes() != x->sizes() || (dres && !(packed2d(dres) && dres->sizes() == x->sizes())))
    return none();
  if (!fits(x->size(0)) || !fits(x->size(1)) || !vector(w, x->size(1)) || !vector(dw, x->size(1)) || !vector(rstd, x->size(0))) return none();
  const int rows = (int)x->size(0), D = (int)x->size(1);
  Tensor dx;
  {
    pybind11::gil_scoped_release no_gil;
    dx = a.empty({rows, D});
    Tensor partial = a.empty({ksa_rmsnorm_bwd_parts(rows), D}, at::kFloat);
    check("ksa_rmsnorm_bwd",
          ksa_rmsnorm_bwd(dy->const_data_ptr(), x->const_data_ptr(), w->const_data_ptr(), rstd->const_data_ptr(),
                          dres ? dres->const_data_ptr() : nullptr, dx.mutable_data_ptr(), partial.mutable_data_ptr(),
                          dw->mutable_data_ptr(), acc, rows, D, a.stream()), 2);
  }
  return wrap(dx);
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(qkv, q_w | None, k_w | None, pos (int32), Hq, Hkv, D, theta, eps, interleaved) -> (out, rstd)
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *qkv = a.tensor(), *qw = a.tensor(at::kBFloat16, true), *kw = a.tensor(at::kBFloat16, true), *pos = a.tensor(at::kInt);
  const long long Hq = a.integer(), Hkv = a.integer(), D = a.integer();
  const float theta = a.real(), eps = a.real();
  const int inter = a.integer() != 0;
  if (!a.ok() || Hq <= 0 || Hkv <= 0 || D <= 0 || !rows2d(qkv) || qkv->size(1) != (Hq + 2 * Hkv) * D || !fits(qkv->size(0)) ||
      !vector(pos, qkv->size(0)) || (qw && !vector(qw, D)) || (kw && !vector(kw, D)))
    return none();
  const int T = (int)qkv->size(0);
  Tensor out, rstd;
  {
    pybind11::gil_scoped_release no_gil;
    out = a.empty({T, qkv->size(1)});
    rstd = a.empty({T, Hq + Hkv}, at::kFloat);
    LAUNCH(ksa_qknorm_rope_fwd, qkv->const_data_ptr(), out.mutable_data_ptr(), qw ? qw->const_data_ptr() : nullptr,
           kw ? kw->const_data_ptr() : nullptr, pos->const_data_ptr(), rstd.mutable_data_ptr(), qkv->stride(0), out.stride(0), T, (int)Hq,
           (int)Hkv, (int)D, theta, eps, inter, 1, a.stream());
  }
  return wrap(out, rstd);
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope_bwd(qkv, d_out, q_w | None, k_w | None, pos, rstd, dq_w (fp32) | None, dk_w | None, Hq, Hkv, D, theta, eps, interleaved)
// -> d_qkv; the weight gradients are added to dq_w and dk_w
PyObject* py_qk_norm_rope_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *qkv = a.tensor(), *g = a.tensor(), *qw = a.tensor(at::kBFloat16, true), *kw = a.tensor(at::kBFloat16, true),
               *pos = a.tensor(at::kInt), *rstd = a.tensor(at::kFloat), *dqw = a.tensor(at::kFloat, true), *dkw = a.tensor(at::kFloat, true);
  const long long Hq = a.integer(), Hkv = a.integer(), D = a.integer();
  const float theta = a.real(), eps = a.real();
  const int inter = a.integer() != 0;
  if (!a.ok() || Hq <= 0 || Hkv <= 0 || D <= 0 || !packed2d(qkv) || qkv->size(1) != (Hq + 2 * Hkv) * D || !fits(qkv->size(0)) ||
      !packed2d(g) || g->sizes() != qkv->sizes() || !vector(pos, qkv->size(0)) || !packed2d(rstd) || rstd->size(0) != qkv->size(0) ||
      rstd->size(1) != Hq + Hkv || (qw && !vector(qw, D)) || (kw && !vector(kw, D)) || (dqw && !vector(dqw, D)) || (dkw && !vector(dkw, D)))
    return none();
  const int T = (int)qkv->size(0);
  Tensor d;
  {
    pybind11::gil_scoped_release no_gil;
    d = a.empty(qkv->sizes());
    LAUNCH(ksa_qknorm_rope_bwd, qkv->const_data_ptr(), g->const_data_ptr(), d.mutable_data_ptr(), qw ? qw->const_data_ptr() : nullptr,
           kw ? kw->const_data_ptr() : nullptr, pos->const_data_ptr(), rstd->const_data_ptr(), dqw ? dqw->mutable_data_ptr() : nullptr,
           dkw ? dkw->mutable_data_ptr() : nullptr, qkv->stride(0), g->stride(0), T, (int)Hq, (int)Hkv, (int)D, theta, eps, inter, 1,
           a.stream());
  }
  return wrap(d);
  END_HANDLE_TH_ERRORS
}

// swiglu(gate | up rows) -> rows of half the width
PyObject* py_swiglu(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor* gu = a.tensor();
  if (!a.ok() || gu->dim() < 1 || !gu->is_contiguous() || gu->size(-1) % 2 != 0 || !fits(gu->size(-1))) return none();
  const long long F = gu->size(-1) / 2, rows = gu->numel() / (2 * F);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    auto sizes = gu->sizes().vec();
    sizes.back() = F;
    out = a.empty(sizes);
    LAUNCH(ksa_swiglu_fwd, gu->const_data_ptr(), out.mutable_data_ptr(), rows, (int)F, a.stream());
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// swiglu_bwd(gate | up rows, dout rows) -> d(gate | up)
PyObject* py_swiglu_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *gu = a.tensor(), *g = a.tensor();
  if (!a.ok() || !packed2d(gu) || !packed2d(g) || gu->size(0) != g->size(0) || gu->size(1) != 2 * g->size(1) || !fits(gu->size(1))) return none();
  Tensor d;
  {
    pybind11::gil_scoped_release no_gil;
    d = a.empty(gu->sizes());
    LAUNCH(ksa_swiglu_bwd, gu->const_data_ptr(), g->const_data_ptr(), d.mutable_data_ptr(), gu->size(0), (int)g->size(1), a.stream());
  }
  return wrap(d);
  END_HANDLE_TH_ERRORS
}

// linear_swiglu(x, w13, pair_min) -> silu(gate) * up where one kernel does it (no gradients wanted), else None
PyObject* py_linear_swiglu(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *w = a.tensor();
  const int pair_min = (int)a.integer();
  if (!a.ok() || !rows2d(x) || !rows2d(w) || x->size(1) != w->size(1) || w->size(0) % 2 != 0 || !fits(x->size(0)) || !fits(w->size(0)) ||
      !fits(x->size(1)) || x->size(1) % 8 != 0 || x->stride(0) % 8 != 0 || w->stride(0) % 8 != 0)
    return none();
  if (c10::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad())) return none();
  const int M = (int)x->size(0), N = (int)w->size(0), K = (int)x->size(1);
  int plan = 0, tall = 0;
  if (M > 16) {
    tall = ksa_gemm_tall_plan(M, N / 2, K, 1, x->stride(0) % 64 != 0 || w->stride(0) % 64 != 0);
    if (tall == 0 && N % 16 == 0) plan = ksa_gemm_narrow_plan(M, N, K, 1, pair_min, (x->stride(0) % 64 != 0) + 2 * (w->stride(0) % 64 != 0));
    if (plan == 0 && tall == 0) return none();
  }
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = a.empty({M, N / 2});
    if (M <= 16)
      LAUNCH(ksa_gemv_swiglu_bf16, x->const_data_ptr(), w->const_data_ptr(), out.mutable_data_ptr(), M, N, K, x->stride(0), w->stride(0),
             out.stride(0), a.stream());
    else if (tall != 0)
      LAUNCH(ksa_gemm_tall_bf16, x->const_data_ptr(), w->const_data_ptr(), out.mutable_data_ptr(), M, N / 2, K, x->stride(0), w->stride(0),
             out.stride(0), 1, tall / 16, 1, a.stream());
    else
      LAUNCH(ksa_gemm_narrow_bf16, x->const_data_ptr(), w->const_data_ptr(), out.mutable_data_ptr(), M, N, K, x->stride(0), w->stride(0),
             out.stride(0), 0, 1, plan / 16, plan % 16, 1.f, a.stream());
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// gemm_swiglu(x, w13, pair_min) -> (silu(gate) * up, gate | up) from one launch of the CTA-pair kernel where that serves the
// product, else None (333 x 19456 x 2560 45.7 us on pairs; on single CTAs with the activation behind 44.4)
PyObject* py_gemm_swiglu(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *w = a.tensor();
  const int pair_min = (int)a.integer();
  if (!a.ok() || !rows2d(x) || !rows2d(w) || x->size(1) != w->size(1) || w->size(0) % 128 != 0 || !fits(x->size(0)) || !fits(w->size(0)) ||
      !fits(x->size(1)) || x->stride(0) % 8 != 0 || w->stride(0) % 8 != 0 || x->size(0) <= 16)
    return none();
  const int M = (int)x->size(0), F = (int)(w->size(0) / 2), K = (int)x->size(1);
  if (!ksa_gemm_on_pairs(M, 2 * F, pair_min) ||
      ksa_gemm_narrow_plan(M, 2 * F, K, 2, pair_min, (x->stride(0) % 64 != 0) + 2 * (w->stride(0) % 64 != 0)) != 0)
    return none();
  Tensor h, gu;
  {
    pybind11::gil_scoped_release no_gil;
    h = a.empty({M, F});
    gu = a.empty({M, 2LL * F});
    LAUNCH(ksa_gemm2_swiglu_bf16, x->const_data_ptr(), w->const_data_ptr(), gu.mutable_data_ptr(), h.mutable_data_ptr(), M, F, K, x->stride(0),
           w->stride(0), 2LL * F, F, a.stream());
  }
  return wrap(h, gu);
  END_HANDLE_TH_ERRORS
}

// norm_linear(x, delta | None, norm_w, eps, w, glu) -> (x + delta, product of the normalised rows), at most four rows, no gradients
PyObject* py_norm_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  PyObject* px = n > 0 ? v[0] : Py_None;
  const Tensor *x = a.tensor(), *d = a.tensor(at::kBFloat16, true), *nw = a.tensor();
  const float eps = a.real();
  const Tensor* w = a.tensor();
  const int glu = a.integer() != 0;
  if (!a.ok() || !rows2d(x) || !rows2d(w) || x->size(0) > 4 || x->numel() > 81920 || x->size(1) != w->size(1) || !vector(nw, x->size(1)) || !fits(w->size(0)) ||
      !fits(x->size(1)) || x->size(1) % 8 != 0 || x->stride(0) % 8 != 0 || w->stride(0) % 8 != 0 || (glu && w->size(0) % 2 != 0))
    return none();
  if (d && !(rows2d(d) && d->size(1) == x->size(1) && d->size(0) <= x->size(0) && d->stride(0) % 8 == 0)) return none();
  if (c10::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad())) return none();
  const int M = (int)x->size(0), K = (int)x->size(1), N = (int)w->size(0);
  Tensor res, out;
  {
    pybind11::gil_scoped_release no_gil;
    if (d) res = a.empty({M, K});
    out = a.empty({M, glu ? N / 2 : N});
    LAUNCH(ksa_gemv_norm_bf16, x->const_data_ptr(), d ? d->const_data_ptr() : nullptr, nw->const_data_ptr(),
           d ? res.mutable_data_ptr() : nullptr, w->const_data_ptr(), out.mutable_data_ptr(), M, N, K, x->stride(0), d ? d->stride(0) : K,
           d ? res.stride(0) : x->stride(0), w->stride(0), out.stride(0), eps, d ? (int)d->size(0) : 0, glu, a.stream());
  }
  if (d) return wrap(res, out);
  Py_INCREF(px);
  return Py_BuildValue("(NN)", px, wrap(out));
  END_HANDLE_TH_ERRORS
}

// Column blocks of packed rows [B*L text rows | B*Ns summary rows], each q heads | k heads | v heads.
struct PackedShape {
  long long B, L, Ns, Hq, Hkv, D, chunk, n_sum, window, tok_window;
  float scale;
  void read(Args& a) {
    B = a.integer(); L = a.integer(); Ns = a.integer(); Hq = a.integer(); Hkv = a.integer(); D = a.integer(); chunk = a.integer();
    n_sum = a.integer(); window = a.integer(); tok_window = a.integer(); scale = a.real();
  }
  bool ok(const Tensor* qkv) const {
    return B > 0 && L > 0 && Ns >= 0 && Hq > 0 && Hkv > 0 && D > 0 && chunk > 0 && rows2d(qkv) && qkv->size(0) == B * (L + Ns) &&
           qkv->size(1) == (Hq + 2 * Hkv) * D;
  }
  long long q_cols() const { return Hq * D; }
  const void* block(const Tensor& t, long long row, long long col) const {
    return static_cast<const char*>(t.const_data_ptr()) + (row * t.stride(0) + col) * 2;
  }
  void* block_mut(Tensor& t, long long row, long long col) const {
    return static_cast<char*>(t.mutable_data_ptr()) + (row * t.stride(0) + col) * 2;
  }
};

// attention(qkv, B, L, Ns, Hq, Hkv, D, chunk, n_sum, window, tok_window, scale) -> (out, lse, summary lse | None)
PyObject* py_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor* x = a.tensor();
  PackedShape s;
  s.read(a);
  if (!a.ok() || !s.ok(x)) return none();
  const int B = (int)s.B, L = (int)s.L, Ns = (int)s.Ns, Hq = (int)s.Hq, Hkv = (int)s.Hkv, D = (int)s.D;
  const long long rs = x->stride(0), text = s.B * s.L, kc = s.q_cols(), vc = kc + s.Hkv * s.D, os = s.q_cols();
  Tensor out, lse, lse_s;
  {
    pybind11::gil_scoped_release no_gil;
    out = a.empty({x->size(0), os});
    lse = a.empty({B, Hq, L}, at::kFloat);
    if (Ns) lse_s = a.empty({B, Hq, Ns}, at::kFloat);      // ahead of the launches: no memory of a kernel that may still run
    const void *k = s.block(*x, 0, kc), *vv = s.block(*x, 0, vc);
    const void *ks = Ns ? s.block(*x, text, kc) : nullptr, *vs = Ns ? s.block(*x, text, vc) : nullptr;
    LAUNCH(ksa_attn_fwd, x->const_data_ptr(), k, vv, ks, vs, out.mutable_data_ptr(), lse.mutable_data_ptr(), B, Hq, Hkv, D, L, L, Ns, rs,
           L * rs, rs, L * rs, rs, L * rs, rs, Ns * rs, rs, Ns * rs, os, L * os, 0, 0, 0, (int)s.chunk, s.n_sum > 1 ? (int)s.n_sum : 1,
           (int)s.window, (int)s.tok_window, s.scale, nullptr, nullptr, a.stream());
    if (Ns) {
      const Beside beside(true);
      LAUNCH(ksa_summary_attn_fwd, s.block(*x, text, 0), k, vv, ks, vs, s.block_mut(out, text, 0), lse_s.mutable_data_ptr(), B, Hq, Hkv,
             D, Ns, L, rs, Ns * rs, rs, L * rs, rs, L * rs, rs, Ns * rs, rs, Ns * rs, os, Ns * os, (int)s.chunk, (int)s.n_sum, 0, 0, 0,
             s.scale, a.stream());
    }
  }
  return Py_BuildValue("(NNN)", wrap(out), wrap(lse), Ns ? wrap(lse_s) : none());
  END_HANDLE_TH_ERRORS
}

// attention_bwd(qkv, out, lse, summary lse | None, dout, B, .., scale) -> dqkv, by the fused kernel (head dim 128)
PyObject* py_attention_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *o = a.tensor(), *lse = a.tensor(at::kFloat), *lse_s = a.tensor(at::kFloat, true), *g = a.tensor();
  PackedShape s;
  s.read(a);
  if (!a.ok() || !s.ok(x) || s.D != 128 || !packed2d(o) || !packed2d(g) || o->size(0) != x->size(0) || o->size(1) != s.q_cols() ||
      g->sizes() != o->sizes() || !lse->is_contiguous() || lse->numel() != s.B * s.Hq * s.L || (s.Ns > 0) != (lse_s != nullptr))
    return none();
  if (lse_s && !(lse_s->is_contiguous() && lse_s->numel() == s.B * s.Hq * s.Ns)) return none();
  if (reinterpret_cast<uintptr_t>(o->const_data_ptr()) % 16 != 0) return none();      // a saved-tensor hook gives any address
  const int B = (int)s.B, L = (int)s.L, Ns = (int)s.Ns, Hq = (int)s.Hq, Hkv = (int)s.Hkv, D = (int)s.D;
  const long long rs = x->stride(0), text = s.B * s.L, kc = s.q_cols(), vc = kc + s.Hkv * s.D, os = s.q_cols();
  Tensor d;
  {
    pybind11::gil_scoped_release no_gil;
    d = a.empty(x->sizes());
    const long long ds = d.stride(0);
    Tensor stats = a.empty({2, B, Hq, (L + 127) / 128 * 128}, at::kFloat), dq32 = a.empty({B, L, Hq, D}, at::kFloat), part_k, part_v;
    if (Ns && ksa_attn_bwd_num_segments(L) > 1) {
      part_k = a.empty({B, Ns, Hkv, D}, at::kFloat).zero_();
      part_v = a.empty({B, Ns, Hkv, D}, at::kFloat).zero_();
    }
    void *pk = part_k.defined() ? part_k.mutable_data_ptr() : nullptr, *pv = part_v.defined() ? part_v.mutable_data_ptr() : nullptr;
    const void *k = s.block(*x, 0, kc), *vv = s.block(*x, 0, vc);
    const void *ks = Ns ? s.block(*x, text, kc) : nullptr, *vs = Ns ? s.block(*x, text, vc) : nullptr;
    void *dk = s.block_mut(d, 0, kc), *dv = s.block_mut(d, 0, vc);
    void *dks = Ns ? s.block_mut(d, text, kc) : nullptr, *dvs = Ns ? s.block_mut(d, text, vc) : nullptr;
    check("ksa_attn_bwd_fused",
          ksa_attn_bwd_fused(x->const_data_ptr(), k, vv, ks, vs, o->const_data_ptr(), g->const_data_ptr(), lse->const_data_ptr(),
                             stats.mutable_data_ptr(), dq32.mutable_data_ptr(), d.mutable_data_ptr(), dk, dv, dks, dvs, B, Hq, Hkv, D, L,
                             L, Ns, rs, L * rs, rs, L * rs, rs, L * rs, rs, Ns * rs, rs, Ns * rs, os, L * os, ds, L * ds, ds, L * ds, ds,
                             L * ds, ds, Ns * ds, ds, Ns * ds, 0, 0, 0, (int)s.chunk, s.n_sum > 1 ? (int)s.n_sum : 1, (int)s.window,
                             (int)s.tok_window, s.scale, pk, pv, nullptr, nullptr, a.stream()), 3);
    if (Ns)
      LAUNCH(ksa_summary_attn_bwd, s.block(*x, text, 0), k, vv, ks, vs, s.block(*o, text, 0), s.block(*g, text, 0), lse_s->const_data_ptr(),
             s.block_mut(d, text, 0), dk, dv, dks, dvs, B, Hq, Hkv, D, Ns, L, rs, Ns * rs, rs, L * rs, rs, L * rs, rs, Ns * rs, rs, Ns * rs,
             os, Ns * os, ds, Ns * ds, ds, L * ds, ds, L * ds, ds, Ns * ds, ds, Ns * ds, (int)s.chunk, (int)s.n_sum, 0, 0, 0, s.scale, pk,
             pv, Ns, a.stream());
  }
  return wrap(d);
  END_HANDLE_TH_ERRORS
}

bool aligned(const Tensor* t) { return (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15) == 0; }

// The four tensors of a cache in four bits: codes [B, H, cap, D / 2], scales [B, H, cap, D / 32, 2].
struct Int4Cache {
  const Tensor *k, *ks, *v, *vs;
  int B = 0, H = 0, cap = 0, D = 0;
  explicit Int4Cache(Args& a) : k(a.tensor(at::kByte)), ks(a.tensor()), v(a.tensor(at::kByte)), vs(a.tensor()) {}
  bool ok() {
    if (k->dim() != 4 || ks->dim() != 5 || k->sizes() != v->sizes() || ks->sizes() != vs->sizes()) return false;
    for (int i = 0; i < 4; ++i)
      if (!fits(k->size(i)) || k->size(i) > INT_MAX / 2) return false;
    B = (int)k->size(0); H = (int)k->size(1); cap = (int)k->size(2); D = (int)(2 * k->size(3));
    if (D % 32 != 0 || cap % 16 != 0 || ks->size(0) != B || ks->size(1) != H || ks->size(2) != cap || ks->size(3) != D / 32 || ks->size(4) != 2)
      return false;
    for (const Tensor* t : {k, ks, v, vs})
      if (!t->is_contiguous() || !aligned(t)) return false;
    return true;
  }
};
bool ints(const Tensor* t, at::IntArrayRef sizes) { return t->sizes() == sizes && t->is_contiguous(); }
bool eights(const Tensor* t) {       // rows of the last dimension, on 16-byte boundaries
  if (t->stride(-1) != 1 || !aligned(t)) return false;
  for (int64_t i = 0; i + 1 < t->dim(); ++i)
    if (t->stride(i) % 8 != 0) return false;
  return true;
}
bool differentiated(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// int4_cache_write(k cache, k scales, v cache, v scales, k_new, v_new, slots, distinct) -> True
PyObject* py_int4_cache_write(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  Int4Cache c(a);
  const Tensor *k = a.tensor(), *x = a.tensor(), *slots = a.tensor(at::kInt);
  const int distinct = a.integer() != 0;
  if (!a.ok() || !c.ok() || k->dim() != 4 || k->sizes() != x->sizes() || k->strides() != x->strides() || !eights(k) || !eights(x) ||
      k->size(0) != c.B || k->size(2) != c.H || k->size(3) != c.D || !fits(k->size(1)) || !ints(slots, {k->size(0), k->size(1)}) ||
      differentiated({k, x}))
    return none();
  const int T = (int)k->size(1);
  {
    pybind11::gil_scoped_release no_gil;
    Tensor last;
    if (!distinct && ksa_int4_cache_write_table(c.B, T, c.H, c.D, c.cap)) last = a.empty({c.B, c.cap}, at::kInt);
    LAUNCH(ksa_int4_cache_write, k->const_data_ptr(), x->const_data_ptr(), c.k->mutable_data_ptr(), c.ks->mutable_data_ptr(),
           c.v->mutable_data_ptr(), c.vs->mutable_data_ptr(), slots->const_data_ptr(), last.defined() ? last.mutable_data_ptr() : nullptr, c.B, T,
           c.H, c.D, c.cap, k->stride(0), k->stride(1), k->stride(2), distinct, a.stream());
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// int4_cache_read(k cache, k scales, v cache, v scales, start, rows) -> (k, v)
PyObject* py_int4_cache_read(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  Int4Cache c(a);
  const Tensor* start = a.tensor(at::kInt);
  const long long rows = a.integer();
  if (!a.ok() || !c.ok() || !vector(start, c.B) || rows <= 0) return none();
  Tensor k, x;
  {
    pybind11::gil_scoped_release no_gil;
    k = a.empty({c.B, c.H, rows, c.D});
    x = a.empty({c.B, c.H, rows, c.D});
    LAUNCH(ksa_int4_cache_read, c.k->const_data_ptr(), c.ks->const_data_ptr(), c.v->const_data_ptr(), c.vs->const_data_ptr(),
           start->const_data_ptr(), k.mutable_data_ptr(), x.mutable_data_ptr(), c.B, c.H, c.D, c.cap, (int)rows, a.stream());
  }
  return wrap(k, x);
  END_HANDLE_TH_ERRORS
}

// int4_decode_attention(q, k cache, k scales, v cache, v scales, start, length, scale) -> out
PyObject* py_int4_decode_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor* q = a.tensor();
  Int4Cache c(a);
  const Tensor *start = a.tensor(at::kInt), *length = a.tensor(at::kInt);
  const float scale = a.real();
  if (!a.ok() || !c.ok() || q->dim() != 4 || !eights(q) || q->size(0) != c.B || q->size(3) != c.D || (c.D != 64 && c.D != 128) || !fits(q->size(1)) ||
      !fits(q->size(2)) || q->size(2) % c.H != 0 || !ints(start, {q->size(0), q->size(1)}) || !ints(length, {q->size(0), q->size(1)}) ||
      differentiated({q}))
    return none();
  const int Tq = (int)q->size(1), Hq = (int)q->size(2);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = a.empty({c.B, Tq, Hq, c.D});
    const long long floats = ksa_int4_attn_workspace(c.B, Tq, Hq, c.H, c.D, c.cap);
    Tensor workspace;
    if (floats > 0) workspace = a.empty({(int64_t)floats}, at::kFloat);
    LAUNCH(ksa_int4_decode_attn, q->const_data_ptr(), c.k->const_data_ptr(), c.ks->const_data_ptr(), c.v->const_data_ptr(),
           c.vs->const_data_ptr(), start->const_data_ptr(), length->const_data_ptr(), floats > 0 ? workspace.mutable_data_ptr() : nullptr, out.mutable_data_ptr(), c.B,
           Tq, Hq, c.H, c.D, c.cap, q->stride(0), q->stride(1), q->stride(2), scale, a.stream());
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// int4_linear(x, codes, scales, glu) -> y [..., N], at most 32 rows (glu: [..., N / 2], at most 16)
PyObject* py_int4_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor *x = a.tensor(), *w = a.tensor(at::kByte), *s = a.tensor();
  const int glu = a.integer() != 0;
  if (!a.ok() || !packed2d(w) || s->dim() != 3 || !s->is_contiguous() || !aligned(w) || !aligned(s) || x->dim() < 1) return none();
  const long long N = w->size(0), K = 2 * w->size(1), groups = s->size(0), pitch = s->size(1), M = x->numel() / K;
  if (K != x->size(-1) || M > (glu || N * K <= 4 << 20 ? 16 : 32) || !fits(N) || !fits(K) || pitch != (N + 3) / 4 * 4 || s->size(2) != 2 || K % groups != 0 ||
      (K / groups != 32 && K / groups != 64 && K / groups != 128) || !(x->is_contiguous() || (x->dim() == 2 && eights(x) && (M <= 16 || x->stride(0) >= K))) || !aligned(x) ||
      (glu && N % 2 != 0) || differentiated({x}))
    return none();
  const long long out = glu ? N / 2 : N;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    auto sizes = x->sizes().vec();
    sizes.back() = out;
    y = a.empty(sizes);
    LAUNCH(ksa_int4_linear, x->const_data_ptr(), w->const_data_ptr(), s->const_data_ptr(), y.mutable_data_ptr(), (int)M, (int)N, (int)K,
           (int)(K / groups), (int)pitch, x->is_contiguous() ? K : x->stride(0), out, glu, a.stream());      // (one row is contiguous at any pitch)
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------------------ post-training
// The differentiated calls of these operators are autograd nodes of this file: through Python a loss and its gradient took 150 us, whatever their size.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int token_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : t.scalar_type() == at::kHalf ? 2 : -1;
}
bool wants_gradient(const Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }
at::TensorOptions on(const Tensor& t, at::ScalarType type) { return at::TensorOptions().dtype(type).device(t.device()); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// What a backward pass of kernels returns: no graph of it exists, so whoever differentiates it again gets an error.
Tensor differentiated_once(const Tensor& t) {
  if (!c10::GradMode::is_enabled() || !t.defined()) return t;
  Tensor leaf = t.detach();
  leaf.set_requires_grad(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that can be differentiated once", 1);
  return (*error)({leaf})[0];
}

// grad_norm(gradients, targets | None, 0: norm | 1: and factor | 2: clip, scale, largest norm) -> norm, or (norm, factor)
PyObject* py_grad_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  PyObject *grads = a.next(), *out = a.next();
  const long long what = a.integer();
  const bool clip = what == 2;
  const float scale = a.real(), most = a.real();
  if (!a.ok() || !(PyList_CheckExact(grads) || PyTuple_CheckExact(grads)) || (out != Py_None && !(PyList_CheckExact(out) || PyTuple_CheckExact(out))))
    return none();
  // (another thread may empty the lists while this one works without the interpreter's lock)
  const auto held_grads = pybind11::reinterpret_steal<pybind11::object>(PySequence_Tuple(grads));
  const auto held_out = out == Py_None ? pybind11::object() : pybind11::reinterpret_steal<pybind11::object>(PySequence_Tuple(out));
  if (!held_grads || (out != Py_None && !held_out)) throw python_error();
  grads = held_grads.ptr();
  if (out != Py_None) out = held_out.ptr();
  const Py_ssize_t count = PyTuple_GET_SIZE(grads);
  if (count == 0 || count > INT_MAX || (out != Py_None && PyTuple_GET_SIZE(out) != count) || !(scale > 0.f && std::isfinite(scale)) || !(most >= 0.f))
    return none();
  std::vector<const void*> src(count);
  std::vector<void*> dst(clip ? count : 0);
  std::vector<long long> meta(count);
  std::vector<const Tensor*> to(dst.size());
  const auto plain = [&](PyObject* o) -> const Tensor* {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (t.numel() > 0 ? !a.dense(t) : !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
    return token_type(t) >= 0 && t.is_non_overlapping_and_dense() ? &t : nullptr;
  };
  const Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor* t = plain(PyTuple_GET_ITEM(grads, i));
    if (!t || (first && t->device() != first->device())) return none();
    if (!first) first = t;
    src[i] = t->const_data_ptr();
    meta[i] = 4 * (long long)t->numel() + token_type(*t);
    if (!clip) continue;
    const Tensor* o = out == Py_None ? t : plain(PyTuple_GET_ITEM(out, i));
    if (!o || o->is_inference() || (o != t && (o->device() != t->device() || o->scalar_type() != t->scalar_type() || o->sizes() != t->sizes() ||
                                               o->strides() != t->strides())))
      return none();
    to[i] = o;
    dst[i] = o->mutable_data_ptr();
  }
  if (first->device().index() != c10::cuda::current_device()) return none();
  if (clip) {                              // memory that is written must not be another tensor's too
    struct Span { uintptr_t lo, hi; bool written; };
    std::vector<Span> spans;
    spans.reserve(out == Py_None ? count : 2 * count);
    bool sorted = true;                    // (as the views of one buffer are)
    const auto add = [&](uintptr_t lo, uintptr_t bytes, bool written) {
      sorted = sorted && (spans.empty() || spans.back().lo <= lo);
      spans.push_back({lo, lo + bytes, written});
    };
    for (Py_ssize_t i = 0; i < count; ++i) {
      const uintptr_t bytes = (uintptr_t)(meta[i] >> 2) * ((meta[i] & 3) == 0 ? 4 : 2), s = reinterpret_cast<uintptr_t>(src[i]), d = reinterpret_cast<uintptr_t>(dst[i]);
      if (bytes == 0) continue;
      add(d, bytes, true);
      if (s != d) add(s, bytes, false);
    }
    if (!sorted) std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.lo < y.lo; });
    uintptr_t any = 0, written = 0;
    for (const Span& s : spans) {
      if (s.lo < (s.written ? any : written)) return none();
      any = std::max(any, s.hi);
      if (s.written) written = std::max(written, s.hi);
    }
  }
  Tensor norm, factor;
  {
    pybind11::gil_scoped_release no_gil;
    const int parts = ksa_grad_norm_parts((int)count);
    const Tensor partial = at::empty({parts + 1}, on(*first, at::kDouble));
    norm = at::empty({}, on(*first, at::kFloat));
    if (what == 1) factor = at::empty({}, on(*first, at::kFloat));
    double* sums = static_cast<double*>(partial.mutable_data_ptr());
    LAUNCH_SEVERAL(2, ksa_grad_norm, src.data(), clip ? dst.data() : nullptr, meta.data(), (int)count, scale, most, sums, norm.mutable_data_ptr(),
                   what == 1 ? factor.mutable_data_ptr() : sums + parts, stream_of(*first));
    for (const Tensor* o : to) o->unsafeGetTensorImpl()->bump_version();
  }
  return what == 1 ? wrap(norm, factor) : wrap(norm);
  END_HANDLE_TH_ERRORS
}

// Tokens as rows or packed: the rules of _sequences in ops/token_losses.py.
struct TokenArgs {
  const Tensor* y = nullptr;
  const Tensor* mask = nullptr;
  const Tensor* cu = nullptr;
  long long n = 0, length = 0;
  int sequences = 0;

  const void* offsets() const { return cu ? cu->const_data_ptr() : nullptr; }
  int wide() const { return cu && cu->scalar_type() == at::kLong; }
};
const Tensor* token_values(Args& a, bool optional = false) {
  PyObject* o = a.next();
  if (optional && o == Py_None) return nullptr;
  if (!THPVariable_CheckExact(o)) { a.plain = false; return nullptr; }
  const Tensor& t = THPVariable_Unpack(o);
  if (!a.dense(t) || token_type(t) < 0 || !t.is_contiguous()) a.plain = false;
  return &t;
}
const Tensor* token_integers(Args& a, std::initializer_list<at::ScalarType> types) {
  PyObject* o = a.next();
  if (o == Py_None) return nullptr;
  if (!THPVariable_CheckExact(o)) { a.plain = false; return nullptr; }
  const Tensor& t = THPVariable_Unpack(o);
  if (!a.dense(t) || std::find(types.begin(), types.end(), t.scalar_type()) == types.end() || !t.is_contiguous()) a.plain = false;
  return &t;
}
bool token_rows(TokenArgs& t) {
  if (t.mask && t.mask->sizes() != t.y->sizes()) return false;
  t.n = t.y->numel();
  if (t.cu) {
    t.sequences = (int)t.cu->numel() - 1;
    return t.cu->dim() == 1 && t.cu->numel() <= INT_MAX && (t.y->dim() == 1 || (t.y->dim() == 2 && t.y->size(0) == 1));
  }
  if (t.y->dim() != 1 && t.y->dim() != 2) return false;
  t.length = t.y->size(-1);
  t.sequences = t.y->dim() == 1 ? 1 : (int)t.y->size(0);
  return t.n / t.length <= INT_MAX;
}
bool same_shape(const Tensor* t, const Tensor* y) { return !t || t->sizes() == y->sizes(); }
double real64(PyObject* o, bool& plain) {
  const double x = PyFloat_Check(o) || PyLong_Check(o) ? PyFloat_AsDouble(o) : (plain = false, 0.0);
  if (PyErr_Occurred()) { PyErr_Clear(); plain = false; }
  return x;
}

struct PolicyCall {
  TokenArgs t;
  const Tensor *old = nullptr, *ref = nullptr, *adv = nullptr;
  int adv_by_sequence = 0, by_sequence = 0;
  double bounds[4] = {0, 0, 0, 0};
  float beta = 0;

  // fp32 values of the buffer in front of the partial sums: gradients up to the normaliser (only where wanted), then normalisers
  static long long inv_at(long long n, bool keep) { return keep ? (n + 3) / 4 * 4 : 0; }
  static long long partial_at(long long n, int sequences, bool keep) { return inv_at(n, keep) + (std::max(sequences, 1) + 3) / 4 * 4; }

  std::tuple<Tensor, Tensor, Tensor> run(bool keep) const {                 // {loss, statistics, buffer}
    const Tensor& y = *t.y;
    const Tensor loss = at::empty({}, on(y, at::kFloat)), stats = at::empty({3}, on(y, at::kFloat));
    const long long sums = partial_at(t.n, t.sequences, keep);
    const Tensor work = at::empty({(int64_t)(sums + 8 * ksa_token_loss_units(t.n, t.sequences))}, on(y, at::kFloat));
    float* at = static_cast<float*>(work.mutable_data_ptr());
    const int types = token_type(y) | token_type(*old) << 4 | (ref ? token_type(*ref) : 0) << 8 | token_type(*adv) << 12;
    LAUNCH_SEVERAL(2, ksa_policy_loss, y.const_data_ptr(), old->const_data_ptr(), ref ? ref->const_data_ptr() : nullptr, adv->const_data_ptr(),
                   t.mask ? t.mask->const_data_ptr() : nullptr, t.offsets(), t.wide(), keep ? at : nullptr, at + sums, at + inv_at(t.n, keep), loss.mutable_data_ptr(), stats.mutable_data_ptr(), types, t.n, t.sequences, t.length,
                   adv_by_sequence, by_sequence, bounds, beta, stream_of(y));
    return {loss, stats, work};
  }
};
struct PolicyNode : public torch::autograd::Function<PolicyNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& y, const PolicyCall* call) {
    auto [loss, stats, work] = call->run(true);
    ctx->save_for_backward({work, call->t.cu ? *call->t.cu : Tensor()});
    ctx->saved_data["sequences"] = (int64_t)call->t.sequences;
    ctx->saved_data["length"] = (int64_t)call->t.length;
    ctx->saved_data["by_sequence"] = (int64_t)call->by_sequence;
    ctx->saved_data["shape"] = y.sizes().vec();
    ctx->saved_data["type"] = (int64_t)y.scalar_type();
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);          // (the statistics' would be zeros in memory of their own)
    return {loss, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &work = saved[0], &cu = saved[1], &dloss = grads[0];
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor dy = at::empty(ctx->saved_data["shape"].toIntVector(), on(work, type));
    const float* at = static_cast<const float*>(work.const_data_ptr());
    const long long n = dy.numel();
    LAUNCH(ksa_policy_loss_bwd, at, at + PolicyCall::inv_at(n, true), dloss.const_data_ptr(), dy.mutable_data_ptr(), token_type(dy),
           cu.defined() ? cu.const_data_ptr() : nullptr, cu.defined() && cu.scalar_type() == at::kLong, n, (int)ctx->saved_data["sequences"].toInt(),
           ctx->saved_data["length"].toInt(), (int)ctx->saved_data["by_sequence"].toInt(), stream_of(work));
    return {differentiated_once(dy), Tensor()};
  }
};

// policy_loss(y, old, advantages, ref | None, mask | None, cu | None, clip_low, clip_high, kl_coef, by_sequence) -> (loss, statistics)
PyObject* py_policy_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  PolicyCall c;
  c.t.y = token_values(a);
  c.old = token_values(a);
  c.adv = token_values(a);
  c.ref = token_values(a, true);
  c.t.mask = token_integers(a, {at::kBool, at::kByte});
  c.t.cu = token_integers(a, {at::kInt, at::kLong});
  const double low = real64(a.next(), a.plain), high = real64(a.next(), a.plain);
  c.beta = a.real();
  c.by_sequence = a.integer() != 0;
  if (!a.ok() || !token_rows(c.t) || !same_shape(c.old, c.t.y) || !same_shape(c.ref, c.t.y) || !(low >= 0 && low <= 1 && high >= 0) || !std::isfinite(c.beta))
    return none();
  c.adv_by_sequence = !same_shape(c.adv, c.t.y);
  if (c.adv_by_sequence && !(c.adv->numel() == c.t.sequences && (c.adv->dim() == 1 || (c.adv->dim() == 2 && c.adv->size(1) == 1)))) return none();
  if (wants_gradient(*c.old) || wants_gradient(*c.adv) || (c.ref && wants_gradient(*c.ref))) return none();
  c.bounds[0] = std::log1p(high);
  c.bounds[1] = low < 1 ? std::log1p(-low) : -INFINITY;
  c.bounds[2] = 1 + high;
  c.bounds[3] = 1 - low;
  Tensor loss, stats;
  {
    pybind11::gil_scoped_release no_gil;
    if (wants_gradient(*c.t.y)) {
      auto made = PolicyNode::apply(*c.t.y, &c);
      loss = made[0];
      stats = made[1];
    } else {
      std::tie(loss, stats, std::ignore) = c.run(false);
    }
  }
  return wrap(loss, stats);
  END_HANDLE_TH_ERRORS
}

struct PreferenceCall {
  TokenArgs t;
  const Tensor* ref = nullptr;
  float beta = 0, smoothing = 0;

  std::tuple<Tensor, Tensor, Tensor> run() const {          // {loss, rewards, coefficients with the partial sums behind them}
    const Tensor& y = *t.y;
    const Tensor loss = at::empty({}, on(y, at::kFloat)), rewards = at::empty({t.sequences / 2, 2}, on(y, at::kFloat));
    const long long sums = (t.sequences + 3) / 4 * 4;
    const Tensor work = at::empty({(int64_t)(sums + 2 * ksa_token_loss_units(t.n, t.sequences))}, on(y, at::kFloat));
    float* at = static_cast<float*>(work.mutable_data_ptr());
    LAUNCH_SEVERAL(2, ksa_preference_loss, y.const_data_ptr(), ref ? ref->const_data_ptr() : nullptr, t.mask ? t.mask->const_data_ptr() : nullptr, t.offsets(), t.wide(),
                   at + sums, at, rewards.mutable_data_ptr(), loss.mutable_data_ptr(),
                   token_type(y) | (ref ? token_type(*ref) : 0) << 4, t.n, t.sequences, t.length, beta, smoothing, stream_of(y));
    return {loss, rewards, work};
  }
};
struct PreferenceNode : public torch::autograd::Function<PreferenceNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& y, const PreferenceCall* call) {
    auto [loss, rewards, work] = call->run();
    ctx->save_for_backward({work, call->t.mask ? *call->t.mask : Tensor(), call->t.cu ? *call->t.cu : Tensor()});
    ctx->saved_data["sequences"] = (int64_t)call->t.sequences;
    ctx->saved_data["length"] = (int64_t)call->t.length;
    ctx->saved_data["shape"] = y.sizes().vec();
    ctx->saved_data["type"] = (int64_t)y.scalar_type();
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &coef = saved[0], &mask = saved[1], &cu = saved[2], &dloss = grads[0];
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor dy = at::empty(ctx->saved_data["shape"].toIntVector(), on(coef, type));
    LAUNCH(ksa_preference_loss_bwd, mask.defined() ? mask.const_data_ptr() : nullptr, coef.const_data_ptr(), dloss.const_data_ptr(), dy.mutable_data_ptr(),
           token_type(dy), cu.defined() ? cu.const_data_ptr() : nullptr, cu.defined() && cu.scalar_type() == at::kLong, dy.numel(), (int)ctx->saved_data["sequences"].toInt(),
           ctx->saved_data["length"].toInt(), stream_of(coef));
    return {differentiated_once(dy), Tensor()};
  }
};

// preference_loss(y, ref | None, mask | None, cu | None, beta, label_smoothing) -> (loss, rewards)
PyObject* py_preference_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  PreferenceCall c;
  c.t.y = token_values(a);
  c.ref = token_values(a, true);
  c.t.mask = token_integers(a, {at::kBool, at::kByte});
  c.t.cu = token_integers(a, {at::kInt, at::kLong});
  c.beta = a.real();
  c.smoothing = a.real();
  if (!a.ok() || !token_rows(c.t) || c.t.sequences % 2 != 0 || c.t.sequences == 0 || !same_shape(c.ref, c.t.y) || !std::isfinite(c.beta) ||
      !(c.smoothing >= 0 && c.smoothing <= 1) || (c.ref && wants_gradient(*c.ref)))
    return none();
  Tensor loss, rewards;
  {
    pybind11::gil_scoped_release no_gil;
    if (wants_gradient(*c.t.y)) {
      auto made = PreferenceNode::apply(*c.t.y, &c);
      loss = made[0];
      rewards = made[1];
    } else {
      std::tie(loss, rewards, std::ignore) = c.run();
    }
  }
  return wrap(loss, rewards);
  END_HANDLE_TH_ERRORS
}

struct LogProbsCall {
  const Tensor* labels = nullptr;
  long long ignore = 0, pad = 0, columns = 0, slab_bytes = 0, plane_bytes = 0, keep_width = 0;
  float tau = 1;
};
struct LogProbsKept {
  Tensor y, dense, kept, codes;            // kept, in words: rows, row_label, place (T each), count (4), log-sums (2 T), maxima of the kept logits
};
// Columns of the vocabulary that the backward pass takes at a time (_slab in ops/log_probs.py).
long long slab_of(long long padded, long long V, long long bytes) {
  return std::min((V + 63) / 64 * 64, std::max(256ll, bytes / (2 * padded) / 256 * 256));
}
LogProbsKept log_probs(const Tensor& h, const Tensor& w, const LogProbsCall& c, bool grad) {
  const long long T = c.labels->numel(), V = w.size(0), D = w.size(1), padded = (T + c.pad - 1) / c.pad * c.pad;
  LogProbsKept k;
  k.y = at::empty(c.labels->sizes(), on(h, at::kFloat));
  k.dense = at::empty({(int64_t)padded, (int64_t)((D + 63) / 64 * 64)}, on(h, at::kBFloat16));
  const long long slab = slab_of(padded, V, c.slab_bytes);
  const bool keep = grad && slab >= V && D >= c.keep_width;
  if (keep) k.codes = at::empty({(int64_t)padded, (int64_t)slab}, on(h, at::kShort));
  k.kept = at::empty({(int64_t)(5 * T + 4 + (keep ? (T + 3) / 4 * 4 * ((V + c.columns - 1) / c.columns) : 0))}, on(h, at::kInt));
  const Tensor work = at::empty({(int64_t)ksa_log_probs_work((int)T, (int)V)}, on(h, at::kFloat));
  int* kept = static_cast<int*>(k.kept.mutable_data_ptr());
  LAUNCH_SEVERAL(3, ksa_log_probs, h.const_data_ptr(), w.const_data_ptr(), c.labels->const_data_ptr(), k.dense.mutable_data_ptr(), kept, kept + T, kept + 2 * T,
                 kept + 3 * T, kept + 3 * T + 4, work.mutable_data_ptr(), k.y.mutable_data_ptr(), keep ? k.codes.mutable_data_ptr() : nullptr,
                 keep ? kept + 5 * T + 4 : nullptr, (int)T, (int)V, (int)D,
                 h.dim() == 2 ? h.stride(0) : D, w.stride(0), c.ignore, c.tau, stream_of(h));
  return k;
}
struct LogProbsNode : public torch::autograd::Function<LogProbsNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const LogProbsCall* call) {
    const LogProbsKept k = log_probs(h, w, *call, true);
    ctx->save_for_backward({k.dense, w, k.kept, k.codes});
    ctx->saved_data["rows"] = (int64_t)call->labels->numel();
    ctx->saved_data["shape"] = h.sizes().vec();
    ctx->saved_data["tau"] = (double)call->tau;
    ctx->saved_data["slab_bytes"] = (int64_t)call->slab_bytes;
    ctx->saved_data["plane_bytes"] = (int64_t)call->plane_bytes;
    return k.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &dense = saved[0], &w = saved[1], &kept = saved[2], &codes = saved[3];
    const long long T = ctx->saved_data["rows"].toInt(), V = w.size(0), D = w.size(1), padded = dense.size(0);
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const Tensor dy = grads[0].contiguous();
    const long long slab = codes.defined() ? codes.size(1) : slab_of(padded, V, ctx->saved_data["slab_bytes"].toInt());
    const Tensor dx = at::empty({(int64_t)padded, (int64_t)slab}, on(w, at::kBFloat16));
    Tensor dh, dh32, dw;
    const long long planes = slab < V ? 1 : std::max(1ll, std::min(64ll, (long long)ctx->saved_data["plane_bytes"].toInt() / (4 * padded * D)));
    if (need_h) {
      dh = at::empty(ctx->saved_data["shape"].toIntVector(), on(w, at::kBFloat16));
      dh32 = at::empty({(int64_t)(planes * padded * D + 1)}, on(w, at::kFloat));               // (the word behind them: how many were used)
    }
    if (need_w) dw = at::empty({(int64_t)V, (int64_t)D}, on(w, at::kBFloat16));
    const int* p = static_cast<const int*>(kept.const_data_ptr());
    LAUNCH_SEVERAL(3, ksa_log_probs_bwd, dense.const_data_ptr(), w.const_data_ptr(), p, p + T, p + 2 * T, p + 3 * T, p + 3 * T + 4, codes.defined() ? codes.const_data_ptr() : nullptr,
                   codes.defined() ? p + 5 * T + 4 : nullptr, dy.const_data_ptr(),
                   dx.mutable_data_ptr(), need_h ? dh32.mutable_data_ptr() : nullptr, need_h ? dh.mutable_data_ptr() : nullptr,
                   need_w ? dw.mutable_data_ptr() : nullptr, (int)T, (int)V, (int)D, w.stride(0), D, 0, 0, (int)slab, need_h ? (int)planes : 1, (float)ctx->saved_data["tau"].toDouble(),
                   stream_of(w));
    return {differentiated_once(dh), differentiated_once(dw), Tensor()};
  }
};

// linear_log_probs(h [..., D], w, labels [...], ignore_index, temperature, row pad, columns of a sum, slab bytes, plane bytes, least width of kept logits) -> y [...]
PyObject* py_linear_log_probs(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(v, n);
  const Tensor* h = a.tensor();
  PyObject* weight = a.next();
  if (!THPVariable_CheckExact(weight)) return none();
  const Tensor& w = THPVariable_Unpack(weight);
  LogProbsCall c;
  c.labels = a.tensor(at::kLong);
  c.ignore = a.integer();
  c.tau = a.real();
  c.pad = a.integer();
  c.columns = a.integer();
  PyObject *slab = a.next(), *planes = a.next();
  c.slab_bytes = PyLong_Check(slab) ? PyLong_AsLongLong(slab) : -1;
  c.plane_bytes = PyLong_Check(planes) ? PyLong_AsLongLong(planes) : -1;
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  c.keep_width = a.integer();
  if (!a.ok() || !a.dense(w) || w.scalar_type() != at::kBFloat16 || !rows2d(&w) || !aligned(&w) || w.size(1) % 8 != 0 || w.stride(0) % 8 != 0 ||
      w.stride(0) < w.size(1) || h->dim() < 1 || h->size(-1) != w.size(1) || c.labels->sizes() != h->sizes().slice(0, h->dim() - 1) ||
      !(h->is_contiguous() || rows2d(h)) || !c.labels->is_contiguous() || !fits(w.size(0)) || c.labels->numel() > INT_MAX / 4 || !(c.tau > 0 && std::isfinite(c.tau)) ||
      c.pad <= 0 || c.columns <= 0 || c.slab_bytes < 0 || c.plane_bytes < 0)
    return none();
  const bool grad = wants_gradient(*h) || wants_gradient(w);
  if (grad && PyObject_HasAttrString(weight, "main_grad")) return none();                  // its gradient goes to a buffer that Python knows
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = grad ? LogProbsNode::apply(*h, w, &c) : log_probs(*h, w, c, false).y;
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* py_launches(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(g_launches.load()); }

#define FN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FN(gemm), FN(linear), FN(linear_dw), FN(dual_linear), FN(rms_norm), FN(rms_norm_bwd), FN(qk_norm_rope),
                           FN(qk_norm_rope_bwd), FN(swiglu), FN(swiglu_bwd), FN(linear_swiglu), FN(gemm_swiglu), FN(norm_linear), FN(attention),
                           FN(attention_bwd), FN(int4_cache_write), FN(int4_cache_read),
                           FN(int4_decode_attention), FN(int4_linear), FN(grad_norm), FN(policy_loss), FN(preference_loss),
                           FN(linear_log_probs), FN(launches), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "ksa_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ksa_native() { return PyModule_Create(&g_module); }
