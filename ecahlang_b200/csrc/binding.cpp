// Python binding of the log-probability, paged-cache and draft entry points
// (include/ecah_sampler.h): checks torch tensors, allocates outputs, fills the
// argument structs and launches on the current torch stream.  A call costs a few
// microseconds of host time, where the same checks in Python cost more than the
// smallest kernels take.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "ecah_sampler.h"

namespace {

// The library's entry points and error class, handed over by bind().
PyObject* g_error = nullptr;
decltype(&ecah_token_logprobs) g_logprobs = nullptr;
decltype(&ecah_paged_append) g_append = nullptr;
decltype(&ecah_paged_decode) g_decode = nullptr;
decltype(&ecah_paged_prefill) g_prefill = nullptr;
decltype(&ecah_paged_copy) g_copy = nullptr;
decltype(&ecah_verify_drafts) g_verify = nullptr;
decltype(&ecah_status_string) g_status_string = nullptr;

[[noreturn]] void refuse(const std::string& why) { throw std::runtime_error(why); }

struct Status {
  int code;
  const char* what;
};

std::string type_name(at::ScalarType t) { return c10::toString(t); }

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// A tensor argument by position; an undefined tensor for None.
struct Args {
  PyObject* const* a;
  Py_ssize_t n;
  const at::Tensor* tensor(int i, const char* name, bool optional = false) const {
    PyObject* o = a[i];
    if (o == Py_None) {
      if (!optional) refuse(std::string(name) + ": a tensor is required");
      return nullptr;
    }
    if (!THPVariable_Check(o)) refuse(std::string(name) + ": expected a tensor");
    return &THPVariable_Unpack(o);
  }
  long integer(int i) const {
    const long v = PyLong_AsLong(a[i]);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); refuse("expected an integer"); }
    return v;
  }
  double real(int i) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); refuse("expected a number"); }
    return v;
  }
  bool truth(int i) const {
    const int v = PyObject_IsTrue(a[i]);
    if (v < 0) { PyErr_Clear(); refuse("expected a truth value"); }
    return v != 0;
  }
};

void need(const at::Tensor& t, const char* name, at::ScalarType type, int64_t numel, at::Device dev) {
  if (t.scalar_type() != type) refuse(std::string(name) + ": expected " + type_name(type) + ", got " + type_name(t.scalar_type()));
  if (t.device() != dev) refuse(std::string(name) + ": expected device " + dev.str() + ", got " + t.device().str());
  if (!t.is_contiguous()) refuse(std::string(name) + ": must be contiguous");
  if (t.numel() != numel)
    refuse(std::string(name) + ": expected " + std::to_string(numel) + " elements, got " + std::to_string(t.numel()));
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}

const void* checked_workspace(const at::Tensor& w, at::Device dev) {
  if (w.device() != dev || w.scalar_type() != at::kByte || !w.is_contiguous())
    refuse("workspace must be a contiguous uint8 tensor on the operands' device");
  if (reinterpret_cast<uintptr_t>(w.data_ptr()) % 16) refuse("workspace must be 16-byte aligned");
  return w.data_ptr();
}

// The entry point with the operands' device current and its current stream.
template <typename A>
void run(int (*entry)(const A*, void*), const A& args, at::Device dev, const char* what) {
  c10::cuda::CUDAGuard guard(dev);
  const int st = entry(&args, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (st != ECAH_OK) throw Status{st, what};
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Status& s) {
    PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "%s failed: %s (status %d)", s.what, g_status_string(s.code), s.code);
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

bool count_is(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

at::Tensor output(const at::Tensor* given, const char* name, at::IntArrayRef shape, at::ScalarType type, at::Device dev) {
  if (!given) return empty(shape, type, dev);
  int64_t n = 1;
  for (int64_t d : shape) n *= d;
  need(*given, name, type, n, dev);
  return *given;
}

// logits, token_ids, workspace, top_n, temperature, row_index, logprobs, entropy,
// top_ids, top_logprobs, vocab (-1: any)
PyObject* logprobs(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor& x = *in.tensor(0, "logits");
    if (x.dim() != 2) refuse("logits must be [R, V], got " + shape_of(x));
    ecah_logprob_args a = {};
    switch (x.scalar_type()) {
      case at::kHalf: a.dtype = ECAH_DTYPE_F16; break;
      case at::kBFloat16: a.dtype = ECAH_DTYPE_BF16; break;
      case at::kFloat: a.dtype = ECAH_DTYPE_F32; break;
      default: refuse("unsupported logits dtype " + type_name(x.scalar_type()));
    }
    if (!x.is_cuda()) refuse("logits must be a CUDA tensor (there is no CPU path)");
    const at::Device dev = x.device();
    const int64_t L = x.size(0), V = x.size(1);
    if (V < 1 || (V > 1 && x.stride(1) != 1)) refuse("logits rows must be contiguous and not empty");
    const long vocab = in.integer(10), top_n = in.integer(3);
    if (vocab >= 0 && V != vocab) refuse("logits must be [R, " + std::to_string(vocab) + "], got " + shape_of(x));
    if (top_n < 0 || top_n > ECAH_MAX_TOP_N) refuse("top_n must be in [0, " + std::to_string(ECAH_MAX_TOP_N) + "], got " + std::to_string(top_n));
    if (V > INT32_MAX || L > INT32_MAX) refuse("logits too large: " + shape_of(x));
    int64_t R = L;
    if (const at::Tensor* t = in.tensor(5, "row_index", true)) {
      R = t->numel();
      need(*t, "row_index", at::kInt, R, dev);
      if (L < 1 && R > 0) refuse("row_index into logits without rows");
      a.row_index = t->data_ptr<int32_t>();
      a.logit_rows = static_cast<int32_t>(L);
    }
    int64_t K = 0, shape[2] = {R, 0};
    int dims = 2;
    const at::Tensor* tok = in.tensor(1, "token_ids", true);
    if (tok) {
      dims = static_cast<int>(tok->dim());
      if (dims < 1 || dims > 2 || tok->size(0) != R)
        refuse("token_ids must be [" + std::to_string(R) + "] or [" + std::to_string(R) + ", K], got " + shape_of(*tok));
      K = dims == 2 ? tok->size(1) : 1;
      shape[1] = K;
      need(*tok, "token_ids", at::kInt, R * K, dev);
      if (K > INT32_MAX) refuse("too many tokens a row");
      a.token_ids = tok->data_ptr<int32_t>();
    }
    if (const at::Tensor* t = in.tensor(4, "temperature", true)) {
      need(*t, "temperature", at::kFloat, R, dev);
      a.temperature = t->data_ptr<float>();
    }
    const at::Tensor& ws = *in.tensor(2, "workspace");
    a.workspace = const_cast<void*>(checked_workspace(ws, dev));
    a.workspace_bytes = static_cast<size_t>(ws.numel());
    at::Tensor lp = output(in.tensor(6, "logprobs", true), "logprobs", at::IntArrayRef(shape, dims), at::kFloat, dev);
    at::Tensor ent = output(in.tensor(7, "entropy", true), "entropy", {R}, at::kFloat, dev);
    at::Tensor ids = output(in.tensor(8, "top_ids", true), "top_ids", {R, top_n}, at::kInt, dev);
    at::Tensor top = output(in.tensor(9, "top_logprobs", true), "top_logprobs", {R, top_n}, at::kFloat, dev);
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.rows = static_cast<int32_t>(R);
    a.vocab = static_cast<int32_t>(V);
    a.row_stride = L > 1 ? x.stride(0) : V;
    a.logits = x.data_ptr();
    a.tokens_per_row = static_cast<int32_t>(K);
    a.top_n = static_cast<int32_t>(top_n);
    a.logprobs = lp.data_ptr<float>();
    a.entropy = ent.data_ptr<float>();
    a.top_ids = ids.data_ptr<int32_t>();
    a.top_logprobs = top.data_ptr<float>();
    run(g_logprobs, a, dev, "ecah_token_logprobs");
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(lp), THPVariable_Wrap(ent), THPVariable_Wrap(ids), THPVariable_Wrap(top));
  });
}

int half_dtype(at::ScalarType t, const char* who) {
  if (t == at::kHalf) return ECAH_DTYPE_F16;
  if (t == at::kBFloat16) return ECAH_DTYPE_BF16;
  refuse("unsupported dtype " + type_name(t) + ": " + who + " takes float16 and bfloat16");
}

// Token and head strides of a [tokens, heads, head_dim] tensor.
void rows(const at::Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t D, at::ScalarType type, at::Device dev,
          int64_t* token_stride, int64_t* head_stride) {
  if (t.scalar_type() != type || t.device() != dev)
    refuse(std::string(name) + ": expected " + type_name(type) + " on " + dev.str() + ", got " + type_name(t.scalar_type()) + " on " + t.device().str());
  if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != D)
    refuse(std::string(name) + ": expected shape [" + std::to_string(tokens) + ", " + std::to_string(heads) + ", " + std::to_string(D) + "], got " + shape_of(t));
  *token_stride = tokens > 1 ? t.stride(0) : 0;
  *head_stride = heads > 1 ? t.stride(1) : 0;
  if (t.stride(2) != 1 || *token_stride % 8 || *head_stride % 8 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
    refuse(std::string(name) + ": rows of head_dim must be contiguous and 16-byte aligned");
}

// Blocks write rows in no order: none may lie on another.
void need_apart(const at::Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) refuse(std::string(name) + ": rows to be written share memory (an expanded tensor)");
}

// What a PagedAttention was made for: (num_qo_heads, num_kv_heads, head_dim,
// page_size, e4m3, max_batch, dtype code), or None.
struct Made {
  long hq = -1, hk, dim, page, e4m3, batch, dtype;
};

Made made_for(PyObject* o) {
  Made m;
  if (o == Py_None) return m;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 7) refuse("layout must be a tuple of 7");
  long v[7];
  for (int i = 0; i < 7; ++i) v[i] = PyLong_AsLong(PyTuple_GET_ITEM(o, i));
  return Made{v[0], v[1], v[2], v[3], v[4], v[5], v[6]};
}

// One layer's cache, without page lists.
void fill_layer(ecah_kv_cache& c, at::ScalarType type, at::Device dev, const at::Tensor& k, const at::Tensor& v,
                const at::Tensor* ks, const at::Tensor* vs, const Made& made) {
  if (k.dim() != 4 || v.sizes() != k.sizes()) refuse("k_cache and v_cache must be [num_pages, page_size, num_kv_heads, head_dim]");
  const at::ScalarType kv = k.scalar_type();
  const bool e4m3 = kv == at::kFloat8_e4m3fn;
  if ((kv != type && !e4m3) || v.scalar_type() != kv)
    refuse("cache must be " + type_name(type) + " or Float8_e4m3fn, got " + type_name(kv) + " and " + type_name(v.scalar_type()));
  if (k.device() != dev || v.device() != dev) refuse("cache must be on " + dev.str());
  const int64_t pages = k.size(0), page = k.size(1), heads = k.size(2), D = k.size(3);
  if (D != 64 && D != 96 && D != 128 && D != 192 && D != 256) refuse("head_dim " + std::to_string(D) + " is not one of 64, 96, 128, 192, 256");
  if (page < 1 || heads < 1) refuse("page_size and num_kv_heads must be positive");
  if (pages > INT32_MAX || page > INT32_MAX || heads > INT32_MAX) refuse("cache too large");
  if (made.hq >= 0 && (page != made.page || heads != made.hk || D != made.dim || e4m3 != (made.e4m3 != 0)))
    refuse("cache must be [pages, " + std::to_string(made.page) + ", " + std::to_string(made.hk) + ", " + std::to_string(made.dim) +
           "], got " + shape_of(k) + " " + type_name(kv));
  const int64_t unit = e4m3 ? 16 : 8;
  auto side = [&](const at::Tensor& t, const char* name, int64_t* p, int64_t* s, int64_t* h) {
    *p = pages > 1 ? t.stride(0) : 0;
    *s = page > 1 ? t.stride(1) : 0;
    *h = heads > 1 ? t.stride(2) : 0;
    if (t.stride(3) != 1 || *p % unit || *s % unit || *h % unit || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
      refuse(std::string(name) + ": rows of head_dim must be contiguous and 16-byte aligned");
  };
  side(k, "k_cache", &c.k_page_stride, &c.k_slot_stride, &c.k_head_stride);
  side(v, "v_cache", &c.v_page_stride, &c.v_slot_stride, &c.v_head_stride);
  if (e4m3) {
    if (!ks || !vs) refuse("an e4m3 cache needs k_scale and v_scale");
    for (const at::Tensor* t : {ks, vs}) {
      if (t->dim() != 3 || t->size(0) != pages || t->size(1) != heads || t->size(2) != page)
        refuse("scales must be [num_pages, num_kv_heads, page_size], got " + shape_of(*t));
      need(*t, "scale", at::kFloat, pages * heads * page, dev);
    }
    c.k_scale = ks->data_ptr<float>();
    c.v_scale = vs->data_ptr<float>();
    c.kv_dtype = ECAH_KV_E4M3;
  } else {
    if (ks || vs) refuse("a cache in the model dtype takes no scales");
    c.kv_dtype = kv == at::kHalf ? ECAH_DTYPE_F16 : ECAH_DTYPE_BF16;
  }
  c.num_pages = static_cast<int32_t>(pages);
  c.page_size = static_cast<int32_t>(page);
  c.num_kv_heads = static_cast<int32_t>(heads);
  c.head_dim = static_cast<int32_t>(D);
  c.k_cache = k.data_ptr();
  c.v_cache = v.data_ptr();
}

void fill_cache(ecah_kv_cache& c, at::ScalarType type, at::Device dev, const at::Tensor& k, const at::Tensor& v,
                const at::Tensor* ks, const at::Tensor* vs, const at::Tensor& indptr, const at::Tensor& indices, const Made& made) {
  fill_layer(c, type, dev, k, v, ks, vs, made);
  const int64_t n = indptr.numel();
  if (n < 1 || n > INT32_MAX) refuse("kv_indptr must have batch + 1 entries");
  need(indptr, "kv_indptr", at::kInt, n, dev);
  need(indices, "kv_indices", at::kInt, indices.numel(), dev);
  c.batch = static_cast<int32_t>(n - 1);
  c.kv_indptr = indptr.data_ptr<int32_t>();
  c.kv_indices = indices.data_ptr<int32_t>();
  c.num_indices = indices.numel();
}

void check_query(const at::Tensor& q, const Made& made, int dtype) {
  if (made.hq >= 0 && (q.dim() != 3 || q.size(1) != made.hq || dtype != made.dtype))
    refuse("q must be [tokens, " + std::to_string(made.hq) + ", " + std::to_string(made.dim) + "] in the model dtype, got " + shape_of(q) + " " +
           type_name(q.scalar_type()));
}

// q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale,
// v_scale, cos_sin, q_norm, k_norm, eps, interleaved, q_out, layout
PyObject* append(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 18)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor &k = *in.tensor(1, "k"), &v = *in.tensor(2, "v");
    const at::Tensor* q = in.tensor(0, "q", true);
    const at::ScalarType type = k.scalar_type();
    ecah_append_args a = {};
    a.dtype = half_dtype(type, "append");
    if (!k.is_cuda()) refuse("append needs CUDA tensors (there is no CPU path)");
    const at::Device dev = k.device();
    const Made made = made_for(raw[17]);
    fill_cache(a.cache, type, dev, *in.tensor(7, "k_cache"), *in.tensor(8, "v_cache"), in.tensor(9, "k_scale", true),
               in.tensor(10, "v_scale", true), *in.tensor(5, "kv_indptr"), *in.tensor(6, "kv_indices"), made);
    need_apart(*in.tensor(7, "k_cache"), "k_cache");
    need_apart(*in.tensor(8, "v_cache"), "v_cache");
    const int64_t heads = a.cache.num_kv_heads, D = a.cache.head_dim;
    if (k.dim() != 3) refuse("k must be [T, num_kv_heads, head_dim], got " + shape_of(k));
    const int64_t T = k.size(0);
    if (T > INT32_MAX) refuse("too many tokens");
    rows(k, "k", T, heads, D, type, dev, &a.k_token_stride, &a.k_head_stride);
    rows(v, "v", T, heads, D, type, dev, &a.v_token_stride, &a.v_head_stride);
    at::Tensor out;
    const at::Tensor *given = in.tensor(16, "q_out", true), *q_norm = in.tensor(12, "q_norm", true), *k_norm = in.tensor(13, "k_norm", true);
    if (q) {
      check_query(*q, made, a.dtype);
      if (q->dim() != 3 || q->size(1) < 1 || q->size(1) > INT32_MAX) refuse("q must be [T, num_qo_heads, head_dim], got " + shape_of(*q));
      const int64_t hq = q->size(1);
      rows(*q, "q", T, hq, D, type, dev, &a.q_token_stride, &a.q_head_stride);
      out = given ? *given : empty({T, hq, D}, type, dev);
      rows(out, "q_out", T, hq, D, type, dev, &a.qo_token_stride, &a.qo_head_stride);
      need_apart(out, "q_out");
      a.q = q->data_ptr();
      a.q_out = out.data_ptr();
      a.num_qo_heads = static_cast<int32_t>(hq);
    } else if (given || q_norm) {
      refuse("q_out and q_norm need q");
    }
    const at::Tensor &pos = *in.tensor(3, "positions"), &batch = *in.tensor(4, "batch_index");
    need(pos, "positions", at::kInt, T, dev);
    need(batch, "batch_index", at::kInt, T, dev);
    if (q_norm) { need(*q_norm, "q_norm", type, D, dev); a.q_norm = q_norm->data_ptr(); }
    if (k_norm) { need(*k_norm, "k_norm", type, D, dev); a.k_norm = k_norm->data_ptr(); }
    if (const at::Tensor* t = in.tensor(11, "cos_sin", true)) {
      if (t->dim() != 2 || t->size(0) < 1 || t->size(1) != D || t->size(0) > INT32_MAX)
        refuse("cos_sin must be [rows, " + std::to_string(D) + "], got " + shape_of(*t));
      need(*t, "cos_sin", at::kFloat, t->numel(), dev);
      a.cos_sin = t->data_ptr<float>();
      a.table_rows = static_cast<int32_t>(t->size(0));
    }
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.tokens = static_cast<int32_t>(T);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.positions = pos.data_ptr<int32_t>();
    a.batch_index = batch.data_ptr<int32_t>();
    a.eps = static_cast<float>(in.real(14));
    a.interleaved = in.truth(15);
    run(g_append, a, dev, "ecah_paged_append");
    if (!q) Py_RETURN_NONE;
    if (given) return Py_NewRef(raw[16]);
    return THPVariable_Wrap(out);
  });
}

// q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace, k_scale,
// v_scale, sm_scale (None: 1 / sqrt(head_dim)), out, lse (True: allocate), layout
PyObject* decode(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 13)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor& q = *in.tensor(0, "q");
    const at::ScalarType type = q.scalar_type();
    ecah_decode_args a = {};
    a.dtype = half_dtype(type, "decode");
    if (!q.is_cuda()) refuse("decode needs CUDA tensors (there is no CPU path)");
    const at::Device dev = q.device();
    const Made made = made_for(raw[12]);
    fill_cache(a.cache, type, dev, *in.tensor(4, "k_cache"), *in.tensor(5, "v_cache"), in.tensor(7, "k_scale", true),
               in.tensor(8, "v_scale", true), *in.tensor(1, "kv_indptr"), *in.tensor(2, "kv_indices"), made);
    const int64_t heads = a.cache.num_kv_heads, D = a.cache.head_dim, B = a.cache.batch;
    check_query(q, made, a.dtype);
    if (q.dim() != 3 || q.size(1) < 1 || q.size(1) % heads || q.size(1) > INT32_MAX)
      refuse("q must be [" + std::to_string(B) + ", num_qo_heads, " + std::to_string(D) + "] with num_qo_heads a multiple of " +
             std::to_string(heads) + ", got " + shape_of(q));
    if (made.hq >= 0 && B > made.batch) refuse(std::to_string(B) + " requests, max_batch is " + std::to_string(made.batch));
    const int64_t hq = q.size(1);
    rows(q, "q", B, hq, D, type, dev, &a.q_token_stride, &a.q_head_stride);
    const at::Tensor* given = in.tensor(10, "out", true);
    at::Tensor out = given ? *given : empty({B, hq, D}, type, dev);
    rows(out, "out", B, hq, D, type, dev, &a.out_token_stride, &a.out_head_stride);
    need_apart(out, "out");
    at::Tensor lse;
    const bool new_lse = raw[11] == Py_True;
    if (new_lse) lse = empty({B, hq}, at::kFloat, dev);
    else if (const at::Tensor* t = in.tensor(11, "lse", true)) lse = *t;
    if (lse.defined()) {
      need(lse, "lse", at::kFloat, B * hq, dev);
      a.lse = lse.data_ptr<float>();
    }
    const at::Tensor& last = *in.tensor(3, "kv_last_page_len");
    need(last, "kv_last_page_len", at::kInt, B, dev);
    const at::Tensor& ws = *in.tensor(6, "workspace");
    a.workspace = const_cast<void*>(checked_workspace(ws, dev));
    a.workspace_bytes = static_cast<size_t>(ws.numel());
    a.sm_scale = raw[9] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D))) : static_cast<float>(in.real(9));
    if (!(a.sm_scale > 0.0f) || std::isinf(a.sm_scale)) refuse("sm_scale must be positive and finite");
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.num_qo_heads = static_cast<int32_t>(hq);
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    a.kv_last_page_len = last.data_ptr<int32_t>();
    run(g_decode, a, dev, "ecah_paged_decode");
    PyObject* o = given ? Py_NewRef(raw[10]) : THPVariable_Wrap(out);
    if (raw[11] == Py_None) return o;
    return Py_BuildValue("(NN)", o, new_lse ? THPVariable_Wrap(lse) : Py_NewRef(raw[11]));
  });
}

// q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace,
// k_scale, v_scale, causal, sm_scale (None: 1 / sqrt(head_dim)), out, lse (True: allocate), layout
PyObject* prefill(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 15)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor& q = *in.tensor(0, "q");
    const at::ScalarType type = q.scalar_type();
    ecah_prefill_args a = {};
    a.dtype = half_dtype(type, "prefill");
    if (!q.is_cuda()) refuse("prefill needs CUDA tensors (there is no CPU path)");
    const at::Device dev = q.device();
    const Made made = made_for(raw[14]);
    fill_cache(a.cache, type, dev, *in.tensor(5, "k_cache"), *in.tensor(6, "v_cache"), in.tensor(8, "k_scale", true),
               in.tensor(9, "v_scale", true), *in.tensor(2, "kv_indptr"), *in.tensor(3, "kv_indices"), made);
    const int64_t heads = a.cache.num_kv_heads, D = a.cache.head_dim, B = a.cache.batch;
    check_query(q, made, a.dtype);
    if (q.dim() != 3 || q.size(1) < 1 || q.size(1) % heads || q.size(1) > INT32_MAX)
      refuse("q must be [T, num_qo_heads, " + std::to_string(D) + "] with num_qo_heads a multiple of " + std::to_string(heads) + ", got " + shape_of(q));
    if (made.hq >= 0 && B > made.batch) refuse(std::to_string(B) + " requests, max_batch is " + std::to_string(made.batch));
    const int64_t T = q.size(0), hq = q.size(1);
    if (T > INT32_MAX) refuse("too many tokens");
    rows(q, "q", T, hq, D, type, dev, &a.q_token_stride, &a.q_head_stride);
    const at::Tensor* given = in.tensor(12, "out", true);
    at::Tensor out = given ? *given : empty({T, hq, D}, type, dev);
    rows(out, "out", T, hq, D, type, dev, &a.out_token_stride, &a.out_head_stride);
    need_apart(out, "out");
    at::Tensor lse;
    const bool new_lse = raw[13] == Py_True;
    if (new_lse) lse = empty({T, hq}, at::kFloat, dev);
    else if (const at::Tensor* t = in.tensor(13, "lse", true)) lse = *t;
    if (lse.defined()) {
      need(lse, "lse", at::kFloat, T * hq, dev);
      a.lse = lse.data_ptr<float>();
    }
    const at::Tensor &qptr = *in.tensor(1, "qo_indptr"), &last = *in.tensor(4, "kv_last_page_len");
    need(qptr, "qo_indptr", at::kInt, B + 1, dev);
    need(last, "kv_last_page_len", at::kInt, B, dev);
    const at::Tensor& ws = *in.tensor(7, "workspace");
    a.workspace = const_cast<void*>(checked_workspace(ws, dev));
    a.workspace_bytes = static_cast<size_t>(ws.numel());
    a.causal = in.truth(10);
    a.sm_scale = raw[11] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D))) : static_cast<float>(in.real(11));
    if (!(a.sm_scale > 0.0f) || std::isinf(a.sm_scale)) refuse("sm_scale must be positive and finite");
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.tokens = static_cast<int32_t>(T);
    a.num_qo_heads = static_cast<int32_t>(hq);
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    a.qo_indptr = qptr.data_ptr<int32_t>();
    a.kv_last_page_len = last.data_ptr<int32_t>();
    run(g_prefill, a, dev, "ecah_paged_prefill");
    PyObject* o = given ? Py_NewRef(raw[12]) : THPVariable_Wrap(out);
    if (raw[13] == Py_None) return o;
    return Py_BuildValue("(NN)", o, new_lse ? THPVariable_Wrap(lse) : Py_NewRef(raw[13]));
  });
}

// src, dst, tokens (or None), caches: a sequence of (k_cache, v_cache, k_scale, v_scale), layout
PyObject* copy_pages(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor &src = *in.tensor(0, "src"), &dst = *in.tensor(1, "dst");
    if (!src.is_cuda()) refuse("copy_pages needs CUDA tensors (there is no CPU path)");
    const at::Device dev = src.device();
    const int64_t pairs = src.numel();
    if (pairs > INT32_MAX) refuse("too many pairs");
    need(src, "src", at::kInt, pairs, dev);
    need(dst, "dst", at::kInt, pairs, dev);
    ecah_copy_args a = {};
    if (const at::Tensor* t = in.tensor(2, "tokens", true)) {
      need(*t, "tokens", at::kInt, pairs, dev);
      a.tokens = t->data_ptr<int32_t>();
    }
    struct Ref {                                             // a new reference, dropped on every way out
      PyObject* o;
      ~Ref() { Py_XDECREF(o); }
    } seq{PySequence_Fast(raw[3], "caches: expected a sequence of (k_cache, v_cache, k_scale, v_scale)")};
    if (!seq.o) { PyErr_Clear(); refuse("caches: expected a sequence of (k_cache, v_cache, k_scale, v_scale)"); }
    const Py_ssize_t layers = PySequence_Fast_GET_SIZE(seq.o);
    const Made made = made_for(raw[4]);
    std::vector<void*> k(layers), v(layers);
    std::vector<float*> ks(layers), vs(layers);
    ecah_kv_cache first = {};
    for (Py_ssize_t i = 0; i < layers; ++i) {
      auto who = [&] { return "caches[" + std::to_string(i) + "]"; };
      PyObject* item = PySequence_Fast_GET_ITEM(seq.o, i);
      if (!(PyTuple_Check(item) || PyList_Check(item)) || PySequence_Fast_GET_SIZE(item) != 4)
        refuse(who() + ": expected (k_cache, v_cache, k_scale, v_scale)");
      const Args c{PySequence_Fast_ITEMS(item), 4};
      const at::Tensor &kc = *c.tensor(0, "k_cache"), &vc = *c.tensor(1, "v_cache");
      if (kc.scalar_type() != at::kHalf && kc.scalar_type() != at::kBFloat16 && kc.scalar_type() != at::kFloat8_e4m3fn)
        refuse(who() + ": unsupported cache dtype " + type_name(kc.scalar_type()));
      need_apart(kc, "k_cache");
      need_apart(vc, "v_cache");
      ecah_kv_cache one = {};
      fill_layer(one, kc.scalar_type(), dev, kc, vc, c.tensor(2, "k_scale", true), c.tensor(3, "v_scale", true), made);
      if (i == 0) {
        first = one;
      } else if (one.kv_dtype != first.kv_dtype || one.num_pages != first.num_pages || one.page_size != first.page_size ||
                 one.num_kv_heads != first.num_kv_heads || one.head_dim != first.head_dim || one.k_page_stride != first.k_page_stride ||
                 one.k_slot_stride != first.k_slot_stride || one.k_head_stride != first.k_head_stride ||
                 one.v_page_stride != first.v_page_stride || one.v_slot_stride != first.v_slot_stride || one.v_head_stride != first.v_head_stride) {
        refuse(who() + ": all layers must have one shape, dtype and set of strides");
      }
      k[i] = one.k_cache; v[i] = one.v_cache; ks[i] = one.k_scale; vs[i] = one.v_scale;
    }
    if (layers == 0) Py_RETURN_NONE;
    if (layers > INT32_MAX) refuse("too many layers");
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.kv_dtype = first.kv_dtype;
    a.num_pages = first.num_pages; a.page_size = first.page_size;
    a.num_kv_heads = first.num_kv_heads; a.head_dim = first.head_dim;
    a.layers = static_cast<int32_t>(layers);
    a.pairs = static_cast<int32_t>(pairs);
    a.k_page_stride = first.k_page_stride; a.k_slot_stride = first.k_slot_stride; a.k_head_stride = first.k_head_stride;
    a.v_page_stride = first.v_page_stride; a.v_slot_stride = first.v_slot_stride; a.v_head_stride = first.v_head_stride;
    a.k_caches = k.data(); a.v_caches = v.data();
    if (first.kv_dtype == ECAH_KV_E4M3) { a.k_scales = ks.data(); a.v_scales = vs.data(); }
    a.src = src.data_ptr<int32_t>();
    a.dst = dst.data_ptr<int32_t>();
    run(g_copy, a, dev, "ecah_paged_copy");
    Py_RETURN_NONE;
  });
}

// target, draft_ids, uniforms, workspace, draft (or None), num_drafts, tokens, accepted,
// vocab (-1: any), max_batch (-1: any)
PyObject* verify(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  if (!count_is(n, 10)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Args in{raw, n};
    const at::Tensor& p = *in.tensor(0, "target_probs");
    if (p.dim() != 3) refuse("target_probs must be [B, N + 1, V], got " + shape_of(p));
    ecah_verify_args a = {};
    switch (p.scalar_type()) {
      case at::kHalf: a.dtype = ECAH_DTYPE_F16; break;
      case at::kBFloat16: a.dtype = ECAH_DTYPE_BF16; break;
      case at::kFloat: a.dtype = ECAH_DTYPE_F32; break;
      default: refuse("unsupported dtype of probabilities " + type_name(p.scalar_type()));
    }
    if (!p.is_cuda()) refuse("target_probs must be a CUDA tensor (there is no CPU path)");
    const at::Device dev = p.device();
    const int64_t B = p.size(0), V = p.size(2);
    if (p.size(1) < 1) refuse("target_probs must have a row after the last draft, got " + shape_of(p));
    const int64_t N = p.size(1) - 1;
    const long vocab = in.integer(8), most = in.integer(9);
    if (vocab >= 0 && V != vocab) refuse("target_probs must be [B, N + 1, " + std::to_string(vocab) + "], got " + shape_of(p));
    if (most >= 0 && B > most) refuse(std::to_string(B) + " requests, max_batch is " + std::to_string(most));
    if (V < 1 || V > INT32_MAX || B > INT32_MAX || N > INT32_MAX - 1) refuse("target_probs too large or empty: " + shape_of(p));
    auto strides = [&](const at::Tensor& t, const char* name, int64_t* b, int64_t* r) {
      if (t.size(2) > 1 && t.stride(2) != 1) refuse(std::string(name) + ": rows of probabilities must be contiguous");
      *b = t.size(0) > 1 ? t.stride(0) : 0;
      *r = t.size(1) > 1 ? t.stride(1) : 0;
    };
    strides(p, "target_probs", &a.target_batch_stride, &a.target_row_stride);
    if (const at::Tensor* q = in.tensor(4, "draft_probs", true)) {
      if (q->scalar_type() != p.scalar_type() || q->device() != dev)
        refuse("draft_probs: expected " + type_name(p.scalar_type()) + " on " + dev.str() + ", got " + type_name(q->scalar_type()) + " on " + q->device().str());
      if (q->dim() != 3 || q->size(0) != B || q->size(1) != N || q->size(2) != V)
        refuse("draft_probs: expected shape [" + std::to_string(B) + ", " + std::to_string(N) + ", " + std::to_string(V) + "], got " + shape_of(*q));
      strides(*q, "draft_probs", &a.draft_batch_stride, &a.draft_row_stride);
      a.draft = N ? q->data_ptr() : nullptr;
    }
    const at::Tensor &ids = *in.tensor(1, "draft_ids"), &u = *in.tensor(2, "uniforms");
    need(ids, "draft_ids", at::kInt, B * N, dev);
    need(u, "uniforms", at::kFloat, B * (N + 1), dev);
    if (const at::Tensor* t = in.tensor(5, "num_drafts", true)) {
      need(*t, "num_drafts", at::kInt, B, dev);
      a.num_drafts = t->data_ptr<int32_t>();
    }
    const at::Tensor& ws = *in.tensor(3, "workspace");
    a.workspace = const_cast<void*>(checked_workspace(ws, dev));
    a.workspace_bytes = static_cast<size_t>(ws.numel());
    at::Tensor tokens = output(in.tensor(6, "tokens", true), "tokens", {B, N + 1}, at::kInt, dev);
    at::Tensor accepted = output(in.tensor(7, "accepted", true), "accepted", {B}, at::kInt, dev);
    a.abi_version = ECAH_SAMPLER_ABI_VERSION;
    a.batch = static_cast<int32_t>(B);
    a.drafts = static_cast<int32_t>(N);
    a.vocab = static_cast<int32_t>(V);
    a.target = p.data_ptr();
    a.draft_ids = ids.data_ptr<int32_t>();
    a.uniforms = u.data_ptr<float>();
    a.tokens = tokens.data_ptr<int32_t>();
    a.accepted = accepted.data_ptr<int32_t>();
    run(g_verify, a, dev, "ecah_verify_drafts");
    return Py_BuildValue("(NN)", THPVariable_Wrap(tokens), THPVariable_Wrap(accepted));
  });
}

// bind(error class, addresses of ecah_token_logprobs, ecah_paged_append,
// ecah_paged_decode, ecah_paged_prefill, ecah_paged_copy, ecah_verify_drafts and
// ecah_status_string)
PyObject* bind(PyObject*, PyObject* const* raw, Py_ssize_t n) {
  constexpr int kEntries = 7;
  if (!count_is(n, 1 + kEntries)) return nullptr;
  void* at[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(raw[i + 1]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "an entry point's address is null");
      return nullptr;
    }
  }
  Py_XDECREF(g_error);
  g_error = Py_NewRef(raw[0]);
  g_logprobs = reinterpret_cast<decltype(g_logprobs)>(at[0]);
  g_append = reinterpret_cast<decltype(g_append)>(at[1]);
  g_decode = reinterpret_cast<decltype(g_decode)>(at[2]);
  g_prefill = reinterpret_cast<decltype(g_prefill)>(at[3]);
  g_copy = reinterpret_cast<decltype(g_copy)>(at[4]);
  g_verify = reinterpret_cast<decltype(g_verify)>(at[5]);
  g_status_string = reinterpret_cast<decltype(g_status_string)>(at[6]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logprobs)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill)), METH_FASTCALL, nullptr},
    {"copy_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(copy_pages)), METH_FASTCALL, nullptr},
    {"verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(verify)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ecah_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ecah_binding(void) { return PyModule_Create(&module); }
