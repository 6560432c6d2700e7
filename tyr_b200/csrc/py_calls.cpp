// The per-call host work of tyr_b200/nn.py in native code: reads sizes, strides and pointers out of
// torch tensors, applies the argument checks, allocates the outputs and calls the C ABI of
// include/tyr_b200_attn.h on torch's current stream.
//
// A single-token step or a short prompt is a few microseconds of device work, and building the
// argument structures from Python cost 14 to 38 us per call (ctypes fields, a device context
// manager, tensor attributes one by one): the host set the pace.  Host time of a pass with the GPU idle, before ->
// after: three prologues and a dense decode 79 -> 23 us, the typed call on a 517-row prompt 21 -> 5.5 us, forward and
// backward 81 -> 18 us, a single-row typed call 35 -> 9.5 us.
// Nothing is cached here: every call reads its tensors anew.
//
// The Python functions keep names, defaults and results; they hand their arguments over by position.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <stdexcept>

#include "../../include/tyr_b200_attn.h"

namespace {

using at::Tensor;

PyObject* g_attn_error = nullptr;  // tyr_b200._lib.AttnError, handed over at import

struct ValueError : std::runtime_error { using std::runtime_error::runtime_error; };
struct CallError { int code; };  // a status of the C ABI

// lets other Python threads run while this one allocates and launches
struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(s); }
};

template <class F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const CallError& e) {
    PyObject* x = g_attn_error ? PyObject_CallFunction(g_attn_error, "i", e.code) : nullptr;
    if (x) {
      PyErr_SetObject(g_attn_error, x);
      Py_DECREF(x);
    } else if (!PyErr_Occurred()) {
      PyErr_SetString(PyExc_RuntimeError, tyr_b200_attn_strerror(e.code));
    }
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

void check_rc(int rc) {
  if (rc != 0) throw CallError{rc};
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw ValueError(std::string(what) + " must be a torch tensor");
  return THPVariable_Unpack(o);
}
// nullptr for None
const Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int64_t integer(PyObject* o) {  // as int(o)
  PyObject* l = PyLong_CheckExact(o) ? Py_NewRef(o) : PyNumber_Long(o);
  if (!l) throw python_error();
  const int64_t v = PyLong_AsLongLong(l);
  Py_DECREF(l);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
float scale_of(PyObject* o) {  // None selects the default in the library
  if (o == Py_None) return 0.0f;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(v);
}

// the launcher checks of Tyr/GPU/Codegen/Attribute.lean:333-336, as exceptions
void require_cuda(const Tensor& t) {
  if (!t.is_cuda()) throw ValueError("tensor must be on a CUDA device");
  if (t.dim() > 4) throw ValueError("tensor rank must be <= 4");
  if (t.dim() < 1 || t.stride(-1) != 1) throw ValueError("tensor must have unit stride on the head dimension");
}
// the kernels follow pointers of one device
void same_device(const Tensor& t, const Tensor& as, const char* what) {
  if (!t.is_cuda() || t.device() != as.device()) throw ValueError(std::string(what) + " must be on the device of the other tensors");
}
void require_count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw ValueError("wrong number of arguments");
}

void strides3(int64_t* s, const Tensor& t) {
  s[0] = t.stride(0);
  s[1] = t.stride(1);
  s[2] = t.stride(2);
}
int32_t i32(int64_t v) { return static_cast<int32_t>(v); }

Tensor new_tensor(at::IntArrayRef size, at::ScalarType dt, at::Device dev) {
  return at::detail::empty_cuda(size, dt, dev, c10::nullopt);
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// The mask as the C ABI takes it, one byte per key; checked only, other types are converted by the Python caller.
Tensor key_bytes(const Tensor& m, int64_t batch, int64_t kv_seq) {
  const bool byte = m.scalar_type() == at::kBool || m.scalar_type() == at::kByte;
  if (!m.is_cuda() || !byte || m.dim() != 2 || m.stride(1) != 1 || m.size(0) != batch || m.size(1) != kv_seq)
    throw ValueError("key_mask must be a uint8/bool CUDA tensor [batch, kv_seq]");
  return m;
}

void fill_prefill(TyrAttnPrefillArgs& a, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor* o) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) throw ValueError("q, k, v must be [batch, heads, seq, head_dim]");
  if (v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3) || (o && o->sizes() != q.sizes()))
    throw ValueError("shape mismatch among q, k, v, out");
  const at::ScalarType dt = q.scalar_type();
  if (k.scalar_type() != dt || v.scalar_type() != dt || (o && o->scalar_type() != dt))
    throw ValueError("q, k, v and out must share one dtype");
  if (dt != at::kBFloat16 && dt != at::kFloat) throw ValueError("dtype must be bfloat16 (float32 in check mode)");
  std::memset(&a, 0, sizeof(a));
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.batch = i32(q.size(0));
  a.n_head = i32(q.size(1));
  a.n_kv_head = i32(k.size(1));
  a.q_seq = i32(q.size(2));
  a.kv_seq = i32(k.size(2));
  a.head_dim = i32(q.size(3));
  strides3(a.q_stride, q);
  strides3(a.k_stride, k);
  strides3(a.v_stride, v);
  a.dtype = dt == at::kBFloat16 ? TYR_ATTN_BF16 : TYR_ATTN_F32;
}

// a window or a number of first tokens: beyond any length is as good as the greatest length
int32_t span_of(PyObject* o) {
  const int64_t v = integer(o);
  return v > INT32_MAX ? INT32_MAX : v < 0 ? -1 : static_cast<int32_t>(v);
}

// q, k, v, is_causal, scale, out, lse, return_lse, check_mode, window_size, key_mask, workspace, n_sink -> (out, lse)
PyObject* attention_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require_count(n, 13);
    const Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k"), &v = tensor(args[2], "v");
    require_cuda(q);
    require_cuda(k);
    require_cuda(v);
    const bool causal = truth(args[3]), return_lse = truth(args[7]), check_mode = truth(args[8]);
    const Tensor *out_in = maybe(args[5], "out"), *lse_in = maybe(args[6], "lse"), *mask = maybe(args[10], "key_mask");
    const bool never_split = args[11] == Py_False;
    const Tensor* ws_in = never_split ? nullptr : maybe(args[11], "workspace");
    TyrAttnPrefillArgs a;
    fill_prefill(a, q, k, v, out_in);
    if (out_in) require_cuda(*out_in);
    same_device(k, q, "k");
    same_device(v, q, "v");
    if (out_in) same_device(*out_in, q, "out");
    if (lse_in) same_device(*lse_in, q, "lse");
    if (mask) same_device(*mask, q, "key_mask");
    a.is_causal = causal;
    a.scale = scale_of(args[4]);
    a.check_mode = check_mode;
    const int32_t n_sink = span_of(args[12]);
    a.window_size = span_of(args[9]);
    if (lse_in && (lse_in->scalar_type() != at::kFloat || !lse_in->is_contiguous() || lse_in->dim() != 3 ||
                   lse_in->size(0) != q.size(0) || lse_in->size(1) != q.size(1) || lse_in->size(2) != q.size(2)))
      throw ValueError("lse must be a contiguous float32 [batch, n_head, q_seq] tensor");
    if (mask) {
      const Tensor m = key_bytes(*mask, k.size(0), k.size(2));
      a.key_mask = static_cast<const uint8_t*>(m.data_ptr());
      a.key_mask_stride = m.stride(0);
    }
    Tensor out, lse, ws;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(q.device());
      out = out_in ? *out_in : new_tensor(q.sizes(), q.scalar_type(), q.device());
      if (lse_in) lse = *lse_in;
      else if (return_lse) lse = new_tensor(q.sizes().slice(0, 3), at::kFloat, q.device());
      a.o = out.data_ptr();
      strides3(a.o_stride, out);
      a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
      // only unmasked, non-causal calls are ever split: no query for the others
      if (!never_split && !causal && a.window_size == 0 && !mask && !check_mode) {
        const int64_t need = tyr_b200_attn_prefill_workspace_bytes(&a);
        if (need > 0) {
          ws = ws_in ? *ws_in : new_tensor({need}, at::kByte, q.device());
          if (ws.scalar_type() != at::kByte || !ws.is_contiguous() || ws.device() != q.device() ||
              reinterpret_cast<uintptr_t>(ws.data_ptr()) % 256 != 0)
            throw ValueError("workspace must be a contiguous uint8 CUDA tensor on q's device, 256-byte aligned");
          a.workspace = ws.data_ptr();
          a.workspace_bytes = ws.numel();
        }
      }
      check_rc(n_sink != 0 ? tyr_b200_attn_prefill_sinks(&a, n_sink, stream_of(q)) : tyr_b200_attn_prefill(&a, stream_of(q)));
    }
    PyObject* t = PyTuple_New(2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(out)));
    if (lse.defined()) {
      PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(lse)));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(t, 1, Py_None);
    }
    return t;
  });
}

// an uninitialised tensor with t's sizes and, where they are dense, its strides
Tensor like(const Tensor& t) {
  return t.is_contiguous() ? new_tensor(t.sizes(), t.scalar_type(), t.device()) : at::empty_like(t);
}

// q, k, v, o, lse, d_o, is_causal, scale, workspace, window_size, key_mask, n_sink -> (d_q, d_k, d_v)
PyObject* attention_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require_count(n, 12);
    const Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k"), &v = tensor(args[2], "v"), &o = tensor(args[3], "o"),
                 &lse = tensor(args[4], "lse"), &d_o = tensor(args[5], "d_o");
    for (const Tensor* t : {&q, &k, &v, &o, &d_o, &lse}) require_cuda(*t);
    if (q.dim() != 4 || k.dim() != 4) throw ValueError("q, k, v must be [batch, heads, seq, head_dim]");
    if (v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3) || o.sizes() != q.sizes() ||
        d_o.sizes() != q.sizes() || lse.sizes() != q.sizes().slice(0, 3))
      throw ValueError("shape mismatch among q, k, v, o, d_o, lse");
    for (const Tensor* t : {&q, &k, &v, &o, &d_o})
      if (t->scalar_type() != at::kBFloat16) throw ValueError("q, k, v, o, d_o must be bfloat16");
    if (lse.scalar_type() != at::kFloat || !lse.is_contiguous())
      throw ValueError("lse must be a contiguous float32 [batch, n_head, q_seq] tensor");
    const Tensor *ws_in = maybe(args[8], "workspace"), *mask = maybe(args[10], "key_mask");
    for (const Tensor* t : {&k, &v, &o, &lse, &d_o}) same_device(*t, q, "k, v, o, lse and d_o");
    if (ws_in) same_device(*ws_in, q, "workspace");
    if (mask) same_device(*mask, q, "key_mask");
    TyrAttnBackwardArgs a;
    std::memset(&a, 0, sizeof(a));
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = o.data_ptr(); a.d_o = d_o.data_ptr();
    a.lse = static_cast<const float*>(lse.data_ptr());
    a.batch = i32(q.size(0)); a.n_head = i32(q.size(1)); a.n_kv_head = i32(k.size(1));
    a.q_seq = i32(q.size(2)); a.kv_seq = i32(k.size(2)); a.head_dim = i32(q.size(3));
    strides3(a.q_stride, q); strides3(a.k_stride, k); strides3(a.v_stride, v); strides3(a.o_stride, o);
    strides3(a.do_stride, d_o);
    a.dtype = TYR_ATTN_BF16;
    a.is_causal = truth(args[6]);
    a.scale = scale_of(args[7]);
    const int32_t n_sink = span_of(args[11]);
    a.window_size = span_of(args[9]);
    if (mask) {
      const Tensor m = key_bytes(*mask, k.size(0), k.size(2));
      a.key_mask = static_cast<const uint8_t*>(m.data_ptr());
      a.key_mask_stride = m.stride(0);
    }
    Tensor ws, d_q, d_k, d_v;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(q.device());
      const int64_t need = n_sink != 0 ? tyr_b200_attn_backward_sinks_workspace_bytes(&a, n_sink)
                                       : (int64_t)tyr_b200_attn_backward_workspace_bytes(a.batch, a.n_head, a.q_seq);
      if (need < 0) throw CallError{(int)need};
      ws = ws_in ? *ws_in : new_tensor({need / 4}, at::kFloat, q.device());
      if (ws.scalar_type() != at::kFloat || !ws.is_contiguous() || ws.numel() * 4 < need)
        throw ValueError("workspace must be a contiguous float32 CUDA tensor of the required size");
      d_q = like(q);
      d_k = like(k);
      d_v = like(v);
      a.d_q = d_q.data_ptr(); a.d_k = d_k.data_ptr(); a.d_v = d_v.data_ptr();
      strides3(a.dq_stride, d_q); strides3(a.dk_stride, d_k); strides3(a.dv_stride, d_v);
      a.workspace = ws.data_ptr();
      a.workspace_bytes = (uint64_t)ws.numel() * 4;
      check_rc(n_sink != 0 ? tyr_b200_attn_backward_sinks(&a, n_sink, stream_of(q)) : tyr_b200_attn_backward(&a, stream_of(q)));
    }
    PyObject* t = PyTuple_New(3);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(d_q)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(d_k)));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(d_v)));
    return t;
  });
}

// The [batch, heads, head_dim] query of a single-token call, given as such or as [batch, heads, 1, head_dim].
struct QueryRows {
  int64_t batch, heads, d, stride_b, stride_h;
};
QueryRows query_rows(const Tensor& q) {
  if (q.dim() != 3 && q.dim() != 4) throw ValueError("q must be bf16 [batch, n_head, head_dim]");
  require_cuda(q);
  return {q.size(0), q.size(1), q.size(-1), q.stride(0), q.stride(1)};
}
PyObject* out_and_lse(Tensor& out, Tensor& lse, bool unsqueeze) {
  PyObject* t = PyTuple_New(2);
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(unsqueeze ? out.unsqueeze(2) : std::move(out)));
  if (lse.defined()) {
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(unsqueeze ? lse.unsqueeze(2) : std::move(lse)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(t, 1, Py_None);
  }
  return t;
}

// q, (batch, n_head, n_kv_head, max_kv_seq, head_dim, max_splits, total_kv_len), k_ptrs, v_ptrs, kv_lens, head_strides,
// workspace or None (the library's own array), workspace_bytes, scale, out, lse, return_lse -> (out, lse)
PyObject* decode_ragged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require_count(n, 18);
    const Tensor& q = tensor(args[0], "q");
    const QueryRows r = query_rows(q);
    TyrAttnDecodeArgs a;
    std::memset(&a, 0, sizeof(a));
    a.batch = i32(integer(args[1]));
    a.n_head = i32(integer(args[2]));
    a.n_kv_head = i32(integer(args[3]));
    a.max_kv_seq = i32(integer(args[4]));
    a.head_dim = i32(integer(args[5]));
    a.max_splits = i32(integer(args[6]));
    a.total_kv_len = integer(args[7]);
    if (q.scalar_type() != at::kBFloat16 || r.batch != a.batch || r.heads != a.n_head || r.d != a.head_dim)
      throw ValueError("q must be bf16 [batch, n_head, head_dim]");
    a.k_ptrs = static_cast<const void* const*>(tensor(args[8], "k_ptrs").data_ptr());
    a.v_ptrs = static_cast<const void* const*>(tensor(args[9], "v_ptrs").data_ptr());
    a.kv_lens = static_cast<const int32_t*>(tensor(args[10], "kv_lens").data_ptr());
    a.kv_head_strides = static_cast<const int64_t*>(tensor(args[11], "head_strides").data_ptr());
    const Tensor* ws = maybe(args[12], "workspace");
    a.workspace = ws ? ws->data_ptr() : nullptr;
    a.workspace_bytes = (size_t)integer(args[13]);
    a.scale = scale_of(args[14]);
    const Tensor *out_in = maybe(args[15], "out"), *lse_in = maybe(args[16], "lse");
    const bool return_lse = truth(args[17]);
    same_device(tensor(args[8], "k_ptrs"), q, "the plan's arrays");
    if (ws) same_device(*ws, q, "the plan's workspace");
    if (out_in) same_device(*out_in, q, "out");
    if (lse_in) same_device(*lse_in, q, "lse");
    if (out_in && (out_in->scalar_type() != at::kBFloat16 || out_in->dim() < 3 || out_in->size(0) != r.batch || out_in->size(1) != r.heads ||
                   out_in->size(-1) != r.d || out_in->stride(-1) != 1 || out_in->numel() != r.batch * r.heads * r.d))
      throw ValueError("out must be bf16 [batch, n_head, head_dim]");
    if (lse_in && (lse_in->scalar_type() != at::kFloat || !lse_in->is_contiguous() || lse_in->numel() != r.batch * r.heads))
      throw ValueError("lse must be a contiguous float32 tensor [batch, n_head]");
    a.q = q.data_ptr();
    a.q_stride[0] = r.stride_b;
    a.q_stride[1] = r.stride_h;
    a.k_stride[2] = a.v_stride[2] = a.head_dim;
    Tensor out, lse;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(q.device());
      out = out_in ? *out_in : new_tensor({r.batch, r.heads, r.d}, at::kBFloat16, q.device());
      if (lse_in) lse = *lse_in;
      else if (return_lse) lse = new_tensor({r.batch, r.heads}, at::kFloat, q.device());
      a.o = out.data_ptr();
      a.o_stride[0] = out.stride(0);
      a.o_stride[1] = out.stride(1);
      a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
      check_rc(ws ? tyr_b200_attn_decode(&a, stream_of(q)) : tyr_b200_attn_decode_static(&a, stream_of(q)));
    }
    return out_and_lse(out, lse, ws && q.dim() == 4);
  });
}

// q, k_cache, v_cache, kv_lens, kv_len, scale, workspace, max_splits -> (out, lse)
PyObject* decode_dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require_count(n, 8);
    const Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k_cache"), &v = tensor(args[2], "v_cache");
    const QueryRows r = query_rows(q);
    require_cuda(k);
    require_cuda(v);
    if (k.dim() != 4 || v.dim() != 4) throw ValueError("k_cache and v_cache must be [batch, n_kv_head, cap, head_dim]");
    const Tensor *lens = maybe(args[3], "kv_lens"), *ws_in = maybe(args[6], "workspace");
    same_device(k, q, "k_cache");
    same_device(v, q, "v_cache");
    if (lens) same_device(*lens, q, "kv_lens");
    if (ws_in) same_device(*ws_in, q, "workspace");
    const int64_t kv_len = args[4] == Py_None ? k.size(2) : integer(args[4]);
    for (const Tensor* t : {&k, &v}) {  // a larger cache than the call needs is fine
      if (t->scalar_type() != at::kBFloat16 || q.scalar_type() != at::kBFloat16) throw ValueError("q and the caches must be bf16");
      if (t->size(0) < r.batch || t->size(1) != k.size(1) || t->size(3) != r.d) throw ValueError("the caches do not match q");
      if (t->size(2) < kv_len) throw ValueError("kv_len " + std::to_string(kv_len) + " exceeds the " + std::to_string(t->size(2)) + " rows of the cache");
    }
    if (lens && (lens->scalar_type() != at::kInt || !lens->is_contiguous() || lens->numel() < r.batch))
      throw ValueError("kv_lens must be a contiguous int32 tensor [batch]");
    TyrAttnDecodeArgs a;
    std::memset(&a, 0, sizeof(a));
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.kv_lens = lens ? static_cast<const int32_t*>(lens->data_ptr()) : nullptr;
    a.batch = i32(r.batch);
    a.n_head = i32(r.heads);
    a.n_kv_head = i32(k.size(1));
    a.max_kv_seq = kv_len < 0 ? -1 : i32(kv_len);
    a.head_dim = i32(r.d);
    a.q_stride[0] = r.stride_b;
    a.q_stride[1] = r.stride_h;
    strides3(a.k_stride, k);
    strides3(a.v_stride, v);
    a.scale = scale_of(args[5]);
    a.max_splits = i32(integer(args[7]));
    a.total_kv_len = 0;  // a shared length is known as it is; per-sequence lengths live on the device
    Tensor out, lse, ws;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(q.device());
      out = new_tensor({r.batch, r.heads, r.d}, q.scalar_type(), q.device());
      lse = new_tensor({r.batch, r.heads}, at::kFloat, q.device());
      a.o = out.data_ptr();
      a.o_stride[0] = r.heads * r.d;
      a.o_stride[1] = r.d;
      a.lse = static_cast<float*>(lse.data_ptr());
      if (ws_in) {
        ws = *ws_in;
      } else {
        const size_t need = tyr_b200_attn_decode_workspace_bytes(a.batch, a.n_head, a.head_dim, a.max_kv_seq, a.max_splits);
        ws = new_tensor({(int64_t)(need > 16 ? need : 16)}, at::kByte, q.device());
      }
      a.workspace = ws.data_ptr();
      a.workspace_bytes = (size_t)ws.numel();
      check_rc(tyr_b200_attn_decode(&a, stream_of(q)));
    }
    return out_and_lse(out, lse, false);
  });
}

// ---- paged cache
// a size or count as the C ABI takes it; what does not fit is refused rather than cut off
int32_t count_of(int64_t v, const char* what) {
  if (v < INT32_MIN || v > INT32_MAX) throw ValueError(std::string(what) + " does not fit 32 bits");
  return static_cast<int32_t>(v);
}
// int32 [batch], contiguous
const int32_t* per_sequence(const Tensor& t, const Tensor& as, int64_t batch, const char* what) {
  same_device(t, as, what);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != batch || !t.is_contiguous())
    throw ValueError(std::string(what) + " must be a contiguous int32 tensor [batch]");
  return static_cast<const int32_t*>(t.data_ptr());
}
void fill_pages(TyrAttnPageTable& p, const Tensor& table, const Tensor& pool, int64_t batch) {
  same_device(table, pool, "page_table");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != batch || (table.size(1) > 1 && table.stride(1) != 1))
    throw ValueError("page_table must be an int32 tensor [batch, max_pages]");
  p.table = static_cast<const int32_t*>(table.data_ptr());
  p.table_stride = table.stride(0);
  p.max_pages = count_of(table.size(1), "page_table");
  p.n_pages = count_of(pool.size(0), "the number of pages");
  p.page_size = count_of(pool.size(2), "the page size");
}
void require_pool(const Tensor& t, const char* what) {
  require_cuda(t);
  if (t.dim() != 4 || t.scalar_type() != at::kBFloat16)
    throw ValueError(std::string(what) + " must be bf16 [n_pages, n_kv_head, page_size, head_dim]");
}
// the pools of K and V and their strides
void fill_pools(const Tensor& k, const Tensor& v, int64_t* k_stride, int64_t* v_stride) {
  require_pool(k, "k_pages");
  require_pool(v, "v_pages");
  if (v.sizes() != k.sizes()) throw ValueError("k_pages and v_pages differ in shape");
  same_device(v, k, "v_pages");
  strides3(k_stride, k);
  strides3(v_stride, v);
}
float* weight_sums(const Tensor& w, const Tensor& as, int64_t batch, int64_t n_kv_head, int64_t* stride) {
  same_device(w, as, "weights");
  if (w.scalar_type() != at::kFloat || w.dim() != 3 || w.size(0) != batch || w.size(1) != n_kv_head || (w.size(2) > 1 && w.stride(2) != 1))
    throw ValueError("weights must be a float32 tensor [batch, n_kv_head, max_kv_seq]");
  stride[0] = w.stride(0);
  stride[1] = w.stride(1);
  return static_cast<float*>(w.data_ptr());
}

// q, k_pages, v_pages, page_table, kv_lens, max_kv_seq, window_size, n_sink, weights, scale, out, lse, workspace, return_lse,
// total_kv_len, max_splits -> (out, lse); with `only_bytes` the workspace the call needs
PyObject* paged_decode_call(PyObject* const* args, Py_ssize_t n, bool only_bytes) {
  require_count(n, 16);
  const Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k_pages"), &v = tensor(args[2], "v_pages"),
               &table = tensor(args[3], "page_table"), &lens = tensor(args[4], "kv_lens");
  const QueryRows r = query_rows(q);
  if (q.scalar_type() != at::kBFloat16 || (q.dim() == 4 && q.size(2) != 1))
    throw ValueError("q must be bf16 [batch, n_head, head_dim] or [batch, n_head, 1, head_dim]");
  TyrAttnPagedDecodeArgs a;
  std::memset(&a, 0, sizeof(a));
  fill_pools(k, v, a.k_stride, a.v_stride);
  same_device(k, q, "k_pages");
  if (k.size(3) != r.d) throw ValueError("q and the pages differ in head_dim");
  fill_pages(a.pages, table, k, r.batch);
  a.kv_lens = per_sequence(lens, q, r.batch, "kv_lens");
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.batch = count_of(r.batch, "the batch");
  a.n_head = count_of(r.heads, "n_head");
  a.n_kv_head = count_of(k.size(1), "n_kv_head");
  a.head_dim = count_of(r.d, "head_dim");
  const Tensor *w = maybe(args[8], "weights"), *out_in = maybe(args[10], "out"), *lse_in = maybe(args[11], "lse"),
               *ws_in = maybe(args[12], "workspace");
  const int64_t cap = (int64_t)a.pages.max_pages * a.pages.page_size;
  a.max_kv_seq = count_of(args[5] == Py_None ? cap : integer(args[5]), "max_kv_seq");
  a.window_size = span_of(args[6]);
  a.n_sink = span_of(args[7]);
  if (w) {
    a.weights = weight_sums(*w, q, r.batch, k.size(1), a.weights_stride);
    if (w->size(2) < a.max_kv_seq)
      throw ValueError("weights holds fewer keys than max_kv_seq (where it is not given, all the page table can hold)");
  }
  a.scale = scale_of(args[9]);
  const bool return_lse = truth(args[13]);
  const int64_t total = integer(args[14]);
  a.total_kv_len = total > 0 ? total : 0;
  a.max_splits = count_of(integer(args[15]), "max_splits");
  a.q_stride[0] = r.stride_b;
  a.q_stride[1] = r.stride_h;
  if (out_in) {
    require_cuda(*out_in);
    same_device(*out_in, q, "out");
    if (out_in->scalar_type() != at::kBFloat16 || out_in->sizes() != q.sizes()) throw ValueError("out must be bf16 and of the shape of q");
  }
  if (lse_in) {
    same_device(*lse_in, q, "lse");
    if (lse_in->scalar_type() != at::kFloat || !lse_in->is_contiguous() || lse_in->sizes() != q.sizes().slice(0, q.dim() - 1))
      throw ValueError("lse must be a contiguous float32 tensor [batch, n_head] (with q's fourth axis, [batch, n_head, 1])");
  }
  if (only_bytes) {
    const int64_t need = r.batch == 0 ? 0 : tyr_b200_attn_paged_decode_workspace_bytes(&a);
    if (need < 0) throw CallError{(int)need};
    return PyLong_FromLongLong(need);
  }
  Tensor out, lse, ws;
  {
    NoGil no_gil;
    c10::cuda::OptionalCUDAGuard guard(q.device());
    out = out_in ? *out_in : new_tensor(q.sizes(), at::kBFloat16, q.device());
    if (lse_in) lse = *lse_in;
    else if (return_lse) lse = new_tensor(q.sizes().slice(0, q.dim() - 1), at::kFloat, q.device());
    a.o = out.data_ptr();
    a.o_stride[0] = out.stride(0);
    a.o_stride[1] = out.stride(1);
    a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
    const int64_t need = r.batch == 0 ? 0 : tyr_b200_attn_paged_decode_workspace_bytes(&a);
    if (need < 0) throw CallError{(int)need};
    if (ws_in) {
      ws = *ws_in;
      if (ws.scalar_type() != at::kByte || !ws.is_contiguous() || ws.device() != q.device())
        throw ValueError("workspace must be a contiguous uint8 tensor on q's device");
    } else if (need > 0) {
      ws = new_tensor({need}, at::kByte, q.device());
    }
    if (ws.defined()) {
      a.workspace = ws.data_ptr();
      a.workspace_bytes = ws.numel();
    }
    check_rc(tyr_b200_attn_paged_decode(&a, stream_of(q)));
  }
  return out_and_lse(out, lse, false);
}
PyObject* decode_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] { return paged_decode_call(args, n, false); });
}
PyObject* decode_paged_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] { return paged_decode_call(args, n, true); });
}

// k_pages, v_pages, page_table, kv_lens, weights, n_keep, n_recent, n_sink, max_kv_seq, new_lens, kept -> (new_lens, kept)
PyObject* evict_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require_count(n, 11);
    const Tensor &k = tensor(args[0], "k_pages"), &v = tensor(args[1], "v_pages"), &table = tensor(args[2], "page_table"),
                 &lens = tensor(args[3], "kv_lens"), &w = tensor(args[4], "weights");
    TyrAttnEvictArgs a;
    std::memset(&a, 0, sizeof(a));
    fill_pools(k, v, a.k_stride, a.v_stride);
    const int64_t batch = lens.dim() == 1 ? lens.size(0) : -1;
    a.kv_lens = per_sequence(lens, k, batch, "kv_lens");
    fill_pages(a.pages, table, k, batch);
    a.weights = weight_sums(w, k, batch, k.size(1), a.weights_stride);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.batch = count_of(batch, "the batch");
    a.n_kv_head = count_of(k.size(1), "n_kv_head");
    a.head_dim = count_of(k.size(3), "head_dim");
    a.n_keep = count_of(integer(args[5]), "n_keep");
    a.n_recent = count_of(integer(args[6]), "n_recent");
    a.n_sink = count_of(integer(args[7]), "n_sink");
    const int64_t cap = (int64_t)a.pages.max_pages * a.pages.page_size;
    a.max_kv_seq = count_of(args[8] == Py_None ? (w.size(2) < cap ? w.size(2) : cap) : integer(args[8]), "max_kv_seq");
    if (w.size(2) < a.max_kv_seq) throw ValueError("weights holds fewer keys than max_kv_seq");
    const Tensor *new_in = maybe(args[9], "new_lens"), *kept_in = maybe(args[10], "kept");
    if (new_in) per_sequence(*new_in, k, batch, "new_lens");
    if (kept_in) {
      same_device(*kept_in, k, "kept");
      if (kept_in->scalar_type() != at::kInt || !kept_in->is_contiguous() || kept_in->dim() != 3 || kept_in->size(0) != batch ||
          kept_in->size(1) != k.size(1) || kept_in->size(2) != a.n_keep)
        throw ValueError("kept must be a contiguous int32 tensor [batch, n_kv_head, n_keep]");
    }
    Tensor new_lens, kept;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(k.device());
      new_lens = new_in ? *new_in : new_tensor({batch}, at::kInt, k.device());
      kept = kept_in ? *kept_in : new_tensor({batch, k.size(1), a.n_keep > 0 ? a.n_keep : 0}, at::kInt, k.device());
      a.new_lens = static_cast<int32_t*>(new_lens.data_ptr());
      a.kept = static_cast<int32_t*>(kept.data_ptr());
      check_rc(tyr_b200_attn_paged_evict(&a, stream_of(k)));
    }
    PyObject* t = PyTuple_New(2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(new_lens)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(kept)));
    return t;
  });
}

// x, out, norm_weight, cos, sin, positions, position0, eps, pe, out_at_row0 [, page_table, rows] -> None
PyObject* qk_prologue(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10) require_count(n, 12);
    const Tensor &x = tensor(args[0], "x"), &out = tensor(args[1], "out");
    require_cuda(x);
    require_cuda(out);
    if (x.dim() != 4 || out.dim() != 4 || x.scalar_type() != at::kBFloat16 || out.scalar_type() != at::kBFloat16)
      throw ValueError("x must be bf16 [B,S,H,D] and out bf16 [B,H,cap,D]");
    const Tensor *table = n == 10 ? nullptr : maybe(args[10], "page_table"), *rows = n == 10 ? nullptr : maybe(args[11], "rows");
    const int64_t B = x.size(0), S = x.size(1), H = x.size(2), D = x.size(3);
    if ((!table && out.size(0) != B) || out.size(1) != H || out.size(3) != D) throw ValueError("out does not match x");
    TyrAttnPageTable pages{};
    if (rows && !table) throw ValueError("rows goes with page_table");
    if (table) {
      fill_pages(pages, *table, out, B);
      if (rows) per_sequence(*rows, x, B, "rows");
      if (args[5] != Py_None) per_sequence(tensor(args[5], "positions"), x, B, "positions");
    }
    const int64_t cap = table ? (int64_t)pages.max_pages * pages.page_size : out.size(2);
    const Tensor *w = maybe(args[2], "norm_weight"), *cos = maybe(args[3], "cos"), *sin = maybe(args[4], "sin"),
                 *pos = maybe(args[5], "positions"), *pe = maybe(args[8], "pe");
    for (const Tensor* t : {w, cos, sin, pe}) {
      if (!t) continue;
      if (t->scalar_type() != at::kFloat || !t->is_contiguous() || !t->is_cuda())
        throw ValueError("norm_weight / cos / sin / pe must be contiguous float32 CUDA tensors");
      same_device(*t, x, "norm_weight / cos / sin / pe");
    }
    if (w && w->numel() < D) throw ValueError("norm_weight must have head_dim elements");
    same_device(out, x, "out");
    if (pe) {
      if (cos || sin) throw ValueError("pass either cos/sin or pe");
      if (pe->dim() != 5 || pe->size(2) != D / 2 || pe->size(3) != 2 || pe->size(4) != 2 ||
          (pe->size(0) != 1 && pe->size(0) != B))
        throw ValueError("pe must be [B or 1, max_pos, D/2, 2, 2]");
    }
    if (cos && (!sin || cos->sizes() != sin->sizes() || cos->dim() != 2 || cos->size(1) != D / 2))
      throw ValueError("cos and sin must both be [max_pos, D/2]");
    const int64_t max_pos = pe ? pe->size(1) : (cos ? cos->size(0) : 0);
    const int64_t position0 = integer(args[6]);
    const bool row0 = truth(args[9]);
    if (row0 && S > cap) throw ValueError(std::to_string(S) + " rows do not fit the " + std::to_string(cap) + " rows of out");
    if (table && row0) throw ValueError("out_at_row0 does not go with page_table");
    if (!pos) {
      if (position0 < 0 || (!row0 && !rows && position0 + S > cap))
        throw ValueError("rows " + std::to_string(position0) + ".." + std::to_string(position0 + S - 1) + " do not fit the " +
                         std::to_string(cap) + " rows of out");
      if (max_pos && position0 + S > max_pos)
        throw ValueError("positions up to " + std::to_string(position0 + S - 1) + " exceed the " + std::to_string(max_pos) +
                         " rows of the rotary table");
    } else {
      if (pos->scalar_type() != at::kInt || !pos->is_cuda()) throw ValueError("positions must be an int32 CUDA tensor");
      same_device(*pos, x, "positions");
      if (pos->numel() < B || !pos->is_contiguous()) throw ValueError("positions must have an element for each sequence");
    }
    TyrAttnPrologueArgs a;
    std::memset(&a, 0, sizeof(a));
    auto f32 = [](const Tensor* t) { return t ? static_cast<const float*>(t->data_ptr()) : nullptr; };
    a.x = x.data_ptr();
    a.out = out.data_ptr();
    a.norm_weight = f32(w);
    a.cos = f32(cos);
    a.sin = f32(sin);
    a.pe = f32(pe);
    a.positions = pos ? static_cast<const int32_t*>(pos->data_ptr()) : nullptr;
    a.position0 = i32(position0);
    a.batch = i32(B);
    a.seq = i32(S);
    a.n_head = i32(H);
    a.head_dim = i32(D);
    strides3(a.x_stride, x);
    strides3(a.out_stride, out);
    const double eps = PyFloat_AsDouble(args[7]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    a.eps = static_cast<float>(eps);
    a.cap = table ? 0 : i32(cap);
    a.max_pos = i32(max_pos);
    a.out_at_row0 = row0;
    a.pe_batch_stride = (pe && pe->size(0) > 1) ? pe->stride(0) : 0;
    {
      NoGil no_gil;
      c10::cuda::OptionalCUDAGuard guard(x.device());
      check_rc(table ? tyr_b200_attn_qk_prologue_paged(&a, &pages, rows ? static_cast<const int32_t*>(rows->data_ptr()) : nullptr,
                                                       stream_of(x))
                     : tyr_b200_attn_qk_prologue(&a, stream_of(x)));
    }
    Py_RETURN_NONE;
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  Py_XSETREF(g_attn_error, cls);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(attention_fwd), FAST(attention_bwd), FAST(decode_ragged), FAST(decode_dense), FAST(qk_prologue),
                           FAST(decode_paged), FAST(decode_paged_workspace), FAST(evict_paged),
                           {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&g_module); }
