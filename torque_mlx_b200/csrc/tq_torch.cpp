// Python binding of the serving operators (paged cache, 4-bit products, draft
// verification) on torch tensors.
//
// These calls are made several times for each generated token, and their
// kernels take a few microseconds, so what the host does around a launch is
// what a small call costs.  Here the argument checks, the output allocation
// and the launch are one native call: about 4 us with one launch, where the
// same steps in Python took 9 to 14.  The compute is libtorque_b200.so's C
// ABI, which this module links.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/torque_b200.h"

namespace {

struct BadArgument : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};

std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}

template <typename... S> [[noreturn]] void refuse(const S&... parts) {
  throw BadArgument((text(parts) + ...));
}

void check(int status, const char* what) {
  if (status == TQ_OK) return;
  std::string msg = std::string(what) + ": " + tq_status_string(status);
  if (status == TQ_E_CUDA) msg += " (cudaError " + std::to_string(tq_last_cuda_error()) + ")";
  switch (status) {
    case TQ_E_BITS: case TQ_E_HEAD_DIM: case TQ_E_SHAPE: case TQ_E_ARG: case TQ_E_SCRATCH_LIMIT: throw BadArgument(msg);
    default: throw std::runtime_error(msg);
  }
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a torch tensor");
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }
int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be an integer");
  }
  return v;
}
double real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a number");
  }
  return v;
}
bool truth(PyObject* o, const char* name) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse(name, " must be true or false");
  }
  return v;
}

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return TQ_F32;
  if (t == at::kHalf) return TQ_F16;
  if (t == at::kBFloat16) return TQ_BF16;
  refuse("unsupported input dtype ", t, " (expected float32, float16 or bfloat16)");
}

bool on(const at::Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

// Whether the slices of `t` along `dim` follow one another without overlap (an
// expanded tensor repeats one).
bool apart(const at::Tensor& t, int64_t dim) {
  int64_t inner = 1;
  for (int64_t d = dim + 1; d < t.dim(); ++d) inner *= t.size(d);
  return t.size(dim) <= 1 || t.stride(dim) >= inner;
}

// `t` with contiguous rows (the first dimension's stride free) at 16-byte
// boundaries, copied only where it has none.
at::Tensor rows_of(const at::Tensor& t) {
  if (!t.is_contiguous()) {
    int64_t inner = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      if (t.size(d) != 1 && t.stride(d) != inner) return t.contiguous();
      inner *= t.size(d);
    }
  }
  const bool aligned = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                       (t.size(0) <= 1 || t.stride(0) * t.element_size() % 16 == 0);
  return aligned && apart(t, 0) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Workspace of one call, from torch's allocator for the current stream and
// given back when the call's launches are queued: what takes the memory next on
// that stream runs after them.  No two calls share one, since two threads may
// be in calls on one stream at once: the interpreter's lock is not held around
// a call's launches, and another call's may come between them.  It costs 0.1 to
// 0.3 us of host time; calls back to back take what they took with a workspace
// kept for each stream (one token over 512: 7.7 us, 32 tokens of 2048 x 8192 in
// 4 bits: 13.9).
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject* wrap_pair(at::Tensor a, at::Tensor b) {
  PyObject* x = wrap(std::move(a));
  PyObject* y = wrap(std::move(b));
  PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

// torch.OutOfMemoryError, as torch's own calls raise it
void out_of_memory(const char* what) {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
  if (!type) PyErr_Clear();
  PyErr_SetString(type ? type : PyExc_RuntimeError, what);
  Py_XDECREF(type);
  Py_XDECREF(torch);
}

// Runs `f`, with C++ errors as Python exceptions.
template <typename F> PyObject* guarded(F f) {
  try {
    return f();
  } catch (const BadArgument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    out_of_memory(e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// A C ABI call without the interpreter's lock: a full launch queue blocks.
template <typename F> int unlocked(F f) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = f();
  Py_END_ALLOW_THREADS
  return status;
}

// ---------------------------------------------------------------------------
// paged cache: the first two arguments of each call are the address of its
// tq_paged_kv and its device
// ---------------------------------------------------------------------------
struct Cache {
  const tq_paged_kv* kv;
  int device;
  Cache(PyObject* const* args)
      : kv(reinterpret_cast<const tq_paged_kv*>(PyLong_AsVoidPtr(args[0]))), device((int)PyLong_AsLong(args[1])) {}
};

tq_paged_batch batch_of(const Cache& c, int64_t rows, PyObject* lengths_o, PyObject* table_o, PyObject* starts_o,
                        PyObject* most_o) {
  const at::Tensor &lengths = tensor(lengths_o, "lengths"), &table = tensor(table_o, "block_table");
  if (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || !on(lengths, c.device) || !lengths.is_contiguous())
    refuse("lengths must be contiguous int32 [seqs] on cuda:", c.device);
  const int64_t seqs = lengths.size(0);
  if (seqs > TQ_PAGED_MAX_SEQS) refuse("at most ", TQ_PAGED_MAX_SEQS, " sequences in a batch, got ", seqs);
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != seqs || !on(table, c.device) ||
      (table.size(1) > 1 && table.stride(1) != 1))
    refuse("block_table must be int32 [", seqs, ", pages] on cuda:", c.device, " with contiguous rows");
  tq_paged_batch b = {};
  b.block_table = table.const_data_ptr<int32_t>();
  b.lengths = lengths.const_data_ptr<int32_t>();
  b.table_width = (int32_t)std::min<int64_t>(table.size(1), INT32_MAX);
  b.table_stride = seqs > 1 ? table.stride(0) : table.size(1);
  b.rows = rows;
  b.seqs = (int32_t)seqs;
  int64_t most = 1;
  if (given(starts_o)) {
    const at::Tensor& starts = tensor(starts_o, "token_starts");
    if (starts.scalar_type() != at::kInt || starts.dim() != 1 || starts.size(0) != seqs + 1 || !on(starts, c.device) ||
        !starts.is_contiguous())
      refuse("token_starts must be contiguous int32 [", seqs + 1, "] on cuda:", c.device);
    b.token_starts = starts.const_data_ptr<int32_t>();
    most = given(most_o) ? integer(most_o, "max_new_tokens") : rows;
    if (most < 0) refuse("max_new_tokens must not be negative");
  } else if (rows != seqs) {
    refuse("without token_starts every sequence brings one row: ", seqs, " sequences, ", rows, " rows");
  }
  b.max_new_tokens = (int32_t)std::min<int64_t>(std::min(most, rows), INT32_MAX);
  return b;
}

at::Tensor output(PyObject* out_o, at::IntArrayRef shape, at::ScalarType type, int device, int align) {
  if (!given(out_o)) return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, device));
  const at::Tensor& out = tensor(out_o, "out");
  if (out.sizes() != shape || out.scalar_type() != type || !on(out, device) || !out.is_contiguous())
    refuse("out must be contiguous ", type, " ", shape, " on cuda:", device);
  if (reinterpret_cast<uintptr_t>(out.data_ptr()) % align) refuse("out must start at a ", align, "-byte boundary");
  return out;
}

// (kv, device, qkv, cos, sin, lengths, block_table, token_starts, max_new_tokens, interleaved, out)
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11) refuse("paged_append takes 11 arguments");
    const Cache c(args);
    at::Tensor qkv = tensor(args[2], "qkv");
    const int64_t d = c.kv->head_dim, heads = c.kv->kv_heads;
    if (qkv.dim() != 2 || !on(qkv, c.device))
      refuse("qkv must be [rows, (q_heads + ", 2 * heads, ") * ", d, "] on cuda:", c.device);
    const int64_t rows = qkv.size(0), width = qkv.size(1), q_heads = width / d - 2 * heads;
    if (width % d || q_heads < 0 || q_heads % heads)
      refuse("qkv width ", width, " must be (q_heads + ", 2 * heads, ") * ", d, " with q_heads a multiple of ", heads);
    const int code = dtype_code(qkv.scalar_type());
    const tq_paged_batch b = batch_of(c, rows, args[5], args[6], args[7], args[8]);
    const float *cos = nullptr, *sin = nullptr;
    int64_t positions = 0, rotary = 0;
    if (given(args[3]) || given(args[4])) {
      if (!given(args[3]) || !given(args[4])) refuse("cos and sin go together");
      const at::Tensor &tc = tensor(args[3], "cos"), &ts = tensor(args[4], "sin");
      if (tc.dim() != 2 || tc.sizes() != ts.sizes() || tc.scalar_type() != at::kFloat || ts.scalar_type() != at::kFloat ||
          !on(tc, c.device) || !on(ts, c.device) || !tc.is_contiguous() || !ts.is_contiguous())
        refuse("cos and sin must be contiguous fp32 tables [positions, rotary_dim / 2] on cuda:", c.device);
      positions = tc.size(0);
      rotary = 2 * tc.size(1);
      if (rotary % 16 || rotary > d) refuse("rotary_dim must be a multiple of 16 up to ", d, ", got ", rotary);
      cos = tc.const_data_ptr<float>();
      sin = ts.const_data_ptr<float>();
    }
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, c.device));
    qkv = rows_of(qkv);
    at::Tensor out = output(args[10], {rows, q_heads, d}, qkv.scalar_type(), c.device, 16);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device);
    const bool interleaved = truth(args[9], "interleaved");
    check(unlocked([&] {
            return tq_paged_append(c.kv, &b, qkv.data_ptr(), code, qkv.stride(0), (int)q_heads, cos, sin, positions,
                                   (int)rotary, interleaved, out.data_ptr(), stream);
          }),
          "paged append");
    return wrap(std::move(out));
  });
}

// (kv, device, q, lengths, block_table, token_starts, max_new_tokens, max_context, lengths_counted, scale, return_lse, out)
PyObject* paged_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 12) refuse("paged_attend takes 12 arguments");
    const Cache c(args);
    at::Tensor q = tensor(args[2], "q");
    const int64_t d = c.kv->head_dim;
    if (q.dim() != 3 || q.size(2) != d || !on(q, c.device)) refuse("q must be [rows, q_heads, ", d, "] on cuda:", c.device);
    const int64_t rows = q.size(0), q_heads = q.size(1);
    if (q_heads == 0 || q_heads % c.kv->kv_heads)
      refuse("q_heads ", q_heads, " must be a positive multiple of kv_heads ", c.kv->kv_heads);
    const at::ScalarType type = q.scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) refuse("q must be float16 or bfloat16, got ", type);
    const tq_paged_batch b = batch_of(c, rows, args[3], args[4], args[5], args[6]);
    int64_t most_context = (int64_t)b.table_width * c.kv->page_size;
    if (given(args[7])) {
      most_context = integer(args[7], "max_context");
      if (most_context < 0) refuse("max_context must not be negative");
    }
    const bool counted = truth(args[8], "lengths_counted"), want_lse = truth(args[10], "return_lse");
    const double scale = given(args[9]) ? real(args[9], "scale") : 1.0 / std::sqrt((double)d);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, c.device));
    q = rows_of(q);
    at::Tensor out = output(args[11], {rows, q_heads, d}, type, c.device, 32), lse;
    if (want_lse) lse = at::empty({rows, q_heads}, q.options().dtype(at::kFloat));
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device);
    size_t need = 0;
    check(tq_paged_attend_workspace_size(c.kv, (int)q_heads, b.max_new_tokens, &need), "paged attend");
    const c10::DataPtr ws = scratch(need);
    check(unlocked([&] {
            return tq_paged_attend(c.kv, &b, q.data_ptr(), dtype_code(type), q.stride(0), (int)q_heads, counted,
                                   (float)scale, most_context, out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr,
                                   ws.get(), need, stream);
          }),
          "paged attend");
    return want_lse ? wrap_pair(std::move(out), std::move(lse)) : wrap(std::move(out));
  });
}

// (kv, device, page_ids, dtype as an empty tensor's)
PyObject* paged_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 4) refuse("paged_dequantize takes 4 arguments");
    const Cache c(args);
    const at::Tensor& ids = tensor(args[2], "page_ids");
    if (ids.scalar_type() != at::kInt || ids.dim() != 1 || !on(ids, c.device) || !ids.is_contiguous())
      refuse("page_ids must be contiguous int32 [n] on cuda:", c.device);
    if (!THPDtype_Check(args[3])) refuse("dtype must be a torch dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
    const int code = dtype_code(type);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, c.device));
    const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, c.device);
    const int64_t shape[4] = {ids.size(0), c.kv->kv_heads, c.kv->page_size, c.kv->head_dim};
    at::Tensor k = at::empty(at::IntArrayRef(shape, 4), options), v = at::empty(at::IntArrayRef(shape, 4), options);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device);
    check(unlocked([&] {
            return tq_paged_dequantize(c.kv, ids.const_data_ptr<int32_t>(), ids.size(0), k.data_ptr(), v.data_ptr(), code,
                                       stream);
          }),
          "paged dequantize");
    return wrap_pair(std::move(k), std::move(v));
  });
}

// ---------------------------------------------------------------------------
// (codes, scales, n, k, group_size, x, mode, norm_weight, eps, residual, out)
PyObject* gemv_w4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 11) refuse("gemv_w4 takes 11 arguments");
    const at::Tensor &codes = tensor(args[0], "codes"), &scales = tensor(args[1], "scales");
    const int64_t n = integer(args[2], "n"), k = integer(args[3], "k"), group = integer(args[4], "group_size");
    at::Tensor x = tensor(args[5], "x");
    const int mode = (int)integer(args[6], "mode"), device = codes.get_device();
    const int64_t width = mode == 3 ? 2 * k : k;
    if (x.dim() < 1 || x.dim() > 2 || x.size(-1) != width || !on(x, device))
      refuse("gemv_w4: x must be [tokens, ", width, "] on cuda:", device, ", got ", x.sizes());
    at::ScalarType type = x.scalar_type();
    if (mode == 1) {
      if (type != at::kFloat) refuse("gemv_w4: x must be float32 in mode 'f32', got ", type);
      type = at::kBFloat16;
    } else if (type != at::kBFloat16 && !(mode == 0 && type == at::kHalf)) {
      refuse("gemv_w4: x must be bfloat16", mode == 0 ? " or float16" : "", " in this mode, got ", type);
    }
    const int64_t tokens = x.dim() == 2 ? x.size(0) : 1;
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, device));
    if ((width > 1 && x.stride(-1) != 1) || (x.dim() == 2 && !apart(x, 0))) x = x.contiguous();
    const void *norm = nullptr, *residual = nullptr;
    if (mode == 2) {
      if (!given(args[7])) refuse("gemv_w4: mode 'rms' needs norm_weight");
      const at::Tensor& w = tensor(args[7], "norm_weight");
      if (w.scalar_type() != at::kBFloat16 || w.numel() != k || !on(w, device) || !w.is_contiguous())
        refuse("gemv_w4: norm_weight must be contiguous bf16 [", k, "] on cuda:", device);
      norm = w.data_ptr();
    }
    if (given(args[9])) {
      const at::Tensor& r = tensor(args[9], "residual");
      if (r.scalar_type() != type || r.numel() != tokens * n || !on(r, device) || !r.is_contiguous())
        refuse("gemv_w4: residual must be contiguous ", type, " of ", tokens, " x ", n, " on cuda:", device);
      residual = r.data_ptr();
    }
    at::Tensor out;
    if (given(args[10])) {
      out = tensor(args[10], "out");
      if (out.scalar_type() != type || out.numel() != tokens * n || !on(out, device) || !out.is_contiguous())
        refuse("gemv_w4: out must be contiguous ", type, " of ", tokens, " x ", n, " on cuda:", device);
    } else {
      const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, device);
      out = x.dim() == 2 ? at::empty({tokens, n}, options) : at::empty({n}, options);
    }
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    size_t need = 0;
    check(tq_gemv_w4_workspace_size(n, k, tokens, &need), "gemv_w4");
    c10::DataPtr ws;
    if (need) ws = scratch(need);
    const float eps = (float)real(args[8], "eps");
    check(unlocked([&] {
            return tq_gemv_w4(codes.data_ptr(), scales.data_ptr(), n, k, (int)group, x.data_ptr(),
                              type == at::kHalf ? TQ_F16 : TQ_BF16, x.dim() == 2 ? x.stride(0) : width, mode, norm, eps,
                              residual, out.data_ptr(), tokens, ws.get(), need, stream);
          }),
          "gemv_w4");
    return wrap(std::move(out));
  });
}

// (target_probs, draft_probs, draft_tokens, uniform, noise, draft_counts)
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6) refuse("verify_drafts takes 6 arguments");
    at::Tensor target = tensor(args[0], "target_probs");
    if (target.dim() != 3 || !target.is_cuda() || target.size(1) < 1 || target.size(2) < 1)
      refuse("target_probs must be a CUDA tensor [seqs, drafts + 1, vocab]");
    const int device = target.get_device();
    const int64_t seqs = target.size(0), rows = target.size(1), vocab = target.size(2), drafts = rows - 1;
    const at::ScalarType type = target.scalar_type();
    const int code = dtype_code(type);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, device));
    if ((vocab > 1 && target.stride(2) != 1) || !apart(target, 1)) target = target.contiguous();
    at::Tensor draft;
    if (given(args[1])) {
      draft = tensor(args[1], "draft_probs");
      if (draft.sizes() != at::IntArrayRef({seqs, drafts, vocab}) || draft.scalar_type() != type || !on(draft, device))
        refuse("draft_probs must be ", type, " [", seqs, ", ", drafts, ", ", vocab, "] on cuda:", device);
      if ((vocab > 1 && draft.stride(2) != 1) || !apart(draft, 1)) draft = draft.contiguous();
    }
    at::Tensor tokens = tensor(args[2], "draft_tokens"), uniform = tensor(args[3], "uniform"),
               noise = tensor(args[4], "noise");
    if (tokens.scalar_type() != at::kInt || tokens.sizes() != at::IntArrayRef({seqs, drafts}) || !on(tokens, device))
      refuse("draft_tokens must be int32 [", seqs, ", ", drafts, "] on cuda:", device);
    if (uniform.scalar_type() != at::kFloat || uniform.sizes() != at::IntArrayRef({seqs, drafts}) || !on(uniform, device))
      refuse("uniform must be fp32 [", seqs, ", ", drafts, "] on cuda:", device);
    if (noise.scalar_type() != at::kFloat || noise.sizes() != at::IntArrayRef({seqs, vocab}) || !on(noise, device))
      refuse("noise must be fp32 [", seqs, ", ", vocab, "] on cuda:", device);
    tokens = tokens.contiguous();
    uniform = uniform.contiguous();
    if ((vocab > 1 && noise.stride(1) != 1) || !apart(noise, 0)) noise = noise.contiguous();
    const int32_t* counts = nullptr;
    if (given(args[5])) {
      const at::Tensor& t = tensor(args[5], "draft_counts");
      if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != seqs || !on(t, device) || !t.is_contiguous())
        refuse("draft_counts must be contiguous int32 [", seqs, "] on cuda:", device);
      counts = t.const_data_ptr<int32_t>();
    }
    const auto options = at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device);
    at::Tensor accepted = at::empty({seqs}, options), out = at::empty({seqs, rows}, options);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    check(unlocked([&] {
            return tq_verify_drafts(target.data_ptr(), target.stride(0), target.stride(1),
                                    draft.defined() ? draft.data_ptr() : nullptr, draft.defined() ? draft.stride(0) : 0,
                                    draft.defined() ? draft.stride(1) : 0, code, tokens.const_data_ptr<int32_t>(), counts,
                                    uniform.const_data_ptr<float>(), noise.const_data_ptr<float>(), noise.stride(0), seqs,
                                    (int)drafts, vocab, accepted.data_ptr<int32_t>(), out.data_ptr<int32_t>(), stream);
          }),
          "verify drafts");
    return wrap_pair(std::move(accepted), std::move(out));
  });
}

PyMethodDef methods[] = {
    {"paged_append", (PyCFunction)(void (*)(void))paged_append, METH_FASTCALL, nullptr},
    {"paged_attend", (PyCFunction)(void (*)(void))paged_attend, METH_FASTCALL, nullptr},
    {"paged_dequantize", (PyCFunction)(void (*)(void))paged_dequantize, METH_FASTCALL, nullptr},
    {"gemv_w4", (PyCFunction)(void (*)(void))gemv_w4, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void (*)(void))verify_drafts, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_bind(void) { return PyModule_Create(&module); }
