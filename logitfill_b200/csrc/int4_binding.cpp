// Python side of the 4-bit paged cache: tensors in, one C ABI call out.
//
// A decode step makes a few calls of a few microseconds on the GPU for every
// layer.  Reading some twenty tensor attributes and filling the argument struct
// costs 8 us from Python and under 1 us here (an attention call, host side: 12.2 us
// through ctypes, 4.9 us so), which is why these functions have a compiled binding
// next to the ctypes one of the rest.  It holds checks and bookkeeping only: the
// kernels are in liblogitfill_b200.so, behind include/logitfill_b200.h.
//
// Errors: ValueError for malformed arguments, NotImplementedError for what the
// kernels do not take, RuntimeError for tensors in the wrong place and CUDA
// failures, TypeError for what is no tensor.  No C++ exception leaves a function.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <mutex>
#include <sstream>
#include <string>
#include <utility>

#include "logitfill_b200.h"

namespace {

struct Fail {
  PyObject* type;
  std::string text;
};
template <typename... A>
[[noreturn]] void fail(PyObject* type, const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Fail{type, s.str()};
}

std::string shape(const at::Tensor& t) {
  std::ostringstream s;
  s << c10::toString(t.scalar_type()) << " [";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << "] on " << t.device();
  return s.str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LF_F32;
    case at::kHalf: return LF_F16;
    case at::kBFloat16: return LF_BF16;
    default:
      fail(PyExc_NotImplementedError, "dtype ", c10::toString(t), " is not supported (float32, float16, bfloat16)");
  }
}

struct Pool {
  lf_int4_pool c;
  int head_dim;
  at::Device device = at::kCPU;
};

Pool make_pool(PyObject* pages_o, PyObject* table_o) {
  const at::Tensor &pages = tensor(pages_o, "pages"), &table = tensor(table_o, "page_table");
  if (pages.dim() != 3 || pages.scalar_type() != at::kInt || pages.stride(2) != 1)
    fail(PyExc_ValueError, "pages must be int32 [n_pages, n_kv, words] with word stride 1, got ", shape(pages));
  if (table.dim() != 2 || table.scalar_type() != at::kInt || table.stride(1) != 1)
    fail(PyExc_ValueError, "page_table must be int32 [batch, width] with entry stride 1, got ", shape(table));
  if (pages.numel() == 0 || table.numel() == 0)
    fail(PyExc_ValueError, "empty pool, batch or page table: pages ", shape(pages), ", page_table ", shape(table));
  if (!pages.is_cuda()) fail(PyExc_RuntimeError, "the 4-bit cache needs CUDA tensors (there is no CPU path)");
  if (table.device() != pages.device())
    fail(PyExc_RuntimeError, "page_table is on ", table.device(), ", pages on ", pages.device());
  const int64_t n = pages.size(0), H = pages.size(1), words = pages.size(2), B = table.size(0), W = table.size(1);
  if (words % 20) fail(PyExc_ValueError, "a record of ", words, " words belongs to no head_dim (20 * head_dim words)");
  for (const int64_t x : {n, H, words, B, W})
    if (x > INT32_MAX) fail(PyExc_NotImplementedError, "an extent of ", x, " is too large");
  Pool p;
  p.c.pages = static_cast<int32_t*>(pages.data_ptr());
  p.c.table = static_cast<const int32_t*>(table.data_ptr());
  p.c.page_stride = n > 1 ? pages.stride(0) : H * words;
  p.c.head_stride = H > 1 ? pages.stride(1) : words;
  p.c.table_stride = B > 1 ? table.stride(0) : W;
  p.c.table_width = static_cast<int32_t>(W);
  p.c.n_pages = static_cast<int32_t>(n);
  p.c.kv_heads = static_cast<int32_t>(H);
  p.c.batch = static_cast<int32_t>(B);
  p.head_dim = static_cast<int>(words / 20);
  p.device = pages.device();
  return p;
}

// int32 [batch] tensor, or None where that is allowed.
const int32_t* per_sequence(PyObject* o, const char* name, const Pool& p, bool optional) {
  if (optional && o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != p.c.batch || t.device() != p.device || !t.is_contiguous())
    fail(PyExc_ValueError, name, " must be a contiguous int32 [", p.c.batch, "] tensor on ", p.device, ", got ", shape(t));
  return static_cast<const int32_t*>(t.data_ptr());
}

int32_t* status_word(PyObject* o, const Pool& p) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "status");
  if (t.scalar_type() != at::kInt || t.numel() < 1 || t.device() != p.device)
    fail(PyExc_ValueError, "status must be an int32 tensor on ", p.device, ", got ", shape(t));
  return static_cast<int32_t*>(t.data_ptr());
}

int8_t* bounds_records(PyObject* o, const Pool& p, int64_t& page_stride, int64_t& head_stride) {
  page_stride = head_stride = 0;
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "bounds");
  const int64_t width = 2 * p.head_dim + 16;
  if (t.scalar_type() != at::kChar || t.dim() != 3 || t.size(0) != p.c.n_pages || t.size(1) != p.c.kv_heads ||
      t.size(2) != width || t.stride(2) != 1 || t.device() != p.device)
    fail(PyExc_ValueError, "bounds must be int8 [", p.c.n_pages, ", ", p.c.kv_heads, ", ", width, "] on ", p.device, ", got ",
         shape(t));
  page_stride = t.size(0) > 1 ? t.stride(0) : t.size(1) * width;
  head_stride = t.size(1) > 1 ? t.stride(1) : width;
  return static_cast<int8_t*>(t.data_ptr());
}

// t [B, H, T, D] with 16-byte aligned rows of channel stride 1 (a copy where it is
// not), and its first three strides (0 where the extent is 1).
at::Tensor aligned_rows(at::Tensor t, int64_t (&s)[3]) {
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    const auto address = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.stride(3) == 1 && address % 16 == 0 && (s[0] | s[1] | s[2]) * static_cast<int64_t>(t.element_size()) % 16 == 0) break;
    t = t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

// The device a call runs on made current, and its stream.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  c10::cuda::CUDAStream stream;
  explicit Launch(at::Device d) : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index())) {}
  lf_stream_t raw() const { return reinterpret_cast<lf_stream_t>(stream.stream()); }
};

void check(int status, const char* what) {
  if (status == LF_OK) return;
  fail(status == LF_ERR_UNSUPPORTED        ? PyExc_NotImplementedError
       : status == LF_ERR_INVALID_ARGUMENT ? PyExc_ValueError
                                           : PyExc_RuntimeError,
       what, ": ", lf_status_string(status), ": ", lf_last_error());
}

// Scratch of attention calls: partial results, then tickets that are zero between
// calls.  Calls on one stream share one buffer (they run in order); a call being
// captured in a CUDA graph gets its own, which the graph keeps and clears, so
// replays on any stream do not meet.
struct Scratch {
  at::Tensor words;
  size_t bytes = 0;
};
Scratch workspace(const lf_int4_query& a, const Launch& on) {
  static std::mutex mu;
  static auto* held = new std::map<std::pair<int, cudaStream_t>, Scratch>;  // outlives the CUDA context's teardown
  const size_t need = lf_int4_workspace_bytes(a.pool.batch, a.pool.kv_heads, a.n_q, a.q_len, a.head_dim);
  const auto options = at::TensorOptions().dtype(at::kByte).device(on.stream.device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    Scratch s{at::empty({static_cast<int64_t>(need)}, options), need};
    s.words.slice(0, static_cast<int64_t>(lf_int4_workspace_clear_from())).zero_();
    return s;
  }
  std::lock_guard<std::mutex> lock(mu);
  Scratch& s = (*held)[{on.stream.device_index(), on.stream.stream()}];
  if (s.bytes < need) {
    const size_t room = need + (size_t{1} << 18);
    s.words = at::zeros({static_cast<int64_t>(room)}, options);
    s.bytes = room;
  }
  return s;
}

template <typename F>
PyObject* guarded(F&& body) noexcept {
  try {
    return body();
  } catch (const Fail& f) {
    PyErr_SetString(f.type, f.text.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) fail(PyExc_TypeError, "expected ", want, " arguments, got ", got);
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    fail(PyExc_TypeError, name, " must be an integer");
  }
  return v;
}

// write(key, value, pages, page_table, start, counts, bounds, status)
PyObject* write(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 8);
    const Pool p = make_pool(v[2], v[3]);
    const at::Tensor &key = tensor(v[0], "key"), &value = tensor(v[1], "value");
    const int64_t B = p.c.batch, H = p.c.kv_heads, D = p.head_dim;
    if (key.dim() != 4 || key.sizes() != value.sizes() || key.size(0) != B || key.size(1) != H || key.size(3) != D)
      fail(PyExc_ValueError, "key and value must be [", B, ", ", H, ", T, ", D, "], got ", shape(key), " and ", shape(value));
    if (key.scalar_type() != value.scalar_type())
      fail(PyExc_ValueError, "key is ", c10::toString(key.scalar_type()), ", value ", c10::toString(value.scalar_type()));
    if (key.device() != p.device || value.device() != p.device)
      fail(PyExc_RuntimeError, "key and value must be on ", p.device);
    if (key.size(2) > INT32_MAX) fail(PyExc_NotImplementedError, "too many tokens");
    lf_int4_tokens a{};
    a.pool = p.c;
    a.dtype = type_code(key.scalar_type());
    int64_t ks[3], vs[3];
    const at::Tensor k = aligned_rows(key, ks), x = aligned_rows(value, vs);
    a.key = k.data_ptr();
    a.value = x.data_ptr();
    a.k_seq_stride = ks[0];
    a.k_head_stride = ks[1];
    a.k_tok_stride = ks[2];
    a.v_seq_stride = vs[0];
    a.v_head_stride = vs[1];
    a.v_tok_stride = vs[2];
    a.start = per_sequence(v[4], "start", p, false);
    a.counts = per_sequence(v[5], "counts", p, true);
    a.bounds = bounds_records(v[6], p, a.bounds_page_stride, a.bounds_head_stride);
    a.status = status_word(v[7], p);
    a.head_dim = p.head_dim;
    a.tokens = static_cast<int32_t>(key.size(2));
    const Launch on(p.device);
    check(lf_int4_write(&a, on.raw()), "lf_int4_write");
    Py_RETURN_NONE;
  });
}

// read(pages, page_table, start, tokens, counts, dtype, status) -> (key, value)
PyObject* read(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 7);
    const Pool p = make_pool(v[0], v[1]);
    const int64_t tokens = integer(v[3], "tokens");
    if (tokens < 0) fail(PyExc_ValueError, "cannot read ", tokens, " tokens");
    if (tokens > INT32_MAX) fail(PyExc_NotImplementedError, "too many tokens");
    if (!THPDtype_Check(v[5])) fail(PyExc_TypeError, "dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(v[5])->scalar_type;
    const int64_t B = p.c.batch, H = p.c.kv_heads, D = p.head_dim;
    lf_int4_tokens a{};
    a.pool = p.c;
    a.dtype = type_code(type);
    const Launch on(p.device);
    const auto options = at::TensorOptions().dtype(type).device(p.device);
    at::Tensor key = at::empty({B, H, tokens, D}, options), value = at::empty({B, H, tokens, D}, options);
    a.key = key.data_ptr();
    a.value = value.data_ptr();
    a.k_seq_stride = a.v_seq_stride = H * tokens * D;
    a.k_head_stride = a.v_head_stride = tokens * D;
    a.k_tok_stride = a.v_tok_stride = D;
    a.start = per_sequence(v[2], "start", p, false);
    a.counts = per_sequence(v[4], "counts", p, true);
    a.status = status_word(v[6], p);
    a.head_dim = p.head_dim;
    a.tokens = static_cast<int32_t>(tokens);
    check(lf_int4_read(&a, on.raw()), "lf_int4_read");
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(key)), THPVariable_Wrap(std::move(value)));
  });
}

// read_bounds(bounds) -> fp32 [n_pages, n_kv, 2, head_dim]
PyObject* read_bounds(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 1);
    const at::Tensor& t = tensor(v[0], "bounds");
    if (t.dim() != 3 || t.scalar_type() != at::kChar || t.stride(2) != 1 || t.size(2) % 2 || t.size(2) < 18)
      fail(PyExc_ValueError, "bounds must be int8 [n_pages, n_kv, 2 * head_dim + 16], got ", shape(t));
    if (!t.is_cuda()) fail(PyExc_RuntimeError, "the 4-bit cache needs CUDA tensors (there is no CPU path)");
    const int64_t P = t.size(0), H = t.size(1), width = t.size(2), D = (width - 16) / 2;
    if (P > INT32_MAX || H > INT32_MAX || D > INT32_MAX) fail(PyExc_NotImplementedError, "too many records");
    const Launch on(t.device());
    at::Tensor out = at::empty({P, H, 2, D}, at::TensorOptions().dtype(at::kFloat).device(t.device()));
    check(lf_int4_read_bounds(static_cast<const int8_t*>(t.data_ptr()), P > 1 ? t.stride(0) : H * width,
                              H > 1 ? t.stride(1) : width, static_cast<int>(P), static_cast<int>(H), static_cast<int>(D),
                              static_cast<float*>(out.data_ptr()), on.raw()),
          "lf_int4_read_bounds");
    return THPVariable_Wrap(std::move(out));
  });
}

// attend(query, pages, page_table, lengths, scaling, counts, out, status) -> out
// With (bounds, top, sink, recent) after these: chosen pages only, -> (out, picked).
// With (bounds, top, sink, recent, True): only the choice, -> picked.
PyObject* attend(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 8 && n != 12 && n != 13) expect(n, 12);
    const bool sparse = n > 8, choose_only = n == 13 && PyObject_IsTrue(v[12]) == 1;
    const Pool p = make_pool(v[1], v[2]);
    const at::Tensor& query = tensor(v[0], "query");
    const int64_t B = p.c.batch, H = p.c.kv_heads, D = p.head_dim;
    if ((query.dim() != 3 && query.dim() != 4) || query.size(0) != B || query.size(-1) != D || query.size(1) < 1 ||
        query.numel() == 0)
      fail(PyExc_ValueError, "query must be [", B, ", n_q, ", D, "] or [", B, ", n_q, q_len, ", D, "], got ", shape(query));
    if (query.size(1) % H) fail(PyExc_ValueError, query.size(1), " query heads do not divide into ", H, " KV heads");
    if (query.scalar_type() != at::kHalf && query.scalar_type() != at::kBFloat16)
      fail(PyExc_NotImplementedError, "the 4-bit cache's attention takes fp16 or bf16 queries, got ",
           c10::toString(query.scalar_type()));
    if (query.device() != p.device) fail(PyExc_RuntimeError, "query is on ", query.device(), ", pages on ", p.device);
    int64_t s[3];
    const at::Tensor q = aligned_rows(query.dim() == 4 ? query : query.unsqueeze(2), s);
    if (q.size(1) > INT32_MAX || q.size(2) > INT32_MAX) fail(PyExc_NotImplementedError, "too many queries");
    lf_int4_query a{};
    a.pool = p.c;
    a.q = q.data_ptr();
    a.q_seq_stride = s[0];
    a.q_head_stride = s[1];
    a.q_tok_stride = s[2];
    a.lengths = per_sequence(v[3], "lengths", p, false);
    a.counts = per_sequence(v[5], "counts", p, true);
    a.status = status_word(v[7], p);
    a.head_dim = p.head_dim;
    a.dtype = type_code(q.scalar_type());
    a.n_q = static_cast<int32_t>(q.size(1));
    a.q_len = static_cast<int32_t>(q.size(2));
    const double scaling = PyFloat_AsDouble(v[4]);
    if (scaling == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      fail(PyExc_TypeError, "scaling must be a number");
    }
    a.scaling = static_cast<float>(scaling);
    const Launch on(p.device);

    at::Tensor picked;
    if (sparse) {
      const int64_t top = integer(v[9], "top_pages"), sink = integer(v[10], "sink_pages"),
                    recent = integer(v[11], "recent_pages");
      if (top < 0 || sink < 0 || recent < 1)
        fail(PyExc_ValueError, "top ", top, " and sink ", sink, " must not be negative, recent ", recent, " at least 1");
      if (top + sink + recent > (1 << 24)) fail(PyExc_ValueError, "a budget of ", top + sink + recent, " pages is too large");
      if (v[8] == Py_None) fail(PyExc_TypeError, "bounds must be a tensor, got None");
      a.bounds = bounds_records(v[8], p, a.bounds_page_stride, a.bounds_head_stride);
      a.slots = static_cast<int32_t>(top + sink + recent);
      a.sink_pages = static_cast<int32_t>(sink);
      a.recent_pages = static_cast<int32_t>(recent);
      picked = at::empty({B, q.size(2), H, a.slots}, at::TensorOptions().dtype(at::kInt).device(p.device));
      a.picked = static_cast<int32_t*>(picked.data_ptr());
      if (choose_only) {
        check(lf_int4_select(&a, on.raw()), "lf_int4_select");
        return THPVariable_Wrap(std::move(picked));
      }
    }

    at::Tensor out;
    if (v[6] == Py_None) {
      out = at::empty(query.sizes(), query.options());
    } else {
      out = tensor(v[6], "out");
      if (out.sizes() != query.sizes() || out.scalar_type() != query.scalar_type() || out.device() != p.device ||
          out.stride(-1) != 1)
        fail(PyExc_ValueError, "out must be like the query (", shape(query), ") with channel stride 1, got ", shape(out));
    }
    a.out = out.data_ptr();
    a.out_seq_stride = B > 1 ? out.stride(0) : 0;
    a.out_head_stride = out.size(1) > 1 ? out.stride(1) : 0;
    a.out_tok_stride = out.dim() == 4 && out.size(2) > 1 ? out.stride(2) : 0;
    const Scratch scratch = workspace(a, on);
    a.workspace = scratch.words.data_ptr();
    a.workspace_bytes = scratch.bytes;
    if (!sparse) {
      check(lf_int4_attend(&a, on.raw()), "lf_int4_attend");
      return THPVariable_Wrap(std::move(out));
    }
    check(lf_int4_attend_sparse(&a, on.raw()), "lf_int4_attend_sparse");
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(picked)));
  });
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"write", fast(write), METH_FASTCALL, nullptr},
                         {"read", fast(read), METH_FASTCALL, nullptr},
                         {"read_bounds", fast(read_bounds), METH_FASTCALL, nullptr},
                         {"attend", fast(attend), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "int4_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_int4_binding(void) { return PyModule_Create(&module_def); }
