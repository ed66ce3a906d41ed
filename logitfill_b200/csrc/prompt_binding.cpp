// Python side of a prompt's operators: tensors in, one C ABI call out.
// (Checks and errors as binding_common.h says; why they are compiled, int4_binding.cpp.)
#include "binding_common.h"

#include <ATen/ops/empty_strided.h>

#include <cmath>

namespace {

float number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    fail(PyExc_TypeError, name, " must be a number");
  }
  return static_cast<float>(v);
}

// A tensor's strides over (sequence, head, token), 0 where the extent is 1: [batch, heads,
// tokens, D], or packed [tokens, heads, D].
struct Rows {
  int64_t seq, head, tok;
  explicit Rows(const at::Tensor& t) {
    const bool packed = t.dim() == 3;
    const auto of = [&](int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; };
    seq = packed ? 0 : of(0);
    head = of(1);
    tok = of(packed ? 0 : 2);
  }
};

at::Tensor channels_last(const at::Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A new tensor like t: with its strides where it has no gaps (a projection's transposed
// view stays one), else contiguous.
at::Tensor new_like(const at::Tensor& t) {
  if (t.is_non_overlapping_and_dense()) return at::empty_strided(t.sizes(), t.strides(), t.options());
  return at::empty(t.sizes(), t.options());
}

// out given by the caller for x: like it, and written once.
void check_out(const at::Tensor& out, const at::Tensor& x, const char* name, const char* of) {
  if (out.sizes() != x.sizes() || out.scalar_type() != x.scalar_type() || out.device() != x.device() || out.stride(-1) != 1)
    fail(PyExc_ValueError, name, " must be like the ", of, " (", shape(x), ") with channel stride 1, got ", shape(out));
  if (at::has_internal_overlap(out) == at::MemOverlap::Yes) fail(PyExc_ValueError, name, " overlaps itself");
}
// The same, where out may be x itself.
void check_out_in_place(const at::Tensor& out, const at::Tensor& x, const char* name, const char* of) {
  check_out(out, x, name, of);
  const bool same = out.data_ptr() == x.data_ptr() && out.strides() == x.strides();
  if (!same && overlap(out, x)) fail(PyExc_ValueError, name, " overlaps the ", of, " without being it");
}

// rotary(query, key, freqs, positions, start, magnitude, interleaved, transposed, out) -> (query, key)
PyObject* rotary(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 9);
    const at::Tensor& query = tensor(v[0], "query");
    const bool with_key = v[1] != Py_None;
    const at::Tensor none;
    const at::Tensor &key = with_key ? tensor(v[1], "key") : none, &freqs = tensor(v[2], "freqs");
    const bool packed = query.dim() == 3;
    if (query.dim() != 3 && query.dim() != 4)
      fail(PyExc_ValueError, "query must be [batch, heads, tokens, head_dim] or [tokens, heads, head_dim], got ", shape(query));
    const int64_t B = packed ? 1 : query.size(0), T = query.size(packed ? 0 : 2), D = query.size(-1);
    if (with_key) {
      bool like = key.dim() == query.dim() && key.size(-1) == D && key.size(0) == query.size(0) && (packed || key.size(2) == T);
      if (!like || key.scalar_type() != query.scalar_type())
        fail(PyExc_ValueError, "key must be like the query but for its heads (", shape(query), "), got ", shape(key));
      if (key.device() != query.device()) fail(PyExc_RuntimeError, "key is on ", key.device(), ", query on ", query.device());
      no_gradient(key, "key");
    }
    no_gradient(query, "query");
    if (v[8] != Py_None && PyTuple_Check(v[8]))
      for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(v[8]); ++i)
        if (PyObject* o = PyTuple_GET_ITEM(v[8], i); o != Py_None) no_gradient(tensor(o, "out"), "out");
    if (!query.is_cuda()) fail(PyExc_RuntimeError, "rotary_embed needs CUDA tensors (there is no CPU path)");
    if (freqs.dim() != 1 || freqs.scalar_type() != at::kLong || !freqs.is_contiguous() || freqs.size(0) < 1 || 2 * freqs.size(0) > D ||
        freqs.device() != query.device())
      fail(PyExc_ValueError, "freqs must be a contiguous int64 [part / 2] tensor on ", query.device(), ", part at most ", D, ", got ",
           shape(freqs));
    for (const int64_t x : {B, T, query.size(1), with_key ? key.size(1) : 0})
      if (x > INT32_MAX) fail(PyExc_NotImplementedError, "an extent of ", x, " is too large");
    lf_rotary a{};
    a.dtype = type_code(query.scalar_type());
    a.head_dim = static_cast<int32_t>(D > INT32_MAX ? INT32_MAX : D);
    a.part = static_cast<int32_t>(2 * freqs.size(0));
    a.batch = static_cast<int32_t>(B);
    a.tokens = static_cast<int32_t>(T);
    a.n_q = static_cast<int32_t>(query.size(1));
    a.n_kv = with_key ? static_cast<int32_t>(key.size(1)) : 0;
    a.freqs = static_cast<const int64_t*>(freqs.data_ptr());
    if ((v[3] == Py_None) == (v[4] == Py_None)) fail(PyExc_ValueError, "give either positions or start");
    if (v[3] != Py_None) {
      const at::Tensor& at_ = tensor(v[3], "positions");
      const bool fits = packed ? at_.dim() == 1 && at_.size(0) == T : at_.dim() == 2 && at_.size(0) == B && at_.size(1) == T;
      if (!fits || (at_.scalar_type() != at::kLong && at_.scalar_type() != at::kInt) || at_.device() != query.device())
        fail(PyExc_ValueError, "positions must be int32 or int64 ", packed ? "[tokens]" : "[batch, tokens]", " on ", query.device(),
             " for ", shape(query), ", got ", shape(at_));
      a.positions = at_.data_ptr();
      a.positions_64 = at_.scalar_type() == at::kLong;
      a.pos_seq_stride = packed ? 0 : at_.stride(0);
      a.pos_tok_stride = at_.stride(-1);
    } else {
      const at::Tensor& at_ = tensor(v[4], "start");
      if (at_.scalar_type() != at::kInt || at_.dim() != 1 || at_.size(0) != B || !at_.is_contiguous() || at_.device() != query.device())
        fail(PyExc_ValueError, "start must be a contiguous int32 [", B, "] tensor on ", query.device(), ", got ", shape(at_));
      a.start = static_cast<const int32_t*>(at_.data_ptr());
    }
    a.magnitude = number(v[5], "magnitude");
    a.interleaved = truth(v[6], "interleaved");
    a.transposed = truth(v[7], "transposed");

    const Launch on(query.device());
    const at::Tensor q = channels_last(query), k = with_key ? channels_last(key) : none;
    at::Tensor q_out, k_out;
    if (v[8] == Py_None) {
      q_out = new_like(q);
      if (with_key) k_out = new_like(k);
    } else {
      if (!PyTuple_Check(v[8]) || PyTuple_GET_SIZE(v[8]) != 2) fail(PyExc_TypeError, "out must be a tuple (query, key)");
      q_out = tensor(PyTuple_GET_ITEM(v[8], 0), "out[0]");
      check_out_in_place(q_out, query, "out[0]", "query");
      if (with_key) {
        k_out = tensor(PyTuple_GET_ITEM(v[8], 1), "out[1]");
        check_out_in_place(k_out, key, "out[1]", "key");
        if (overlap(q_out, k_out) || overlap(q_out, key) || overlap(k_out, query))
          fail(PyExc_ValueError, "query and key, or their outputs, share memory");
      }
    }
    const auto place = [](const at::Tensor& x, int64_t& seq, int64_t& head, int64_t& tok) {
      const Rows r(x);
      seq = r.seq;
      head = r.head;
      tok = r.tok;
      return x.data_ptr();
    };
    a.q = place(q, a.q_seq_stride, a.q_head_stride, a.q_tok_stride);
    a.q_out = place(q_out, a.q_out_seq_stride, a.q_out_head_stride, a.q_out_tok_stride);
    if (with_key) {
      a.k = place(k, a.k_seq_stride, a.k_head_stride, a.k_tok_stride);
      a.k_out = place(k_out, a.k_out_seq_stride, a.k_out_head_stride, a.k_out_tok_stride);
    }
    check(lf_rotary_embed(&a, on.raw()), "lf_rotary_embed");
    if (!with_key) return Py_BuildValue("NO", THPVariable_Wrap(std::move(q_out)), Py_None);
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(q_out)), THPVariable_Wrap(std::move(k_out)));
  });
}

// t with 16-byte aligned rows of channel stride 1 and no stride of 0 over more than one
// row (a copy where it is not so).
at::Tensor plain_rows(const at::Tensor& t) {
  bool fits = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.size(d) > 1) fits = fits && t.stride(d) > 0 && t.stride(d) * static_cast<int64_t>(t.element_size()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

const int32_t* small_ints(PyObject* o, const char* name, int64_t count, const at::Device& on) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || (count >= 0 ? t.size(0) != count : t.size(0) < 1) || t.device() != on ||
      !t.is_contiguous())
    fail(PyExc_ValueError, name, " must be a contiguous int32 [", count >= 0 ? std::to_string(count) : "batch + 1", "] tensor on ", on,
         ", got ", shape(t));
  return static_cast<const int32_t*>(t.data_ptr());
}

// attend(query, key, value, scaling, starts, counts, out, status) -> out
PyObject* attend(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 8);
    const at::Tensor &query = tensor(v[0], "query"), &key = tensor(v[1], "key"), &value = tensor(v[2], "value");
    const bool packed = query.dim() == 3;
    if (query.dim() != 3 && query.dim() != 4)
      fail(PyExc_ValueError, "query must be [batch, heads, tokens, head_dim] or [tokens, heads, head_dim], got ", shape(query));
    const int64_t T = query.size(packed ? 0 : 2), D = query.size(-1), nq = query.size(1);
    const bool like = key.dim() == query.dim() && key.size(-1) == D && key.size(0) == query.size(0) && (packed || key.size(2) == T);
    if (!like || key.sizes() != value.sizes() || key.scalar_type() != query.scalar_type() || value.scalar_type() != query.scalar_type())
      fail(PyExc_ValueError, "key and value must be like the query but for their heads (", shape(query), "), got ", shape(key), " and ",
           shape(value));
    const int64_t nkv = key.size(1);
    if (nq < 1 || nkv < 1 || nq % nkv) fail(PyExc_ValueError, nq, " query heads do not divide into ", nkv, " KV heads");
    if (query.scalar_type() != at::kHalf && query.scalar_type() != at::kBFloat16)
      fail(PyExc_NotImplementedError, "prompt attention takes fp16 or bf16, got ", c10::toString(query.scalar_type()));
    no_gradient(query, "query");
    no_gradient(key, "key");
    no_gradient(value, "value");
    if (v[6] != Py_None) no_gradient(tensor(v[6], "out"), "out");
    if (!query.is_cuda()) fail(PyExc_RuntimeError, "prompt_attention needs CUDA tensors (there is no CPU path)");
    if (key.device() != query.device() || value.device() != query.device())
      fail(PyExc_RuntimeError, "key and value must be on ", query.device());
    for (const int64_t x : {query.size(0), T, nq, D})
      if (x > INT32_MAX) fail(PyExc_NotImplementedError, "an extent of ", x, " is too large");
    lf_prompt a{};
    a.batch = static_cast<int32_t>(packed ? 1 : query.size(0));
    if (packed) {
      if (v[5] != Py_None) fail(PyExc_ValueError, "packed sequences take starts, a padded batch counts");
      if (v[4] != Py_None) {
        a.starts = small_ints(v[4], "starts", -1, query.device());
        const int64_t b = tensor(v[4], "starts").size(0) - 1;
        if (b > INT32_MAX) fail(PyExc_NotImplementedError, "an extent of ", b, " is too large");
        a.batch = static_cast<int32_t>(b);
      }
    } else {
      if (v[4] != Py_None) fail(PyExc_ValueError, "packed sequences take starts, a padded batch counts");
      if (v[5] != Py_None) a.counts = small_ints(v[5], "counts", query.size(0), query.device());
    }
    a.scaling = number(v[3], "scaling");
    if (v[7] != Py_None) {
      const at::Tensor& t = tensor(v[7], "status");
      if (t.scalar_type() != at::kInt || t.numel() < 1 || t.device() != query.device())
        fail(PyExc_ValueError, "status must be an int32 tensor on ", query.device(), ", got ", shape(t));
      a.status = static_cast<int32_t*>(t.data_ptr());
    }
    const Launch on(query.device());
    at::Tensor out;
    if (v[6] == Py_None) {
      out = new_like(query);
      if (plain_rows(out).data_ptr() != out.data_ptr()) out = at::empty(query.sizes(), query.options());
    } else {
      out = tensor(v[6], "out");
      check_out(out, query, "out", "query");
      if (overlap(out, query) || overlap(out, key) || overlap(out, value)) fail(PyExc_ValueError, "out shares memory with an input");
    }
    if (query.numel() == 0) return THPVariable_Wrap(std::move(out));
    const at::Tensor q = plain_rows(query), k = plain_rows(key), x = plain_rows(value);
    const auto place = [](const at::Tensor& y, int64_t& seq, int64_t& head, int64_t& tok) {
      const Rows r(y);
      seq = r.seq;
      head = r.head;
      tok = r.tok;
      return y.data_ptr();
    };
    a.q = place(q, a.q_seq_stride, a.q_head_stride, a.q_tok_stride);
    a.k = place(k, a.k_seq_stride, a.k_head_stride, a.k_tok_stride);
    a.v = place(x, a.v_seq_stride, a.v_head_stride, a.v_tok_stride);
    a.out = place(out, a.out_seq_stride, a.out_head_stride, a.out_tok_stride);
    a.head_dim = static_cast<int32_t>(D);
    a.dtype = type_code(q.scalar_type());
    a.tokens = static_cast<int32_t>(T);
    a.n_q = static_cast<int32_t>(nq);
    a.n_kv = static_cast<int32_t>(nkv);
    check(lf_prompt_attend(&a, on.raw()), "lf_prompt_attend");
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef methods[] = {{"rotary", fast(rotary), METH_FASTCALL, nullptr},
                         {"attend", fast(attend), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "prompt_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_prompt_binding(void) { return PyModule_Create(&module_def); }
