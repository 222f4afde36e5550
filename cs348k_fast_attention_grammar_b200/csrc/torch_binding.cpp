// Torch side of the rotary and paged operators: checks of arguments, output and
// workspace allocation and the call of the C ABI (include/fa_b200.h), as a plain
// CPython module.
//
// These operators are called per layer and step on a few rows, where the host
// decides how fast a program runs: the same checks written in Python took 10 to
// 17 us of a call's 14 to 21, here they take about one.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <exception>

#include "../../include/fa_b200.h"

namespace {

// The C ABI's functions, from the library that the package has loaded, and the
// package's check(status, where), which raises FaError.
struct Library {
  int (*rotary)(const fa_rotary_args*, void*);
  int (*paged_append)(const fa_paged_append_args*, void*);
  int64_t (*paged_attn_workspace)(const fa_paged_attn_args*);
  int (*paged_attn)(const fa_paged_attn_args*, void*, int64_t, void*);
  PyObject* check;
} lib = {};

// A Python error has been set.
struct Raised : std::exception {};

template <typename... A>
[[noreturn]] void raise(PyObject* kind, const char* format, A... args) {
  PyErr_Format(kind, format, args...);
  throw Raised();
}

// One tensor argument.
struct Arg {
  const char* name = nullptr;
  PyObject* obj = nullptr;
  const at::Tensor* t = nullptr;
  const at::Tensor* operator->() const { return t; }
  explicit operator bool() const { return t != nullptr; }
  int64_t stride(int d) const { return t->strides()[d < 0 ? d + t->dim() : d]; }
  int64_t size(int d) const { return t->sizes()[d < 0 ? d + t->dim() : d]; }
};

enum : unsigned { kBF16 = 1, kF16 = 2, kF32 = 4, kF64 = 8, kI32 = 16, kI64 = 32 };

unsigned type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return kBF16;
    case at::kHalf: return kF16;
    case at::kFloat: return kF32;
    case at::kDouble: return kF64;
    case at::kInt: return kI32;
    case at::kLong: return kI64;
    default: return 0;
  }
}

PyObject* attribute(PyObject* o, const char* name) {
  PyObject* a = PyObject_GetAttrString(o, name);
  if (a == nullptr) throw Raised();
  return a;
}

[[noreturn]] void wrong_type(const Arg& a, unsigned types) {
  static const char* const names[] = {"bfloat16", "float16", "float32", "float64", "int32", "int64"};
  std::string want;
  for (int i = 0; i < 6; ++i)
    if (types >> i & 1) want += (want.empty() ? "" : " or ") + std::string(names[i]);
  PyObject* got = attribute(a.obj, "dtype");
  PyErr_Format(PyExc_TypeError, "%s must be %s (got %S)", a.name, want.c_str(), got);
  Py_DECREF(got);
  throw Raised();
}

// Raises `text` with the tensor's shape behind it.
[[noreturn]] void wrong_shape(const Arg& a, const std::string& text) {
  PyObject* got = attribute(a.obj, "shape");
  PyErr_Format(PyExc_ValueError, "%s (got %S)", text.c_str(), got);
  Py_DECREF(got);
  throw Raised();
}

// `dims`: a bit for each number of dimensions that is taken.
Arg tensor(const char* name, PyObject* o, unsigned types, unsigned dims) {
  Arg a{name, o, nullptr};
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a torch.Tensor", name);
  a.t = &THPVariable_Unpack(o);
  if (!(type_of(*a.t) & types)) wrong_type(a, types);
  const int64_t d = a->dim();
  if (d > 30 || !(dims >> d & 1)) {
    std::string want;
    for (int i = 0; i < 8; ++i)
      if (dims >> i & 1) want += (want.empty() ? "" : " or ") + std::to_string(i) + "-D";
    wrong_shape(a, std::string(name) + " must be " + want);
  }
  return a;
}

Arg rows(const char* name, PyObject* o, unsigned types, unsigned dims) {
  const Arg a = tensor(name, o, types, dims);
  if (a.stride(-1) != 1 && a.size(-1) > 1)
    raise(PyExc_ValueError, "%s must be contiguous along its last dimension", name);
  return a;
}

// A contiguous int32 tensor of n entries.
Arg list(const char* name, PyObject* o, int64_t n) {
  const Arg a = tensor(name, o, kI32, 1u << 1);
  if (a.size(0) != n || (a.stride(0) != 1 && n > 1))
    wrong_shape(a, std::string(name) + " must be a contiguous [" + std::to_string(n) + "] tensor");
  return a;
}

void same_shape(const Arg& a, const Arg& b) {
  if (a->sizes() != b->sizes()) raise(PyExc_ValueError, "%s must have %s's shape", a.name, b.name);
}

template <typename... A>
void devices(const c10::Device& device, const A&... args) {
  auto one = [&](const Arg& a) {
    if (!a) return;
    if (!a->is_cuda())
      raise(PyExc_ValueError, "%s must be a CUDA tensor (got device %s)", a.name,
            a->device().str().c_str());
    if (a->device() != device)
      raise(PyExc_ValueError, "%s must be on %s like the others (got %s)", a.name,
            device.str().c_str(), a->device().str().c_str());
  };
  (one(args), ...);
}

int64_t dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? FA_BF16 : t.scalar_type() == at::kHalf ? FA_F16 : FA_F32;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v != 0;
}

void check(int rc, const char* where) {
  if (rc == FA_OK) return;
  PyObject* r = PyObject_CallFunction(lib.check, "is", rc, where);
  Py_XDECREF(r);
  if (r != nullptr) PyErr_Format(PyExc_RuntimeError, "%s: status %d", where, rc);
  throw Raised();
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const c10::Device& device) {
  return at::detail::empty_cuda(sizes, type, device, c10::nullopt);
}

PyObject* given(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// Frequencies and, where there are any, sections and positions.
Arg frequencies(PyObject* o, int64_t* R) {
  const Arg f = tensor("inv_freq", o, kF32 | kF64, 1u << 1);
  if (!f->is_contiguous()) raise(PyExc_ValueError, "inv_freq must be contiguous");
  *R = 2 * f.size(0);
  return f;
}

int64_t sections(PyObject* o, int64_t planes, int64_t (&ends)[4]) {
  ends[0] = planes;
  ends[1] = ends[2] = ends[3] = 0;
  if (o == Py_None) return 1;
  PyObject* seq = PySequence_Fast(o, "sections must be a sequence of whole numbers");
  if (seq == nullptr) throw Raised();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  int64_t total = 0;
  bool whole = true;
  for (Py_ssize_t i = 0; i < n && whole; ++i) {
    PyObject* x = PySequence_Fast_GET_ITEM(seq, i);
    const long v = PyLong_Check(x) && !PyBool_Check(x) ? PyLong_AsLong(x) : 0;
    if (v <= 0 || v > INT_MAX) whole = false;
    total += v;
    if (i < 4) ends[i] = total;
  }
  Py_DECREF(seq);
  PyErr_Clear();
  if (!whole) raise(PyExc_ValueError, "sections must be positive whole numbers (got %S)", o);
  if (n < 1 || n > 4 || total != planes)
    raise(PyExc_ValueError,
          "sections must be 1 to 4 numbers that add up to %lld, the number of frequencies (got %S)",
          static_cast<long long>(planes), o);
  return n;
}

// rotary(x, positions, inv_freq, sections, interleaved, inverse, out)
PyObject* rotary(PyObject* const* in) {
  const Arg x = rows("x", in[0], kBF16 | kF16 | kF32, 1u << 3 | 1u << 4);
  fa_rotary_args a;
  const Arg freq = frequencies(in[2], &a.R);
  a.axes = sections(in[3], a.R / 2, a.section_end);
  const bool packed = x->dim() == 3;
  const int lead = in[3] == Py_None ? 0 : 1;
  a.B = packed ? 1 : x.size(0);
  a.H = x.size(1);
  a.S = packed ? x.size(0) : x.size(2);
  a.D = x.size(-1);
  const unsigned dims = packed ? 1u << 1 : 1u << 1 | 1u << 2;
  const Arg pos = tensor("positions", in[1], kI32 | kI64, dims << lead);
  const bool per_batch = pos->dim() - lead == 2;
  if ((lead && pos.size(0) != a.axes) || pos.size(-1) != a.S || (per_batch && pos.size(-2) != a.B))
    wrong_shape(pos, "positions do not match x" +
                         (lead ? " and its " + std::to_string(a.axes) + " axes" : std::string()));
  a.pos_strides[0] = lead ? pos.stride(0) : 0;
  a.pos_strides[1] = per_batch ? pos.stride(-2) : 0;
  a.pos_strides[2] = pos.stride(-1);
  Arg out;
  if (in[6] != Py_None) {
    out = rows("out", in[6], type_of(*x.t), 1u << x->dim());
    same_shape(out, x);
  }
  devices(x->device(), x, pos, freq, out);
  at::Tensor made;
  if (!out) {
    made = make(x->sizes(), x->scalar_type(), x->device());
    out.t = &made;
  }
  auto strides = [&](const Arg& t, int64_t(&s)[3]) {
    s[0] = packed ? 0 : t.stride(0);
    s[1] = t.stride(1);
    s[2] = packed ? t.stride(0) : t.stride(2);
  };
  if (x->numel() > 0) {
    strides(x, a.x_strides);
    strides(out, a.out_strides);
    a.x = x->data_ptr();
    a.out = out->data_ptr();
    a.positions = pos->data_ptr();
    a.inv_freq = freq->data_ptr();
    a.dtype = dtype_code(*x.t);
    a.pos_is_i64 = pos->scalar_type() == at::kLong;
    a.freq_is_f64 = freq->scalar_type() == at::kDouble;
    a.interleaved = truth(in[4]);
    a.inverse = truth(in[5]);
    const c10::cuda::CUDAGuard guard(x->device());
    check(lib.rotary(&a, c10::cuda::getCurrentCUDAStream().stream()), "fa_rotary");
  }
  return out.obj ? given(out.obj) : THPVariable_Wrap(std::move(made));
}

// What append and attention check alike.
struct Paged {
  Arg k_cache, v_cache, table, lens, cu;
};
Paged paged(int64_t T, unsigned type, int64_t D, PyObject* k, PyObject* v, PyObject* table,
            PyObject* lens, PyObject* cu) {
  Paged p;
  p.k_cache = rows("k_cache", k, type, 1u << 4);
  p.v_cache = rows("v_cache", v, type, 1u << 4);
  if (p.k_cache->sizes() != p.v_cache->sizes() || p.k_cache.size(3) != D)
    wrong_shape(p.k_cache, "caches must both be [pages, page_size, Hkv, " + std::to_string(D) + "]");
  p.table = tensor("block_table", table, kI32, 1u << 2);
  if (p.table.stride(1) != 1 && p.table.size(1) > 1)
    raise(PyExc_ValueError, "block_table must be contiguous along its last dimension");
  const int64_t B = p.table.size(0);
  p.lens = list("kv_lens", lens, B);
  if (cu != Py_None) {
    p.cu = list("cu_seqlens", cu, B + 1);
  } else if (T != B) {
    raise(PyExc_ValueError,
          "without cu_seqlens every sequence has one new token: %lld tokens, %lld sequences",
          static_cast<long long>(T), static_cast<long long>(B));
  }
  return p;
}

// The members that both argument structs share.
template <typename Args>
void fill(Args& a, const Paged& p) {
  a.block_table = static_cast<const int32_t*>(p.table->data_ptr());
  a.kv_lens = static_cast<const int32_t*>(p.lens->data_ptr());
  a.cu_seqlens = p.cu ? static_cast<const int32_t*>(p.cu->data_ptr()) : nullptr;
  a.k_cache = p.k_cache->data_ptr();
  a.v_cache = p.v_cache->data_ptr();
  a.B = p.table.size(0);
  a.pages = p.k_cache.size(0);
  a.page_size = p.k_cache.size(1);
  a.max_pages = p.table.size(1);
  a.table_stride = p.table.stride(0);
  for (int i = 0; i < 3; ++i) {
    a.k_cache_strides[i] = p.k_cache.stride(i);
    a.v_cache_strides[i] = p.v_cache.stride(i);
  }
}

// paged_kv_append(k, v, k_cache, v_cache, block_table, kv_lens, cu_seqlens, q, inv_freq,
//                 positions, sections, interleaved, q_out)
PyObject* paged_kv_append(PyObject* const* in) {
  const Arg k = rows("k", in[0], kBF16 | kF16, 1u << 3);
  const unsigned type = type_of(*k.t);
  const Arg v = rows("v", in[1], type, 1u << 3);
  if (k->sizes() != v->sizes()) wrong_shape(v, "k and v shapes differ: v");
  fa_paged_append_args a = {};
  a.T = k.size(0);
  a.Hkv = k.size(1);
  a.D = k.size(2);
  if (a.Hkv == 0) raise(PyExc_ValueError, "k and v must have at least one head");
  const Paged p = paged(a.T, type, a.D, in[2], in[3], in[4], in[5], in[6]);
  if (p.k_cache.size(2) != a.Hkv)
    raise(PyExc_ValueError, "the caches have %lld heads, k has %lld",
          static_cast<long long>(p.k_cache.size(2)), static_cast<long long>(a.Hkv));
  Arg q, q_out, pos, freq;
  if (in[7] != Py_None) {
    q = rows("q", in[7], type, 1u << 3);
    if (q.size(0) != a.T || q.size(2) != a.D)
      wrong_shape(q, "q must be [" + std::to_string(a.T) + ", Hq, " + std::to_string(a.D) + "]");
    a.Hq = q.size(1);
    if (in[12] != Py_None) {
      q_out = rows("q_out", in[12], type, 1u << 3);
      same_shape(q_out, q);
    }
  } else if (in[12] != Py_None) {
    raise(PyExc_ValueError, "q_out needs q");
  }
  a.axes = 1;
  if (in[8] != Py_None) {
    freq = frequencies(in[8], &a.R);
    a.axes = sections(in[10], a.R / 2, a.section_end);
    if (in[9] != Py_None) {
      const int lead = in[10] == Py_None ? 0 : 1;
      pos = tensor("positions", in[9], kI32 | kI64, 1u << (1 + lead));
      if (pos.size(-1) != a.T || (lead && pos.size(0) != a.axes))
        wrong_shape(pos, "positions must be [" + (lead ? std::to_string(a.axes) + ", " : "") +
                             std::to_string(a.T) + "]");
      a.pos_strides[0] = lead ? pos.stride(0) : 0;
      a.pos_strides[1] = pos.stride(-1);
    } else if (a.axes > 1) {
      raise(PyExc_ValueError, "several axes need positions");
    }
  } else if (in[9] != Py_None || in[10] != Py_None) {
    raise(PyExc_ValueError, "positions and sections need inv_freq");
  }
  devices(k->device(), k, v, p.k_cache, p.v_cache, p.table, p.lens, p.cu, q, q_out, pos, freq);
  at::Tensor made;
  if (q && !q_out) {
    made = make(q->sizes(), q->scalar_type(), q->device());
    q_out.t = &made;
  }
  if (k->numel() > 0) {
    fill(a, p);
    a.k = k->data_ptr();
    a.v = v->data_ptr();
    a.dtype = dtype_code(*k.t);
    for (int i = 0; i < 2; ++i) {
      a.k_strides[i] = k.stride(i);
      a.v_strides[i] = v.stride(i);
    }
    if (a.Hq > 0) {
      a.q = q->data_ptr();
      a.q_out = q_out->data_ptr();
      for (int i = 0; i < 2; ++i) {
        a.q_strides[i] = q.stride(i);
        a.q_out_strides[i] = q_out.stride(i);
      }
    }
    if (freq) {
      a.inv_freq = freq->data_ptr();
      a.freq_is_f64 = freq->scalar_type() == at::kDouble;
    }
    if (pos) {
      a.positions = pos->data_ptr();
      a.pos_is_i64 = pos->scalar_type() == at::kLong;
    }
    a.interleaved = truth(in[11]);
    const c10::cuda::CUDAGuard guard(k->device());
    check(lib.paged_append(&a, c10::cuda::getCurrentCUDAStream().stream()), "fa_paged_append");
  }
  if (!q) Py_RETURN_NONE;
  return q_out.obj ? given(q_out.obj) : THPVariable_Wrap(std::move(made));
}

// paged_attention(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, max_q_len, causal,
//                 scale, out)
PyObject* paged_attention(PyObject* const* in) {
  const Arg q = rows("q", in[0], kBF16 | kF16, 1u << 3);
  const unsigned type = type_of(*q.t);
  fa_paged_attn_args a;
  a.T = q.size(0);
  a.Hq = q.size(1);
  a.D = q.size(2);
  const Paged p = paged(a.T, type, a.D, in[1], in[2], in[3], in[4], in[5]);
  a.Hkv = p.k_cache.size(2);
  if (a.Hkv == 0 || a.Hq % a.Hkv)
    raise(PyExc_ValueError, "%lld query heads cannot share %lld key heads evenly",
          static_cast<long long>(a.Hq), static_cast<long long>(a.Hkv));
  if (in[6] == Py_None) {
    a.max_q_len = p.cu ? a.T : 1;
  } else {
    a.max_q_len = PyLong_AsLongLong(in[6]);
    if (a.max_q_len == -1 && PyErr_Occurred()) throw Raised();
    if (a.max_q_len < 0) raise(PyExc_ValueError, "max_q_len must not be negative");
  }
  if (a.max_q_len == 0) a.max_q_len = 1;
  a.scale = a.D > 0 ? 1.0 / std::sqrt(static_cast<double>(a.D)) : 1.0;
  if (in[8] != Py_None) {
    a.scale = PyFloat_AsDouble(in[8]);
    if (PyErr_Occurred()) throw Raised();
  }
  a.causal = truth(in[7]);
  Arg out;
  if (in[9] != Py_None) {
    out = rows("out", in[9], type, 1u << 3);
    same_shape(out, q);
  }
  devices(q->device(), q, p.k_cache, p.v_cache, p.table, p.lens, p.cu, out);
  at::Tensor made;
  if (!out) {
    made = make(q->sizes(), q->scalar_type(), q->device());
    out.t = &made;
  }
  if (q->numel() > 0) {
    fill(a, p);
    a.q = q->data_ptr();
    a.o = out->data_ptr();
    a.dtype = dtype_code(*q.t);
    for (int i = 0; i < 2; ++i) {
      a.q_strides[i] = q.stride(i);
      a.o_strides[i] = out.stride(i);
    }
    const c10::cuda::CUDAGuard guard(q->device());
    const int64_t size = lib.paged_attn_workspace(&a);
    if (size < 0) check(static_cast<int>(-size), "fa_paged_attn");
    // The workspace is this call's own: on one stream the allocator hands it
    // out again in order, and a captured graph keeps its own.
    at::Tensor ws;
    if (size > 0) ws = make({size}, at::kByte, q->device());
    check(lib.paged_attn(&a, size > 0 ? ws.data_ptr() : nullptr, size, c10::cuda::getCurrentCUDAStream().stream()),
          "fa_paged_attn");
  }
  return out.obj ? given(out.obj) : THPVariable_Wrap(std::move(made));
}

// Entry: argument count, and C++ exceptions to torch's Python errors (one for
// memory that is out).
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
  if (lib.check == nullptr) return PyErr_Format(PyExc_RuntimeError, "the library is not bound");
  HANDLE_TH_ERRORS
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(fa_rotary, fa_paged_append, fa_paged_attn_workspace, fa_paged_attn, check):
// addresses as whole numbers.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "5 arguments expected, got %zd", n);
  void* at[4];
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  lib.rotary = reinterpret_cast<decltype(lib.rotary)>(at[0]);
  lib.paged_append = reinterpret_cast<decltype(lib.paged_append)>(at[1]);
  lib.paged_attn_workspace = reinterpret_cast<decltype(lib.paged_attn_workspace)>(at[2]);
  lib.paged_attn = reinterpret_cast<decltype(lib.paged_attn)>(at[3]);
  Py_INCREF(args[4]);
  lib.check = args[4];
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, nullptr},
    {"rotary", fast(entry<rotary, 7>), METH_FASTCALL, nullptr},
    {"paged_kv_append", fast(entry<paged_kv_append, 13>), METH_FASTCALL, nullptr},
    {"paged_attention", fast(entry<paged_attention, 10>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fa_torch", nullptr, -1, methods,
                      nullptr,               nullptr,     nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fa_torch() { return PyModule_Create(&module); }
