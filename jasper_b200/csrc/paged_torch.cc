// paged_torch.cc -- the Python boundary of the paged cache: torch tensors in,
// C ABI calls (include/jasper_b200.h) out.
//
// A decode step makes several of these calls a layer and its kernels take a
// few microseconds each, so what the boundary costs is part of the operator:
// checking the tensors and passing some 20 arguments from Python took 10 to 17
// us a call, here it takes about one.  The C functions come from the library
// that jasper_b200._lib has loaded (init()); no torch type crosses that ABI.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <memory>
#include <sstream>
#include <stdexcept>
#include <string>

#include "../../include/jasper_b200.h"

namespace {

using at::Tensor;

PyObject* g_jasper_error = nullptr;
const char* (*g_last_error)() = nullptr;
decltype(&jb_rotary) g_rotary;
decltype(&jb_kv_append) g_append;
decltype(&jb_pages_extend) g_extend;
decltype(&jb_pages_fork) g_fork;
decltype(&jb_pages_free) g_free;
decltype(&jb_pages_adopt) g_adopt;
decltype(&jb_pages_compact) g_compact;
decltype(&jb_pages_copy) g_copy;
decltype(&jb_paged_attention) g_attention;

struct ValueError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct PythonError {};  // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw ValueError(s.str());
}

// Runs one call; C++ exceptions become Python's.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const PythonError&) {
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void check_call(int rc) {
  if (rc == JB_OK) return;
  const char* msg = g_last_error();
  if (rc == JB_ERR_INVALID_ARGUMENT) throw ValueError(msg);
  PyObject* e = PyObject_CallFunction(g_jasper_error, "is", rc, msg);
  if (e) {
    PyErr_SetObject(g_jasper_error, e);
    Py_DECREF(e);
  }
  throw PythonError{};
}

void need_args(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("expected ", want, " arguments, got ", n);
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return v;
}

bool truth(PyObject* o) { return PyObject_IsTrue(o) == 1; }

const jb_page_cache& cache_at(PyObject* o) {
  return *reinterpret_cast<const jb_page_cache*>(static_cast<uintptr_t>(integer(o)));
}

at::ScalarType type_of(const jb_page_cache& c) {
  return c.dtype == JB_F16 ? at::kHalf : at::kBFloat16;
}

c10::Device device_of(const jb_page_cache& c) {
  return c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(c.device));
}

void* stream_of(int device) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

uint32_t layer_of(PyObject* o) {
  const int64_t v = integer(o);
  if (v < 0 || v > 0xFFFFFFFFll) refuse("layer out of range");
  return uint32_t(v);
}

// [tokens, heads, dim] with dim contiguous, on the device.
Tensor heads(const Tensor& t, const char* name, int64_t n_heads, int64_t dim, at::ScalarType type,
             c10::Device dev) {
  if (t.dim() != 3 || t.size(2) != dim || (n_heads >= 0 && t.size(1) != n_heads))
    refuse(name, " must be [n, ", n_heads < 0 ? std::string("heads") : std::to_string(n_heads), ", ",
           dim, "], got ", t.sizes());
  if (t.scalar_type() != type) refuse(name, " must be ", type, ", got ", t.scalar_type());
  if (t.device() != dev) refuse(name, " must be on ", dev, ", got ", t.device());
  return t.stride(2) == 1 || dim == 1 ? t : t.contiguous();
}

// A 1D int32 tensor of n entries (n < 0: any number) on the device.
Tensor ints(PyObject* o, const char* name, int64_t n, c10::Device dev) {
  const Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.device() != dev)
    refuse(name, " must be a 1D int32 tensor on ", dev, ", got ", t.dim(), "D ", t.scalar_type(), " on ",
           t.device());
  if (n >= 0 && t.size(0) != n) refuse(name, " must have ", n, " entries, got ", t.size(0));
  return t.is_contiguous() ? t : t.contiguous();
}

// Positions of n tokens, int32 or int64.
Tensor positions_of(const Tensor& t, int64_t n, c10::Device dev) {
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
    refuse("positions must be int32 or int64, got ", t.scalar_type());
  if (t.dim() != 1 || t.size(0) != n || t.device() != dev)
    refuse("positions must be [", n, "] on ", dev, ", got ", t.sizes(), " on ", t.device());
  return t.is_contiguous() ? t : t.contiguous();
}

void check_out(const Tensor& out, const Tensor& like, const char* name) {
  if (out.sizes() != like.sizes() || out.scalar_type() != like.scalar_type() ||
      out.device() != like.device() || (out.stride(-1) != 1 && out.size(-1) != 1))
    refuse(name, " must have the input's shape, type and device, and contiguous heads");
  if ((out.requires_grad() && at::GradMode::is_enabled()) || out._fw_grad(0).defined())
    refuse(name, " must not require a gradient: what is written to it is not recorded");
}

// A tensor of the caller's was written to: autograd sees that by its version.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A call without derivatives: its results, made from q, raise in a backward pass
// that reaches them, and tangents are refused.
void check_tangent(const Tensor& q, const char* call) {
  if (q._fw_grad(0).defined()) refuse(call, " has no forward-mode derivative");
}
template <typename... R>
void not_differentiable(const char* call, const Tensor& q, const R&... results) {
  if (!torch::autograd::compute_requires_grad(q)) return;
  const std::shared_ptr<torch::autograd::Node> fn(
      new torch::autograd::NotImplemented(call, torch::autograd::collect_next_edges(q)), torch::autograd::deleteNode);
  (torch::autograd::set_history(results, fn), ...);
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

uint32_t count32(int64_t n) {
  if (n > 0xFFFFFFFFll) refuse("too many entries");
  return uint32_t(n);
}

// rotary(x, positions, out, inverse, freq, head_dim, rot_dim, scale, interleaved) -> out
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 9);
    const Tensor& freq = THPVariable_Unpack(a[4]);
    const c10::Device dev = freq.device();
    if (!dev.is_cuda()) refuse("this Rotary is on ", dev, ": apply() needs one on a CUDA device");
    const Tensor& given = tensor(a[0], "x");
    const at::ScalarType type = given.scalar_type();
    const int dtype = type == at::kHalf ? JB_F16 : type == at::kBFloat16 ? JB_BF16 : JB_F32;
    if (dtype == JB_F32 && type != at::kFloat) refuse("Unsupported tensor dtype: ", type);
    Tensor x = given, out, flat_out, pos = tensor(a[1], "positions");
    if (a[2] != Py_None) {
      out = tensor(a[2], "out");
      check_out(out, x, "out");
    } else if (dev == x.device()) {
      out = empty(x.sizes(), type, dev);
    } else {
      refuse("x must be on ", dev, ", got ", x.device());
    }
    flat_out = out;
    if (x.dim() == 4) {
      if (pos.dim() < 1 || pos.dim() > 2 || pos.size(-1) != x.size(1) || (pos.dim() == 2 && pos.size(0) != x.size(0)))
        refuse("positions must be [", x.size(0), ", ", x.size(1), "] or [", x.size(1), "], got ", pos.sizes());
      pos = pos.expand({x.size(0), x.size(1)}).reshape({-1});
      flat_out = out.flatten(0, 1);
      if (flat_out.const_data_ptr() != out.const_data_ptr()) refuse("out's batch and tokens must be one run of tokens");
      x = x.flatten(0, 1);
    }
    const int64_t dim = integer(a[5]);
    x = heads(x, "x", -1, dim, type, dev);
    pos = positions_of(pos, x.size(0), dev);
    c10::cuda::OptionalCUDAGuard on(dev);
    check_call(g_rotary(x.const_data_ptr(), x.stride(0), x.stride(1), flat_out.mutable_data_ptr(),
                        flat_out.stride(0), flat_out.stride(1), dtype, x.size(0), uint32_t(x.size(1)),
                        uint32_t(dim), uint32_t(integer(a[6])), pos.const_data_ptr(),
                        pos.scalar_type() == at::kLong, static_cast<const int64_t*>(freq.const_data_ptr()),
                        float(real(a[7])), truth(a[8]), truth(a[3]), stream_of(dev.index())));
    if (a[2] != Py_None) written(out);
    return THPVariable_Wrap(out);
  });
}

// append(cache, layer, k, v, rows, index, q, positions, q_out, freq, head_dim, rot_dim, scale,
//        interleaved) -> q_out or None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 14);
    const jb_page_cache& c = cache_at(a[0]);
    const c10::Device dev = device_of(c);
    const at::ScalarType type = type_of(c);
    const Tensor k = heads(tensor(a[2], "k"), "k", c.n_kv_heads, c.head_dim, type, dev);
    const Tensor v = heads(tensor(a[3], "v"), "v", c.n_kv_heads, c.head_dim, type, dev);
    const int64_t n = k.size(0);
    if (v.size(0) != n) refuse("v must have ", n, " tokens, got ", v.size(0));
    const Tensor rows = ints(a[4], "rows", n, dev);
    Tensor index, q, q_out, pos;
    if (a[5] != Py_None) index = ints(a[5], "index", n, dev);
    const bool turn = a[9] != Py_None;
    if (turn) {
      const Tensor& freq = THPVariable_Unpack(a[9]);
      if (integer(a[10]) != int64_t(c.head_dim) || freq.device() != dev)
        refuse("rotary must be for heads of ", c.head_dim, " on ", dev);
    }
    if (a[6] != Py_None) {
      if (!turn) refuse("q is only taken to be rotated: pass rotary");
      q = heads(tensor(a[6], "q"), "q", -1, c.head_dim, type, dev);
      if (q.size(0) != n) refuse("q must have ", n, " tokens, got ", q.size(0));
      check_tangent(q, "PagedCache.append");
      if (a[8] != Py_None) {
        q_out = tensor(a[8], "q_out");
        check_out(q_out, q, "q_out");
      } else {
        q_out = empty(q.sizes(), type, dev);
      }
    }
    if (a[7] != Py_None) pos = positions_of(tensor(a[7], "positions"), n, dev);
    const bool has_q = q.defined();
    check_call(g_append(
        &c, layer_of(a[1]), n, has_q ? q.const_data_ptr() : nullptr, has_q ? q.stride(0) : 0,
        has_q ? q.stride(1) : 0, has_q ? q_out.mutable_data_ptr() : nullptr, has_q ? q_out.stride(0) : 0,
        has_q ? q_out.stride(1) : 0, has_q ? uint32_t(q.size(1)) : 0, k.const_data_ptr(), k.stride(0),
        k.stride(1), v.const_data_ptr(), v.stride(0), v.stride(1), i32(rows),
        index.defined() ? i32(index) : nullptr, pos.defined() ? pos.const_data_ptr() : nullptr,
        pos.defined() && pos.scalar_type() == at::kLong,
        turn ? static_cast<const int64_t*>(THPVariable_Unpack(a[9]).const_data_ptr()) : nullptr,
        turn ? uint32_t(integer(a[11])) : 0, turn ? float(real(a[12])) : 1.0f, turn && truth(a[13]),
        stream_of(c.device)));
    if (!has_q) Py_RETURN_NONE;
    if (a[8] != Py_None) written(q_out);
    else not_differentiable("PagedCache.append", q, q_out);
    return THPVariable_Wrap(q_out);
  });
}

// attend(cache, layer, q, rows, scale, window, mask, return_lse, out) -> out or (out, lse)
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 9);
    const jb_page_cache& c = cache_at(a[0]);
    const c10::Device dev = device_of(c);
    Tensor q = heads(tensor(a[2], "q"), "q", -1, c.head_dim, type_of(c), dev);
    check_tangent(q, "PagedCache.attend");
    const int64_t n = q.size(0), n_heads = q.size(1);
    if (c.n_kv_heads && n_heads % c.n_kv_heads)  // a cache without heads is refused below, with its other limits
      refuse("q's heads (", n_heads, ") must be a multiple of the cache's (", c.n_kv_heads, ")");
    if (q.stride(0) % 8 || q.stride(1) % 8 || reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16)
      q = q.clone(at::MemoryFormat::Contiguous);
    Tensor rows, mask, out, lse;
    if (a[3] != Py_None) rows = ints(a[3], "rows", n, dev);
    else if (n > int64_t(c.n_rows)) refuse("q has ", n, " rows, the cache ", c.n_rows);
    const int64_t window = integer(a[5]);
    if (window < 0 || window > 0xFFFFFFFFll) refuse("window must not be negative, got ", window);
    if (a[6] != Py_None) {
      mask = tensor(a[6], "mask");
      if (mask.scalar_type() != at::kBool || mask.dim() != 2 || mask.size(0) != n || mask.device() != dev)
        refuse("mask must be bool [", n, ", width] on ", dev);
      if (mask.size(1) > 1 && mask.stride(1) != 1) mask = mask.contiguous();
    }
    if (a[8] != Py_None) {
      out = tensor(a[8], "out");
      check_out(out, q, "out");
    } else {
      out = empty(q.sizes(), q.scalar_type(), dev);
    }
    const bool return_lse = truth(a[7]);
    if (return_lse) lse = empty({n, n_heads}, at::kFloat, dev);
    const double scale = a[4] == Py_None ? 1.0 / std::sqrt(double(c.head_dim)) : real(a[4]);
    const bool masked = mask.defined() && mask.size(1) > 0;
    check_call(g_attention(&c, layer_of(a[1]), q.const_data_ptr(), q.stride(0), q.stride(1),
                           out.mutable_data_ptr(), out.stride(0), out.stride(1), count32(n),
                           count32(n_heads), rows.defined() ? i32(rows) : nullptr,
                           masked ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr,
                           masked ? mask.stride(0) : 0, masked ? count32(mask.size(1)) : 0,
                           uint32_t(window), float(scale),
                           return_lse ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr,
                           stream_of(c.device)));
    if (a[8] != Py_None) written(out);
    else not_differentiable("PagedCache.attend", q, out);
    if (return_lse) not_differentiable("PagedCache.attend", q, lse);
    if (!return_lse) return THPVariable_Wrap(out);
    PyObject *o = THPVariable_Wrap(out), *l = THPVariable_Wrap(lse);
    PyObject* pair = o && l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(l);
    return pair;
  });
}

// Calls over two lists of equal length.
template <typename F>
PyObject* two_lists(PyObject* const* a, Py_ssize_t n_args, F call, const char* first, const char* second) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 3);
    const jb_page_cache& c = cache_at(a[0]);
    const c10::Device dev = device_of(c);
    const Tensor x = ints(a[1], first, -1, dev), y = ints(a[2], second, x.size(0), dev);
    check_call(call(&c, i32(x), i32(y), count32(x.size(0)), stream_of(c.device)));
    Py_RETURN_NONE;
  });
}

PyObject* py_extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return two_lists(a, n, g_extend, "rows", "tokens");
}
PyObject* py_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return two_lists(a, n, g_fork, "parents", "children");
}
PyObject* py_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return two_lists(a, n, g_copy, "src", "dst");
}

PyObject* py_free(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 2);
    const jb_page_cache& c = cache_at(a[0]);
    const Tensor rows = ints(a[1], "rows", -1, device_of(c));
    check_call(g_free(&c, i32(rows), count32(rows.size(0)), stream_of(c.device)));
    Py_RETURN_NONE;
  });
}

// adopt(cache, rows, pages, lengths)
PyObject* py_adopt(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 4);
    const jb_page_cache& c = cache_at(a[0]);
    const c10::Device dev = device_of(c);
    const Tensor rows = ints(a[1], "rows", -1, dev);
    Tensor pages = tensor(a[2], "pages"), lengths;
    if (pages.scalar_type() != at::kInt || pages.dim() != 2 || pages.device() != dev)
      refuse("pages must be a 2D int32 tensor on ", dev);
    if (pages.size(0) != rows.size(0)) refuse("pages must have ", rows.size(0), " rows, got ", pages.size(0));
    if (pages.size(1) > 1 && pages.stride(1) != 1) pages = pages.contiguous();
    if (a[3] != Py_None) lengths = ints(a[3], "lengths", rows.size(0), dev);
    check_call(g_adopt(&c, i32(rows), i32(pages), pages.stride(0), count32(pages.size(1)),
                       lengths.defined() ? i32(lengths) : nullptr, count32(rows.size(0)),
                       stream_of(c.device)));
    Py_RETURN_NONE;
  });
}

PyObject* py_compact(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 1);
    const jb_page_cache& c = cache_at(a[0]);
    Tensor remap = empty({int64_t(c.n_pages)}, at::kInt, device_of(c));
    check_call(g_compact(&c, static_cast<int32_t*>(remap.mutable_data_ptr()), stream_of(c.device)));
    return THPVariable_Wrap(remap);
  });
}

// init(JasperError, {name: address})
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need_args(n_args, 2);
    auto load = [&](auto& fn, const char* name) {
      PyObject* v = PyDict_GetItemString(a[1], name);
      if (!v) refuse("no address for ", name);
      fn = reinterpret_cast<std::decay_t<decltype(fn)>>(static_cast<uintptr_t>(integer(v)));
    };
    load(g_last_error, "jb_last_error");
    load(g_rotary, "jb_rotary");
    load(g_append, "jb_kv_append");
    load(g_extend, "jb_pages_extend");
    load(g_fork, "jb_pages_fork");
    load(g_free, "jb_pages_free");
    load(g_adopt, "jb_pages_adopt");
    load(g_compact, "jb_pages_compact");
    load(g_copy, "jb_pages_copy");
    load(g_attention, "jb_paged_attention");
    Py_INCREF(a[0]);
    Py_XDECREF(g_jasper_error);
    g_jasper_error = a[0];
    Py_RETURN_NONE;
  });
}

#define JB_METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {
    JB_METHOD(init),   JB_METHOD(rotary), JB_METHOD(append), JB_METHOD(attend),
    JB_METHOD(extend), JB_METHOD(fork),   JB_METHOD(free),   JB_METHOD(adopt),
    JB_METHOD(compact), JB_METHOD(copy_pages), {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "jasper_paged_torch", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_jasper_paged_torch() {
  return PyModule_Create(&g_module);
}
