// mr_torch.cpp — the short way from torch tensors to the C ABI for the calls
// whose GPU time is less than their way through ctypes: sorted tokens and 4-bit
// products. A CPython module; the functions of libminirun_moe come to it as
// addresses (bind), so it works on whichever build of the library is loaded.
//
// Every function takes the plain case: CUDA tensors on the context's device, of
// the right types and shapes, contiguous. It returns the results, an int (the
// mr_status of a failed call), or None for anything else, which the Python
// function of that name then checks, copies or refuses. A call takes 4 to 6 us
// this way, 7 to 13 through ctypes: each allocation from Python is 2 us, here
// 0.7.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/api/include/torch/version.h>

#include <algorithm>
#include <exception>

#include "minirun_moe.h"

namespace {

struct Api {
  decltype(&mr_moe_sort) sort;
  decltype(&mr_moe_dispatch) dispatch;
  decltype(&mr_moe_dispatch_backward) dispatch_backward;
  decltype(&mr_moe_combine) combine;
  decltype(&mr_moe_combine_backward) combine_backward;
  decltype(&mr_mxfp4_quantize) quantize;
  decltype(&mr_mxfp4_quantize_swiglu) quantize_swiglu;
  decltype(&mr_mxfp4_scaled_mm) scaled_mm;
  decltype(&mr_mxfp4_grouped_mm) grouped_mm;
} api;

// A Python exception is set already (an argument that is no number or truth value).
struct Raised : std::exception {};

// A C++ exception (an allocation that failed) becomes a Python one.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, wrap(std::move(a)));
  PyTuple_SET_ITEM(r, 1, wrap(std::move(b)));
  return r;
}

struct Args {
  PyObject* const* v;
  int64_t num(int i) const {
    const long long n = PyLong_AsLongLong(v[i]);
    if (n == -1 && PyErr_Occurred()) throw Raised();
    return n;
  }
  bool flag(int i) const {
    const int b = PyObject_IsTrue(v[i]);
    if (b < 0) throw Raised();
    return b != 0;
  }
  template <typename T>
  T* at(int i) const {
    return static_cast<T*>(PyLong_AsVoidPtr(v[i]));
  }
  // A contiguous CUDA tensor on `device`, or nullptr.
  const at::Tensor* tensor(int i, int64_t device) const {
    if (!THPVariable_Check(v[i])) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(v[i]);
    return t.is_cuda() && t.get_device() == device && t.is_contiguous() ? &t : nullptr;
  }
};

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int64_t device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::DeviceType::CUDA, (int8_t)device),
                                std::nullopt);
}

void* stream_of(int64_t device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

bool row_type(const at::Tensor& t, mr_dtype* out) {
  switch (t.scalar_type()) {
    case at::kBFloat16: *out = MR_DTYPE_BF16; return true;
    case at::kHalf: *out = MR_DTYPE_F16; return true;
    case at::kFloat: *out = MR_DTYPE_F32; return true;
    default: return false;
  }
}

#define FUNC(name) PyObject* name(PyObject*, PyObject* const* argv, Py_ssize_t argc)
#define NEEDS(n) \
  if (argc != (n)) return none(); \
  const Args a { argv }

// bind(addresses of the functions of Api, in its order)
FUNC(bind) {
  if (argc != (Py_ssize_t)(sizeof(Api) / sizeof(void*))) {
    PyErr_SetString(PyExc_TypeError, "bind takes the address of every function");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < argc; ++i) {
    void* p = PyLong_AsVoidPtr(argv[i]);
    memcpy(reinterpret_cast<char*>(&api) + i * sizeof p, &p, sizeof p);
  }
  return none();
}

// sort(ctx, device, ids, experts) -> int32 [2 P + experts + 1]: order, inverse, offsets
FUNC(sort) {
  NEEDS(4);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1), E = a.num(3);
    const at::Tensor* ids = a.tensor(2, dev);
    if (!ids || ids->scalar_type() != at::kInt || ids->dim() != 2 || E <= 0 || E > INT32_MAX)
      return none();
    const int64_t T = ids->size(0), k = ids->size(1), P = T * k;
    if (k > INT32_MAX) return none();
    // (more than 1024 experts are refused)
    at::Tensor mem = empty({2 * P + std::min<int64_t>(E, 1024) + 1}, at::kInt, dev);
    int32_t* m = mem.mutable_data_ptr<int32_t>();
    const mr_status st = api.sort(a.at<mr_ctx>(0), ids->const_data_ptr<int32_t>(), T, (int32_t)k,
                                  (int32_t)E, m, m + P, m + 2 * P, stream_of(dev));
    return st ? PyLong_FromLong(st) : wrap(std::move(mem));
  });
}

// views(mem, tokens, top_k, experts) -> (order, inverse, offsets)
FUNC(views) {
  NEEDS(4);
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(argv[0])) return none();
    const at::Tensor& mem = THPVariable_Unpack(argv[0]);
    const int64_t T = a.num(1), k = a.num(2), E = a.num(3), P = T * k;
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, wrap(mem.as_strided({P}, {1}, 0)));
    PyTuple_SET_ITEM(r, 1, wrap(mem.as_strided({T, k}, {k, 1}, P)));
    PyTuple_SET_ITEM(r, 2, wrap(mem.as_strided({E + 1}, {1}, 2 * P)));
    return r;
  });
}

// dispatch / dispatch_backward(ctx, device, rows, plan): the result's rows are the plan's others
template <bool BACK>
FUNC(move_rows) {
  NEEDS(4);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    const at::Tensor* x = a.tensor(2, dev);
    const mr_sorted* plan = a.at<mr_sorted>(3);
    mr_dtype dt;
    const int64_t P = plan->tokens * plan->top_k;
    if (!x || x->dim() != 2 || !row_type(*x, &dt) || x->size(0) != (BACK ? P : plan->tokens))
      return none();
    const int64_t H = x->size(1);
    at::Tensor out = empty({BACK ? plan->tokens : P, H}, x->scalar_type(), dev);
    const mr_status st =
        (BACK ? api.dispatch_backward : api.dispatch)(a.at<mr_ctx>(0), x->const_data_ptr(), dt, H,
                                                      H, plan, out.mutable_data_ptr(),
                                                      stream_of(dev));
    return st ? PyLong_FromLong(st) : wrap(std::move(out));
  });
}

bool plan_weights(const at::Tensor* w, const mr_sorted* plan) {
  return w && w->scalar_type() == at::kFloat && w->dim() == 2 && w->size(0) == plan->tokens &&
         w->size(1) == plan->top_k;
}

// combine(ctx, device, ys, weights, plan)
FUNC(combine) {
  NEEDS(5);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    const at::Tensor *ys = a.tensor(2, dev), *w = a.tensor(3, dev);
    const mr_sorted* plan = a.at<mr_sorted>(4);
    mr_dtype dt;
    if (!ys || ys->dim() != 2 || !row_type(*ys, &dt) ||
        ys->size(0) != plan->tokens * plan->top_k || !plan_weights(w, plan))
      return none();
    const int64_t H = ys->size(1);
    at::Tensor out = empty({plan->tokens, H}, ys->scalar_type(), dev);
    const mr_status st = api.combine(a.at<mr_ctx>(0), ys->const_data_ptr(), dt, H, H,
                                     w->const_data_ptr<float>(), nullptr, plan,
                                     out.mutable_data_ptr(), stream_of(dev));
    return st ? PyLong_FromLong(st) : wrap(std::move(out));
  });
}

// combine_backward(ctx, device, dout, ys, weights, plan) -> (dys, dweights)
FUNC(combine_backward) {
  NEEDS(6);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    const at::Tensor *g = a.tensor(2, dev), *ys = a.tensor(3, dev), *w = a.tensor(4, dev);
    const mr_sorted* plan = a.at<mr_sorted>(5);
    mr_dtype dt;
    const int64_t P = plan->tokens * plan->top_k;
    if (!g || !ys || ys->dim() != 2 || g->dim() != 2 || !row_type(*ys, &dt) ||
        g->scalar_type() != ys->scalar_type() || ys->size(0) != P ||
        g->size(0) != plan->tokens || g->size(1) != ys->size(1) || !plan_weights(w, plan))
      return none();
    const int64_t H = ys->size(1);
    at::Tensor dys = empty({P, H}, ys->scalar_type(), dev);
    at::Tensor dw = empty({plan->tokens, plan->top_k}, at::kFloat, dev);
    const mr_status st = api.combine_backward(
        a.at<mr_ctx>(0), g->const_data_ptr(), H, ys->const_data_ptr(), H, dt, H,
        w->const_data_ptr<float>(), plan, dys.mutable_data_ptr(), dw.mutable_data_ptr<float>(),
        stream_of(dev));
    return st ? PyLong_FromLong(st) : pair(std::move(dys), std::move(dw));
  });
}

// quantize(ctx, device, x [rows, in], values) -> (packed, scales[, values])
FUNC(quantize) {
  NEEDS(4);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    const at::Tensor* x = a.tensor(2, dev);
    mr_dtype dt;
    if (!x || x->dim() != 2 || !row_type(*x, &dt)) return none();
    const int64_t rows = x->size(0), n = x->size(1);
    if (n <= 0 || n % 32) return none();
    at::Tensor packed = empty({rows, n / 8}, at::kInt, dev);
    at::Tensor scales = empty({rows, n / 32}, at::kByte, dev);
    at::Tensor values;
    const bool want = a.flag(3);
    if (want) values = empty({rows, n}, x->scalar_type(), dev);
    const mr_status st = api.quantize(
        a.at<mr_ctx>(0), x->const_data_ptr(), dt, rows, n, n,
        reinterpret_cast<uint32_t*>(packed.mutable_data_ptr<int32_t>()),
        scales.mutable_data_ptr<uint8_t>(), want ? values.mutable_data_ptr() : nullptr,
        stream_of(dev));
    if (st) return PyLong_FromLong(st);
    if (!want) return pair(std::move(packed), std::move(scales));
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, wrap(std::move(packed)));
    PyTuple_SET_ITEM(r, 1, wrap(std::move(scales)));
    PyTuple_SET_ITEM(r, 2, wrap(std::move(values)));
    return r;
  });
}

// quantize_swiglu(ctx, device, gate_up [rows, 2 inter], limit) -> (packed, scales)
FUNC(quantize_swiglu) {
  NEEDS(4);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    const at::Tensor* x = a.tensor(2, dev);
    mr_dtype dt;
    if (!x || x->dim() != 2 || !row_type(*x, &dt)) return none();
    const int64_t rows = x->size(0), n = x->size(1) / 2;
    if (n <= 0 || x->size(1) % 64) return none();
    const double limit = PyFloat_AsDouble(argv[3]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor packed = empty({rows, n / 8}, at::kInt, dev);
    at::Tensor scales = empty({rows, n / 32}, at::kByte, dev);
    const mr_status st = api.quantize_swiglu(
        a.at<mr_ctx>(0), x->const_data_ptr(), dt, rows, n, 2 * n, (float)limit,
        reinterpret_cast<uint32_t*>(packed.mutable_data_ptr<int32_t>()),
        scales.mutable_data_ptr<uint8_t>(), stream_of(dev));
    return st ? PyLong_FromLong(st) : pair(std::move(packed), std::move(scales));
  });
}

// An MXFP4 operand: packed int32 [experts?, rows, in / 8], scales uint8 [.., in / 32].
bool operand(const at::Tensor* p, const at::Tensor* s, bool stack, mr_mxfp4_desc* d) {
  const int64_t dims = stack ? 3 : 2;
  if (!p || !s || p->scalar_type() != at::kInt || s->scalar_type() != at::kByte ||
      p->dim() != dims || s->dim() != dims)
    return false;
  for (int64_t i = 0; i + 1 < dims; ++i)
    if (p->size(i) != s->size(i)) return false;
  if (p->size(-1) != 4 * s->size(-1) || (stack && p->size(0) > INT32_MAX)) return false;
  d->packed = reinterpret_cast<const uint32_t*>(p->const_data_ptr<int32_t>());
  d->scales = s->const_data_ptr<uint8_t>();
  d->experts = stack ? (int32_t)p->size(0) : 0;
  d->out_features = p->size(-2);
  d->in_features = 8 * p->size(-1);
  return true;
}

// scaled_mm(ctx, device, a packed, a scales, w packed, w scales, f32)
// grouped_mm(the same, plan, by_token)
template <bool GROUPED>
FUNC(product) {
  NEEDS(GROUPED ? 9 : 7);
  return guarded([&]() -> PyObject* {
    const int64_t dev = a.num(1);
    mr_mxfp4_desc x, w;
    if (!operand(a.tensor(2, dev), a.tensor(3, dev), false, &x) ||
        !operand(a.tensor(4, dev), a.tensor(5, dev), GROUPED, &w) ||
        x.in_features != w.in_features)
      return none();
    const bool f32 = a.flag(6);
    const mr_sorted* plan = GROUPED ? a.at<mr_sorted>(7) : nullptr;
    const bool by_token = GROUPED && a.flag(8);
    int64_t rows = x.out_features;
    if (GROUPED) {
      rows = plan->tokens * plan->top_k;
      if (w.experts != plan->experts || x.out_features != (by_token ? plan->tokens : rows))
        return none();
    }
    at::Tensor out = empty({rows, w.out_features}, f32 ? at::kFloat : at::kBFloat16, dev);
    const mr_dtype dt = f32 ? MR_DTYPE_F32 : MR_DTYPE_BF16;
    mr_ctx* ctx = a.at<mr_ctx>(0);
    const mr_status st =
        GROUPED ? api.grouped_mm(ctx, &x, &w, plan, by_token, dt, out.mutable_data_ptr(),
                                 stream_of(dev))
                : api.scaled_mm(ctx, &x, &w, dt, out.mutable_data_ptr(), stream_of(dev));
    return st ? PyLong_FromLong(st) : wrap(std::move(out));
  });
}

#define ENTRY(name, f) \
  { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {
    ENTRY("bind", bind),
    ENTRY("sort", sort),
    ENTRY("views", views),
    ENTRY("dispatch", move_rows<false>),
    ENTRY("dispatch_backward", move_rows<true>),
    ENTRY("combine", combine),
    ENTRY("combine_backward", combine_backward),
    ENTRY("quantize", quantize),
    ENTRY("quantize_swiglu", quantize_swiglu),
    ENTRY("scaled_mm", product<false>),
    ENTRY("grouped_mm", product<true>),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_minirun_torch", nullptr, -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__minirun_torch() {
  PyObject* m = PyModule_Create(&module_def);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
