// Calls of the operators beside frozen weights in native code: the second part of `wave_b200._fast`.
//
// A decode step's adapters run for 6 microseconds on the GPU and a router for 3, and the Python code that leads to them took 22 to 27, a
// Python autograd function with its backward 110. Here the same checks are made on the tensors themselves; a call that passes them goes
// straight to the C ABI of include/wave_b200.h, through an autograd node of its own where a gradient is wanted. Whatever does not pass
// returns None, and the Python code does what it does without this module: copies of what is laid out otherwise, other devices, error
// messages. Nothing is kept from one call for the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "fast.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kF32 = 0, kBF16 = 1;  // WB200_F32, WB200_BF16

struct Abi {
  int (*adapters_forward)(int, int, int, int, int, const void*, long long, const void*, const void*, const void*, int, const float*, const void*, long long,
                          void*, long long, int, void*, size_t, void*);
  int (*adapters_backward)(int, int, int, int, int, const void*, long long, const void*, const void*, const void*, int, const float*, const void*, long long,
                           const void*, size_t, void*, long long, int, void*, void*, void*, size_t, void*);
  int (*input_grad)(int, int, int, const void*, long long, const void*, const void*, long long, void*, long long, void*);
  size_t (*router_workspace_bytes)(int, int);
  int (*router)(int, int, int, const void*, int, long long, const void*, const void*, int, int, float*, int*, int*, float*, float*, void*, size_t, void*);
  int (*router_grad)(int, int, int, const void*, int, long long, const void*, const int*, const float*, const float*, int, const int*, const float*, void*,
                     long long, void*);
  int (*combine)(const void*, long long, int, const int*, const float*, int, int, int, void*, long long, void*);
  int (*combine_grad)(const void*, long long, const void*, long long, int, const int*, int, int, int, float*, void*);
  const char* (*last_error)();
  size_t (*adapters_backward_workspace_bytes)(int, int, int);
} entry;

void check(int rc) { TORCH_CHECK(rc == 0, "wave_b200: ", entry.last_error(), " (status ", rc, ")"); }

Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int dtype_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? kF32 : t.scalar_type() == at::kBFloat16 ? kBF16 : -1; }
// Rows of unit column stride that do not overlap.
bool row_major(const Tensor& t) { return t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)); }
Tensor rows_of(const Tensor& t) { return row_major(t) ? t : t.contiguous(); }
long long pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
bool fits(int64_t n) { return n > 0 && n <= 0x7fffffff; }
// A tensor on the current device that needs nothing from the Python code; false leaves the call to it.
bool here(PyObject* o, Tensor* t) {
  if (!wbfast::plain_or_parameter(o)) return false;
  *t = THPVariable_Unpack(o);
  return t->device().index() == c10::cuda::current_device() && !t->_fw_grad(0).defined();  // (a forward-mode derivative is refused there)
}

// The interpreter lock is given back while a call allocates, launches and builds its node, and taken again where the scope ends: a launch waits where the
// queue is full, and what the stream waits for may be a host function that needs the lock.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The gradients of a node whose backward is a kernel: differentiating them again is an error that is raised if it is done.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<size_t> at;
  variable_list defined;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      at.push_back(i);
      defined.push_back(grads[i].detach().requires_grad_());
    }
  auto error = std::make_shared<torch::autograd::DelayedError>("wave_b200: this gradient cannot be differentiated again", int64_t(defined.size()));
  defined = (*error)(std::move(defined));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = defined[i];
  return grads;
}

// ---------------------------------------------------------------------------------------------
// adapters
// ---------------------------------------------------------------------------------------------
Tensor run_adapters(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& ids, const Tensor& scale, const Tensor& out) {
  const int64_t rank = a.size(1), padded = (rank + 15) / 16 * 16;
  const Tensor hidden = fresh({x.size(0) * padded * (y.scalar_type() == at::kFloat ? 6 : 4)}, at::kByte, x);  // wb200_adapters_hidden_bytes
  check(entry.adapters_forward(int(x.size(0)), int(x.size(1)), int(y.size(1)), int(rank), int(a.size(0)), x.data_ptr(), pitch(x), a.data_ptr(), b.data_ptr(),
                             ids.data_ptr(), ids.scalar_type() == at::kLong, static_cast<const float*>(ptr(scale)), y.data_ptr(), pitch(y), out.data_ptr(),
                             pitch(out), dtype_code(out), hidden.data_ptr(), size_t(hidden.numel()), stream_of(x)));
  return hidden;
}

struct AdaptersNode : torch::autograd::Function<AdaptersNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& ids,
                        const std::optional<Tensor>& given_scale) {  // (an undefined tensor is no input of a node)
    const Tensor scale = given_scale.value_or(Tensor());
    const Tensor out = fresh(y.sizes(), y.scalar_type(), y);
    const Tensor hidden = run_adapters(y, x, a, b, ids, scale, out);
    ctx->save_for_backward({x, a, b, ids, scale, hidden});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &a = saved[1], &b = saved[2], &ids = saved[3], &scale = saved[4], &hidden = saved[5];
    variable_list result(6);
    if (!grads[0].defined()) return result;
    const c10::cuda::CUDAGuard guard(x.device());
    if (ctx->needs_input_grad(0)) result[0] = grads[0];
    const Tensor g = rows_of(grads[0].detach());
    Tensor dx, da, db;
    if (ctx->needs_input_grad(1)) dx = fresh(x.sizes(), at::kBFloat16, x);
    if (ctx->needs_input_grad(2)) da = fresh(a.sizes(), at::kBFloat16, x);
    if (ctx->needs_input_grad(3)) db = fresh(b.sizes(), at::kBFloat16, x);
    if (dx.defined() || da.defined() || db.defined()) {
      const size_t bytes = entry.adapters_backward_workspace_bytes(int(x.size(0)), int(b.size(1)), int(a.size(1)));
      const Tensor ws = fresh({int64_t(bytes)}, at::kByte, x);
      check(entry.adapters_backward(int(x.size(0)), int(x.size(1)), int(b.size(1)), int(a.size(1)), int(a.size(0)), x.data_ptr(), pitch(x), a.data_ptr(),
                                  b.data_ptr(), ids.data_ptr(), ids.scalar_type() == at::kLong, static_cast<const float*>(ptr(scale)), g.data_ptr(), pitch(g),
                                  hidden.data_ptr(), size_t(hidden.numel()), ptr(dx), x.size(1), 0, ptr(da), ptr(db), ws.data_ptr(),
                                  bytes, stream_of(x)));
      variable_list mine = once({dx, da, db});
      for (int i = 0; i < 3; ++i) result[1 + i] = mine[i];
    }
    return result;
  }
};

// ---------------------------------------------------------------------------------------------
// router
// ---------------------------------------------------------------------------------------------
struct Routed {
  Tensor weight, ids, counts, loss, unit;
};
Routed run_router(const Tensor& logits, const Tensor& mask, int64_t top_k, bool renormalize) {
  const int64_t rows = logits.size(0), E = logits.size(1);
  const size_t bytes = entry.router_workspace_bytes(int(rows), int(E));
  Routed r;
  r.weight = fresh({rows, top_k}, at::kFloat, logits);
  r.ids = fresh({rows, top_k}, at::kInt, logits);
  r.counts = fresh({E}, at::kInt, logits);
  r.loss = fresh({}, at::kFloat, logits);
  r.unit = fresh({1 + int64_t(bytes) / 4}, at::kFloat, logits);  // and the partial sums behind it
  check(entry.router(int(rows), int(E), int(top_k), logits.data_ptr(), dtype_code(logits), pitch(logits), ptr(mask), nullptr, 0, renormalize,
                   static_cast<float*>(r.weight.data_ptr()), static_cast<int*>(r.ids.data_ptr()), static_cast<int*>(r.counts.data_ptr()),
                   static_cast<float*>(r.unit.data_ptr()), static_cast<float*>(r.loss.data_ptr()), static_cast<float*>(r.unit.data_ptr()) + 1, bytes,
                   stream_of(logits)));
  return r;
}

struct RouterNode : torch::autograd::Function<RouterNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const std::optional<Tensor>& given_mask, int64_t top_k, bool renormalize) {
    const Tensor mask = given_mask.value_or(Tensor());
    const Routed r = run_router(logits, mask, top_k, renormalize);
    ctx->save_for_backward({logits, mask, r.ids, r.counts, r.unit});
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({r.ids, r.counts});
    ctx->set_materialize_grads(false);
    return {r.weight, r.ids, r.counts, r.loss};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &mask = saved[1], &ids = saved[2], &counts = saved[3], &unit = saved[4];
    variable_list result(4);
    if (!grads[0].defined() && !grads[3].defined()) return result;
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor gw = grads[0].defined() ? grads[0].detach().contiguous() : Tensor(), gl = grads[3].defined() ? grads[3].detach() : Tensor();
    const Tensor dz = fresh(logits.sizes(), logits.scalar_type(), logits);
    check(entry.router_grad(int(logits.size(0)), int(logits.size(1)), int(ctx->saved_data["top_k"].toInt()), logits.data_ptr(), dtype_code(logits),
                          pitch(logits), ptr(mask), static_cast<const int*>(ids.data_ptr()), static_cast<const float*>(ptr(gw)),
                          static_cast<const float*>(ptr(gl)), ctx->saved_data["renormalize"].toBool(), static_cast<const int*>(counts.data_ptr()),
                          static_cast<const float*>(unit.data_ptr()), dz.data_ptr(), logits.size(1), stream_of(logits)));
    result[0] = once({dz})[0];
    return result;
  }
};

// ---------------------------------------------------------------------------------------------
// the weighted sum of experts' rows
// ---------------------------------------------------------------------------------------------
Tensor run_combine(const Tensor& y, const Tensor& row_of, const Tensor& weight) {
  const Tensor out = fresh({row_of.size(0), y.size(1)}, y.scalar_type(), y);
  check(entry.combine(y.data_ptr(), pitch(y), dtype_code(y), static_cast<const int*>(row_of.data_ptr()), static_cast<const float*>(weight.data_ptr()),
                    int(row_of.size(0)), int(row_of.size(1)), int(y.size(1)), out.data_ptr(), y.size(1), stream_of(y)));
  return out;
}

struct CombineNode : torch::autograd::Function<CombineNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& row_of, const Tensor& weight) {
    ctx->save_for_backward({y, row_of});
    return run_combine(y, row_of, weight);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &row_of = saved[1];
    variable_list result(3);
    if (!grads[0].defined()) return result;
    const c10::cuda::CUDAGuard guard(y.device());
    const Tensor g = rows_of(grads[0].detach());
    const Tensor gw = fresh(row_of.sizes(), at::kFloat, y);
    check(entry.combine_grad(g.data_ptr(), pitch(g), y.data_ptr(), pitch(y), dtype_code(y), static_cast<const int*>(row_of.data_ptr()), int(row_of.size(0)),
                           int(row_of.size(1)), int(y.size(1)), static_cast<float*>(gw.data_ptr()), stream_of(y)));
    result[2] = once({gw})[0];
    return result;
  }
};

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

bool wanted(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}

}  // namespace

namespace wbfast {

// adapters(y, x, a, b, ids, scale or None, out or None) -> the output, or None: left to the Python code
PyObject* adapters(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "adapters takes 7 arguments");
    return nullptr;
  }
  try {
    Tensor y, x, a, b, ids, scale, out;
    if (!here(args[0], &y) || !here(args[1], &x) || !here(args[2], &a) || !here(args[3], &b) || !here(args[4], &ids) ||
        (args[5] != Py_None && !here(args[5], &scale)) || (args[6] != Py_None && !here(args[6], &out)))
      Py_RETURN_NONE;
    if (x.scalar_type() != at::kBFloat16 || a.scalar_type() != at::kBFloat16 || b.scalar_type() != at::kBFloat16 || dtype_code(y) < 0 || !row_major(x) ||
        !row_major(y) || a.dim() != 3 || b.dim() != 3 || !a.is_contiguous() || !b.is_contiguous() || ids.dim() != 1 || !ids.is_contiguous() ||
        (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong))
      Py_RETURN_NONE;
    const int64_t rows = x.size(0), K = x.size(1), N = y.size(1), pool = a.size(0), rank = a.size(1);
    if (!fits(rows) || !fits(K) || !fits(N) || !fits(pool) || rank < 1 || rank > 256 || K % 8 || y.size(0) != rows || a.size(2) != K || b.size(0) != pool ||
        b.size(1) != N || b.size(2) != rank || ids.size(0) != rows)
      Py_RETURN_NONE;
    if (scale.defined() && (scale.scalar_type() != at::kFloat || scale.dim() != 1 || scale.size(0) != pool || !scale.is_contiguous() || scale.requires_grad()))
      Py_RETURN_NONE;
    if (out.defined() && (out.scalar_type() != y.scalar_type() || out.sizes() != y.sizes() || !row_major(out))) Py_RETURN_NONE;
    if (wanted({&y, &x, &a, &b})) {
      if (out.defined() || y.scalar_type() != at::kBFloat16 || pool > 65535) Py_RETURN_NONE;
      Tensor result;
      {
        const Unlocked scope;
        result = AdaptersNode::apply(y, x, a, b, ids, given(scale));
      }
      return THPVariable_Wrap(result);
    }
    if (out.defined() && out.requires_grad()) Py_RETURN_NONE;
    const bool given_out = out.defined();
    {
      const Unlocked scope;
      if (!given_out) out = fresh(y.sizes(), y.scalar_type(), y);
      run_adapters(y, x, a, b, ids, scale, out);
    }
    if (given_out && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();  // autograd may hold what it was
    return THPVariable_Wrap(out);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    return fail(e);
  }
}

// router(logits, top_k, mask or None, renormalize) -> (weight, ids, counts, loss), or None
PyObject* router(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "router takes 4 arguments");
    return nullptr;
  }
  try {
    Tensor logits, mask;
    if (!here(args[0], &logits) || (args[2] != Py_None && !here(args[2], &mask)) || !PyLong_Check(args[1])) Py_RETURN_NONE;
    const long long top_k = PyLong_AsLongLong(args[1]);
    const int renormalize = PyObject_IsTrue(args[3]);
    if (PyErr_Occurred()) return nullptr;
    if (dtype_code(logits) < 0 || !row_major(logits) || !fits(logits.size(0)) || logits.size(1) < 1 || logits.size(1) > 256 || top_k < 1 ||
        top_k > std::min<int64_t>(32, logits.size(1)))
      Py_RETURN_NONE;
    if (mask.defined() && (mask.scalar_type() != at::kBool || mask.dim() != 1 || mask.size(0) != logits.size(0) || !mask.is_contiguous())) Py_RETURN_NONE;
    variable_list r;
    {
      const Unlocked scope;
      if (wanted({&logits})) {
        r = RouterNode::apply(logits, given(mask), int64_t(top_k), renormalize != 0);
      } else {
        const Routed v = run_router(logits, mask, top_k, renormalize != 0);
        r = {v.weight, v.ids, v.counts, v.loss};
      }
    }
    PyObject* result = PyTuple_New(4);
    if (!result) return nullptr;
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(r[i]));
    return result;
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    return fail(e);
  }
}

// combine_rows(y, row_of, weight) -> the output, or None
PyObject* combine_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "combine_rows takes 3 arguments");
    return nullptr;
  }
  try {
    Tensor y, row_of, weight;
    if (!here(args[0], &y) || !here(args[1], &row_of) || !here(args[2], &weight)) Py_RETURN_NONE;
    if (dtype_code(y) < 0 || !row_major(y) || row_of.scalar_type() != at::kInt || weight.scalar_type() != at::kFloat || row_of.dim() != 2 ||
        weight.sizes() != row_of.sizes() || !row_of.is_contiguous() || !weight.is_contiguous() || !fits(row_of.size(0)) || !fits(row_of.size(1)) ||
        !fits(y.size(1)) || y.size(0) == 0 || (at::GradMode::is_enabled() && y.requires_grad()))
      Py_RETURN_NONE;
    Tensor result;
    {
      const Unlocked scope;
      result = wanted({&weight}) ? CombineNode::apply(y, row_of, weight) : run_combine(y, row_of, weight);
    }
    return THPVariable_Wrap(result);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    return fail(e);
  }
}

// input_grad(g, codes, scales) -> the gradient, or None
PyObject* input_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "input_grad takes 3 arguments");
    return nullptr;
  }
  try {
    Tensor g, codes, scales;
    if (!here(args[0], &g) || !here(args[1], &codes) || !here(args[2], &scales)) Py_RETURN_NONE;
    if (g.scalar_type() != at::kBFloat16 || codes.element_size() != 1 || scales.element_size() != 1 || !row_major(g) || codes.dim() != 2 ||
        !codes.is_contiguous() || scales.dim() != 2 || !row_major(scales) || at::isFloatingType(codes.scalar_type()) || at::isFloatingType(scales.scalar_type()) ||
        codes.scalar_type() == at::kBool || scales.scalar_type() == at::kBool)
      Py_RETURN_NONE;
    const int64_t M = g.size(0), N = g.size(1), K = codes.size(1) * 2;
    auto aligned = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; };
    if (!fits(M) || !fits(N) || !fits(K) || K % 32 || codes.size(0) != N || scales.size(0) != N || scales.size(1) != K / 32 || !aligned(g) || !aligned(codes) ||
        (M > 1 ? g.stride(0) : N) % 8 || N % 8)
      Py_RETURN_NONE;
    Tensor dx;
    {
      const Unlocked scope;
      dx = fresh({M, K}, at::kBFloat16, g);
      check(entry.input_grad(int(M), int(N), int(K), g.data_ptr(), pitch(g), codes.data_ptr(), scales.data_ptr(), pitch(scales), dx.data_ptr(), K, stream_of(g)));
    }
    return THPVariable_Wrap(dx);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    return fail(e);
  }
}

// bind_adapt(adapters_forward, adapters_backward, input_grad, router_workspace_bytes, router, router_grad, combine, combine_grad, last_error,
//            adapters_backward_workspace_bytes)
PyObject* bind_adapt(PyObject*, PyObject* args) {
  unsigned long long p[10];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7], &p[8], &p[9])) return nullptr;
  entry.adapters_forward = reinterpret_cast<decltype(entry.adapters_forward)>(p[0]);
  entry.adapters_backward = reinterpret_cast<decltype(entry.adapters_backward)>(p[1]);
  entry.input_grad = reinterpret_cast<decltype(entry.input_grad)>(p[2]);
  entry.router_workspace_bytes = reinterpret_cast<decltype(entry.router_workspace_bytes)>(p[3]);
  entry.router = reinterpret_cast<decltype(entry.router)>(p[4]);
  entry.router_grad = reinterpret_cast<decltype(entry.router_grad)>(p[5]);
  entry.combine = reinterpret_cast<decltype(entry.combine)>(p[6]);
  entry.combine_grad = reinterpret_cast<decltype(entry.combine_grad)>(p[7]);
  entry.last_error = reinterpret_cast<decltype(entry.last_error)>(p[8]);
  entry.adapters_backward_workspace_bytes = reinterpret_cast<decltype(entry.adapters_backward_workspace_bytes)>(p[9]);
  Py_RETURN_NONE;
}

}  // namespace wbfast
