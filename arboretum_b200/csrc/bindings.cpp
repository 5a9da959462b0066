// The Python side of the operators on torch tensors: arguments are checked and turned into a call of
// the C entry points here rather than in Python, whose share of a small call was four times the
// launch's (16.6 us for a lookup, 4.8 here; 333 us for the addresses of 500 gradients, 15 here with the
// whole step, 11 where the gradients are given once).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <memory>
#include <string>
#include <vector>

#include "../../include/arboretum_b200.h"

namespace {

PyObject *g_error = nullptr;  // arboretum_b200.ArboretumError

// an error message of the C library
struct LibraryError {
  std::string message;
};
void call(const char *message) {
  if (message) throw LibraryError{message};
}

#define ARB_BEGIN \
  HANDLE_TH_ERRORS \
  try {
#define ARB_END                                                                          \
  }                                                                                      \
  catch (const LibraryError &e) {                                                        \
    PyObject *inner = PyObject_CallFunction(PyExc_ValueError, "y", e.message.c_str());   \
    if (inner) {                                                                         \
      PyErr_SetObject(g_error, inner);                                                   \
      Py_DECREF(inner);                                                                  \
    }                                                                                    \
    return nullptr;                                                                      \
  }                                                                                      \
  END_HANDLE_TH_ERRORS

// elements from a tensor's first to its last, both included
int64_t reach(const at::Tensor &t) {
  if (t.numel() == 0) return 0;
  int64_t n = 1;
  for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  return n;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch tensor");
  const at::Tensor &t = THPVariable_Unpack(o);
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.has_storage(), name, " must be a tensor with memory of its own");
  // a storage can be freed or shrunk under its tensors (untyped_storage().resize_)
  TORCH_CHECK_VALUE((t.storage_offset() + reach(t)) * int64_t(t.element_size()) <= int64_t(t.storage().nbytes()) || t.numel() == 0, name,
                    " lies outside its memory");
  // of such a view the memory holds the values with their signs turned
  TORCH_CHECK_VALUE(!t.is_neg(), name, " is a view to be negated: pass its resolve_neg()");
  return t;
}

int float_type(const at::Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
  }
}

// Nothing here is recorded for derivatives: a tensor that carries one is refused, not stripped of it.
// Tangents live in the dual level that is entered; without one no tensor is asked (20 ns each, more than
// the rest of a gradient's checks).
bool tangents() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const at::Tensor &t, const char *name, bool any = tangents()) {
  TORCH_CHECK_VALUE(!any || !t._fw_grad(0).defined(), name, " carries a tangent, which is not followed here: pass its primal");
}
void no_grad(const at::Tensor &t, const char *name) {
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), name,
                    " requires grad, which is not recorded here: pass it detached and use embedding_grad for the backward pass");
  no_tangent(t, name);
}

// autograd has to see that this was written in place; an inference tensor has no version
void written(const at::Tensor &t) {
  c10::TensorImpl *impl = t.unsafeGetTensorImpl();
  if (impl->version_counter().enabled()) impl->bump_version();
}

void on_device(const at::Tensor &t, const char *name, c10::Device device) {
  TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device().str(), ", the others are on ", device.str());
}

int cuda_index(const at::Tensor &t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "the tensors must be CUDA tensors");
  return t.get_device();
}

struct Extent {
  uintptr_t first, last;
};
Extent extent(const at::Tensor &t) {
  if (t.numel() == 0) return {0, 0};
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {at, at + uintptr_t(reach(t)) * t.element_size()};
}
void apart(const at::Tensor &out, const char *name, const at::Tensor &t) {
  const Extent a = extent(out), b = extent(t);
  TORCH_CHECK_VALUE(!(a.first < b.last && b.first < a.last), "out shares memory with ", name);
}

struct Bags {
  at::Tensor tokens;
  int bytes;
  int64_t bags, per_bag, bag_stride, token_stride;
};
Bags bags_of(PyObject *o, bool pooled) {
  const at::Tensor &t = tensor(o, "tokens");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "tokens must be int32 or int64, not ", t.scalar_type());
  const int bytes = t.scalar_type() == at::kInt ? 4 : 8;
  if (pooled) {
    TORCH_CHECK_VALUE(t.dim() == 2, "pooled tokens must have two dimensions: bags x tokens");
    return {t, bytes, t.size(0), t.size(1), t.stride(0), t.stride(1)};
  }
  const at::Tensor flat = t.dim() == 1 ? t : t.reshape({-1});
  return {flat, bytes, flat.size(0), 1, flat.stride(0), 0};
}

c10::optional<at::ScalarType> dtype_of(PyObject *o) {
  if (o == Py_None) return c10::nullopt;
  TORCH_CHECK_TYPE(THPDtype_Check(o), "out_dtype must be a torch dtype");
  return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// The output as a matrix of rows: a new tensor, or the caller's.
struct Out {
  at::Tensor whole, rows;
  int type;
  bool given;
};
Out output(PyObject *o, at::IntArrayRef shape, const at::Tensor &like, PyObject *out_dtype) {
  const c10::optional<at::ScalarType> want = dtype_of(out_dtype);
  Out r;
  r.given = o != Py_None;
  if (!r.given) {
    r.whole = at::empty(shape, like.options().dtype(want.value_or(like.scalar_type())));
  } else {
    r.whole = tensor(o, "out");
    TORCH_CHECK_VALUE(r.whole.sizes() == shape, "out must have shape ", shape, ", not ", r.whole.sizes());
    TORCH_CHECK_TYPE(!want || r.whole.scalar_type() == *want, "out is ", r.whole.scalar_type(), ", out_dtype is ", want.value_or(at::kFloat));
    no_grad(r.whole, "out");
  }
  r.rows = r.whole;
  if (r.rows.dim() != 2) {
    TORCH_CHECK_VALUE(r.rows.is_contiguous(), "an out of more than two dimensions must be contiguous");
    const int64_t dim = shape.back();
    int64_t n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
    r.rows = r.rows.view({n, dim});
  }
  TORCH_CHECK_VALUE(r.rows.numel() == 0 || r.rows.size(1) <= 1 || r.rows.stride(1) == 1, "the last dimension of out must be contiguous");
  TORCH_CHECK_TYPE(r.rows.scalar_type() == like.scalar_type() || r.rows.scalar_type() == at::kFloat, "out must be ", like.scalar_type(),
                   " or float32, not ", r.rows.scalar_type());
  r.type = float_type(r.rows, "out");
  return r;
}

void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// A trace would not see the call: the result would stand in it as a constant, or as memory nobody filled.
void not_traced() {
  const bool traced = at::tracer::impl::is_dispatch_enabled() ||
                      (c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                       c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK_VALUE(!traced, "the operators on learned tables cannot be traced");
}

void need(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n); }
double number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
int64_t whole_number(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// embedding(tokens, table, scale, pooled, out, out_dtype)
PyObject *embedding(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 6);
  not_traced();
  const at::Tensor &table = tensor(args[1], "table");
  const int type = float_type(table, "table");
  TORCH_CHECK_VALUE(table.dim() == 2, "table must have two dimensions: rows x columns");
  TORCH_CHECK_VALUE(table.numel() == 0 || table.size(1) <= 1 || table.stride(1) == 1, "the columns of table must be contiguous");
  no_grad(table, "table");
  const bool pooled = truth(args[3]);
  const Bags b = bags_of(args[0], pooled);
  const int device = cuda_index(table);
  on_device(b.tokens, "tokens", table.device());
  const int64_t rows = table.size(0), dim = table.size(1);
  at::DimVector shape;
  if (pooled) {
    shape.push_back(b.bags);
  } else {
    const at::IntArrayRef sizes = THPVariable_Unpack(args[0]).sizes();
    shape.append(sizes.begin(), sizes.end());
  }
  shape.push_back(dim);
  const Out out = output(args[4], shape, table, args[5]);
  if (out.given) {
    on_device(out.whole, "out", table.device());
    apart(out.whole, "table", table);
    apart(out.whole, "tokens", b.tokens);
  }
  call(AEmbedding(table.const_data_ptr(), type, rows, dim, table.stride(0), b.tokens.const_data_ptr(), b.bytes, b.bags, b.per_bag,
                  b.bag_stride, b.token_stride, number(args[2]), out.rows.data_ptr(), out.type, out.rows.stride(0), device,
                  stream_of(device)));
  if (out.given) written(out.whole);
  return THPVariable_Wrap(out.whole);
  ARB_END
}

at::Tensor memory(int64_t bytes, c10::Device device) {
  return at::empty({std::max<int64_t>(256, bytes)}, at::TensorOptions().dtype(at::kByte).device(device));
}

// token_order(tokens, rows, pooled) -> (memory, bags, tokens a bag, stream)
PyObject *token_order(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 3);
  not_traced();
  const Bags b = bags_of(args[0], truth(args[2]));
  const int64_t rows = whole_number(args[1]);
  int64_t order_bytes = 0, scratch_bytes = 0;
  call(ATokenOrderBytes(b.bags, b.per_bag, rows, &order_bytes, &scratch_bytes));
  const int device = cuda_index(b.tokens);
  const at::Tensor data = memory(order_bytes, b.tokens.device()), scratch = memory(scratch_bytes, b.tokens.device());
  void *stream = stream_of(device);
  call(ATokenOrder(b.tokens.const_data_ptr(), b.bytes, b.bags, b.per_bag, b.bag_stride, b.token_stride, rows, data.data_ptr(),
                   scratch.data_ptr(), device, stream));
  return Py_BuildValue("(NLLK)", THPVariable_Wrap(data), (long long)b.bags, (long long)b.per_bag,
                       (unsigned long long)reinterpret_cast<uintptr_t>(stream));
  ARB_END
}

// embedding_grad(grad, tokens, rows, scale, pooled, out, out_dtype, accumulate, order): order is None
// or (memory, bags, tokens a bag, stream), and tokens then the shape of its tokens
PyObject *embedding_grad(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 9);
  not_traced();
  at::Tensor grad = tensor(args[0], "grad");
  const int type = float_type(grad, "grad");
  no_grad(grad, "grad");
  const bool pooled = truth(args[4]), accumulate = truth(args[7]);
  const int64_t rows = whole_number(args[2]);
  const bool sorted = args[8] != Py_None;
  Bags b{};
  at::Tensor order;
  unsigned long long order_stream = 0;
  at::DimVector shape;  // of grad without its columns
  if (sorted) {
    PyObject *data = nullptr;
    long long bags = 0, per_bag = 0;
    if (!PyArg_ParseTuple(args[8], "OLLK", &data, &bags, &per_bag, &order_stream)) throw python_error();
    order = tensor(data, "order");
    b.bags = bags, b.per_bag = per_bag;
    for (Py_ssize_t i = 0; i < PyTuple_Size(args[1]); ++i) shape.push_back(whole_number(PyTuple_GetItem(args[1], i)));
  } else {
    b = bags_of(args[1], pooled);
    const at::IntArrayRef sizes = THPVariable_Unpack(args[1]).sizes();
    shape.append(sizes.begin(), sizes.end());
  }
  if (pooled) shape = at::DimVector{b.bags};
  TORCH_CHECK_VALUE(grad.dim() >= 1 && grad.sizes().slice(0, grad.dim() - 1) == at::IntArrayRef(shape), "grad must have shape ",
                    at::IntArrayRef(shape), " x columns, not ", grad.sizes());
  const int64_t dim = grad.size(-1);
  TORCH_CHECK_VALUE(!accumulate || args[5] != Py_None, "accumulate needs the gradient to add to: out");
  int64_t order_bytes = 0, sort_bytes = 0, scratch_bytes = 0;
  call(ATokenOrderBytes(b.bags, b.per_bag, rows, &order_bytes, &sort_bytes));
  const int device = cuda_index(grad);
  on_device(sorted ? order : b.tokens, "tokens", grad.device());
  call(AEmbeddingGradBytes(b.bags, b.per_bag, rows, dim, device, &scratch_bytes));
  if (grad.dim() != 2) grad = grad.reshape({b.bags, dim});
  if (grad.numel() != 0 && dim > 1 && grad.stride(1) != 1) grad = grad.contiguous();
  const int64_t out_shape[2] = {rows, dim};
  const Out out = output(args[5], out_shape, grad, args[6]);
  if (out.given) {
    on_device(out.whole, "out", grad.device());
    apart(out.whole, "grad", grad);
    apart(out.whole, sorted ? "the order" : "tokens", sorted ? order : b.tokens);
  }
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  at::Tensor scratch;
  char *order_at = nullptr, *scratch_at = nullptr;
  if (sorted) {
    // its memory must not be handed out again before this stream is done
    if (reinterpret_cast<uintptr_t>(stream.stream()) != order_stream) order.record_stream(stream);
    scratch = memory(scratch_bytes, grad.device());
    order_at = static_cast<char *>(order.data_ptr());
    scratch_at = static_cast<char *>(scratch.data_ptr());
  } else {
    scratch = memory(order_bytes + std::max(sort_bytes, scratch_bytes), grad.device());
    order_at = static_cast<char *>(scratch.data_ptr());
    scratch_at = order_at + order_bytes;
    call(ATokenOrder(b.tokens.const_data_ptr(), b.bytes, b.bags, b.per_bag, b.bag_stride, b.token_stride, rows, order_at, scratch_at,
                     device, stream.stream()));
  }
  call(AEmbeddingGrad(grad.const_data_ptr(), type, b.bags, dim, grad.stride(0), order_at, b.per_bag, rows, number(args[3]),
                      out.rows.data_ptr(), out.type, out.rows.stride(0), accumulate, scratch_at, device, stream.stream()));
  if (out.given) written(out.whole);
  return THPVariable_Wrap(out.whole);
  ARB_END
}

// ---- AdamW -----------------------------------------------------------------------------------
struct Optimizer {
  std::vector<at::Tensor> params, buffers;
  std::vector<const void *> at;     // where the parameters lie
  std::vector<const void *> grads;  // where the gradients given at construction lie (nullptr: None or empty)
  std::vector<at::Tensor> bound;    // they, one for every parameter (undefined: None)
  std::vector<c10::Storage> memory; // of both: stays as long as the device's table names it
  bool has_bound = false, bound_fp32 = false;
  VoidPointer handle = nullptr;
  int device = 0;
  void *stream = nullptr;
  ~Optimizer() { AFreeAdamW(handle); }
};
const char *kOptimizer = "arboretum_b200.AdamW";
Optimizer &optimizer(PyObject *o) {
  void *p = PyCapsule_GetPointer(o, kOptimizer);
  if (!p) throw python_error();
  return *static_cast<Optimizer *>(p);
}

void stays(const Optimizer &o, size_t i) {
  TORCH_CHECK_VALUE(o.params[i].unsafeGetTensorImpl()->data() == o.at[i], "a parameter's memory has moved since the optimizer was made");
}

// addresses of one gradient, or None, for every parameter; whether all are float32 (else each has its
// parameter's type)
bool addresses(const Optimizer &o, PyObject *list, std::vector<const void *> &at, std::vector<at::Tensor> *keep) {
  THPObjectPtr fast(PySequence_Fast(list, "grads must be a sequence"));
  if (!fast) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.get());
  TORCH_CHECK_VALUE(size_t(n) == o.params.size(), n, " gradients for ", o.params.size(), " parameters");
  at.resize(size_t(n));
  bool same = true, single = true;
  const bool dual = tangents();
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *item = PySequence_Fast_GET_ITEM(fast.get(), i);
    const at::Tensor &p = o.params[size_t(i)];
    stays(o, size_t(i));
    at[size_t(i)] = nullptr;
    if (keep) keep->emplace_back();
    if (item == Py_None) continue;
    TORCH_CHECK_VALUE(THPVariable_CheckExact(item) || THPVariable_Check(item), "a gradient must be a contiguous tensor of its parameter's shape");
    const at::Tensor &g = THPVariable_Unpack(item);
    const c10::TensorImpl *gi = g.unsafeGetTensorImpl(), *pi = p.unsafeGetTensorImpl();
    TORCH_CHECK_VALUE(gi->sizes() == pi->sizes() && gi->is_contiguous(), "a gradient must be a contiguous tensor of its parameter's shape");
    TORCH_CHECK_VALUE(gi->device() == pi->device(), "a gradient is on ", g.device().str(), ", its parameter on ", p.device().str());
    TORCH_CHECK_VALUE(gi->numel() == 0 || (gi->storage_offset() + gi->numel()) * int64_t(gi->itemsize()) <= int64_t(gi->unsafe_storage().nbytes()),
                      "a gradient lies outside its memory");
    TORCH_CHECK_VALUE(!g.is_neg(), "a gradient is a view to be negated: pass its resolve_neg()");
    no_tangent(g, "a gradient", dual);
    single = single && gi->dtype() == caffe2::TypeMeta::Make<float>();
    same = same && gi->dtype() == pi->dtype();
    at[size_t(i)] = gi->data();
    if (keep) keep->back() = g;
  }
  TORCH_CHECK_TYPE(same || single, "gradients must have their parameters' types, or all be float32");
  return !same;
}

// adamw(params, config bytes, buffers, grads): buffers = (moment1, moment2, scale1, scale2, master,
// workspace), None where there is none
PyObject *adamw(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 4);
  std::unique_ptr<Optimizer> o(new Optimizer());
  std::vector<AAdamWParam> table;
  THPObjectPtr params(PySequence_Fast(args[0], "params must be a sequence"));
  if (!params) throw python_error();
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(params.get()); ++i) {
    const at::Tensor &p = tensor(PySequence_Fast_GET_ITEM(params.get(), i), "a parameter");
    no_tangent(p, "a parameter");
    o->params.push_back(p);
    o->at.push_back(p.const_data_ptr());
    o->memory.push_back(p.storage());
    table.push_back(AAdamWParam{p.data_ptr(), p.numel(), float_type(p, "a parameter")});
  }
  AAdamWConfig config;
  TORCH_CHECK_TYPE(PyBytes_Check(args[1]) && PyBytes_Size(args[1]) == Py_ssize_t(sizeof config), "bad configuration");
  std::memcpy(&config, PyBytes_AsString(args[1]), sizeof config);
  std::vector<void *> at;
  for (Py_ssize_t i = 0; i < 6; ++i) {
    PyObject *b = PyTuple_GetItem(args[2], i);
    if (!b) throw python_error();
    at.push_back(b == Py_None ? nullptr : tensor(b, "a buffer").data_ptr());
    if (b != Py_None) o->buffers.push_back(THPVariable_Unpack(b));
  }
  config.moment1 = at[0], config.moment2 = at[1];
  config.scale1 = static_cast<float *>(at[2]), config.scale2 = static_cast<float *>(at[3]);
  config.master = static_cast<float *>(at[4]);
  o->device = cuda_index(o->params.at(0));
  o->stream = stream_of(o->device);
  if (args[3] != Py_None) {
    o->bound_fp32 = addresses(*o, args[3], o->grads, &o->bound);
    o->has_bound = true;
    for (const at::Tensor &g : o->bound)
      if (g.defined()) o->memory.push_back(g.storage());
  }
  call(AAdamWCreate(table.data(), int(table.size()), &config, at[5], o->device, &o->handle));
  PyObject *capsule = PyCapsule_New(o.get(), kOptimizer, [](PyObject *c) {
    delete static_cast<Optimizer *>(PyCapsule_GetPointer(c, kOptimizer));
  });
  if (capsule) o.release();
  return capsule;
  ARB_END
}

const float *scalar(PyObject *t, const char *name, const Optimizer &o) {
  const at::Tensor &x = tensor(t, name);
  TORCH_CHECK_TYPE(x.scalar_type() == at::kFloat && x.numel() == 1, name, " must be a float32 tensor of one element");
  on_device(x, name, o.params[0].device());
  no_tangent(x, name);
  return x.const_data_ptr<float>();
}

// adamw_step(optimizer, grads, lr, grad_scale)
PyObject *adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 4);
  not_traced();
  Optimizer &o = optimizer(args[0]);
  // one look at every parameter and its gradient: 500 of them are further apart than the first-level cache is large
  std::vector<const void *> given;
  const std::vector<const void *> *grads = &o.grads;
  bool fp32 = o.bound_fp32;
  if (args[1] != Py_None) {
    fp32 = addresses(o, args[1], given, nullptr);
    grads = &given;
  } else {
    TORCH_CHECK_VALUE(o.has_bound, "no gradients: pass grads to step() or to the constructor");
    for (size_t i = 0; i < o.grads.size(); ++i) {
      stays(o, i);
      TORCH_CHECK_VALUE(!o.bound[i].defined() || o.bound[i].unsafeGetTensorImpl()->data() == o.grads[i],
                        "a gradient's memory has moved since the optimizer was made");
    }
  }
  double lr = 0.0;
  const float *lr_device = nullptr;
  if (THPVariable_Check(args[2])) lr_device = scalar(args[2], "lr", o);
  else lr = number(args[2]);
  const float *grad_scale = args[3] == Py_None ? nullptr : scalar(args[3], "grad_scale", o);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(o.device);
  if (stream.stream() != o.stream)  // the optimizer's memory must not be handed out again before that stream is done with it
    for (const at::Tensor &b : o.buffers) b.record_stream(stream);
  call(AAdamWStep(o.handle, grads->data(), int(grads->size()), fp32, lr, lr_device, grad_scale, stream.stream()));
  // also a parameter that was passed detached: it shares its counter (6 ns each, a locked addition)
  for (size_t i = 0; i < o.params.size(); ++i)
    if ((*grads)[i] != nullptr) written(o.params[i]);
  Py_RETURN_NONE;
  ARB_END
}

// adamw_count(optimizer, step or None) -> the step count
PyObject *adamw_count(PyObject *, PyObject *const *args, Py_ssize_t n) {
  ARB_BEGIN
  need(n, 2);
  Optimizer &o = optimizer(args[0]);
  int64_t step = 0;
  if (args[1] != Py_None) {
    step = whole_number(args[1]);
    call(AAdamWSetStep(o.handle, step, stream_of(o.device)));
  } else {
    call(AAdamWGetStep(o.handle, &step, stream_of(o.device)));
  }
  return PyLong_FromLongLong(step);
  ARB_END
}

PyObject *set_error(PyObject *, PyObject *cls) {
  Py_XDECREF(g_error);
  Py_INCREF(cls);
  g_error = cls;
  Py_RETURN_NONE;
}

#define ARB_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef kMethods[] = {
    {"embedding", ARB_FAST(embedding), nullptr},           {"embedding_grad", ARB_FAST(embedding_grad), nullptr},
    {"token_order", ARB_FAST(token_order), nullptr},       {"adamw", ARB_FAST(adamw), nullptr},
    {"adamw_step", ARB_FAST(adamw_step), nullptr},         {"adamw_count", ARB_FAST(adamw_count), nullptr},
    {"set_error", set_error, METH_O, nullptr},             {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&kModule); }
