// The usual calls of model_b200/train_ops.py without the interpreter's share:
// argument checks, outputs, workspace and the C ABI call in one extension
// function each.  A small layer norm spends 11 us in Python and ctypes around
// a 3 us launch; here it is 5.
//
// A function returns None for every call it does not take (other layouts,
// types, devices or errors of any kind); train_ops.py then goes its general
// way, which also raises what there is to raise.  Nothing has been written by
// then but tensors nobody holds.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "memlayer.h"

namespace {

// A call that the general way takes.
struct Decline {};

void need(bool ok) {
  if (!ok) throw Decline{};
}

// A contiguous CUDA tensor; on the device of `like`, or on the current one.
const at::Tensor& tensor(PyObject* o, const at::Tensor* like) {
  need(THPVariable_CheckExact(o));
  const at::Tensor& t = THPVariable_Unpack(o);
  need(t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg() && !t.is_conj());
  need(like ? t.device() == like->device() : t.get_device() == c10::cuda::current_device());
  return t;
}

const at::Tensor& same(PyObject* o, const at::Tensor& like) {
  const at::Tensor& t = tensor(o, &like);
  need(t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes());
  return t;
}

const float* vector(PyObject* o, int64_t n, const at::Tensor& like) {
  const at::Tensor& t = tensor(o, &like);
  need(t.scalar_type() == at::kFloat && t.numel() == n);
  return static_cast<const float*>(t.const_data_ptr());
}

int32_t dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MEMLAYER_F32;
    case at::kHalf: return MEMLAYER_F16;
    case at::kBFloat16: return MEMLAYER_BF16;
    default: throw Decline{};
  }
}

double number(PyObject* o) {
  need(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
  const double v = PyFloat_AsDouble(o);
  need(!PyErr_Occurred());
  return v;
}

int32_t int32(PyObject* o) {
  need(PyLong_CheckExact(o));
  const long long v = PyLong_AsLongLong(o);
  need(!PyErr_Occurred() && v >= INT32_MIN && v <= INT32_MAX);
  return static_cast<int32_t>(v);
}

int32_t dim(int64_t n) {
  need(n > 0 && n <= INT32_MAX);
  return static_cast<int32_t>(n);
}

at::Tensor floats(at::IntArrayRef sizes, const at::Tensor& like) {
  return at::empty(sizes, like.options().dtype(at::kFloat).requires_grad(false));
}
at::Tensor like_of(const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }
at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(n < 256 ? 256 : n)},
                   like.options().dtype(at::kByte).requires_grad(false));
}

void* stream(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void done(int32_t status) { need(status == MEMLAYER_OK); }

PyObject* tuple(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

template <class F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F f) {
  try {
    need(have == want);
    return f();
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (x, scale, bias, residual or None, eps)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor& x = tensor(a[0], nullptr);
    need(x.dim() > 0);
    const int32_t d = dim(x.size(-1));
    const memlayer_norm_config cfg{x.numel() / d, d, dtype(x), static_cast<float>(number(a[4]))};
    memlayer_norm_args g{};
    g.x = x.const_data_ptr();
    g.x_stride = d;
    g.scale = vector(a[1], d, x);
    g.bias = vector(a[2], d, x);
    const bool two = a[3] != Py_None;
    if (two) {
      g.residual = same(a[3], x).const_data_ptr();
      g.residual_stride = d;
    }
    at::Tensor y = like_of(x), sum;
    g.y = y.data_ptr();
    if (two) {
      sum = like_of(x);
      g.sum = sum.data_ptr();
    }
    done(memlayer_layer_norm(&cfg, &g, stream(x)));
    return two ? tuple({y, sum}) : THPVariable_Wrap(y);
  });
}

// (dy, x, scale, dresidual or None, eps)
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor& dy = tensor(a[0], nullptr);
    need(dy.dim() > 0);
    const int32_t d = dim(dy.size(-1));
    const memlayer_norm_config cfg{dy.numel() / d, d, dtype(dy), static_cast<float>(number(a[4]))};
    memlayer_norm_grads g{};
    g.dy = dy.const_data_ptr();
    g.dy_stride = g.x_stride = d;
    g.x = same(a[1], dy).const_data_ptr();
    g.scale = vector(a[2], d, dy);
    if (a[3] != Py_None) {
      g.dresidual = same(a[3], dy).const_data_ptr();
      g.dresidual_stride = d;
    }
    size_t nb = 0;
    done(memlayer_layer_norm_backward_workspace_size(&cfg, &nb));
    at::Tensor dx = like_of(dy), ds = floats({d}, dy), db = floats({d}, dy), ws = bytes(nb, dy);
    g.dx = dx.data_ptr();
    g.dscale = static_cast<float*>(ds.data_ptr());
    g.dbias = static_cast<float*>(db.data_ptr());
    done(memlayer_layer_norm_backward(&cfg, &g, ws.data_ptr(), nb, stream(dy)));
    return tuple({dx, ds, db});
  });
}

struct Loss {
  const at::Tensor &h, &w, &y;
  memlayer_loss_config cfg;
  memlayer_loss_args args;
  Loss(PyObject* const* a, PyObject* ignore)
      : h(tensor(a[0], nullptr)), w(tensor(a[1], &h)), y(tensor(a[2], &h)), cfg{}, args{} {
    need(h.dim() > 0 && w.dim() == 2 && w.scalar_type() == h.scalar_type() && w.size(1) == h.size(-1));
    need(y.scalar_type() == at::kInt && y.sizes() == h.sizes().slice(0, h.dim() - 1));
    cfg = {y.numel(), dim(h.size(-1)), dim(w.size(0)), dtype(h), int32(ignore)};
    args.h = h.const_data_ptr();
    args.weight = w.const_data_ptr();
    args.h_stride = args.weight_stride = cfg.d_model;
    args.targets = static_cast<const int32_t*>(y.const_data_ptr());
  }
  at::Tensor workspace(int32_t backward, size_t* nb) {
    done(memlayer_cross_entropy_workspace_size(&cfg, backward, nb));
    return bytes(*nb, h);
  }
};

// (h, weight, targets, ignore_index)
PyObject* linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    Loss l(a, a[3]);
    size_t nb = 0;
    at::Tensor ws = l.workspace(0, &nb), loss = floats(l.y.sizes(), l.h), lse = floats(l.y.sizes(), l.h);
    l.args.loss = static_cast<float*>(loss.data_ptr());
    l.args.lse = static_cast<float*>(lse.data_ptr());
    done(memlayer_cross_entropy(&l.cfg, &l.args, ws.data_ptr(), nb, stream(l.h)));
    return tuple({loss, lse});
  });
}

// (h, weight, targets, lse, dloss, dlse or None, ignore_index)
PyObject* linear_cross_entropy_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    Loss l(a, a[6]);
    memlayer_loss_grads g{};
    g.lse = vector(a[3], l.cfg.tokens, l.h);
    g.dloss = vector(a[4], l.cfg.tokens, l.h);
    if (a[5] != Py_None) g.dlse = vector(a[5], l.cfg.tokens, l.h);
    size_t nb = 0;
    at::Tensor ws = l.workspace(1, &nb), dh = like_of(l.h), dw = like_of(l.w);
    g.dh = dh.data_ptr();
    g.dweight = dw.data_ptr();
    done(memlayer_cross_entropy_backward(&l.cfg, &l.args, &g, ws.data_ptr(), nb, stream(l.h)));
    return tuple({dh, dw});
  });
}

// (update, steps, a, b, c, eps)
PyObject* orthogonalize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const at::Tensor& u = tensor(a[0], nullptr);
    need(u.dim() >= 2);
    memlayer_orth_config cfg{};
    cfg.rows = dim(u.size(-2));
    cfg.cols = dim(u.size(-1));
    cfg.batch = u.numel() / (static_cast<int64_t>(cfg.rows) * cfg.cols);
    cfg.dtype = dtype(u);
    cfg.steps = int32(a[1]);
    cfg.a = static_cast<float>(number(a[2]));
    cfg.b = static_cast<float>(number(a[3]));
    cfg.c = static_cast<float>(number(a[4]));
    cfg.epsilon = static_cast<float>(number(a[5]));
    size_t nb = 0;
    done(memlayer_orthogonalize_workspace_size(&cfg, &nb));
    at::Tensor out = like_of(u), ws = bytes(nb, u);
    done(memlayer_orthogonalize(&cfg, u.const_data_ptr(), out.data_ptr(), ws.data_ptr(), nb, stream(u)));
    return THPVariable_Wrap(out);
  });
}

#define FAST(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {FAST(layer_norm),           FAST(layer_norm_backward),
                         FAST(linear_cross_entropy), FAST(linear_cross_entropy_backward),
                         FAST(orthogonalize),        {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// train_ops.py uses the module with the torch it was compiled against only.
PyMODINIT_FUNC PyInit__fast() {
  if (memlayer_abi_version() != MEMLAYER_ABI_VERSION) {
    PyErr_SetString(PyExc_ImportError, "_fast was built for another version of libmemlayer.so's interface");
    return nullptr;
  }
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", MEMLAYER_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
