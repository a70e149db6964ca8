// mlx_vit_b200._tensors: the host-side reading of lists of torch tensors, in C++.
//
// A step over a model's parameters looks at some hundred tensors five times (parameter,
// gradient, two states, shadow) before its one launch.  From Python that is about 0.1 us an
// attribute and 2.5 us a tensor, longer than the kernel for all but the largest models; here it is some
// ten nanoseconds a tensor.  Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/kda_b200.h"

namespace {

struct Refused {
  std::string why;
};
void need(bool ok, const char *why) {
  if (!ok) throw Refused{why};
}

// borrowed items of a list or tuple (the caller keeps the sequence alive)
struct Items {
  PyObject **p;
  Py_ssize_t n;
  Items(PyObject *o, const char *name) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) throw Refused{std::string(name) + ": expected a list"};
    n = PySequence_Fast_GET_SIZE(o);
    p = PySequence_Fast_ITEMS(o);
  }
};
const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) throw Refused{std::string(name) + ": expected torch tensors"};
  return THPVariable_Unpack(o);
}
int32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? KDA_F32 : t == at::kBFloat16 ? KDA_BF16 : t == at::kHalf ? KDA_F16 : -1;
}
const at::Tensor &state_part(PyObject *o, const char *name, at::ScalarType type, const at::Device &dev, int64_t numel) {
  const at::Tensor &t = tensor(o, name);
  if (t.device() != dev) throw Refused{std::string(name) + ": every tensor must be on the parameters' CUDA device"};
  if (t.scalar_type() != type) throw Refused{std::string(name) + (type == at::kByte ? ": must be uint8" : ": must be float32")};
  if (!t.is_contiguous()) throw Refused{std::string(name) + ": every tensor must be contiguous"};
  if (t.numel() != numel) throw Refused{std::string(name) + ": sizes do not match the parameters'"};
  return t;
}

template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const Refused &r) {
    PyErr_SetString(PyExc_ValueError, r.why.c_str());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// adamw_table(params, grads, exp_avgs, exp_avg_sqs, emas or None, bits) -> (KdaAdamWTensor array as
// bytes, device index).  ValueError for operands that the kernel does not take.  The versions
// of what the step writes are advanced, as torch's own in-place operations do.
PyObject *adamw_table(PyObject *, PyObject *args) {
  PyObject *po, *go, *mo, *vo, *eo;
  int bits;
  if (!PyArg_ParseTuple(args, "OOOOOi", &po, &go, &mo, &vo, &eo, &bits)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Items p(po, "params"), g(go, "grads"), m(mo, "exp_avgs"), v(vo, "exp_avg_sqs");
    const bool ema = eo != Py_None;
    const Items e(ema ? eo : po, "emas");
    need(p.n > 0, "no parameters");
    need(g.n == p.n && m.n == p.n && v.n == p.n && e.n == p.n, "every list must hold one entry a parameter");
    const at::Device dev = tensor(p.p[0], "params").device();
    need(dev.is_cuda(), "adamw_step takes CUDA tensors; there is no CPU path");
    std::vector<KdaAdamWTensor> rows(p.n);
    std::vector<const void *> written;
    written.reserve(4 * p.n);
    std::vector<const at::Tensor *> bump;
    bump.reserve(4 * p.n);
    for (Py_ssize_t i = 0; i < p.n; ++i) {
      const at::Tensor &pt = tensor(p.p[i], "params"), &gt = tensor(g.p[i], "grads");
      need(pt.device() == dev && gt.device() == dev,
           "params and grads must all be on one CUDA device; there is no CPU path");
      need(pt.layout() == at::kStrided && gt.layout() == at::kStrided, "params and grads must be dense tensors");
      need(pt.sizes() == gt.sizes(), "grads: shapes do not match the parameters'");
      need(pt.scalar_type() == gt.scalar_type(), "grads: dtypes do not match the parameters'");
      need(pt.is_non_overlapping_and_dense(), "params must be dense in memory");
      need((pt.is_contiguous() && gt.is_contiguous()) || pt.strides() == gt.strides(),
           "grads: not laid out in memory as the parameters");
      KdaAdamWTensor &r = rows[i];
      r = {};
      r.dtype = code_of(pt.scalar_type());
      need(r.dtype >= 0, "params must be float32, bfloat16 or float16");
      r.numel = pt.numel();
      r.p = pt.data_ptr();
      r.g = gt.data_ptr();
      const at::Tensor *mt, *vt;
      if (bits == 8) {
        const int64_t blocks = (r.numel + 255) / 256;
        const Items mp(m.p[i], "exp_avgs"), vp(v.p[i], "exp_avg_sqs");
        need(mp.n == 2 && vp.n == 2, "8-bit states are (codes, exponents) pairs, all of them");
        mt = &state_part(mp.p[0], "exp_avgs", at::kByte, dev, r.numel);
        vt = &state_part(vp.p[0], "exp_avg_sqs", at::kByte, dev, r.numel);
        const at::Tensor &me = state_part(mp.p[1], "exp_avgs' exponents", at::kByte, dev, blocks);
        const at::Tensor &ve = state_part(vp.p[1], "exp_avg_sqs' exponents", at::kByte, dev, blocks);
        r.m_exp = static_cast<uint8_t *>(me.data_ptr());
        r.v_exp = static_cast<uint8_t *>(ve.data_ptr());
        if (r.numel) written.insert(written.end(), {r.m_exp, r.v_exp});
        bump.insert(bump.end(), {&me, &ve});
      } else {
        mt = &state_part(m.p[i], "exp_avgs", at::kFloat, dev, r.numel);
        vt = &state_part(v.p[i], "exp_avg_sqs", at::kFloat, dev, r.numel);
      }
      r.m = mt->data_ptr();
      r.v = vt->data_ptr();
      bump.insert(bump.end(), {&pt, mt, vt});
      if (ema) {
        const at::Tensor &et = state_part(e.p[i], "emas", at::kFloat, dev, r.numel);
        r.ema = static_cast<float *>(et.data_ptr());
        bump.push_back(&et);
      }
      if (r.numel) {
        written.insert(written.end(), {r.p, r.m, r.v});
        if (ema) written.push_back(r.ema);
      }
    }
    std::sort(written.begin(), written.end());
    need(std::adjacent_find(written.begin(), written.end()) == written.end(), "the same tensor is passed twice");
    for (const at::Tensor *t : bump)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return Py_BuildValue("(y#i)", reinterpret_cast<const char *>(rows.data()),
                         (Py_ssize_t)(rows.size() * sizeof(KdaAdamWTensor)), (int)dev.index());
  });
}

// grad_table(grads) -> (KdaAdamWTensor array as bytes, device index), for the norm alone
PyObject *grad_table(PyObject *, PyObject *args) {
  PyObject *go;
  if (!PyArg_ParseTuple(args, "O", &go)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Items g(go, "grads");
    need(g.n > 0, "no gradients");
    const at::Device dev = tensor(g.p[0], "grads").device();
    need(dev.is_cuda(), "grad_norm takes CUDA tensors; there is no CPU path");
    std::vector<KdaAdamWTensor> rows(g.n);
    for (Py_ssize_t i = 0; i < g.n; ++i) {
      const at::Tensor &t = tensor(g.p[i], "grads");
      need(t.device() == dev, "grads must all be on one CUDA device; there is no CPU path");
      need(t.layout() == at::kStrided && t.is_non_overlapping_and_dense(), "grads must be dense in memory");
      rows[i] = {};
      rows[i].dtype = code_of(t.scalar_type());
      need(rows[i].dtype >= 0, "grads must be float32, bfloat16 or float16");
      rows[i].g = t.data_ptr();
      rows[i].numel = t.numel();
    }
    return Py_BuildValue("(y#i)", reinterpret_cast<const char *>(rows.data()),
                         (Py_ssize_t)(rows.size() * sizeof(KdaAdamWTensor)), (int)dev.index());
  });
}

// unlike(params, grads) -> indices of the strided gradients that lie in memory otherwise than their parameters
PyObject *unlike(PyObject *, PyObject *args) {
  PyObject *po, *go;
  if (!PyArg_ParseTuple(args, "OO", &po, &go)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Items p(po, "params"), g(go, "grads");
    need(g.n == p.n, "every list must hold one entry a parameter");
    PyObject *out = PyList_New(0);
    for (Py_ssize_t i = 0; out && i < p.n; ++i) {
      const at::Tensor &pt = tensor(p.p[i], "params"), &gt = tensor(g.p[i], "grads");
      if (pt.layout() != at::kStrided || gt.layout() != at::kStrided || pt.strides() == gt.strides() ||
          (pt.is_contiguous() && gt.is_contiguous()))
        continue;
      PyObject *k = PyLong_FromSsize_t(i);
      if (!k || PyList_Append(out, k)) {
        Py_XDECREF(k);
        Py_CLEAR(out);
        break;
      }
      Py_DECREF(k);
    }
    return out;
  });
}

PyMethodDef methods[] = {{"adamw_table", adamw_table, METH_VARARGS, nullptr},
                         {"grad_table", grad_table, METH_VARARGS, nullptr},
                         {"unlike", unlike, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
