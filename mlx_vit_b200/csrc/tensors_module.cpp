// mlx_vit_b200._tensors: the host side of the operators whose launches are shorter than Python's way
// to them, in C++: the optimizer's step over a model's tensor lists, and the linear products with
// their autograd functions.
//
// An optimizer step over a model's parameters looks at some hundred tensors five times (parameter,
// gradient, two states, shadow) before its one launch.  From Python that is about 0.1 us an
// attribute and 2.5 us a tensor, longer than the kernel for all but the largest models; here it is some
// ten nanoseconds a tensor.  Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/CUDAContextLight.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

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
  } catch (python_error &e) {
    e.restore();
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// The KdaAdamWTensor array of a step's lists, after their checks, their device, and the tensors that the
// step writes.
std::vector<KdaAdamWTensor> adamw_table(PyObject *po, PyObject *go, PyObject *mo, PyObject *vo, PyObject *eo, int &bits,
                                        at::Device &dev, std::vector<const at::Tensor *> &bump) {
  const Items p(po, "params"), g(go, "grads"), m(mo, "exp_avgs"), v(vo, "exp_avg_sqs");
  const bool ema = eo != Py_None;
  const Items e(ema ? eo : po, "emas");
  need(p.n > 0, "no parameters");
  need(g.n == p.n && m.n == p.n && v.n == p.n && e.n == p.n, "every list must hold one entry a parameter");
  dev = tensor(p.p[0], "params").device();
  bits = PyTuple_Check(m.p[0]) || PyList_Check(m.p[0]) ? 8 : 32;
  need(dev.is_cuda(), "adamw_step takes CUDA tensors; there is no CPU path");
  std::vector<KdaAdamWTensor> rows(p.n);
  std::vector<const void *> written;
  written.reserve(4 * p.n);
  bump.reserve(4 * p.n + 1);
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
  return rows;
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

void done(int status, const char *where) {
  TORCH_CHECK(status == 0, where, ": ", kda_strerror(status));
}
void *stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
bool capturing(void *st) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(static_cast<cudaStream_t>(st), &s) == cudaSuccess) return s != cudaStreamCaptureStatusNone;
  (void)cudaGetLastError();  // not a question for this stream now: the launch will say
  return false;
}
at::Tensor adamw_workspace(int64_t count, const at::Device &dev) {
  return at::empty({(int64_t)kda_adamw_workspace_bytes(count)}, at::TensorOptions().dtype(at::kByte).device(dev));
}
// a step, learning rate or norm that lies on the device
const at::Tensor *scalar(PyObject *o, const char *name, at::ScalarType type, const at::Device &dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (t.device() != dev || t.scalar_type() != type || t.numel() != 1)
    throw Refused{std::string(name) + " as a tensor must be one " + (type == at::kLong ? "int64" : "float32") +
                  " value on the parameters' device"};
  return &t;
}

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, emas or None, step, lr, beta1, beta2, eps, weight_decay,
//            bias_correction, max_grad_norm (0: none), ema_decay, seed, norm or None, first_tensor) -> norm or None.
// ValueError for operands that the kernel does not take.
PyObject *adamw_step(PyObject *, PyObject *args) {
  PyObject *po, *go, *mo, *vo, *eo, *so, *lo, *no;
  KdaAdamW a = {};
  int bias;
  unsigned int seed, first;
  if (!PyArg_ParseTuple(args, "OOOOOOOddddpddIOI", &po, &go, &mo, &vo, &eo, &so, &lo, &a.beta1, &a.beta2, &a.eps, &a.weight_decay,
                        &bias, &a.max_grad_norm, &a.ema_decay, &seed, &no, &first))
    return nullptr;
  return guarded([&]() -> PyObject * {
    need(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1, "betas must lie in [0, 1)");
    need(a.eps >= 0, "eps must not be negative");
    need(a.ema_decay >= 0 && a.ema_decay <= 1, "ema_decay must lie in [0, 1]");
    need(no == Py_None || a.max_grad_norm > 0, "norm is used with max_grad_norm only");
    at::Device dev(at::kCPU);
    std::vector<const at::Tensor *> written;
    const std::vector<KdaAdamWTensor> rows = adamw_table(po, go, mo, vo, eo, a.state_bits, dev, written);
    need(a.state_bits == 32 || a.eps >= 1e-30, "8-bit states need an eps of at least 1e-30");
    const at::Tensor *step = scalar(so, "step", at::kLong, dev), *lr = scalar(lo, "lr", at::kFloat, dev);
    const at::Tensor *given = no == Py_None ? nullptr : scalar(no, "norm", at::kFloat, dev);
    need(no == Py_None || given, "norm must be a tensor");
    if (!step) {
      a.step = PyLong_AsLongLong(so);
      if (PyErr_Occurred()) return nullptr;
      need(a.step >= 1, "step counts from 1");
    }
    if (!lr) {
      a.lr = PyFloat_AsDouble(lo);
      if (PyErr_Occurred()) return nullptr;
    }
    a.seed = seed;
    a.first_tensor = first;
    a.bias_correction = bias;
    a.use_ema = eo != Py_None;
    a.norm_given = given != nullptr;
    const c10::cuda::CUDAGuard guard(dev);
    void *st = stream();
    need((step && lr) || !capturing(st), "step and lr must be CUDA tensors while a graph is captured");
    const bool clip = a.max_grad_norm > 0;
    at::Tensor ws, norm;
    if (clip || step || lr) ws = adamw_workspace((int64_t)rows.size(), dev);
    if (clip) norm = given ? *given : at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    done(kda_adamw_step(&a, rows.data(), (int64_t)rows.size(), step ? step->data_ptr<int64_t>() : nullptr,
                        lr ? lr->data_ptr<float>() : nullptr, clip ? norm.data_ptr<float>() : nullptr,
                        ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0, st),
         "kda_adamw_step");
    // the versions of what was written advance, as under torch's own in-place operations
    if (step) written.push_back(step);
    for (const at::Tensor *t : written)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    if (clip) return THPVariable_Wrap(norm);
    Py_RETURN_NONE;
  });
}

// grad_norm(grads) -> their 2-norm, a float32 scalar on their device
PyObject *grad_norm(PyObject *, PyObject *args) {
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
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor ws = adamw_workspace((int64_t)rows.size(), dev);
    const at::Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    done(kda_grad_norm(rows.data(), (int64_t)rows.size(), norm.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream()),
         "kda_grad_norm");
    return THPVariable_Wrap(norm);
  });
}

// ---- linear products ----
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int dtype_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? KDA_BF16 : KDA_F16; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
// elements from row to row of a matrix with contiguous rows
int64_t pitch(const Tensor &t) {
  return !t.defined() ? 0 : t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
}
// a matrix that the products can read: a row pitch of whole 16-byte units
Tensor matrix(int64_t rows, int64_t cols, const Tensor &like) {
  const int64_t ld = (cols + 7) / 8 * 8;
  Tensor t = at::empty({rows, ld}, like.options());
  return ld == cols ? t : t.narrow(1, 0, cols);
}
// a tensor as a matrix with contiguous rows, in place where its strides allow it
Tensor rows_of(const Tensor &x, int64_t cols) {
  Tensor t = x.dim() == 2 ? x : x.reshape({x.numel() / cols, cols});
  if ((cols > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < cols)) t = t.contiguous();
  return t;
}
struct Workspace {
  Tensor t;
  size_t n;
  Workspace(int op, int64_t m, int64_t n_, int64_t k, bool db, const Tensor &like) : n(kda_linear_workspace_bytes(op, m, n_, k, db)) {
    if (n) t = at::empty({(int64_t)n}, like.options().dtype(at::kByte));
  }
};
// dz (undefined: not wanted) = dy act'(z), and its column sums
void act_grad(int act, const Tensor &dy, const Tensor &z, const Tensor &dz, const Tensor &db) {
  const Workspace ws(KDA_LINEAR_ACT_GRAD, dy.size(0), dy.size(1), 1, db.defined(), dy);
  done(kda_act_grad(dtype_of(dy), act, dy.size(0), dy.size(1), ptr(dy), pitch(dy), ptr(z), pitch(z), ptr(dz), pitch(dz), ptr(db),
                    ptr(ws.t), ws.n, stream()),
       "kda_act_grad");
}
bool is_readable(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && pitch(t) % 8 == 0; }
// the matrix itself where the products can read it, else a copy with padded rows
Tensor readable(const Tensor &t) {
  if (is_readable(t)) return t;
  Tensor out = matrix(t.size(0), t.size(1), t);
  act_grad(KDA_ACT_NONE, t, Tensor(), out, Tensor());
  return out;
}
// the gradient at a layer's sum from the one at its result (z undefined: no activation), as the products
// read it, and with want_db its column sums: in one pass, or none where neither is asked for
Tensor gradient_at_sum(int act, const Tensor &dy, const Tensor &z, bool want_db, Tensor &db) {
  const bool copy = act || !is_readable(dy);
  if (want_db) db = at::empty({dy.size(1)}, dy.options());
  const Tensor dz = copy ? matrix(dy.size(0), dy.size(1), dy) : Tensor();
  if (copy || want_db) act_grad(act, dy, z, dz, db);
  return copy ? dz : dy;
}
void product(int act, const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, const Tensor &y, const Tensor &z) {
  const Workspace ws(KDA_LINEAR_FWD, x.size(0), w.size(0), w.size(1), false, x);
  done(kda_linear_fwd(dtype_of(x), act, x.size(0), w.size(0), w.size(1), ptr(x), pitch(x), ptr(w), pitch(w), ptr(b),
                      ptr(r), pitch(r), ptr(y), pitch(y), ptr(z), pitch(z), ptr(ws.t), ws.n, stream()),
       "kda_linear_fwd");
}
void dgrad(int act, const Tensor &dz, const Tensor &w, const Tensor &z, const Tensor &dx, const Tensor &db) {
  const Workspace ws(KDA_LINEAR_DGRAD, dz.size(0), w.size(0), w.size(1), db.defined(), dz);
  done(kda_linear_dgrad(dtype_of(dz), act, dz.size(0), w.size(0), w.size(1), ptr(dz), pitch(dz), ptr(w), pitch(w), ptr(z),
                        pitch(z), ptr(dx), pitch(dx), ptr(db), ptr(ws.t), ws.n, stream()),
       "kda_linear_dgrad");
}
Tensor wgrad(const Tensor &dz, const Tensor &x) {
  const int64_t m = dz.size(0), n = dz.size(1), k = x.size(1);
  Tensor dw = at::empty({n, k}, x.options());
  const Workspace ws(KDA_LINEAR_WGRAD, m, n, k, false, x);
  done(kda_linear_wgrad(dtype_of(x), m, n, k, ptr(dz), pitch(dz), ptr(x), pitch(x), ptr(dw), k, ptr(ws.t), ws.n, stream()),
       "kda_linear_wgrad");
  return dw;
}
std::vector<int64_t> with_last(const Tensor &x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}
// the results of a backward pass that has no derivative of its own
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (Tensor &g : grads)
    if (g.defined()) in.push_back(g = g.detach().requires_grad_());
  variable_list out = torch::autograd::DelayedError("the linear products are differentiable once", (int)in.size())(variable_list(in));
  size_t i = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor plain(const Maybe &t) { return t ? *t : Tensor(); }
// A leaf's accumulating node keeps the stream on which the leaf first entered a graph that still lives.  Where
// that is the default stream, a backward pass that is being captured would have to wait on it, which invalidates
// the capture inside torch's engine and ends the process: refused before.
void refuse_uncapturable_leaves(const at::Device &dev) {
  const c10::cuda::CUDAGuard guard(dev);
  const c10::cuda::CUDAStream now = c10::cuda::getCurrentCUDAStream();
  if (!capturing(now.stream())) return;
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const torch::autograd::Edge &e = node->next_edge(i);
    if (!e.function || !node->task_should_compute_output(i) || !dynamic_cast<torch::autograd::AccumulateGrad *>(e.function.get()))
      continue;
    const std::optional<c10::Stream> s = e.function->stream();
    TORCH_CHECK(!s || *s != c10::cuda::getDefaultCUDAStream(now.device_index()).unwrap(),
                "linear products: an operand entered a graph on the default stream that is still alive, so that its gradient "
                "cannot be captured; release that graph's results, or run it on another stream");
  }
}
// which of the tensor arguments need a gradient; an absent one has no edge in the graph
struct Needs {
  const AutogradContext *ctx;
  size_t edge = 0;
  bool operator()(bool present) { return present && ctx->needs_input_grad(edge++); }
};

struct LinearAct : public torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext *ctx, Tensor x, Tensor w, Maybe bias, Maybe residual, int64_t act, bool save) {
    const int64_t n = w.size(0), k = w.size(1);
    const Tensor b = plain(bias), r = plain(residual);
    Tensor y = at::empty(with_last(x, n), x.options()), z;
    if (x.numel()) {
      const c10::cuda::CUDAGuard guard(x.device());
      Tensor x2 = readable(rows_of(x, k)), w2 = readable(rows_of(w, k));
      if (save && act) z = matrix(x2.size(0), n, x);
      product((int)act, x2, w2, b.defined() ? b.contiguous() : b, r.defined() ? rows_of(r, n) : r, y.view({-1, n}), z);
      if (save) ctx->save_for_backward({x2, w2, z});
    } else if (save) {
      ctx->save_for_backward({x, w, z});
    }
    if (save) {
      ctx->saved_data["act"] = act;
      ctx->saved_data["sizes"] = x.sizes().vec();
      ctx->saved_data["bias"] = b.defined();
      ctx->saved_data["residual"] = r.defined();
    }
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list dys) {
    refuse_uncapturable_leaves(dys[0].device());
    const variable_list saved = ctx->get_saved_variables();
    Tensor x = saved[0].detach(), w = saved[1].detach(), z = saved[2];
    const Tensor dy = dys[0].detach();
    const int64_t n = w.size(0), k = w.size(1);
    const int act = (int)ctx->saved_data["act"].toInt();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    Needs needs{ctx};
    const bool need_x = needs(true), need_w = needs(true), need_b = needs(ctx->saved_data["bias"].toBool());
    variable_list g(6);
    // dys[0] itself, whose owners torch counts before it keeps a gradient: dy, a tensor of its own over the same
    // memory, would be kept as it is and then written to
    if (needs(ctx->saved_data["residual"].toBool())) g[3] = dys[0];
    if (x.numel() == 0) {
      if (need_x) g[0] = at::zeros(sizes, x.options());
      if (need_w) g[1] = at::zeros_like(w);
      if (need_b) g[2] = at::zeros({n}, w.options());
    } else if (need_x || need_w || need_b) {
      const c10::cuda::CUDAGuard guard(x.device());
      // a hook on saved tensors (save_on_cpu) gives them back without their padded rows
      x = readable(rows_of(x, k));
      w = readable(rows_of(w, k));
      if (z.defined()) z = rows_of(z, n);
      const Tensor dz = gradient_at_sum(act, rows_of(dy, n), z, need_b, g[2]);
      if (need_x) {
        g[0] = at::empty(sizes, x.options());
        dgrad(KDA_ACT_NONE, dz, w, Tensor(), g[0].view({-1, k}), Tensor());
      }
      if (need_w) g[1] = wgrad(dz, x);
    }
    return once(g);
  }
};

struct Mlp : public torch::autograd::Function<Mlp> {
  static Tensor forward(AutogradContext *ctx, Tensor x, Tensor w1, Maybe bias1, Tensor w2, Maybe bias2, Maybe residual,
                        int64_t act, bool save) {
    const int64_t n = w1.size(0), k = w1.size(1), out = w2.size(0);
    const Tensor b1 = plain(bias1), b2 = plain(bias2), r = plain(residual);
    Tensor y = at::empty(with_last(x, out), x.options()), h, z;
    if (x.numel()) {
      const c10::cuda::CUDAGuard guard(x.device());
      const Tensor x2 = readable(rows_of(x, k)), u1 = readable(rows_of(w1, k)), u2 = readable(rows_of(w2, n));
      h = matrix(x2.size(0), n, x);
      if (save && act) z = matrix(x2.size(0), n, x);
      product((int)act, x2, u1, b1.defined() ? b1.contiguous() : b1, Tensor(), h, z);
      product(KDA_ACT_NONE, h, u2, b2.defined() ? b2.contiguous() : b2, r.defined() ? rows_of(r, out) : r, y.view({-1, out}),
              Tensor());
      if (save) ctx->save_for_backward({x2, u1, u2, h, z});
    } else if (save) {
      ctx->save_for_backward({x, w1, w2, h, z});
    }
    if (save) {
      ctx->saved_data["act"] = act;
      ctx->saved_data["sizes"] = x.sizes().vec();
      ctx->saved_data["bias1"] = b1.defined();
      ctx->saved_data["bias2"] = b2.defined();
      ctx->saved_data["residual"] = r.defined();
    }
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list dys) {
    refuse_uncapturable_leaves(dys[0].device());
    const variable_list saved = ctx->get_saved_variables();
    Tensor x = saved[0].detach(), w1 = saved[1].detach(), w2 = saved[2].detach(), h = saved[3], z = saved[4];
    const Tensor dy = dys[0].detach();
    const int64_t n = w1.size(0), k = w1.size(1), out = w2.size(0);
    const int act = (int)ctx->saved_data["act"].toInt();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    Needs needs{ctx};
    const bool need_x = needs(true), need_w1 = needs(true), need_b1 = needs(ctx->saved_data["bias1"].toBool()),
               need_w2 = needs(true), need_b2 = needs(ctx->saved_data["bias2"].toBool());
    variable_list g(8);
    // as in LinearAct
    if (needs(ctx->saved_data["residual"].toBool())) g[5] = dys[0];
    if (x.numel() == 0) {
      if (need_x) g[0] = at::zeros(sizes, x.options());
      if (need_w1) g[1] = at::zeros_like(w1);
      if (need_b1) g[2] = at::zeros({n}, w1.options());
      if (need_w2) g[3] = at::zeros_like(w2);
      if (need_b2) g[4] = at::zeros({out}, w2.options());
    } else if (need_x || need_w1 || need_b1 || need_w2 || need_b2) {
      const c10::cuda::CUDAGuard guard(x.device());
      // as in LinearAct
      x = readable(rows_of(x, k));
      w1 = readable(rows_of(w1, k));
      w2 = readable(rows_of(w2, n));
      h = readable(rows_of(h, n));
      if (z.defined()) z = rows_of(z, n);
      const Tensor dy2 = gradient_at_sum(KDA_ACT_NONE, rows_of(dy, out), Tensor(), need_b2, g[4]);
      if (need_w2) g[3] = wgrad(dy2, h);
      if (need_x || need_w1 || need_b1) {
        const Tensor dz = matrix(dy2.size(0), n, x);
        if (need_b1) g[2] = at::empty({n}, x.options());
        dgrad(act, dy2, w2, z, dz, g[2]);
        if (need_x) {
          g[0] = at::empty(sizes, x.options());
          dgrad(KDA_ACT_NONE, dz, w1, Tensor(), g[0].view({-1, k}), Tensor());
        }
        if (need_w1) g[1] = wgrad(dz, x);
      }
    }
    return once(g);
  }
};

std::string shape_of(const Tensor &t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
Tensor operand(PyObject *o, const char *name, bool optional) {
  if (optional && o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) throw Refused{std::string(name) + ": expected a torch tensor"};
  return THPVariable_Unpack(o);
}
struct Layer {
  const char *name;
  const Tensor &w, &b;
};
// a tangent is not carried along, and a result without one would count as constant
void refuse_tangent(const Tensor &t) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "linear products: no forward-mode derivatives");
}
void check_operands(const Tensor &x, const Tensor &r, std::initializer_list<Layer> layers) {
  // a tracer (torch.jit.trace, make_fx) would record the results' allocation and not what fills them
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
              "linear products cannot be traced");
  refuse_tangent(x);
  refuse_tangent(r);
  for (const Layer &l : layers) {
    refuse_tangent(l.w);
    refuse_tangent(l.b);
  }
  need(x.is_cuda(), "linear products take CUDA tensors; there is no CPU path");
  need(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "linear products take bfloat16 or float16");
  need(x.dim() >= 1, "x must have at least one dimension");
  int64_t k = x.size(-1);
  auto like_x = [&](const Tensor &t) {
    need(t.device() == x.device() && t.scalar_type() == x.scalar_type(), "all operands must share x's dtype and device");
  };
  for (const Layer &l : layers) {
    if (l.w.dim() != 2 || l.w.size(1) != k || l.w.size(0) < 1 || k < 1)
      throw Refused{std::string(l.name) + " must be (out_features, " + std::to_string(k) + "), got " + shape_of(l.w)};
    like_x(l.w);
    k = l.w.size(0);
    if (!l.b.defined()) continue;
    if (l.b.dim() != 1 || l.b.size(0) != k)
      throw Refused{"the bias of " + std::string(l.name) + " must be (" + std::to_string(k) + "), got " + shape_of(l.b)};
    like_x(l.b);
  }
  if (!r.defined()) return;
  like_x(r);
  if (r.sizes() != at::IntArrayRef(with_last(x, k)))
    throw Refused{"residual must have x's leading dimensions and " + std::to_string(k) + " columns, got " + shape_of(r)};
}
template <typename... T>
bool grads_wanted(const T &...t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// linear_act(x, w, b or None, act, residual or None) -> y
PyObject *linear_act(PyObject *, PyObject *args) {
  PyObject *xo, *wo, *bo, *ro;
  int act;
  if (!PyArg_ParseTuple(args, "OOOiO", &xo, &wo, &bo, &act, &ro)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Tensor x = operand(xo, "x", false), w = operand(wo, "weight", false), b = operand(bo, "bias", true),
                 r = operand(ro, "residual", true);
    check_operands(x, r, {{"weight", w, b}});
    // nothing to record: the computation alone
    if (!grads_wanted(x, w, b, r)) return THPVariable_Wrap(LinearAct::forward(nullptr, x, w, maybe(b), maybe(r), act, false));
    return THPVariable_Wrap(LinearAct::apply(x, w, maybe(b), maybe(r), (int64_t)act, true));
  });
}
// mlp(x, w1, b1 or None, w2, b2 or None, act, residual or None) -> y
PyObject *mlp(PyObject *, PyObject *args) {
  PyObject *xo, *w1o, *b1o, *w2o, *b2o, *ro;
  int act;
  if (!PyArg_ParseTuple(args, "OOOOOiO", &xo, &w1o, &b1o, &w2o, &b2o, &act, &ro)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Tensor x = operand(xo, "x", false), w1 = operand(w1o, "w1", false), b1 = operand(b1o, "b1", true),
                 w2 = operand(w2o, "w2", false), b2 = operand(b2o, "b2", true), r = operand(ro, "residual", true);
    check_operands(x, r, {{"w1", w1, b1}, {"w2", w2, b2}});
    if (!grads_wanted(x, w1, b1, w2, b2, r))
      return THPVariable_Wrap(Mlp::forward(nullptr, x, w1, maybe(b1), w2, maybe(b2), maybe(r), act, false));
    return THPVariable_Wrap(Mlp::apply(x, w1, maybe(b1), w2, maybe(b2), maybe(r), (int64_t)act, true));
  });
}

PyMethodDef methods[] = {{"adamw_step", adamw_step, METH_VARARGS, nullptr},
                         {"grad_norm", grad_norm, METH_VARARGS, nullptr},
                         {"unlike", unlike, METH_VARARGS, nullptr},
                         {"linear_act", linear_act, METH_VARARGS, nullptr},
                         {"mlp", mlp, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
