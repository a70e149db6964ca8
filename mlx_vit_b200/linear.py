"""Linear products with bias, activation and residual in one kernel (bf16 or fp16), with autograd:
``linear_act`` is act(x W^T + b) + r, one layer of the blocks around the KDA recurrence; ``mlp`` the
blocks' MLP of two layers, residual included (HybridBlock, nope_gdn_mlx.py:4009-4090), whose
backward takes the activation's derivative in the epilogue of the product that feeds it.  Products
run on the tensor cores with float32 accumulation (``kda_linear_*`` in include/kda_b200.h); what is
rounded to 16 bits on the way are the results, the saved pre-activation z, the MLP's hidden
activation and the gradient at z.  No CPU path."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": _lib.KDA_ACT_NONE, "relu": _lib.KDA_ACT_RELU, "silu": _lib.KDA_ACT_SILU,
               "gelu": _lib.KDA_ACT_GELU, "gelu_tanh": _lib.KDA_ACT_GELU_TANH}
_DTYPES = {torch.bfloat16: _lib.KDA_BF16, torch.float16: _lib.KDA_F16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _pitch(t):
    """Elements from row to row of a 2-D tensor whose rows are contiguous."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _new(rows, cols, like):
    """A matrix that the products can read: a row pitch of whole 16-byte units."""
    return torch.empty((rows, -(-cols // 8) * 8), dtype=like.dtype, device=like.device)[:, :cols]


def _rows(t, cols):
    """A tensor as a matrix with contiguous rows, in place where its strides allow it."""
    t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _readable(t):
    """The matrix itself where the products can read it, else a copy with padded rows."""
    if t.data_ptr() % 16 == 0 and _pitch(t) % 8 == 0:
        return t
    out = _new(t.shape[0], t.shape[1], t)
    _act_grad(_lib.KDA_ACT_NONE, t, None, out)
    return out


def _act_grad(act, dy, z, dz):
    _lib.check(_lib.lib().kda_act_grad(_DTYPES[dy.dtype], act, dy.shape[0], dy.shape[1], dy.data_ptr(), _pitch(dy),
                                       _ptr(z), 0 if z is None else _pitch(z), dz.data_ptr(), _pitch(dz), _stream()),
               "kda_act_grad")


def _fwd(act, x, w, b, r, y, z):
    _lib.check(_lib.lib().kda_linear_fwd(
        _DTYPES[x.dtype], act, x.shape[0], w.shape[0], w.shape[1], x.data_ptr(), _pitch(x), w.data_ptr(), _pitch(w),
        _ptr(b), _ptr(r), 0 if r is None else _pitch(r), y.data_ptr(), _pitch(y), _ptr(z),
        0 if z is None else _pitch(z), _stream()), "kda_linear_fwd")


def _dgrad(act, dz, w, z, dx):
    _lib.check(_lib.lib().kda_linear_dgrad(
        _DTYPES[dz.dtype], act, dz.shape[0], w.shape[0], w.shape[1], dz.data_ptr(), _pitch(dz), w.data_ptr(), _pitch(w),
        _ptr(z), 0 if z is None else _pitch(z), dx.data_ptr(), _pitch(dx), _stream()), "kda_linear_dgrad")


def _wgrad(dz, x, want_db):
    m, n, k = dz.shape[0], dz.shape[1], x.shape[1]
    dw = torch.empty((n, k), dtype=x.dtype, device=x.device)
    db = torch.empty((n,), dtype=x.dtype, device=x.device) if want_db else None
    L = _lib.lib()
    nws = L.kda_linear_wgrad_workspace_bytes(m, n, k) if want_db else 0
    ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws else None
    _lib.check(L.kda_linear_wgrad(_DTYPES[x.dtype], m, n, k, dz.data_ptr(), _pitch(dz), x.data_ptr(), _pitch(x),
                                  dw.data_ptr(), k, _ptr(db), _ptr(ws), nws, _stream()), "kda_linear_wgrad")
    return dw, db


def _check(x, activation, residual, out_features, layers):
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("linear products take CUDA tensors; there is no CPU path")
    if x.dtype not in _DTYPES:
        raise ValueError(f"linear products take bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    k = x.shape[-1]
    for name, w, b in layers:
        if w.dim() != 2 or w.shape[1] != k or w.shape[0] < 1 or k < 1:
            raise ValueError(f"{name} must be (out_features, {k}), got {tuple(w.shape)}")
        if b is not None and tuple(b.shape) != (w.shape[0],):
            raise ValueError(f"the bias of {name} must be ({w.shape[0]},), got {tuple(b.shape)}")
        k = w.shape[0]
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], out_features):
        raise ValueError(f"residual must be {(*x.shape[:-1], out_features)}, got {tuple(residual.shape)}")
    for t in (residual, *(t for _, w, b in layers for t in (w, b))):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"all operands must share x's dtype and device ({x.dtype}, {x.device}), got {t.dtype}, "
                             f"{t.device}")


class LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act, save):
        n, k = w.shape
        y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
        ctx.act, ctx.x_shape = act, x.shape
        with torch.cuda.device(x.device):
            x2 = _rows(x, k)
            m = x2.shape[0]
            ctx.empty = m == 0
            if m:
                x2, w2 = _readable(x2), _readable(_rows(w, k))
                z = _new(m, n, x) if save and act else None
                _fwd(act, x2, w2, None if b is None else b.contiguous(), None if r is None else _rows(r, n),
                     y.view(m, n), z)
                ctx.save_for_backward(x2, w2, z)
            else:
                ctx.save_for_backward(x2, w, None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        n, k = w.shape
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dr = dy if need_r else None
        if ctx.empty:
            return (x.new_zeros(ctx.x_shape) if need_x else None, torch.zeros_like(w) if need_w else None,
                    w.new_zeros(n) if need_b else None, dr, None, None)
        dx = dw = db = None
        with torch.cuda.device(x.device):
            if need_x or need_w or need_b:
                dz = _rows(dy, n)
                if ctx.act:
                    out = _new(dz.shape[0], n, dz)
                    _act_grad(ctx.act, dz, z, out)
                    dz = out
                else:
                    dz = _readable(dz)
                if need_x:
                    dx = torch.empty(ctx.x_shape, dtype=x.dtype, device=x.device)
                    _dgrad(_lib.KDA_ACT_NONE, dz, w, None, dx.view(-1, k))
                if need_w or need_b:
                    dw, db = _wgrad(dz, x, need_b)
        return dx, dw if need_w else None, db, dr, None, None


class MLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, r, act, save):
        (n, k), out = w1.shape, w2.shape[0]
        y = torch.empty((*x.shape[:-1], out), dtype=x.dtype, device=x.device)
        ctx.act, ctx.x_shape = act, x.shape
        with torch.cuda.device(x.device):
            x2 = _rows(x, k)
            m = x2.shape[0]
            ctx.empty = m == 0
            if m:
                x2, w1, w2 = _readable(x2), _readable(_rows(w1, k)), _readable(_rows(w2, n))
                h = _new(m, n, x)
                z = _new(m, n, x) if save and act else None
                _fwd(act, x2, w1, None if b1 is None else b1.contiguous(), None, h, z)
                _fwd(_lib.KDA_ACT_NONE, h, w2, None if b2 is None else b2.contiguous(),
                     None if r is None else _rows(r, out), y.view(m, out), None)
                ctx.save_for_backward(x2, w1, w2, h, z)
            else:
                ctx.save_for_backward(x2, w1, w2, None, None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w1, w2, h, z = ctx.saved_tensors
        (n, k), out = w1.shape, w2.shape[0]
        need_x, need_w1, need_b1, need_w2, need_b2, need_r = ctx.needs_input_grad[:6]
        dr = dy if need_r else None
        if ctx.empty:
            return (x.new_zeros(ctx.x_shape) if need_x else None, torch.zeros_like(w1) if need_w1 else None,
                    w1.new_zeros(n) if need_b1 else None, torch.zeros_like(w2) if need_w2 else None,
                    w2.new_zeros(out) if need_b2 else None, dr, None, None)
        dx = dw1 = db1 = dw2 = db2 = None
        with torch.cuda.device(x.device):
            dy2 = _readable(_rows(dy, out))
            if need_w2 or need_b2:
                dw2, db2 = _wgrad(dy2, h, need_b2)
            if need_x or need_w1 or need_b1:
                dz = _new(dy2.shape[0], n, x)
                _dgrad(ctx.act, dy2, w2, z, dz)
                if need_x:
                    dx = torch.empty(ctx.x_shape, dtype=x.dtype, device=x.device)
                    _dgrad(_lib.KDA_ACT_NONE, dz, w1, None, dx.view(-1, k))
                if need_w1 or need_b1:
                    dw1, db1 = _wgrad(dz, x, need_b1)
        return (dx, dw1 if need_w1 else None, db1, dw2 if need_w2 else None, db2, dr, None, None)


def _grad_wanted(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual.

    x is (..., in_features), weight (out_features, in_features), bias (out_features,), residual
    (..., out_features); all bf16 or all fp16, on one device, any strides.  ``activation`` is "none",
    "relu", "silu", "gelu" (exact) or "gelu_tanh".  Sizes or strides that 16 bytes do not divide are
    taken through padded copies.  Differentiable once in every tensor."""
    _check(x, activation, residual, weight.shape[0] if weight.dim() else 0, (("weight", weight, bias),))
    return LinearAct.apply(x, weight, bias, residual, ACTIVATIONS[activation], _grad_wanted(x, weight, bias, residual))


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
        activation: str = "gelu", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w1^T + b1) w2^T + b2 + residual: a block's MLP, operands as for ``linear_act``."""
    _check(x, activation, residual, w2.shape[0] if w2.dim() else 0, (("w1", w1, b1), ("w2", w2, b2)))
    return MLP.apply(x, w1, b1, w2, b2, residual, ACTIVATIONS[activation], _grad_wanted(x, w1, b1, w2, b2, residual))
