"""Linear products with bias, activation and residual in one kernel (bf16 or fp16), with autograd:
``linear_act`` is act(x W^T + b) + r, one layer of the blocks around the KDA recurrence; ``mlp`` the
blocks' MLP of two layers, residual included (HybridBlock, nope_gdn_mlx.py:4009-4090), whose
backward takes the activation's derivative in the epilogue of the product that feeds it.  Products
run on the tensor cores with float32 accumulation (``kda_linear_*`` in include/kda_b200.h); what is
rounded to 16 bits on the way are the results, the saved pre-activation z, the MLP's hidden
activation and the gradient at z.  Both are C++ autograd functions (csrc/tensors_module.cpp).  No
CPU path."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

ACTIVATIONS = {"none": _lib.KDA_ACT_NONE, "relu": _lib.KDA_ACT_RELU, "silu": _lib.KDA_ACT_SILU,
               "gelu": _lib.KDA_ACT_GELU, "gelu_tanh": _lib.KDA_ACT_GELU_TANH}


def _act(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual.

    x is (..., in_features), weight (out_features, in_features), bias (out_features,), residual
    (..., out_features); all bf16 or all fp16, on one device, any strides.  ``activation`` is "none",
    "relu", "silu", "gelu" (exact) or "gelu_tanh".  Sizes or strides that 16 bytes do not divide are
    taken through padded copies.  Differentiable once in every tensor, in reverse mode; forward-mode
    tangents, ``torch.func``'s transforms and tracers raise."""
    return _lib.tensors().linear_act(x, weight, bias, _act(activation), residual)


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
        activation: str = "gelu", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w1^T + b1) w2^T + b2 + residual: a block's MLP, operands as for ``linear_act``."""
    return _lib.tensors().mlp(x, w1, b1, w2, b2, _act(activation), residual)
