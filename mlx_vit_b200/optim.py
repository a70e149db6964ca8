"""AdamW over a model's tensors in one kernel launch, with float32 or 8-bit states.

``AdamW`` is a ``torch.optim.Optimizer`` for the training step around the KDA layers; the
reference trainers' optimizer, gradient clipping and shadow average (train_mlx_k400.py:176-222,
:379-408) are one pass here:

    g   <- g min(1, max_grad_norm / (||g|| + 1e-6))
    m   <- beta1 m + (1 - beta1) g
    v   <- beta2 v + (1 - beta2) g^2
    p   <- p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
    ema <- ema_decay ema + (1 - ema_decay) p

``adamw_step`` is the same step on lists of tensors, ``grad_norm`` the global gradient norm alone.
All launches go on the current torch CUDA stream; there is no CPU path.

With ``state_bits=8`` m and v are held as one byte an element plus one exponent byte per
``STATE_BLOCK`` consecutive elements: e is float32's exponent field of the block's largest
magnitude plus one, and a code's magnitude 8 k + f stands for (1 + f / 8) 2^(k - L + e - 127),
zero for zero; m has a sign in bit 7 and L = 15, v has L = 31.  Values are rounded to their three
bits of mantissa stochastically (to nearest, v could never decay by beta2 = 0.999 a step), by bits
that a hash of (seed, step, the tensor's number in the step, element) gives: the same call gives the
same states.  Magnitudes below the least code become it or zero for m, unbiased, and the least code
for v.  A block that holds a value that is not finite reads back as NaN.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib

STATE_BLOCK = 256

State8 = Tuple[torch.Tensor, torch.Tensor]


def zeros_state8(p: torch.Tensor) -> State8:
    """The zero 8-bit state of a tensor: (codes, exponents)."""
    n = p.numel()
    return (torch.zeros(n, dtype=torch.uint8, device=p.device),
            torch.zeros(-(-n // STATE_BLOCK), dtype=torch.uint8, device=p.device))


def decode_state8(codes: torch.Tensor, exps: torch.Tensor, signed: bool) -> torch.Tensor:
    """The values of an 8-bit state as bf16, which holds them exactly, in the codes' shape."""
    _need(codes.is_cuda and exps.is_cuda and codes.device == exps.device, "an 8-bit state lies on one CUDA device")
    _need(codes.dtype == torch.uint8 and exps.dtype == torch.uint8, "codes and exponents are uint8")
    _need(codes.is_contiguous() and exps.is_contiguous(), "codes and exponents must be contiguous")
    n = codes.numel()
    _need(exps.numel() == -(-n // STATE_BLOCK), f"{n} codes take {-(-n // STATE_BLOCK)} exponents, got {exps.numel()}")
    out = torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device)
    with torch.cuda.device(codes.device):
        _lib.check(_lib.lib().kda_decode_state8(n, int(signed), codes.data_ptr(), exps.data_ptr(), out.data_ptr(),
                                                torch.cuda.current_stream().cuda_stream), "kda_decode_state8")
    return out


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _same_order(p, stride):
    """Whether a dense tensor of p's shape with these strides lies in memory as p does."""
    return all(a == b for a, b, n in zip(p.stride(), stride, p.shape) if n > 1)


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all gradients together, a float32 scalar on their device (sums in 64 bits)."""
    return _lib.tensors().grad_norm(list(grads))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[Union[torch.Tensor, State8]], exp_avg_sqs: Sequence[Union[torch.Tensor, State8]], *,
               step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor], betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, bias_correction: bool = True, max_grad_norm: Optional[float] = None,
               emas: Optional[Sequence[torch.Tensor]] = None, ema_decay: Optional[float] = None, seed: int = 0,
               norm: Optional[torch.Tensor] = None, first_tensor: int = 0) -> Optional[torch.Tensor]:
    """One AdamW step over lists of CUDA tensors, in place.

    ``params`` and ``grads`` are float32, bfloat16 or float16, dense in memory and each pair laid
    out alike.  The states are contiguous float32 tensors, or (codes, exponents) pairs
    (``zeros_state8``) for 8 bits, in the parameter's order in memory.  ``step`` is this
    step's number from 1, or an int64 CUDA scalar that the call advances; ``lr`` a number or a
    float32 CUDA scalar.  A captured graph needs both as tensors: numbers would be frozen in it.
    With ``max_grad_norm`` the gradients are scaled as they are read (``grads`` keep their values)
    by their global norm, or by ``norm``, a float32 CUDA scalar, where that is given.  ``emas``
    (float32) follow the parameters with ``ema_decay``.  Tensors must not overlap one another.
    ``first_tensor`` numbers the lists' first tensor where several calls make one step, so that 8-bit
    states in different calls are rounded by different bits.
    Returns the gradients' norm (float32 scalar) with ``max_grad_norm``, else None.
    """
    _need((emas is None) == (ema_decay is None), "emas and ema_decay go together")
    _need(max_grad_norm is None or max_grad_norm > 0.0, "max_grad_norm must be positive")
    _need(0 <= first_tensor < 1 << 31, "first_tensor counts from 0")
    return _lib.tensors().adamw_step(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs),
                                     None if emas is None else list(emas), step, lr, betas[0], betas[1], eps, weight_decay,
                                     bias_correction, max_grad_norm or 0.0, ema_decay or 0.0, seed & 0xFFFFFFFF, norm,
                                     first_tensor)


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with every tensor of a group updated by one launch.

    ``state_bits`` 32 or 8; ``max_grad_norm`` clips the global norm over all groups (the last
    step's norm is ``self.grad_norm``); ``ema_decay`` keeps a float32 shadow of every parameter
    (``ema_of``), started at the parameter's first step, or the first after states without a shadow
    were loaded.  ``capturable`` keeps the step's number and the learning rate on the device, so that
    ``step`` can be captured into a CUDA graph after one eager step; the parameters of a group then
    share one step number and all need gradients, and ``lr`` is the tensor ``group["lr"]`` (fill it
    to change it).
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 bias_correction: bool = True, state_bits: int = 32, max_grad_norm: Optional[float] = None,
                 ema_decay: Optional[float] = None, seed: int = 0, capturable: bool = False):
        _need(state_bits in (8, 32), f"state_bits must be 8 or 32, got {state_bits}")
        _need(max_grad_norm is None or max_grad_norm > 0.0, f"max_grad_norm must be positive, got {max_grad_norm}")
        _need(ema_decay is None or 0.0 <= ema_decay <= 1.0, f"ema_decay must lie in [0, 1], got {ema_decay}")
        self.state_bits, self.max_grad_norm, self.ema_decay = state_bits, max_grad_norm, ema_decay
        self.seed, self.capturable = int(seed), bool(capturable)
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      bias_correction=bias_correction))

    def __getstate__(self):
        names = ("state_bits", "max_grad_norm", "ema_decay", "seed", "capturable", "grad_norm")
        return {**super().__getstate__(), **{n: getattr(self, n) for n in names}}

    def ema_of(self, p: torch.Tensor) -> torch.Tensor:
        """The shadow average of a parameter, in its shape (float32)."""
        return self.state[p]["ema"].as_strided(p.shape, p.stride())

    def _init_state(self, p):
        """The state of a parameter that has none, and the shadow of one whose loaded state has none."""
        st = self.state[p]
        if not st:
            st["stride"] = tuple(p.stride())  # the order in memory that the states lie in
            if not self.capturable:
                st["step"] = 0
            for name in ("exp_avg", "exp_avg_sq"):
                if self.state_bits == 8:
                    st[name], st[name + "_exp"] = zeros_state8(p)
                else:
                    st[name] = torch.zeros(p.numel(), dtype=torch.float32, device=p.device)
        if self.ema_decay is not None:  # in the parameter's order in memory, as every state
            st["ema"] = p.detach().as_strided((p.numel(),), (1,)).float().clone()
        return st

    def _states(self, ps, name):
        if self.state_bits == 8:
            return [(self.state[p][name], self.state[p][name + "_exp"]) for p in ps]
        return [self.state[p][name] for p in ps]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        shadow = self.ema_decay is not None
        calls = []  # (group, parameters, gradients in memory order, step number)
        for group in self.param_groups:
            live = [p for p in group["params"] if p.grad is not None]
            if not live:
                continue
            capturing = live[0].is_cuda and torch.cuda.is_current_stream_capturing()
            if capturing and not self.capturable:
                raise ValueError("AdamW: a step is captured into a graph with capturable=True only")
            for p in live:
                st = self.state[p]
                if not st or (shadow and "ema" not in st):
                    if capturing:
                        raise ValueError("AdamW: take one step before a step is captured into a graph")
                    self._init_state(p)
            grads = [p.grad for p in live]
            for i in _lib.tensors().unlike(live, grads):
                grads[i] = torch.empty_like(live[i]).copy_(grads[i])
            if self.capturable:
                _need(len(live) == len(group["params"]), "a capturable AdamW needs every parameter's gradient")
                dev = live[0].device
                for name, dt in (("step", torch.int64), ("lr", torch.float32)):
                    t = group.get(name, 0)
                    if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != dt:
                        if capturing:
                            raise ValueError("AdamW: take one step before a step is captured into a graph")
                        group[name] = torch.as_tensor(t, dtype=dt, device=dev).clone()
                calls.append((group, live, grads, group["step"]))
            else:
                by_step = {}
                for p, g in zip(live, grads):
                    at = by_step.setdefault(self.state[p]["step"] + 1, ([], []))
                    at[0].append(p)
                    at[1].append(g)
                calls += [(group, ps, gs, n) for n, (ps, gs) in by_step.items()]
        norm = None
        if self.max_grad_norm is not None and len(calls) > 1:
            norm = grad_norm([g for c in calls for g in c[2]])
        first = 0  # tensors of the calls before
        for group, ps, gs, n in calls:
            out = adamw_step(ps, gs, self._states(ps, "exp_avg"),
                             self._states(ps, "exp_avg_sq"), step=n,
                             lr=group["lr"] if self.capturable else float(group["lr"]), betas=group["betas"],
                             eps=group["eps"], weight_decay=group["weight_decay"],
                             bias_correction=group["bias_correction"], max_grad_norm=self.max_grad_norm,
                             emas=None if self.ema_decay is None else [self.state[p]["ema"] for p in ps],
                             ema_decay=self.ema_decay, seed=self.seed, norm=norm, first_tensor=first)
            self.grad_norm = out
            first += len(ps)
            if not self.capturable:
                for p in ps:
                    self.state[p]["step"] = n
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but the states are not cast to the parameters' dtypes.  The states of a
        ``torch.optim.AdamW`` can be loaded into one of 32 bits (in float32, whatever they were), unless
        its groups ask for another rule than this one's (``maximize``, ``amsgrad``, decay that is not
        decoupled).  A capturable group takes states of one step number only.  States lie in their
        parameter's order in memory: float32 ones are reordered for a parameter that lies otherwise,
        8-bit ones refused."""
        for g in state_dict["param_groups"]:
            for name in ("maximize", "amsgrad"):
                _need(not g.get(name), f"the loaded states are of an optimizer with {name}, which this one has not")
            _need(g.get("decoupled_weight_decay", True) or not g.get("weight_decay"),
                  "the loaded states are of an optimizer whose weight decay is not decoupled")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            held = state_dict["state"].get(i)
            _need(not held or ("exp_avg_exp" in held) == (self.state_bits == 8),
                  f"the loaded states are not those of an optimizer with state_bits={self.state_bits}")
            _need(self.state_bits == 32 or not held or _same_order(p, held.get("stride", p.stride())),
                  "8-bit states cannot be loaded into a parameter that lies otherwise in memory than theirs")
        for g in state_dict["param_groups"] if self.capturable else ():
            steps = {int(state_dict["state"][i]["step"]) for i in g["params"] if "step" in state_dict["state"].get(i, ())}
            _need(len(steps) <= 1 or "step" in g, "the parameters of a capturable group have one step number, those loaded "
                  f"have {len(steps)}: {sorted(steps)}")
        super().load_state_dict(state_dict)
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            if i in state_dict["state"]:
                held = state_dict["state"][i]
                self.state[p] = {k: self._own(k, v, p, held.get("stride", p.stride())) for k, v in held.items()}
                if held:
                    self.state[p]["stride"] = tuple(p.stride())
        for group in self.param_groups:
            for name, value in self.defaults.items():
                group.setdefault(name, value)
            held = [self.state[p] for p in group["params"] if self.state[p]]
            # the step's number: a group's where it is capturable, else a parameter's
            if self.capturable:
                steps = [st.pop("step") for st in held if "step" in st]
                if "step" not in group and steps:
                    group["step"] = steps[0]
            elif "step" in group:
                n = int(group.pop("step"))
                group["lr"] = float(group["lr"])
                for st in held:
                    st["step"] = n

    def _own(self, name, v, p, stride):
        """A loaded state entry as this optimizer holds it: tensors flat, in the parameter's order in memory
        (``stride``: the order of those that came flat), codes and exponents as they are, others in float32."""
        if name == "step":
            return int(v)
        if not isinstance(v, torch.Tensor):
            return v
        if v.dtype == torch.uint8:
            return v.to(p.device, copy=True)
        if v.dim() != 1 and v.shape == p.shape:
            return torch.empty_like(p, dtype=torch.float32).copy_(v).as_strided((p.numel(),), (1,))
        if v.shape == (p.numel(),) and not _same_order(p, stride):
            return self._own(name, v.as_strided(p.shape, stride), p, stride)
        return v.to(p.device, torch.float32, copy=True)
