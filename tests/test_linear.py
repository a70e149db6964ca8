"""CPU: argument checks of the linear products."""
import ctypes

import pytest
import torch

from mlx_vit_b200 import _lib, linear


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        linear.linear_act(x, w)
    with pytest.raises(ValueError, match="no CPU path"):
        linear.mlp(x, w, None, w.t(), None)


def test_unknown_activation():
    with pytest.raises(ValueError, match="unknown activation"):
        linear.linear_act(torch.zeros(2, 16), torch.zeros(8, 16), activation="tanh")


A = 1 << 20


def fwd(**kw):
    a = dict(dtype=_lib.KDA_BF16, act=0, M=4, N=8, K=16, x=A, ldx=16, w=A, ldw=16, b=None, r=None, ldr=0, y=A, ldy=8, z=None,
             ldz=0, ws=None, nws=0, st=None)
    a.update(kw)
    return _lib.STATUS[_lib.lib().kda_linear_fwd(*a.values())]


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=_lib.KDA_F32), "DTYPE"), (dict(act=5), "INVALID_ARG"), (dict(act=-1), "INVALID_ARG"),
    (dict(M=0), "INVALID_ARG"), (dict(K=-3), "INVALID_ARG"), (dict(N=1 << 31, ldy=1 << 31), "UNSUPPORTED"),
    (dict(x=None), "INVALID_ARG"), (dict(y=None), "INVALID_ARG"), (dict(ldx=8), "INVALID_ARG"),
    (dict(ldy=7), "INVALID_ARG"), (dict(r=A, ldr=4), "INVALID_ARG"), (dict(x=A + 2), "MISALIGNED"),
    (dict(ldw=17), "MISALIGNED"), (dict(z=A, ldz=9), "MISALIGNED"), (dict(b=A + 1), "MISALIGNED"),
    (dict(y=A + 1), "MISALIGNED")])
def test_forward_refusals(kw, status):
    assert fwd(**kw) == "KDA_ERR_" + status


def test_backward_refusals():
    L, n = _lib.lib(), ctypes.c_void_p(None)
    st = lambda s: _lib.STATUS[s].replace("KDA_ERR_", "")  # noqa: E731
    bf = _lib.KDA_BF16
    assert st(L.kda_linear_dgrad(bf, 3, 4, 8, 16, A, 8, A, 16, n, 0, A, 16, n, n, 0, n)) == "INVALID_ARG"  # no z
    assert st(L.kda_linear_dgrad(bf, 0, 4, 8, 16, A, 12, A, 16, n, 0, A, 16, n, n, 0, n)) == "MISALIGNED"
    assert st(L.kda_linear_dgrad(bf, 0, 4, 8, 16, A, 8, A, 16, n, 0, A, 16, A, n, 0, n)) == "WORKSPACE"
    assert st(L.kda_linear_wgrad(bf, 4, 8, 16, A, 8, A, 16, A, 15, n, 0, n)) == "INVALID_ARG"
    assert st(L.kda_linear_wgrad(bf, 4, 8, 16, A, 8, A, 12, A, 16, n, 0, n)) == "INVALID_ARG"
    assert st(L.kda_linear_wgrad(bf, 4, 8, 16, A, 8, A + 2, 16, A, 16, n, 0, n)) == "MISALIGNED"
    for op in (_lib.KDA_LINEAR_FWD, _lib.KDA_LINEAR_DGRAD, _lib.KDA_LINEAR_WGRAD):
        assert L.kda_linear_workspace_bytes(op, 0, 8, 16, 1) == 0
        assert L.kda_linear_workspace_bytes(op, 1000, 8, 1 << 20, 1) >= 0
    assert L.kda_linear_workspace_bytes(_lib.KDA_LINEAR_DGRAD, 4, 8, 16, 1) >= 16 * 4
    assert L.kda_linear_workspace_bytes(_lib.KDA_LINEAR_ACT_GRAD, 4, 8, 1, 1) >= 8 * 4
    assert L.kda_linear_workspace_bytes(_lib.KDA_LINEAR_ACT_GRAD, 4, 8, 1, 0) == 0
    assert L.kda_linear_workspace_bytes(_lib.KDA_LINEAR_WGRAD, 12544, 2304, 768, 0) > 2304 * 768 * 4  # split
    assert L.kda_linear_workspace_bytes(7, 4, 8, 16, 1) == 0
    assert st(L.kda_act_grad(bf, 1, 4, 8, A, 8, n, 0, A, 8, n, n, 0, n)) == "INVALID_ARG"
    assert st(L.kda_act_grad(bf, 0, 4, 8, A, 8, n, 0, n, 0, n, n, 0, n)) == "INVALID_ARG"  # neither dz nor db
    assert st(L.kda_act_grad(bf, 0, 4, 8, A + 1, 8, n, 0, A, 8, n, n, 0, n)) == "MISALIGNED"
    assert st(L.kda_act_grad(bf, 0, 4, 8, A, 8, n, 0, n, 0, A, n, 0, n)) == "WORKSPACE"
