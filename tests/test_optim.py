"""CPU: the optimizer's argument checks and its 8-bit state format (restated)."""
import copy
import ctypes

import numpy as np
import pytest
import torch

from mlx_vit_b200 import _lib, optim
from optim_testutil import decode, encode, mix


def test_cpu_tensors_are_refused():
    p, g, m, v = (torch.zeros(4) for _ in range(4))
    with pytest.raises(ValueError, match="no CPU path"):
        optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="no CPU path"):
        optim.grad_norm([g])
    with pytest.raises(ValueError, match="CUDA"):
        optim.decode_state8(torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), True)
    w = torch.nn.Parameter(torch.zeros(4))
    w.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="no CPU path"):
        optim.AdamW([w]).step()


@pytest.mark.parametrize("kw", [dict(state_bits=4), dict(max_grad_norm=0.0), dict(ema_decay=1.5)])
def test_bad_options_are_refused(kw):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4))], **kw)


@pytest.mark.parametrize("kw", [dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(max_grad_norm=-1.0), dict(ema_decay=0.5)])
def test_bad_step_arguments_are_refused(kw):
    p, g, m, v = (torch.zeros(4) for _ in range(4))
    with pytest.raises(ValueError):
        optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-3, **kw)


def call(rows=(), count=None, step_dev=None, ws=None, nws=0, norm=None, **kw):
    a = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, max_grad_norm=0.0, ema_decay=0.0, step=1,
             seed=0, state_bits=32, bias_correction=1, use_ema=0, norm_given=0, reserved=0)
    a.update(kw)
    table = (ctypes.c_int64 * max(1, 9 * len(rows)))(*[x for r in rows for x in r])
    return _lib.STATUS[_lib.lib().kda_adamw_step(ctypes.byref(_lib.KdaAdamW(**a)), table,
                                                 len(rows) if count is None else count, step_dev, None, norm, ws, nws,
                                                 None)]


def test_c_entry_refuses_bad_arguments_before_any_launch():
    a = 1 << 20
    good = (a, a, a, a, 0, 0, 0, 16, _lib.KDA_F32)

    def row(**kw):
        names = ("p", "g", "m", "v", "me", "ve", "ema", "n", "dtype")
        return tuple(kw.get(n, x) for n, x in zip(names, good))

    assert _lib.STATUS[_lib.lib().kda_adamw_step(None, None, 0, None, None, None, None, 0, None)] == "KDA_ERR_INVALID_ARG"
    assert call([row(p=0)]) == "KDA_ERR_INVALID_ARG"
    assert call([row(g=0)]) == "KDA_ERR_INVALID_ARG"
    assert call([row(n=-1)]) == "KDA_ERR_INVALID_ARG"
    assert call([row(dtype=9)]) == "KDA_ERR_DTYPE"
    assert call([row(m=a + 2)]) == "KDA_ERR_MISALIGNED"
    assert call([row(g=a + 1)]) == "KDA_ERR_MISALIGNED"
    assert call([row()], state_bits=16) == "KDA_ERR_UNSUPPORTED"
    assert call([row()], state_bits=8) == "KDA_ERR_INVALID_ARG"  # no exponent bytes
    assert call([row()], use_ema=1) == "KDA_ERR_INVALID_ARG"
    assert call([row()], step=0) == "KDA_ERR_INVALID_ARG"
    assert call([row()], beta2=1.0) == "KDA_ERR_INVALID_ARG"
    assert call([row()], eps=float("nan")) == "KDA_ERR_INVALID_ARG"
    assert call([row()], lr=float("inf")) == "KDA_ERR_INVALID_ARG"
    assert call([row()], count=-1) == "KDA_ERR_INVALID_ARG"
    assert call([row()], max_grad_norm=1.0, norm_given=1) == "KDA_ERR_INVALID_ARG"
    assert call([]) == "KDA_OK"
    L = _lib.lib()
    assert _lib.STATUS[L.kda_decode_state8(4, 1, None, None, None, None)] == "KDA_ERR_INVALID_ARG"
    assert L.kda_decode_state8(0, 1, None, None, None, None) == 0
    assert L.kda_adamw_workspace_bytes(0) == 0 and L.kda_adamw_workspace_bytes(1) > 256


@pytest.mark.parametrize("low,signed", [(15, True), (31, False)])
def test_format_round_trip_and_bracket(low, signed):
    """Every value a code stands for is kept by any random bits, and a rounded value is one of its
    two neighbours: at most one eighth of its binade away."""
    rng = np.random.default_rng(low)
    code = np.arange(256, dtype=np.uint8)
    code = code[(code & (127 if signed else 255)) <= 8 * low - 1]
    code = np.concatenate([code, np.zeros(256 - code.size, np.uint8)])
    exp = np.array([130], np.uint8)
    x = decode(code, exp, low, signed)
    c2, e2 = encode(x.astype(np.float32), rng.integers(0, 65536, 256), low, signed)
    assert e2[0] == 130 and np.array_equal(decode(c2, e2, low, signed), x)
    y = (rng.standard_normal(4096) * np.exp2(rng.uniform(-12, 0, 4096))).astype(np.float32)
    y = y if signed else np.abs(y)
    c, e = encode(y, rng.integers(0, 65536, 4096), low, signed)
    d = decode(c, e, low, signed)
    assert (np.abs(d - y) <= np.maximum(np.abs(y) / 8, 1.125 * np.exp2(np.repeat(e, 256) - 127.0 - low))).all()


def test_hash_spreads():
    h = mix(np.arange(1 << 16, dtype=np.uint64))
    assert len(set(h.tolist())) == 1 << 16
    assert abs((h & np.uint64(0xFFFF)).mean() / 65535 - 0.5) < 0.01


def torch_states(opt, *ps, **kw):
    """The state dict of a torch optimizer after one step over parameters like these."""
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for q in qs:
        q.grad = torch.ones_like(q)
    old = opt(qs, **kw)
    old.step()
    return old.state_dict()


@pytest.mark.parametrize("opt,kw,name", [(torch.optim.AdamW, dict(maximize=True), "maximize"),
                                         (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
                                         (torch.optim.Adam, dict(weight_decay=0.1), "decoupled")])
def test_states_of_another_rule_are_refused(opt, kw, name):
    """What a loaded group asks for and the step does not do; nothing is loaded."""
    p = torch.nn.Parameter(torch.randn(6))
    new = optim.AdamW([p], lr=0.5)
    with pytest.raises(ValueError, match=name):
        new.load_state_dict(torch_states(opt, p, **kw))
    assert not new.state and new.param_groups[0]["lr"] == 0.5
    new.load_state_dict(torch_states(torch.optim.AdamW, p, lr=0.25))
    new.load_state_dict(torch_states(torch.optim.Adam, p, lr=0.25))  # without decay the two are one rule
    assert new.state[p]["step"] == 1 and new.param_groups[0]["lr"] == 0.25


def test_a_loaded_state_without_a_shadow_starts_one():
    """The shadow starts at the parameter's next step, from what the parameter is then."""
    p = torch.nn.Parameter(torch.randn(6))
    new = optim.AdamW([p], ema_decay=0.9)
    new.load_state_dict(torch_states(torch.optim.AdamW, p))
    p.data.fill_(2.0)  # a model's weights may be loaded after its optimizer's states
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="no CPU path"):
        new.step()
    assert (new.ema_of(p) == 2).all() and new.state[p]["step"] == 1 and (new.state[p]["exp_avg"] != 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_loaded_states_are_float32(dtype):
    """torch holds a 16-bit parameter's states in 16 bits, those of biases and norms, of one dimension, too."""
    ps = [torch.nn.Parameter(torch.randn(s).to(dtype)) for s in ((6,), (3, 4), (), (2, 1, 5))]
    states = torch_states(torch.optim.AdamW, *ps)
    assert states["state"][0]["exp_avg"].dtype == dtype
    new = optim.AdamW(ps)
    new.load_state_dict(states)
    for i, p in enumerate(ps):
        for name in ("exp_avg", "exp_avg_sq"):
            held = new.state[p][name]
            assert held.dtype == torch.float32 and held.shape == (p.numel(),)
            assert torch.equal(held, states["state"][i][name].float().reshape(-1))
    again = optim.AdamW(ps)
    again.load_state_dict(new.state_dict())
    assert all(torch.equal(again.state[p][n], new.state[p][n]) for p in ps for n in ("exp_avg", "exp_avg_sq"))


def test_capturable_refuses_states_of_several_steps():
    """A capturable group has one step number: parameters that have taken 1 and 2 steps would be corrected by one."""
    a, b = (torch.nn.Parameter(torch.randn(6)) for _ in range(2))
    old = torch.optim.AdamW([a, b])
    a.grad = torch.ones_like(a)
    old.step()
    b.grad = torch.ones_like(b)
    old.step()
    new = optim.AdamW([a, b], capturable=True)
    with pytest.raises(ValueError, match="step"):
        new.load_state_dict(old.state_dict())
    assert not new.state
    plain = optim.AdamW([a, b])
    plain.load_state_dict(old.state_dict())
    assert [plain.state[p]["step"] for p in (a, b)] == [2, 1]
    apart = optim.AdamW([dict(params=[a]), dict(params=[b])], capturable=True)
    states = old.state_dict()
    g = states["param_groups"][0]
    states["param_groups"] = [dict(g, params=[0]), dict(g, params=[1])]
    apart.load_state_dict(states)
    assert [int(g["step"]) for g in apart.param_groups] == [2, 1]


@pytest.mark.parametrize("swap", [False, True])
def test_states_follow_the_parameter_s_layout(swap):
    """States lie in their parameter's order in memory: loaded into a parameter laid out otherwise, float32 ones are
    reordered and 8-bit ones, whose blocks are of that order, refused."""
    a, b = (torch.nn.Parameter(torch.randn(2, 3, 4, 5).to(memory_format=f))
            for f in (torch.contiguous_format, torch.channels_last)[::-1 if swap else 1])
    g = torch.randn(2, 3, 4, 5)
    old = torch.optim.AdamW([a])
    a.grad = g.clone()
    old.step()
    one, two, same = optim.AdamW([a], ema_decay=0.5), optim.AdamW([b], ema_decay=0.5), optim.AdamW([a], ema_decay=0.5)
    one.load_state_dict(old.state_dict())
    one._init_state(a)
    states = copy.deepcopy(one.state_dict())
    two.load_state_dict(states)
    same.load_state_dict(states)
    for name, want in (("exp_avg", old.state[a]["exp_avg"]), ("exp_avg_sq", old.state[a]["exp_avg_sq"]), ("ema", a.detach())):
        for o, p in ((one, a), (two, b), (same, a)):
            held = o.state[p][name]
            assert held.shape == (120,) and torch.equal(held.as_strided(p.shape, p.stride()), want)
    assert torch.equal(two.ema_of(b), a.detach())
    for st in states["state"].values():  # states from before the layout was kept: the parameter's own
        del st["stride"]
    two.load_state_dict(states)
    assert torch.equal(two.state[b]["exp_avg"], one.state[a]["exp_avg"])
    codes = optim.AdamW([a], state_bits=8)
    codes._init_state(a)
    optim.AdamW([a], state_bits=8).load_state_dict(codes.state_dict())
    with pytest.raises(ValueError, match="memory"):
        optim.AdamW([b], state_bits=8).load_state_dict(codes.state_dict())


def test_layouts_that_differ_in_name_only():
    """Strides of dimensions of one element say nothing."""
    a = torch.nn.Parameter(torch.randn(4, 1, 3))
    b = torch.nn.Parameter(a.detach().as_strided((4, 1, 3), (3, 7, 1)))
    codes = optim.AdamW([a], state_bits=8)
    codes._init_state(a)
    optim.AdamW([b], state_bits=8).load_state_dict(codes.state_dict())


def test_c_entries_refuse_misaligned_scalars():
    a = 1 << 20
    row = (a, a, a, a, 0, 0, 0, 16, _lib.KDA_F32)
    L = _lib.lib()

    def status(step=None, lr=None, norm=None):
        args = _lib.KdaAdamW(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_grad_norm=1.0, step=1, state_bits=32)
        return _lib.STATUS[L.kda_adamw_step(ctypes.byref(args), (ctypes.c_int64 * 9)(*row), 1, step, lr, norm, a, 1 << 20, None)]

    assert status(step=a + 4) == "KDA_ERR_MISALIGNED"
    assert status(lr=a + 2) == "KDA_ERR_MISALIGNED"
    assert status(norm=a + 2) == "KDA_ERR_MISALIGNED"
