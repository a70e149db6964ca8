"""GPU: the AdamW step against its formulas in 64 bits and, for the 8-bit states, code by code
against a restatement of the format."""
import copy
import ctypes

import numpy as np
import pytest
import torch

from mlx_vit_b200 import _lib, optim
from optim_testutil import BLOCK, adamw64, decode, encode, moments32, random_bits

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}  # half a step, relative
TINY = {"fp32": 0.0, "bf16": 0.0, "fp16": 2.0 ** -25}  # half the least subnormal
SIZES = [(1,), (255,), (16, 16), (257,), (2047,), (2048,), (2049,), (3, 5, 7), (0,), (70, 131)]
HYP = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def np64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def make(cuda, dtype, bits, sizes=SIZES, seed=0, offset=0):
    """Lists of tensors; with ``offset`` every one starts that many elements into its storage."""
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)

    def tensor(s, dt, scale):
        n = int(np.prod(s))
        t = torch.empty(n + offset, dtype=dt, device=cuda)[offset:].view(s)
        return t.copy_(torch.randn(s, generator=g, device=cuda) * scale)

    p = [tensor(s, DT[dtype], 0.5) for s in sizes]
    gr = [tensor(s, DT[dtype], 10.0 ** (-i % 4)) for i, s in enumerate(sizes)]
    m, v = [], []
    for s in sizes:
        n = int(np.prod(s))
        a = (torch.randn(n, generator=g, device=cuda) * 0.1).cpu().numpy().astype(np.float32)
        b = (a * a * 1.5 + 1e-4).astype(np.float32)
        if bits == 8:
            half = np.full(n, 1 << 15)
            for x, low, signed, out in ((a, 15, True, m), (b, 31, False, v)):
                c, e = encode(x, half, low, signed)
                code = torch.empty(n + offset, dtype=torch.uint8, device=cuda)[offset:]
                out.append((code.copy_(torch.from_numpy(c)), torch.from_numpy(e).to(cuda)))
        else:
            m.append(tensor(s, torch.float32, 0).copy_(torch.from_numpy(a).view(s)))
            v.append(tensor(s, torch.float32, 0).copy_(torch.from_numpy(b).view(s)))
    return p, gr, m, v


def values(state, signed):
    """A state tensor's float64 values."""
    if isinstance(state, tuple):
        return decode(state[0].cpu().numpy(), state[1].cpu().numpy(), 15 if signed else 31, signed)
    return np64(state)


def check_step(p, g, m, v, run, dtype, bits, step, seed=0, coef=1.0, emas=None, ema_decay=None):
    """Runs a step and compares all it wrote.  m, v: equal to the separately rounded float32
    operations (or their codes).  p, with u = 2^-24: the update's m errs by 4 u (|b1 m| + |(1-b1) g|)
    (constants, products, the coefficient, the sum), the root of v by 3 u and 2 u of its own, the
    constants, products and the sum around it by 5 u, the quotient by 4 u and c1 m by 2 u: 20 u of
    the update with both parts of m counted positive; then 2 u of p (1 - lr wd), 1 u of the sum, and
    half a step of the stored type."""
    hyp = dict(lr=HYP["lr"], b1=0.9, b2=0.999, eps=HYP["eps"], wd=HYP["weight_decay"])
    before = [(np64(a), np64(b), values(c, True), values(d, False)) for a, b, c, d in zip(p, g, m, v)]
    held = None if emas is None else [np64(e) for e in emas]
    run()
    for i, (p0, g0, m0, v0) in enumerate(before):
        m32, v32 = moments32(g0, m0, v0, 0.9, 0.999, coef)
        pe, _, _ = adamw64(p0, g0, m0, v0, step, coef=coef, **hyp)
        if bits == 8:
            r = random_bits(seed, step, i, p0.size)
            for state, x, low, signed, r16 in ((m[i], m32, 15, True, r & np.uint64(0xFFFF)),
                                               (v[i], v32, 31, False, r >> np.uint64(16))):
                code, exp = encode(x, r16, low, signed)
                assert np.array_equal(state[1].cpu().numpy(), exp), i
                assert np.array_equal(state[0].cpu().numpy(), code), i
        else:
            assert np.array_equal(m[i].cpu().numpy().reshape(-1), m32), i
            assert np.array_equal(v[i].cpu().numpy().reshape(-1), v32), i
        pa, _, _ = adamw64(0 * p0, np.abs(g0), np.abs(m0), v0, step, coef=coef, **hyp)
        got, upd = np64(p[i]), np.abs(pa)
        tol = 20 * 2.0 ** -24 * upd + 2 * 2.0 ** -24 * (np.abs(p0) + np.abs(pe)) + HALF[dtype] * np.abs(pe) * 1.01
        assert (np.abs(got - pe) <= tol + TINY[dtype]).all(), (i, np.abs(got - pe).max())
        if emas is not None:  # of the parameter as stored; three float32 roundings
            want = ema_decay * held[i] + (1 - ema_decay) * got
            assert (np.abs(np64(emas[i]) - want) <= 4 * 2.0 ** -24 * (np.abs(held[i]) + np.abs(got))).all(), i


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_step_matches_the_formulas(cuda, dtype, bits, offset):
    p, g, m, v = make(cuda, dtype, bits, offset=offset)
    emas = [x.float() + 0.01 for x in p] if bits == 32 or offset else None
    for step in (1, 2, 1000):
        def run():
            out = optim.adamw_step(p, g, m, v, step=step, seed=7, emas=emas, ema_decay=None if emas is None else 0.99,
                                   **HYP)
            assert out is None
        check_step(p, g, m, v, run, dtype, bits, step, 7, emas=emas, ema_decay=0.99)


@pytest.mark.parametrize("bits", [8, 32])
def test_large_tensor_of_many_binades(cuda, bits):
    """Millions of elements that differ by many binades: values below the least code, and one rounding
    too few in m or v would show in some codes of a million."""
    n, gen = 6_000_000, torch.Generator(device=cuda).manual_seed(17)
    spread = torch.exp2(torch.randn(n, generator=gen, device=cuda) * 2)
    p, g = torch.randn(n, generator=gen, device=cuda), torch.randn(n, generator=gen, device=cuda) * spread
    if bits == 8:
        m, v = optim.zeros_state8(p), optim.zeros_state8(p)
    else:
        m, v = torch.zeros_like(p), torch.zeros_like(p)
    for step in (1, 2, 3):
        g = g * torch.randn(n, generator=gen, device=cuda)
        check_step([p], [g], [m], [v], lambda: optim.adamw_step([p], [g], [m], [v], step=step, seed=9, **HYP), "fp32", bits,
                   step, 9)


@pytest.mark.parametrize("count", [1, 64, 65, 449, 1000])
def test_tables_of_many_tensors(cuda, count):
    """More tensors than a launch holds; the hash goes by the index in the whole list."""
    sizes = [(1 + (37 * i) % 700,) for i in range(count)]
    p, g, m, v = make(cuda, "fp32", 8, sizes)
    check_step(p, g, m, v, lambda: optim.adamw_step(p, g, m, v, step=3, seed=1, **HYP), "fp32", 8, 3, 1)


@pytest.mark.parametrize("dtype,bits,limit", [("fp32", 32, 0.5), ("bf16", 8, 0.5), ("fp16", 32, 1e6)])
def test_clipping(cuda, dtype, bits, limit):
    p, g, m, v = make(cuda, dtype, bits)
    norm = np.sqrt(sum((np64(x) ** 2).sum() for x in g))
    coef = np.float32(min(1.0, limit / (norm + 1e-6)))
    got = []
    check_step(p, g, m, v, lambda: got.append(optim.adamw_step(p, g, m, v, step=2, max_grad_norm=limit, **HYP)), dtype,
               bits, 2, coef=coef)
    # one rounding to float32, and sums in 64 bits
    assert abs(float(got[0]) - norm) <= 1.01 * 2.0 ** -24 * norm
    assert float(optim.grad_norm(g)) == float(got[0])


def test_no_bias_correction_and_given_norm(cuda):
    p, g, m, v = make(cuda, "fp32", 32, [(300,)])
    q, m2, v2 = p[0].clone(), m[0].clone(), v[0].clone()
    optim.adamw_step(p, g, m, v, step=5, bias_correction=False, max_grad_norm=1.0,
                     norm=torch.tensor(4.0, device=cuda), **HYP)
    want, _, _ = adamw64(np64(q), np64(g[0]), np64(m2), np64(v2), 5, 3e-3, 0.9, 0.999, 1e-8, 0.1, bias=False,
                         coef=np.float32(1 / (4 + 1e-6)))
    assert np.allclose(np64(p[0]), want, rtol=0, atol=8 * 2.0 ** -23 * np.abs(want).max())


def test_codes_stay_inside_their_tensors(cuda):
    """Bytes before and behind every tensor keep their values."""
    n = 1000
    for off in (8, 3):
        buf = {k: torch.full((n + 64,), 77, dtype=d, device=cuda) for k, d in
               (("p", torch.bfloat16), ("m", torch.uint8), ("v", torch.uint8))}
        ex = {k: torch.full((4 + 2,), 99, dtype=torch.uint8, device=cuda) for k in "mv"}
        cut = {k: b[off:off + n] for k, b in buf.items()}
        for k in "mv":
            cut[k].zero_()
            ex[k][1:5] = 0
        g = torch.randn(n, device=cuda).to(torch.bfloat16)
        optim.adamw_step([cut["p"]], [g], [(cut["m"], ex["m"][1:5])], [(cut["v"], ex["v"][1:5])], step=1, **HYP)
        for b in buf.values():
            assert (b[:off] == 77).all() and (b[off + n:] == 77).all()
        for e in ex.values():
            assert e[0] == 99 and e[5] == 99


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 1e30])
def test_values_that_are_not_finite(cuda, bad):
    """m follows g, v its square (1e30 squared is infinite); an 8-bit block with such a value reads
    back as NaN, the other blocks are as without it."""
    n, at = 1024, 300
    g = torch.randn(n, device=cuda)
    g[at] = bad
    for bits in (32, 8):
        p = torch.randn(n, device=cuda)
        if bits == 8:
            m, v = optim.zeros_state8(p), optim.zeros_state8(p)
        else:
            m, v = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
        p0 = p.clone()
        optim.adamw_step([p], [g], [m], [v], step=1, **HYP)
        fine = torch.ones(n, dtype=torch.bool, device=cuda)
        fine[at] = False
        assert torch.isfinite(p[fine]).all()
        if bad == 1e30:  # m finite over an infinite root: no step but the decay
            assert abs(float(p[at]) - float(p0[at]) * (1 - 3e-4)) <= 2.0 ** -22 * abs(float(p0[at]))
        else:
            assert torch.isnan(p[at])
        if bits == 8:
            block = torch.zeros(n, dtype=torch.bool, device=cuda)
            block[256:512] = True
            vv = optim.decode_state8(*v, signed=False)
            assert torch.isnan(vv[block]).all() and (vv[~block] > 0).all()
            mm = optim.decode_state8(*m, signed=True)
            assert torch.isfinite(mm[~block]).all()
            assert torch.isnan(mm[block]).all() == (bad != 1e30)
        else:
            assert torch.isfinite(m[fine]).all() and torch.isfinite(v[fine]).all()
            assert not torch.isfinite(v[at])


def test_zero_and_subnormal_gradients(cuda):
    """Zero blocks keep zero states; magnitudes under 2^-126 count as zero in 8 bits."""
    n = 600
    p = torch.ones(n, device=cuda)
    g = torch.zeros(n, device=cuda)
    g[300] = 1e-25  # its square is zero, m = 1e-26
    m, v = optim.zeros_state8(p), optim.zeros_state8(p)
    optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-3, weight_decay=0.0)
    mm, vv = optim.decode_state8(*m, signed=True).float(), optim.decode_state8(*v, signed=False).float()
    assert (vv == 0).all() and mm.nonzero().flatten().tolist() == [300]
    assert abs(float(mm[300]) - 1e-26) <= 1e-26 / 8
    assert (p[:300] == 1).all() and (p[301:] == 1).all() and torch.isfinite(p).all()


@pytest.mark.parametrize("signed", [True, False])
def test_decoding_every_code(cuda, signed):
    exp = torch.tensor([0, 1, 40, 127, 254, 255], dtype=torch.uint8, device=cuda)
    code = torch.arange(256, dtype=torch.uint8, device=cuda).repeat(6)[:-5].contiguous()
    got = optim.decode_state8(code, exp, signed).double().cpu().numpy()
    low = 15 if signed else 31
    want = decode(code.cpu().numpy(), exp.cpu().numpy(), low, signed)
    # codes that the encoder gives: a magnitude of at least 2^-126 and below 2^128
    a = np.abs(want)
    ok = np.isnan(want) | (want == 0) | ((a >= 2.0 ** -126) & (a < 2.0 ** 128))
    assert ok.mean() > 0.5 and np.array_equal(got[ok], want[ok], equal_nan=True)


def test_rounding_is_unbiased_and_v_decays(cuda):
    """With no gradient v has to fall by beta2 a step: 400 steps of rounding to nearest with three
    bits would leave it where it was.  The mean over n elements deviates by at most five of its
    standard deviations: a step rounds with a deviation of at most 1/16 of a value, relatively."""
    n, steps = 1 << 16, 400
    p, g = torch.zeros(n, device=cuda), torch.randn(n, device=cuda).abs() + 0.5
    m, v = optim.zeros_state8(p), optim.zeros_state8(p)
    optim.adamw_step([p], [g], [m], [v], step=1, lr=0.0)
    first = optim.decode_state8(*v, signed=False).double().mean()
    zero = torch.zeros_like(g)
    for t in range(2, steps + 2):
        optim.adamw_step([p], [zero], [m], [v], step=t, lr=0.0)
    left = float(optim.decode_state8(*v, signed=False).double().mean() / first)
    want = 0.999 ** steps
    assert abs(left - want) <= 5 * (steps ** 0.5 / 16) * 3 / n ** 0.5, (left, want)


def test_runs_are_equal_and_seeds_differ(cuda):
    outs = []
    for seed in (1, 1, 2):
        p, g, m, v = make(cuda, "bf16", 8)
        for t in (1, 2, 3):
            optim.adamw_step(p, g, m, v, step=t, max_grad_norm=0.3, seed=seed, **HYP)
        outs.append([x.clone() for x in p] + [c.clone() for c, _ in m] + [c.clone() for c, _ in v])
    assert all(torch.equal(a, b) for a, b in zip(outs[0], outs[1]))
    assert not all(torch.equal(a, b) for a, b in zip(outs[0], outs[2]))


def test_refusals(cuda):
    p, g, m, v = (torch.zeros(8, 4, device=cuda) for _ in range(4))
    ok = dict(step=1, lr=1e-3)
    for bad in ([[p], [g.t().contiguous()], [m], [v]], [[p], [g.bfloat16()], [m], [v]], [[p], [g], [m.bfloat16()], [v]],
                [[p], [g], [m[:4]], [v]], [[p[:, :2]], [g[:, :2]], [m[:, :2]], [v[:, :2]]], [[p.t()], [g.t().contiguous()], [m], [v]], [[p, p], [g, g], [m, m], [v, v]],
                [[p], [g], [m], [m]], [[p], [g, g], [m], [v]], [[p.double()], [g.double()], [m], [v]],
                [[p], [g], [optim.zeros_state8(p)], [v]], [[p], [g.cpu()], [m], [v]], [[], [], [], []]):
        with pytest.raises(ValueError):
            optim.adamw_step(*bad, **ok)
    for kw in (dict(step=0, lr=1e-3), dict(step=1, lr=1e-3, emas=[m.clone()]), dict(step=1, lr=1e-3, norm=m[0, 0]),
               dict(step=torch.ones((), device=cuda), lr=1e-3)):
        with pytest.raises(ValueError):
            optim.adamw_step([p], [g], [m], [v], **kw)
    with pytest.raises(ValueError, match="eps"):
        optim.adamw_step([p], [g], [optim.zeros_state8(p)], [optim.zeros_state8(p)], step=1, lr=1e-3, eps=0.0)
    code, exp = optim.zeros_state8(p)
    with pytest.raises(ValueError):
        optim.decode_state8(code, exp[:0], True)


def params_of(cuda, dtype=torch.float32):
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.Flatten(), torch.nn.Linear(8 * 36, 33),
                              torch.nn.LayerNorm(33)).to(cuda, dtype)
    net[0].to(memory_format=torch.channels_last)  # a parameter that is dense in another order
    return net


def backward(net, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(4, 3, 8, 8, generator=gen, device="cuda", dtype=next(net.parameters()).dtype)
    net(x).float().square().sum().backward()


@pytest.mark.parametrize("clip", [None, 1.0])
def test_optimizer_follows_torch_in_fp32(cuda, clip):
    """Against torch.optim.AdamW with clip_grad_norm_; both round differently in float32: each step
    moves a parameter by about lr and errs by at most 16 units of 2^-24 of that and of p, and the
    norms differ by at most 2^-20 relative."""
    a, b = params_of(cuda), params_of(cuda)
    groups = lambda n: [dict(params=list(n[0].parameters()) + list(n[2].parameters()), weight_decay=0.1),  # noqa: E731
                        dict(params=list(n[3].parameters()), weight_decay=0.0, lr=5e-3)]
    o1 = optim.AdamW(groups(a), lr=1e-2, max_grad_norm=clip, ema_decay=0.9)
    o2 = torch.optim.AdamW(groups(b), lr=1e-2)
    ema = None
    for t in range(4):
        for n, o in ((a, o1), (b, o2)):
            o.zero_grad(set_to_none=True)
            for q, w in zip(n.parameters(), a.parameters()):  # the same gradients for both
                q.grad = torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(t), device=cuda)
                if q.dim() == 4:
                    q.grad = q.grad.to(memory_format=torch.channels_last) if t % 2 else q.grad
        if clip:
            want = torch.nn.utils.clip_grad_norm_(b.parameters(), clip)
            o1.step()
            assert abs(float(o1.grad_norm) - float(want)) <= 2.0 ** -18 * float(want)
        else:
            o1.step()
        o2.step()
        now = [q.detach().clone() for q in a.parameters()]
        if ema is None:
            ema = [q.clone() for q in params_of(cuda).parameters()]
        ema = [0.9 * e.detach() + 0.1 * q for e, q in zip(ema, now)]
    for p, q, e in zip(a.parameters(), b.parameters(), ema):
        tol = 4 * (16 * 2.0 ** -24 * (q.abs() + 1) + 1e-2 * 2.0 ** -16)
        assert ((p - q).abs() <= tol).all()
        assert ((o1.ema_of(p) - e).abs() <= tol).all()


def test_optimizer_steps_count_per_parameter(cuda):
    """A parameter without a gradient is left alone and keeps its own step number."""
    a, b = params_of(cuda), params_of(cuda)
    o1, o2 = optim.AdamW(a.parameters(), lr=1e-2), torch.optim.AdamW(b.parameters(), lr=1e-2)
    for t in range(3):
        for n, o in ((a, o1), (b, o2)):
            o.zero_grad(set_to_none=True)
            backward(n, t)
            if t == 1:
                n[2].weight.grad = None
            o.step()
    assert o1.state[a[2].weight]["step"] == 2 and o1.state[a[2].bias]["step"] == 3
    for p, q in zip(a.parameters(), b.parameters()):
        assert ((p - q).abs() <= 1e-4 * (1 + q.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_round_trip(cuda, bits):
    """Saved, loaded into another optimizer (bf16 parameters, states of other types) and copied:
    the next steps are the same bit for bit."""
    a = params_of(cuda, torch.bfloat16)
    o = optim.AdamW(a.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, ema_decay=0.9, seed=5)
    for t in range(2):
        o.zero_grad()
        backward(a, t)
        o.step()
    b = copy.deepcopy(a)
    o2 = optim.AdamW(b.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, ema_decay=0.9, seed=5)
    o2.load_state_dict(o.state_dict())
    both = copy.deepcopy((a, o))
    for n, q in ((a, o), (b, o2), both):
        q.zero_grad()
        backward(n, 9)
        q.step()
    for p, q, r in zip(a.parameters(), b.parameters(), both[0].parameters()):
        assert torch.equal(p, q) and torch.equal(p, r)
        for s1, s2 in ((o.state[p], o2.state[q]),):
            assert s1.keys() == s2.keys()
            for k in s1:
                assert torch.equal(s1[k], s2[k]) if torch.is_tensor(s1[k]) else s1[k] == s2[k]


def test_states_of_torch_adamw_load(cuda):
    """A run that torch.optim.AdamW began goes on: the next step moves every parameter as torch's would,
    a channels-last one among them, within float32's roundings of the update (see above)."""
    a, b = params_of(cuda), params_of(cuda)
    old = torch.optim.AdamW(a.parameters(), lr=1e-2)
    for t in range(3):
        old.zero_grad()
        backward(a, t)
        old.step()
    b.load_state_dict(a.state_dict())
    b[0].to(memory_format=torch.channels_last)
    new = optim.AdamW(b.parameters(), lr=1e-2)
    new.load_state_dict(old.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        g = torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(5), device=cuda)
        p.grad, q.grad = g, g.clone()
    old.step(), new.step()
    assert all(new.state[p]["step"] == 4 for p in b.parameters())
    for p, q in zip(a.parameters(), b.parameters()):
        assert ((p - q).abs() <= 16 * 2.0 ** -24 * (q.abs() + 1) + 1e-2 * 2.0 ** -16).all()
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW(b.parameters(), state_bits=8).load_state_dict(new.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(cuda, bits):
    """A captured step advances its own counter and reads the learning rate that is set between
    replays: equal to the eager capturable step bit for bit.  Two graphs of two optimizers do not
    disturb one another."""
    def build(seed):
        torch.manual_seed(seed)
        ps = [torch.nn.Parameter(torch.randn(s, device=cuda)) for s in ((300, 7), (64,))]
        gs = [torch.randn_like(p) for p in ps]
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        return ps, optim.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=2.0, ema_decay=0.9, capturable=True)

    sets = [(build(1), build(1)), (build(2), build(2))]
    graphs = []
    for (ps, o), (qs, o2) in sets:
        o.step(), o2.step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o.step()
        graphs.append(g)
    for t in range(3):
        for ((ps, o), (qs, o2)), g in zip(sets, graphs):
            for a, b in zip(ps, qs):
                a.grad.copy_(torch.randn(a.shape, generator=torch.Generator(device="cuda").manual_seed(t), device=cuda))
                b.grad.copy_(a.grad)
            for opt in (o, o2):
                opt.param_groups[0]["lr"].fill_(1e-2 / (t + 1))
            g.replay()
            o2.step()
    torch.cuda.synchronize()
    for (ps, o), (qs, o2) in sets:
        assert int(o.param_groups[0]["step"]) == int(o2.param_groups[0]["step"]) == 4
        for p, q in zip(ps, qs):
            assert torch.equal(p, q)
            assert torch.equal(o.ema_of(p), o2.ema_of(q))


def test_capturable_state_round_trip(cuda):
    """Step counter and learning rate of a capturable optimizer go through its state dict."""
    def build():
        torch.manual_seed(4)
        ps = [torch.nn.Parameter(torch.randn(40, 9, device=cuda)), torch.nn.Parameter(torch.randn(3, device=cuda))]
        for p in ps:
            p.grad = torch.ones_like(p) * 0.1
        return ps, optim.AdamW([dict(params=ps[:1]), dict(params=ps[1:], lr=3e-3)], lr=1e-2, state_bits=8, capturable=True)

    ps, o = build()
    for _ in range(3):
        o.step()
    o.param_groups[0]["lr"].fill_(5e-3)
    qs, o2 = build()
    o2.load_state_dict(copy.deepcopy(o.state_dict()))
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    o.step(), o2.step()
    assert [int(g["step"]) for g in o2.param_groups] == [4, 4]
    assert abs(float(o2.param_groups[0]["lr"]) - 5e-3) <= 2.0 ** -24 * 5e-3
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_captured_step_of_many_tensors(cuda):
    """More tensors than the small table holds: the captured launch carries the whole table itself."""
    def build():
        torch.manual_seed(8)
        ps = [torch.nn.Parameter(torch.randn(30 + i, device=cuda)) for i in range(500)]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps, optim.AdamW(ps, lr=1e-2, max_grad_norm=3.0, capturable=True)

    (ps, o), (qs, o2) = build(), build()
    o.step(), o2.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.step()
    junk = [torch.randn(1 << 16, device=cuda) for _ in range(8)]  # memory that the host's lists might have held
    for _ in range(3):
        graph.replay()
        o2.step()
    del junk
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and int(o.param_groups[0]["step"]) == 4


@pytest.mark.parametrize("first", [False, True])
def test_state_between_capturable_and_not(cuda, first):
    """The step's number goes along whichever of the two saved it: the next step is the same."""
    w = torch.nn.Parameter(torch.randn(500, device=cuda))
    w.grad = torch.randn_like(w)
    a = optim.AdamW([w], lr=1e-2, capturable=first)
    for _ in range(3):
        a.step()
    v = torch.nn.Parameter(w.detach().clone())
    v.grad = w.grad.clone()
    b = optim.AdamW([v], lr=1e-2, capturable=not first)
    b.load_state_dict(a.state_dict())
    a.step(), b.step()
    # the constants of the step come from lr as float32 on one side: one rounding of the update
    assert ((w - v).abs() <= 4 * 2.0 ** -24 * (w.abs() + 1)).all()
    n = b.param_groups[0]["step"] if not first else b.state[v]["step"]
    assert int(n) == 4


def test_capture_refuses_frozen_numbers(cuda):
    ps = [torch.nn.Parameter(torch.randn(10, device=cuda))]
    ps[0].grad = torch.randn(10, device=cuda)
    plain, fresh = optim.AdamW(ps), optim.AdamW(ps, capturable=True)
    plain.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError, match="captured"):
            plain.step()
        with pytest.raises(ValueError, match="captured"):
            fresh.step()
        ps[0].grad.mul_(1.0)


def test_side_stream_and_version(cuda):
    """The step runs on the current stream, and tells autograd that the parameters changed."""
    p = torch.nn.Parameter(torch.randn(1 << 20, device=cuda))
    y = (p * p).sum()
    p.grad = torch.zeros_like(p)
    o = optim.AdamW([p], lr=1e-2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            p.grad.fill_(1.0)
            o.step()
        out = p.detach().clone()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, p.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_offsets_past_32_bits(cuda):
    """One tensor of more than 2^31 elements: its last elements are updated as those of a small one,
    and their random bits go by the index modulo 2^32."""
    n = (1 << 31) + 1000
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=cuda), torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g[-1000:] = torch.randn(1000, generator=torch.Generator(device="cuda").manual_seed(0), device=cuda).to(g.dtype)
    m, v = optim.zeros_state8(p), optim.zeros_state8(p)
    optim.adamw_step([p], [g], [m], [v], step=1, seed=3, **HYP)
    i = np.arange(n - 1000, n, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    from optim_testutil import mix
    r = mix(i ^ mix(mix((3 + 0x9E3779B9) & 0xFFFFFFFF) ^ np.uint64(0)))
    m32, v32 = moments32(np64(g[-1000:]), np.zeros(1000), np.zeros(1000), 0.9, 0.999)
    assert (n - 1000) % BLOCK == 0
    code, exp = encode(m32, r & np.uint64(0xFFFF), 15, True)
    assert np.array_equal(m[0][-1000:].cpu().numpy(), code) and np.array_equal(m[1][-4:].cpu().numpy(), exp)
    code, exp = encode(v32, r >> np.uint64(16), 31, False)
    assert np.array_equal(v[0][-1000:].cpu().numpy(), code) and np.array_equal(v[1][-4:].cpu().numpy(), exp)
    want, _, _ = adamw64(np.zeros(1000), np64(g[-1000:]), 0.0, 0.0, 1, 3e-3, 0.9, 0.999, 1e-8, 0.1)
    assert (np.abs(np64(p[-1000:]) - want) <= 1.01 * 2.0 ** -8 * np.abs(want)).all()
    assert int(m[0][:-1000].max()) == 0 and int(v[1][:-4].max()) == 0


def test_a_torch_state_gets_a_shadow(cuda):
    """A run that torch.optim.AdamW began goes on with a shadow average, which starts at its next step; a captured step
    wants that start behind it."""
    a, b = params_of(cuda), params_of(cuda)
    old = torch.optim.AdamW(a.parameters(), lr=1e-2)
    backward(a, 0)
    old.step()
    b.load_state_dict(a.state_dict())
    for capturable in (False, True):
        new = optim.AdamW(b.parameters(), lr=1e-2, ema_decay=0.9, capturable=capturable)
        new.load_state_dict(old.state_dict())
        before = [p.detach().clone() for p in b.parameters()]
        b.zero_grad()
        backward(b, 1)
        if capturable:
            for g in new.param_groups:
                g["step"], g["lr"] = torch.tensor(g["step"], device=cuda), torch.tensor(g["lr"], device=cuda)
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                with pytest.raises(ValueError, match="captured"):
                    new.step()
                next(b.parameters()).grad.mul_(1.0)
        new.step()
        for p, q in zip(b.parameters(), before):
            want = 0.9 * q.double() + 0.1 * p.detach().double()
            assert ((new.ema_of(p).double() - want).abs() <= 4 * 2.0 ** -24 * (p.detach().abs() + q.abs())).all()



def test_torch_states_in_16_bits_load(cuda):
    """States that torch keeps in the parameter's 16 bits, biases' among them, are taken on in float32."""
    a, b = params_of(cuda, torch.bfloat16), params_of(cuda, torch.bfloat16)
    old = torch.optim.AdamW(a.parameters(), lr=1e-2)
    backward(a, 0)
    old.step()
    b.load_state_dict(a.state_dict())
    new = optim.AdamW(b.parameters(), lr=1e-2)
    new.load_state_dict(old.state_dict())
    backward(b, 1)
    want = []
    for p, q in zip(b.parameters(), a.parameters()):
        st = old.state[q]
        want.append(adamw64(np64(p), np64(p.grad), np64(st["exp_avg"]), np64(st["exp_avg_sq"]), 2, 1e-2, 0.9, 0.999, 1e-8, 1e-2)[0])
    new.step()
    for p, x in zip(b.parameters(), want):
        # half a step of bf16; m, v, the update and the sum some roundings of float32 (the update is below 1)
        assert (np.abs(np64(p) - x) <= 2.0 ** -8 * 1.01 * np.abs(x) + 32 * 2.0 ** -24 * (1 + np.abs(x))).all()


def test_c_calls_of_no_tensors(cuda):
    """The size query asks for no workspace and the calls take none: the device's step number is advanced, and the
    norm of nothing is zero."""
    L = _lib.lib()
    nws = L.kda_adamw_workspace_bytes(0)
    assert nws == 0
    step, norm = torch.full((), 4, dtype=torch.int64, device=cuda), torch.full((2,), 7.0, device=cuda)
    a = _lib.KdaAdamW(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_grad_norm=1.0, state_bits=32)
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(L.kda_adamw_step(ctypes.byref(a), None, 0, step.data_ptr(), None, norm.data_ptr(), None, nws, s), "step")
    _lib.check(L.kda_grad_norm(None, 0, norm[1:].data_ptr(), None, nws, s), "norm")
    assert int(step) == 5 and norm.tolist() == [0.0, 0.0]
    a.max_grad_norm = 0.0
    _lib.check(L.kda_adamw_step(ctypes.byref(a), None, 0, step.data_ptr(), None, None, None, 0, s), "step")
    assert int(step) == 6


def test_a_refused_step_leaves_versions_alone(cuda):
    """A call that writes nothing does not tell autograd that something changed: a living graph's backward runs."""
    p = torch.randn(64, device=cuda, requires_grad=True)
    g, m, v, e = (torch.zeros(64, device=cuda) for _ in range(4))
    y = (p * p).sum()
    was = [t._version for t in (p, m, v, e)]
    kw = dict(emas=[e], ema_decay=0.9)
    for bad in (dict(step=0, lr=1e-3), dict(step=1, lr=float("inf")), dict(step=torch.ones((), device=cuda), lr=1e-3),
                dict(step=1, lr=1e-3, max_grad_norm=1.0, norm=m[:2]), dict(step=1, lr=m), dict(step="1", lr=1e-3)):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            optim.adamw_step([p], [g], [m], [v], **bad, **kw)
    assert [t._version for t in (p, m, v, e)] == was
    y.backward()
    assert torch.equal(p.grad, 2 * p.detach())
    optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-3, **kw)
    assert all(t._version > n for t, n in zip((p, m, v, e), was))


@pytest.mark.parametrize("capturable", [False, True])
def test_groups_round_by_bits_of_their_own(cuda, capturable):
    """Equal tensors with equal gradients in two groups, and in two subsets of one group with step numbers of their
    own, are rounded apart; the codes are the restated ones of the tensor's place in the whole step."""
    torch.manual_seed(9)
    w, grad = torch.randn(40, 50, device=cuda), torch.randn(40, 50, device=cuda)

    def run(groups, late=None):
        ps = [torch.nn.Parameter(w.clone()) for _ in range(4)]
        o = optim.AdamW([dict(params=[ps[i] for i in g]) for g in groups], lr=1e-3, state_bits=8, seed=3, capturable=capturable)
        for t in range(2):
            for i, p in enumerate(ps):
                p.grad = None if t == 0 and i == late else grad.clone()
            o.step()
        return ps, [o.state[p] for p in ps]

    m32, v32 = moments32(grad.cpu().numpy().reshape(-1), np.zeros(2000), np.zeros(2000), 0.9, 0.999)

    def first_codes(tensor):  # both states after a first step from zero
        r = random_bits(3, 1, tensor, 2000)
        return encode(m32, r & np.uint64(0xFFFF), 15, True), encode(v32, r >> np.uint64(16), 31, False)

    ps = [torch.nn.Parameter(w.clone()) for _ in range(4)]
    o = optim.AdamW([dict(params=ps[:1]), dict(params=ps[1:3]), dict(params=ps[3:])], lr=1e-3, state_bits=8, seed=3,
                    capturable=capturable)
    for p in ps:
        p.grad = grad.clone()
    o.step()
    for i, p in enumerate(ps):
        for name, (code, exp) in zip(("exp_avg", "exp_avg_sq"), first_codes(i)):
            assert np.array_equal(o.state[p][name].cpu().numpy(), code), (i, name)
            assert np.array_equal(o.state[p][name + "_exp"].cpu().numpy(), exp), (i, name)
    _, one = run([[0, 1, 2, 3]])
    _, two = run([[0, 1], [2, 3]])
    for a, b in zip(one, two):  # how the parameters are grouped changes nothing
        assert torch.equal(a["exp_avg"], b["exp_avg"]) and torch.equal(a["exp_avg_sq"], b["exp_avg_sq"])
    assert all(not torch.equal(two[i]["exp_avg"], two[j]["exp_avg"]) for i in range(4) for j in range(i))
    if not capturable:
        _, st = run([[0, 1, 2, 3]], late=1)  # 1 is at its first step while the others are at their second
        assert [s["step"] for s in st] == [2, 1, 2, 2]


def test_first_tensor_of_a_call(cuda):
    """Lists stepped in two calls with ``first_tensor`` give the codes of one call."""
    outs = []
    for cut in (None, 4):
        p, g, m, v = make(cuda, "bf16", 8)
        for part in ([slice(None)] if cut is None else [slice(0, cut), slice(cut, None)]):
            optim.adamw_step(p[part], g[part], m[part], v[part], step=2, seed=5, first_tensor=part.start or 0, **HYP)
        outs.append([x.clone() for x in p] + [c.clone() for c, _ in m] + [c.clone() for c, _ in v])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    for bad in (-1, 1 << 31):
        with pytest.raises((ValueError, OverflowError)):
            optim.adamw_step(p, g, m, v, step=2, first_tensor=bad, **HYP)
