"""GPU: the linear products against the formulas in 64 bits.

Tolerances, with h = finfo.eps / 2 (half a step of the 16-bit type) and u = 2^-24.  A product of
length K accumulates in float32 with an error of at most (K + 2) u sum |a||b| (operands are exact),
far under h at these sizes but carried along.  y: that error times the activation's slope (at
most 1.13), the activation's own error (3.0e-5 relative of the normal tail, which is at most that of the
result, and 2e-9 where the tail is cut; a few u else), and h of the result.  z and the gradient at z are stored in 16 bits: h of each, through the
second derivative (at most 0.8) and the next product."""
import gc
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from mlx_vit_b200 import _lib
from mlx_vit_b200.linear import ACTIVATIONS, linear_act, mlp

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
SLOPE = 1.13   # largest |act'|
CURVE = 0.8    # largest |act''|
U = 2.0 ** -24


def act64(z, kind):
    if kind == "relu":
        return torch.relu(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def grad64(z, kind):
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        act64(z, kind).sum().backward()
    return z.grad


def rnd(g, *s, dt, scale=1.0):
    return (torch.randn(*s, generator=g, device="cuda") * scale).to(dt)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def near(got, want, tol, name):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float(err[bad].max()), tuple(bad.nonzero()[0].tolist()))


def product(a, b):
    """a b^T in 64 bits and the bound of its float32 accumulation."""
    return a @ b.t(), (a.shape[1] + 2) * U * (a.abs() @ b.abs().t())


def check_linear(m, n, k, dtype, act, bias, residual, seed=0, pad=0, train=True):
    dt, h = DT[dtype], torch.finfo(DT[dtype]).eps / 2
    tiny = float(torch.finfo(dt).tiny) * torch.finfo(dt).eps  # half a subnormal step and more
    g = gen(seed)
    x = rnd(g, m, k + pad, dt=dt)[:, :k]
    w = rnd(g, n, k, dt=dt, scale=k ** -0.5)
    b = rnd(g, n, dt=dt, scale=0.5) if bias else None
    r = rnd(g, m, n + pad, dt=dt)[:, pad:] if residual else None
    dy = rnd(g, m, n, dt=dt)
    leaves = [t for t in (x, w, b, r) if t is not None]
    if train:
        for t in leaves:
            t.requires_grad_()
    y = linear_act(x, w, b, act, r)
    assert y.shape == (m, n) and y.dtype == dt
    X, W, DY = x.detach().double(), w.detach().double(), dy.double()
    z, ez = product(X, W)
    if bias:
        z = z + b.detach().double()
        ez = ez + U * z.abs()
    a = act64(z, act)
    want = a + (r.detach().double() if residual else 0)
    ea = SLOPE * ez + 3.1e-5 * a.abs() + 2e-9 + 8 * U * z.abs()
    near(y, want, ea + h * want.abs() * 1.01 + tiny, "y")
    if not train:
        return
    grads = dict(zip([i for i, t in enumerate((x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    s = grad64(z, act)
    dz = DY * s
    if act == "none":
        edz = torch.zeros_like(dz)
    elif act == "relu":  # the sign of z may differ where z is within its own error of zero
        edz = h * dz.abs() + DY.abs() * (z.abs() <= ez + h * z.abs() + tiny)
    else:
        edz = DY.abs() * (CURVE * (ez + h * z.abs() * 1.01 + tiny) + 2e-5) + h * dz.abs() * 1.01
    edz = edz + (0 if act == "none" else tiny)
    dx, e = product(dz, W.t())
    near(grads[0], dx, e * 1.01 + edz @ W.abs() + h * dx.abs() * 1.01 + tiny, "dx")
    dw, e = product(dz.t(), X.t())
    near(grads[1], dw, e * 1.01 + edz.t() @ X.abs() + h * dw.abs() * 1.01 + tiny, "dw")
    if bias:
        db = dz.sum(0)
        near(grads[2], db, (m + 2) * U * dz.abs().sum(0) + edz.sum(0) + h * db.abs() * 1.01 + tiny, "db")
    if residual:
        assert torch.equal(grads[3], dy)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (1, 1, 1), (3, 5, 7), (64, 64, 64), (128, 128, 64), (129, 65, 72), (31, 400, 768),
                                   (257, 255, 129), (500, 1000, 520), (16, 2304, 200)])
def test_shapes(cuda, dtype, m, n, k):
    check_linear(m, n, k, dtype, "none", True, True)


@pytest.mark.parametrize("m,n,k", [(2048, 2304, 768), (3000, 2560, 136), (1900, 4100, 60), (4096, 1024, 4096), (5001, 2111, 333)])
def test_large_tiles(cuda, m, n, k):
    """Enough tiles for pairs of CTAs, whole and ragged."""
    check_linear(m, n, k, "bf16", "gelu", True, True)


@pytest.mark.parametrize("m,n,k,act", [(300, 200, 5000, "gelu"), (200, 6000, 100, "silu"), (20000, 130, 200, "none"),
                                       (9000, 700, 260, "gelu_tanh"), (40, 33, 9001, "relu"), (333, 1027, 3001, "none")])
def test_split_sums(cuda, m, n, k, act):
    """Long sums over few tiles: k in parts, joined with every epilogue, in each of the three products."""
    check_linear(m, n, k, "bf16", act, True, True, seed=4)
    check_linear(m, n, k, "fp16", act, False, False, seed=5, pad=8)


def test_unsplit_without_workspace(cuda):
    g = gen(15)
    x, w = rnd(g, 200, 4096, dt=torch.bfloat16), rnd(g, 72, 4096, dt=torch.bfloat16, scale=0.02)
    L = _lib.lib()
    assert L.kda_linear_workspace_bytes(_lib.KDA_LINEAR_FWD, 200, 72, 4096, 0) > 0
    y = torch.empty(200, 72, dtype=torch.bfloat16, device=cuda)
    args = (_lib.KDA_BF16, 0, 200, 72, 4096, x.data_ptr(), 4096, w.data_ptr(), 4096, None, None, 0, y.data_ptr(), 72, None, 0)
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(L.kda_linear_fwd(*args, None, 0, s), "fwd")
    want, e = product(x.double(), w.double())
    near(y, want, e + 2.0 ** -8 * want.abs() * 1.01, "y")
    ws = torch.empty(64, dtype=torch.uint8, device=cuda)
    assert _lib.STATUS[L.kda_linear_fwd(*args, ws.data_ptr(), 64, s)] == "KDA_ERR_WORKSPACE"


def test_wgrad_large_tiles(cuda):
    check_linear(300, 2600, 4200, "bf16", "none", True, False)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False), (True, False), (False, True)])
def test_epilogues(cuda, act, dtype, bias, residual):
    check_linear(200, 136, 96, dtype, act, bias, residual, seed=1)


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_strided_views(cuda, pad, act):
    check_linear(77, 90, 101, "bf16", act, True, True, seed=2, pad=pad)


@pytest.mark.parametrize("m", [1, 2, 4, 7, 8, 9, 15, 16, 17, 32, 33, 100])
def test_few_rows(cuda, m):
    check_linear(m, 1000, 2056, "bf16", "gelu", True, True, seed=m, train=False)
    check_linear(m, 130, 4097, "fp16", "silu", True, True, seed=m, train=False)


@pytest.mark.parametrize("n,k", [(1185, 264), (2369, 104), (3001, 40), (9001, 72), (11008, 520), (40003, 136)])
@pytest.mark.parametrize("m", [1, 9, 16, 17, 32])
def test_few_rows_by_many_outputs(cuda, m, n, k):
    """Every split of k over the warps of a CTA, 8 and 16 outputs a warp."""
    check_linear(m, n, k, "bf16", "silu", True, True, seed=m, train=False)


def check_mlp(m, k, n, out, dtype, act, bias, residual, seed=0):
    dt, h = DT[dtype], torch.finfo(DT[dtype]).eps / 2
    tiny = float(torch.finfo(dt).tiny) * torch.finfo(dt).eps
    g = gen(seed)
    x, w1, w2 = rnd(g, m, k, dt=dt), rnd(g, n, k, dt=dt, scale=k ** -0.5), rnd(g, out, n, dt=dt, scale=n ** -0.5)
    b1 = rnd(g, n, dt=dt, scale=0.5) if bias else None
    b2 = rnd(g, out, dt=dt, scale=0.5) if bias else None
    r = rnd(g, m, out, dt=dt) if residual else None
    dy = rnd(g, m, out, dt=dt)
    leaves = [t.requires_grad_() for t in (x, w1, b1, w2, b2, r) if t is not None]
    y = mlp(x, w1, b1, w2, b2, act, r)
    got = list(torch.autograd.grad(y, leaves, dy))
    X, W1, W2, DY = (t.detach().double() for t in (x, w1, w2, dy))
    z, ez = product(X, W1)
    if bias:
        z = z + b1.detach().double()
        ez = ez + U * z.abs()
    a = act64(z, act)
    ea = SLOPE * ez + 3.1e-5 * a.abs() + 2e-9 + 8 * U * z.abs() + h * a.abs() * 1.01 + tiny  # h is stored in 16 bits
    want, e = product(a, W2)
    ey = e * 1.01 + ea @ W2.abs().t()
    if bias:
        want = want + b2.detach().double()
        ey = ey + U * want.abs()  # the sum with the bias is rounded before the residual may cancel it
    if residual:
        want = want + r.detach().double()
    near(y, want, ey + 2 * U * want.abs() + h * want.abs() * 1.01 + tiny, "y")
    dh, e = product(DY, W2.t())
    s = grad64(z, act)
    dz = dh * s
    es = (z.abs() <= ez + h * z.abs() + tiny).double() if act == "relu" else \
        CURVE * (ez + h * z.abs() * 1.01 + tiny) + 2e-5 if act != "none" else torch.zeros_like(z)
    edz = SLOPE * e + dh.abs() * es + h * dz.abs() * 1.02 + tiny
    checks = []
    dx, e = product(dz, W1.t())
    checks.append((dx, e * 1.01 + edz @ W1.abs()))
    dw1, e = product(dz.t(), X.t())
    checks.append((dw1, e * 1.01 + edz.t() @ X.abs()))
    if bias:
        checks.append((dz.sum(0), (m + 2) * U * dz.abs().sum(0) + edz.sum(0)))
    dw2, e = product(DY.t(), a.t())
    checks.append((dw2, e * 1.01 + DY.abs().t() @ ea))
    if bias:
        checks.append((DY.sum(0), (m + 2) * U * DY.abs().sum(0)))
    for i, (v, e) in enumerate(checks):
        near(got[i], v, e + h * v.abs() * 1.01 + tiny, i)
    if residual:
        assert torch.equal(got[-1], dy)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("m,k,n,out", [(50, 72, 200, 72), (1, 64, 256, 64), (131, 33, 77, 21)])
def test_mlp(cuda, act, m, k, n, out):
    check_mlp(m, k, n, out, "bf16", act, True, True)


@pytest.mark.parametrize("dtype,bias,residual", [("fp16", True, True), ("bf16", False, False), ("bf16", False, True)])
def test_mlp_large(cuda, dtype, bias, residual):
    check_mlp(1568, 512, 2048, 512, dtype, "gelu", bias, residual)


def test_leading_dimensions_and_layouts(cuda):
    """(B, T, K) inputs, transposed and expanded views, gradients for some operands only."""
    g = gen(5)
    x = rnd(g, 3, 7, 40, dt=torch.bfloat16)
    w = rnd(g, 40, 24, dt=torch.bfloat16, scale=0.2).t()       # column-major weight
    r = rnd(g, 24, dt=torch.bfloat16).expand(3, 7, 24)          # broadcast residual
    y = linear_act(x.transpose(0, 1), w, None, "none", r.transpose(0, 1))
    want = x.transpose(0, 1).double() @ w.double().t() + r.double().transpose(0, 1)
    assert y.shape == (7, 3, 24)
    near(y, want, 2.0 ** -8 * want.abs() * 1.01 + 50 * U * 40, "y")
    row = rnd(g, 1, 40, dt=torch.bfloat16).expand(5, 40)
    near(linear_act(row, w), row.double() @ w.double().t(), 2.0 ** -8 * (row.double() @ w.double().t()).abs() * 1.01 + 50 * U * 40, "e")
    one = linear_act(x[0, 0], w)
    assert one.shape == (24,) and torch.equal(one, linear_act(x[:1, :1], w)[0, 0])
    b = rnd(g, 24, dt=torch.bfloat16).requires_grad_()
    linear_act(x, w, b, "gelu").sum().backward()
    assert b.grad is not None and w.grad is None
    rr = torch.zeros(3, 7, 24, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    linear_act(x, w, None, "none", rr).sum().backward()
    assert (rr.grad == 1).all()


def test_broadcast_leaf_gradients(cuda):
    """A residual and an input that broadcast: their gradients are summed by autograd."""
    g = gen(6)
    x0, r0 = rnd(g, 1, 64, dt=torch.bfloat16).requires_grad_(), rnd(g, 32, dt=torch.bfloat16).requires_grad_()
    w = rnd(g, 32, 64, dt=torch.bfloat16, scale=0.125)
    dy = rnd(g, 6, 32, dt=torch.bfloat16)
    linear_act(x0.expand(6, 64), w, None, "none", r0.expand(6, 32)).backward(dy)
    want = dy.double().sum(0)
    near(r0.grad, want, 6 * 2.0 ** -8 * dy.double().abs().sum(0), "r")
    want = (dy.double() @ w.double())
    near(x0.grad[0], want.sum(0), 7 * 2.0 ** -8 * want.abs().sum(0) + 1e-5, "x")


def test_no_rows(cuda):
    w = torch.ones(8, 16, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    x = torch.empty(2, 0, 16, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    b = torch.ones(8, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    y = linear_act(x, w, b, "gelu")
    y.sum().backward()
    assert y.shape == (2, 0, 8) and (w.grad == 0).all() and (b.grad == 0).all() and x.grad.shape == x.shape
    w2 = torch.ones(16, 8, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    w.grad = None
    y = mlp(x, w, b, w2, None, "gelu", x)
    y.sum().backward()
    assert y.shape == x.shape and (w.grad == 0).all() and (w2.grad == 0).all()


@pytest.mark.parametrize("m,k,n,out", [(3000, 64, 1024, 512), (700, 40, 1001, 96), (300, 64, 136, 5000)])
def test_bias_gradients_are_sums_of_unrounded_values(cuda, m, k, n, out):
    """db1 and db2 are rounded once: what they sum, the gradient at z before it is stored, carries only
    z's rounding (through act'') and the accumulation's; last case: the product below is split."""
    g = gen(16)
    x, dy = rnd(g, m, k, dt=torch.bfloat16), rnd(g, m, out, dt=torch.bfloat16)
    w1, w2 = rnd(g, n, k, dt=torch.bfloat16, scale=k ** -0.5), rnd(g, out, n, dt=torch.bfloat16, scale=n ** -0.5)
    b1 = rnd(g, n, dt=torch.bfloat16, scale=0.5).requires_grad_()
    b2 = rnd(g, out, dt=torch.bfloat16).requires_grad_()
    d1, d2 = torch.autograd.grad(mlp(x, w1, b1, w2, b2, "none"), (b1, b2), dy)
    want = dy.double().sum(0)
    near(d2, want, (m + 2) * U * dy.double().abs().sum(0) + 2.0 ** -8 * 1.01 * want.abs(), "db2")
    dh, e = product(dy.double(), w2.double().t())
    want = dh.sum(0)
    near(d1, want, e.sum(0) + (m + 2) * U * dh.abs().sum(0) + 2.0 ** -8 * 1.01 * want.abs(), "db1")


def test_bias_gradient_with_infinite_weights(cuda):
    """The hidden bias gradient sums the rows there are: those behind the last, zeros in the products, would
    turn an infinite weight into NaN."""
    x, dy = torch.ones(33, 16, dtype=torch.bfloat16, device=cuda), torch.ones(33, 8, dtype=torch.bfloat16, device=cuda)
    w1 = torch.eye(16, dtype=torch.bfloat16, device=cuda)
    w2 = torch.ones(8, 16, dtype=torch.bfloat16, device=cuda)
    w2[3, 5] = float("inf")
    b1 = torch.zeros(16, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    mlp(x, w1, b1, w2, None, "relu").backward(dy)
    want = torch.full((16,), 33 * 8.0, device=cuda)
    want[5] = float("inf")
    assert torch.equal(b1.grad.float(), want)


def test_values_that_are_not_finite_stay_in_their_rows(cuda):
    g = gen(8)
    x = rnd(g, 40, 72, dt=torch.bfloat16)
    w = rnd(g, 24, 72, dt=torch.bfloat16)
    clean = linear_act(x, w, None, "relu")
    x[3, 5], x[9, 0] = float("nan"), float("inf")
    y = linear_act(x, w, None, "relu")
    keep = torch.ones(40, dtype=torch.bool, device=cuda)
    keep[[3, 9]] = False
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all()
    assert torch.equal(torch.isinf(y[9]), w[:, 0] > 0)


def test_rows_behind_the_last_are_left_alone(cuda):
    """Outputs written through TMA and element by element end where the matrix ends."""
    g = gen(9)
    for n in (72, 75):
        x, w = rnd(g, 70, 64, dt=torch.bfloat16), rnd(g, n, 64, dt=torch.bfloat16)
        buf = torch.full((80, n), 7.0, dtype=torch.bfloat16, device=cuda)
        L = _lib.lib()
        _lib.check(L.kda_linear_fwd(_lib.KDA_BF16, 0, 70, n, 64, x.data_ptr(), 64, w.data_ptr(), 64, None, None, 0,
                                    buf.data_ptr(), n, None, 0, None, 0, torch.cuda.current_stream().cuda_stream), "fwd")
        assert (buf[70:] == 7).all() and torch.equal(buf[:70], linear_act(x, w))


def test_refusals(cuda):
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16, device=cuda), torch.zeros(8, 16, dtype=torch.bfloat16, device=cuda)
    b, r = torch.zeros(8, dtype=torch.bfloat16, device=cuda), torch.zeros(4, 8, dtype=torch.bfloat16, device=cuda)
    for bad in ((x.float(), w.float()), (x, w.half()), (x, w[:, :8]), (x, w[0]), (x, w, b[:4]), (x, w, b.float()),
                (x, w, b, "swish"), (x, w, b, "gelu", r[:3]), (x, w.cpu()), (x, w[:0])):
        with pytest.raises(ValueError):
            linear_act(*bad)
    with pytest.raises(ValueError):
        mlp(x, w, None, w, None)
    y = linear_act(x.requires_grad_(), w, b, "gelu")
    (gx,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_same_results_every_time(cuda):
    g = gen(10)
    x, w1, w2 = rnd(g, 900, 256, dt=torch.bfloat16), rnd(g, 1024, 256, dt=torch.bfloat16, scale=0.06), rnd(g, 256, 1024, dt=torch.bfloat16, scale=0.03)
    b1, b2 = rnd(g, 1024, dt=torch.bfloat16), rnd(g, 256, dt=torch.bfloat16)
    outs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (x, w1, b1, w2, b2)]
        y = mlp(*leaves, "gelu", x)
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, x)])
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


def test_capture_and_two_streams(cuda):
    """A training step captured into a graph and replayed on new inputs, two graphs one after the other,
    and two streams at once: the same as eager."""
    g = gen(11)
    w1, w2 = rnd(g, 512, 128, dt=torch.bfloat16, scale=0.09), rnd(g, 128, 512, dt=torch.bfloat16, scale=0.04)
    b1 = rnd(g, 512, dt=torch.bfloat16)

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, w1, b1, w2)]
        y = mlp(leaves[0], leaves[1], leaves[2], leaves[3], None, "gelu", leaves[0])
        return [y.detach(), *torch.autograd.grad(y, leaves, x)]

    xs = [rnd(g, 300 + 20 * i, 128, dt=torch.bfloat16) for i in range(2)]
    eager = [step(x) for x in xs]
    graphs = []
    for x in xs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(x)
        torch.cuda.current_stream().wait_stream(s)
        graph, buf = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph):
            out = step(buf)
        graphs.append((graph, buf, out))
    for _ in range(2):
        for (graph, buf, out), x, want in zip(graphs, xs, eager):
            buf.copy_(x)
            graph.replay()
        for (graph, buf, out), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x in zip(streams, xs):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(step(x))
    torch.cuda.synchronize()
    for o, want in zip(got, eager):
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    assert _lib.lib().kda_device_status(0) == 0


@pytest.mark.parametrize("which", ["linear_act", "mlp", "residual"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_capture_beside_an_eager_graph_is_refused(cuda, which, accumulate):
    """A leaf whose eager graph on the default stream is alive: its captured backward raises, nothing is left
    invalid, and once that graph is gone the same step is captured and replays as eager."""
    g = gen(12)
    x, w = rnd(g, 70, 64, dt=torch.bfloat16), rnd(g, 64, 64, dt=torch.bfloat16, scale=0.1)
    r = rnd(g, 70, 64, dt=torch.bfloat16)
    leaves = [r] if which == "residual" else [x, w]
    for t in leaves:
        t.requires_grad_()

    def forward():
        return linear_act(x, w, None, "silu", r) if which != "mlp" else mlp(x, w, None, w, None, "silu", r)

    def step():
        y = forward()
        if accumulate:
            y.backward(torch.ones_like(y))
            return [t.grad for t in leaves]
        return torch.autograd.grad(y, leaves, torch.ones_like(y))

    def captured():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out

    alive = forward()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        captured()
    torch.cuda.synchronize()
    want = [t.clone() for t in torch.autograd.grad(alive, leaves, torch.ones_like(alive))]
    del alive
    gc.collect()
    for t in leaves:
        t.grad = None
    graph, out = captured()
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert _lib.lib().kda_device_status(0) == 0


def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements in x, y and dy: the last rows are those of a small product."""
    m, k, n = (1 << 25) + 40, 64, 72
    w = rnd(gen(12), n, k, dt=torch.bfloat16, scale=0.125)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda)
    x[-300:] = rnd(gen(13), 300, k, dt=torch.bfloat16)
    y = linear_act(x, w, None, "none")
    assert torch.equal(y[-300:], linear_act(x[-300:].contiguous(), w))
    assert (y[:100] == 0).all()
    leaf = w.clone().requires_grad_()
    out = linear_act(x, leaf)
    (dw,) = torch.autograd.grad(out, leaf, y)
    X, Y = x[-300:].double(), y[-300:].double()
    want = Y.t() @ X
    near(dw, want, 2.0 ** -8 * want.abs() * 1.01 + 400 * U * (Y.abs().t() @ X.abs()), "dw")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(cuda, act):
    """Central differences of the 64-bit formula along the returned gradient's direction."""
    g = gen(14)
    x, w = rnd(g, 20, 48, dt=torch.float16).requires_grad_(), rnd(g, 40, 48, dt=torch.float16, scale=0.15).requires_grad_()
    dy = rnd(g, 20, 40, dt=torch.float16)
    gx, gw = torch.autograd.grad(linear_act(x, w, None, act), (x, w), dy)
    f = lambda a, b: float((act64(a @ b.t(), act) * dy.double()).sum())  # noqa: E731
    X, W = x.detach().double(), w.detach().double()
    for grad, move in ((gx, lambda e, d: f(X + e * d, W)), (gw, lambda e, d: f(X, W + e * d))):
        d = grad.double() / grad.double().norm()
        diff = (move(1e-4, d) - move(-1e-4, d)) / 2e-4
        assert abs(diff - float((grad.double() * d).sum())) <= 4e-3 * abs(diff)


@pytest.mark.parametrize("which", ["linear_act", "mlp"])
def test_residual_gradient_is_its_own(cuda, which):
    """A leaf residual's gradient accumulates in memory of its own, beside the dy that the caller keeps and
    beside the gradient of another leaf that the same dy reaches."""
    g = gen(17)
    x, w = rnd(g, 40, 64, dt=torch.bfloat16), rnd(g, 64, 64, dt=torch.bfloat16, scale=0.1)
    r, other = (torch.zeros(40, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True) for _ in range(2))

    def forward():
        return linear_act(x, w, None, "none", r) if which == "linear_act" else mlp(x, w, None, w, None, "relu", r)

    dy = torch.ones(40, 64, dtype=torch.bfloat16, device=cuda)
    for n in (1, 2, 3):
        forward().backward(dy)
        assert (r.grad == n).all() and (dy == 1).all()
    r.grad.zero_()
    assert (dy == 1).all()
    for y in (lambda: forward() + other, lambda: other + forward()):
        r.grad = other.grad = None
        y().sum().backward()
        r.grad.mul_(5)
        assert (other.grad == 1).all()
        y().backward(dy)
        assert (other.grad == 2).all() and (r.grad == 6).all() and (dy == 1).all()
    gr, = torch.autograd.grad(forward(), r, dy)
    assert torch.equal(gr, dy)


def test_forward_mode_is_refused(cuda):
    """A tangent at any operand is refused, whether gradients are recorded or not: no result without one."""
    g = gen(18)
    x, w, b, r = (rnd(g, *s, dt=torch.bfloat16) for s in ((40, 64), (64, 64), (64,), (40, 64)))
    with fwd_ad.dual_level():
        for i in range(4):
            ops = [fwd_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((x, w, b, r))]
            calls = [lambda: linear_act(*ops[:3], "gelu", ops[3]), lambda: mlp(ops[0], w, None, ops[1], ops[2], "gelu", ops[3]),
                     lambda: mlp(ops[0], ops[1], ops[2], w, None, "gelu", ops[3])]
            for call in calls:
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert fwd_ad.unpack_dual(linear_act(x, w, b, "gelu", r)).tangent is None
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: linear_act(t, w), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: linear_act(t, w))(x.view(4, 10, 64))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: linear_act(t, w).float().sum())(x)


def test_tracers_are_refused(cuda):
    """A tracer sees the allocation of the result and not the kernels that fill it: what it recorded would return
    memory that no one wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx

    g = gen(19)
    x, w = rnd(g, 40, 64, dt=torch.bfloat16), rnd(g, 64, 64, dt=torch.bfloat16)
    for f in (lambda t: linear_act(t, w), lambda t: mlp(t, w, None, w, None, "relu", t)):
        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(f, (leaf,))
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(f)(leaf)
            with pytest.raises(RuntimeError):
                make_fx(f, tracing_mode="fake")(leaf)
        compiled = torch.compile(f, backend="eager")  # leaves the graph around the call
        assert torch.equal(compiled(x), f(x))


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("m,n", [(9, 8), (100, 8), (100, 13)])
def test_far_from_zero(cuda, act, m, n):
    """Results and gradients at pre-activations up to 2^122, where z^2 and z^3 are past float32: z is a power of
    two, exact in every form.  dz is stored in 16 bits; each product below is of powers of two."""
    g = gen(20)
    h = 2.0 ** -8
    x = torch.zeros(m, 16, dtype=torch.bfloat16, device=cuda)
    x[:, 0] = torch.exp2(torch.arange(m, device=cuda) % 9 * 7.0) * torch.where(torch.arange(m, device=cuda) % 2 == 0, 1.0, -1.0)
    w1 = torch.zeros(n, 16, dtype=torch.bfloat16, device=cuda)
    w1[:, 0] = torch.exp2(torch.arange(n, device=cuda) % 8 * 9.5).log2().round().exp2()
    eye = torch.eye(n, dtype=torch.bfloat16, device=cuda)
    z = x.double() @ w1.double().t()
    assert z.abs().max() > 2.0 ** 100
    s = grad64(z, act)
    want_y, dy = act64(z, act), rnd(g, m, n, dt=torch.bfloat16)
    dz = dy.double() * s
    for which in ("linear_act", "mlp"):
        a, b = x.clone().requires_grad_(), w1.clone().requires_grad_()
        bias = torch.zeros(n, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        y = linear_act(a, b, bias, act) if which == "linear_act" else mlp(a, b, bias, eye, None, act)
        near(y, want_y, (h + 3.1e-5) * 1.01 * want_y.abs() + 2e-9, "y")
        dx, dw, db = torch.autograd.grad(y, (a, b, bias), dy)
        edz = 1.01 * h * dz.abs() + 2e-5 * dy.double().abs()
        for got, left, right, name in ((dx, dz, w1.double(), "dx"), (dw, dz.t(), x.double(), "dw")):
            want = left @ right
            e = edz if name == "dx" else edz.t()
            near(got, want, e @ right.abs() + (m + n + 2) * U * (left.abs() @ right.abs()) + 1.01 * h * want.abs(), name)
        near(db, dz.sum(0), edz.sum(0) + (m + 2) * U * dz.abs().sum(0) + 1.01 * h * dz.sum(0).abs(), "db")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", [a for a in ACTIVATIONS if a != "none"])
@pytest.mark.parametrize("m,k", [(3, 16), (70, 16), (70, 9008)])
def test_pre_activations_past_the_type(cuda, dtype, act, m, k):
    """z is finite in float32 and past the 16-bit type: the derivative is 1 or 0 as at the type's largest value, in
    the kernel for few rows, in tiles and joined from parts.  Every value below is exact."""
    if k > 16:
        assert _lib.lib().kda_linear_workspace_bytes(_lib.KDA_LINEAR_FWD, m, 16, k, 0) > 0
    dt = DT[dtype]
    x, w = torch.zeros(m, k, dtype=dt, device=cuda), torch.zeros(16, k, dtype=dt, device=cuda)
    if dtype == "fp16":
        x[:, 0], w[:8, 0], w[8:, 0] = 400.0, 250.0, -250.0
    else:  # 2^127 (2 - 2^-8): above the largest bf16, which is 2^127 (2 - 2^-7), by half a step
        x[:, :2] = 2.0 ** 64
        w[:8, 0], w[:8, 1] = (2 - 2.0 ** -7) * 2.0 ** 63, 2.0 ** 55
        w[8:] = -w[:8]
    x.requires_grad_(), w.requires_grad_()
    b = torch.zeros(16, dtype=dt, device=cuda, requires_grad=True)
    y = linear_act(x, w, b, act)
    assert torch.isinf(y[:, :8]).all() and (y[:, 8:] == 0).all()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert torch.equal(dx, 8 * w[:1].detach().expand(m, k))
    assert torch.equal(dw[:8], (m * x[:1].detach()).expand(8, k)) and (dw[8:] == 0).all()
    assert (db[:8] == m).all() and (db[8:] == 0).all()
    w1, w2 = w.detach()[8:].clone().requires_grad_(), torch.ones(4, 8, dtype=dt, device=cuda, requires_grad=True)
    y = mlp(x, w1, None, w2, None, act)
    assert (y == 0).all()
    for t in torch.autograd.grad(y, (x, w1, w2), torch.ones_like(y)):
        assert (t == 0).all()


@pytest.mark.parametrize("n", [64, 75])
def test_relu_gradient_selects(cuda, n):
    """Behind a dead unit an infinite or NaN gradient is dropped, and a NaN's passes, as torch's ReLU does it: in the
    activation-gradient pass and in the epilogue of the product below, whole and joined from parts."""
    g = gen(21)
    m, k = 70, 64
    x, w = rnd(g, m, k, dt=torch.bfloat16), rnd(g, n, k, dt=torch.bfloat16, scale=0.1)
    b = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    b[5], b[6], b[7] = -1e4, 1e4, float("nan")
    dy = rnd(g, m, n, dt=torch.bfloat16)
    dy[3, 5], dy[4, 5] = float("inf"), float("nan")
    for t in (x, w, b):
        t.requires_grad_()
    got = torch.autograd.grad(linear_act(x, w, b, "relu"), (x, b), dy)
    clean = dy.clone()
    clean[:, 5] = 0
    with torch.no_grad():
        b[7] = 1e4
    want = torch.autograd.grad(linear_act(x, w, b, "relu"), (x, b), clean)
    assert all(torch.isfinite(t).all() for t in want)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for out in (40, 5000):  # 5000: the sum over out is in parts
        if out > 40:
            plain = -(-m // 32) * n * 4
            assert _lib.lib().kda_linear_workspace_bytes(_lib.KDA_LINEAR_DGRAD, m, out, n, 1) > plain + m * n * 4
        w2, dy2 = rnd(g, out, n, dt=torch.bfloat16, scale=0.1), rnd(g, m, out, dt=torch.bfloat16).abs()
        with torch.no_grad():
            b[7] = float("nan")
            w2[1, 5], w2[2, 5] = float("inf"), float("nan")
        got = torch.autograd.grad(mlp(x, w, b, w2, None, "relu"), (x, w, b), dy2)
        with torch.no_grad():
            b[7] = 1e4
            w2[1, 5] = w2[2, 5] = 0
        want = torch.autograd.grad(mlp(x, w, b, w2, None, "relu"), (x, w, b), dy2)
        assert all(torch.isfinite(t).all() for t in want)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("m,k,n,out", [(200, 64, 512, 2048), (131, 40, 137, 3001)])
def test_mlp_split_hidden_gradient(cuda, dtype, act, m, k, n, out):
    """The gradient at the hidden activation summed in parts: the join takes the activation's derivative, with the
    bias's sums and without."""
    sums = -(-m // 32) * n * 4
    assert _lib.lib().kda_linear_workspace_bytes(_lib.KDA_LINEAR_DGRAD, m, out, n, 1) >= sums + 2 * m * n * 4
    check_mlp(m, k, n, out, dtype, act, True, True, seed=22)
    check_mlp(m, k, n, out, dtype, act, False, False, seed=23)


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("k,n", [(64, 72), (75, 37), (64, 37), (75, 72)])
def test_hooks_on_saved_tensors(cuda, k, n, act):
    """What a hook gives back for a saved tensor has its values and not its padded rows, nor their order in memory."""
    g = gen(24)
    x, w, b = rnd(g, 100, k, dt=torch.bfloat16), rnd(g, n, k, dt=torch.bfloat16, scale=0.1), rnd(g, n, dt=torch.bfloat16)
    w2, r, dy = (rnd(g, *s, dt=torch.bfloat16) for s in ((k, n), (100, n), (100, n)))
    for t in (x, w, b, w2, r):
        t.requires_grad_()
    calls = [(lambda: linear_act(x, w, b, act, r), (x, w, b, r), dy), (lambda: mlp(x, w, b, w2, None, act, x), (x, w, b, w2), x)]
    turned = torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous() if t.dim() == 2 else t,
                                                      lambda t: t.t() if t.dim() == 2 else t)
    for call, leaves, d in calls:
        want = torch.autograd.grad(call(), leaves, d)
        for hook in (torch.autograd.graph.save_on_cpu(), turned):
            with hook:
                y = call()
            assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, d), want))
