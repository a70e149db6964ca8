"""GPU: the training operators together, as a training program uses them: the video model with its
linear products fused, the AdamW step with clipping, 8-bit states and the shadow average, eager and in
a captured graph."""
import pytest
import torch
import torch.nn.functional as F

from mlx_vit_b200 import _lib, optim
from mlx_vit_b200.checkpoint import load_checkpoint, save_checkpoint
from mlx_vit_b200.nope_gdn import KDABlock, NoPEGDNVideo

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_fused_block_agrees_with_the_torch_block(cuda):
    """Both round to bf16 at the same places but for sums and the MLP's inner results: output and
    gradients differ by some bf16 roundings in the 2-norm."""
    torch.manual_seed(0)
    a = KDABlock(128, 2).to(cuda)
    with torch.no_grad():
        a.layer.A_log.fill_(0.4)
    b = KDABlock(128, 2, fused_linear=True).to(cuda)
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 100, 128, device=cuda).bfloat16()
    dy = torch.randn_like(x)
    out = []
    for blk in (a, b):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = blk(leaf)
        y.backward(dy.to(y.dtype))
        out.append((y.detach(), leaf.grad))
    assert out[1][0].dtype == torch.bfloat16
    assert rel(out[1][0], out[0][0]) <= 4 * 2.0 ** -8 and rel(out[1][1], out[0][1]) <= 8 * 2.0 ** -8
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        if "A_log" in n or "dt_bias" in n or "f_proj" in n:
            continue  # sums of decay gradients with cancellation: any two bf16 paths differ in them
        assert q.grad is not None and rel(q.grad, p.grad) <= 8 * 2.0 ** -8, n


def model(cuda, **kw):
    torch.manual_seed(1)
    return NoPEGDNVideo(img_size=64, frames=8, dim=128, depth=2, heads=2, num_classes=10, fused_linear=True, **kw).to(cuda)


def data(cuda, n=2):
    g = torch.Generator(device=cuda).manual_seed(2)
    return torch.rand(n, 8, 64, 64, 3, generator=g, device=cuda), torch.arange(n, device=cuda) * 4 % 10


def loss_of(net, clips, labels):
    with torch.autocast("cuda", dtype=torch.bfloat16):
        return F.cross_entropy(net(clips).float(), labels)


@pytest.mark.parametrize("bits", [32, 8])
def test_model_steps(cuda, bits, tmp_path):
    """Every parameter gets a finite gradient and moves; the shadow goes through a checkpoint."""
    net = model(cuda)
    opt = optim.AdamW([dict(params=[p for p in net.parameters() if p.dim() > 1], weight_decay=0.05),
                       dict(params=[p for p in net.parameters() if p.dim() <= 1], weight_decay=0.0)], lr=1e-3,
                      state_bits=bits, max_grad_norm=1.0, ema_decay=0.9)
    clips, labels = data(cuda)
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(4):
        opt.zero_grad(set_to_none=True)
        loss_of(net, clips, labels).backward()
        want = torch.sqrt(sum(p.grad.double().square().sum() for p in net.parameters()))
        opt.step()
        assert abs(float(opt.grad_norm) - float(want)) <= 2.0 ** -23 * float(want)
    for (n, p), q in zip(net.named_parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, q), n
        assert torch.isfinite(opt.ema_of(p)).all() and opt.ema_of(p).shape == p.shape
    ema = {n: opt.ema_of(p) for n, p in net.named_parameters()}
    path = str(tmp_path / "m.safetensors")
    save_checkpoint(path, net, ema=ema)
    other = {n: torch.zeros_like(v) for n, v in ema.items()}
    load_checkpoint(path, model(cuda), ema=other)
    assert all(torch.equal(ema[n].cpu(), other[n].cpu()) for n in ema)
    assert _lib.lib().kda_device_status(0) == 0


def test_whole_step_in_a_graph(cuda):
    """Forward, loss, backward and the optimizer's step captured together and replayed: losses and
    parameters as the eager steps give them."""
    def fresh():
        net = model(cuda)
        return net, optim.AdamW(net.parameters(), lr=1e-3, max_grad_norm=1.0, state_bits=8, capturable=True)

    clips, labels = data(cuda)

    def step(net, opt):
        opt.zero_grad(set_to_none=False)
        loss = loss_of(net, clips, labels)
        loss.backward()
        opt.step()
        return loss

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        net, opt = fresh()
        for _ in range(3):
            step(net, opt)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        loss = step(net, opt)
    got = []
    for _ in range(3):
        graph.replay()
        got.append(float(loss.detach()))
    assert int(opt.param_groups[0]["step"]) == 6
    net2, opt2 = fresh()
    want = [float(step(net2, opt2).detach()) for _ in range(6)][3:]
    # the model's other kernels add some gradients by atomics: the paths agree to bf16, not bit for bit
    assert all(abs(a - b) <= 0.05 * abs(b) for a, b in zip(got, want)), (got, want)
