"""The feed-forward sublayer on the omarchy_mac_torch device: autograd, modules, a small language model trained and then
served in 8 bits, against the same mathematics in plain torch on the CPU (float64 where gradients are compared).

8-bit checkpoints: an e4m3 value is within 2^-4 of what it stands for (uniformly spread rounding: 2.6% rms), so a
gradient through them is within 2^-4 of the exact one, relative 2-norm, per rounded factor."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def omt(cuda):
    import omarchy_mac_torch
    return omarchy_mac_torch


def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


def plain_block(m, x, residual=None):
    h = x if residual is None else x + residual
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + m.norm.eps) * m.norm.weight
    act = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[m.ffn.act]
    return (act(y @ m.ffn.gate.T) * (y @ m.ffn.up.T)) @ m.ffn.down.weight.T, h


def plain_lm(m, tokens):
    e = m.embed(tokens)
    n = tokens.shape[1] - m.context + 1
    x, stream = torch.cat([e[:, i:i + n] for i in range(m.context)], -1), None
    for b in m.blocks:
        x, stream = plain_block(b, x, stream)
    h = x + stream
    return m.head(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + m.norm.eps) * m.norm.weight)


@pytest.mark.parametrize("checkpoint,tol", [("full", 2e-5), ("fp8", 2 ** -4)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_sublayer_gradients(omt, checkpoint, tol, act):
    from omarchy_mac_torch import ffn
    torch.manual_seed(3)
    ref = ffn.FeedForward(96, 260, act, checkpoint)
    dev = ffn.FeedForward(96, 260, act, checkpoint)
    dev.load_state_dict(ref.state_dict())
    ref, dev = ref.double(), dev.to(omt.DEVICE)
    x, r = torch.randn(3, 50, 96), torch.randn(3, 50, 96)
    go, gs = torch.randn(3, 50, 96), torch.randn(3, 50, 96)
    inputs = [[t.double().requires_grad_(True) for t in (x, r)], [t.to(omt.DEVICE).requires_grad_(True) for t in (x, r)]]
    want = plain_block(ref, *inputs[0])
    got = dev(*inputs[1])
    for a, b in zip(got, want):
        assert rel(a, b) <= 2e-5
    torch.autograd.backward(want, [go.double(), gs.double()])
    torch.autograd.backward(got, [go.to(omt.DEVICE), gs.to(omt.DEVICE)])
    for a, b in zip(inputs[1], inputs[0]):
        assert rel(a.grad, b.grad) <= tol
    for (name, a), b in zip(dev.named_parameters(), ref.parameters()):
        assert rel(a.grad, b.grad) <= tol, name


def test_frozen_parameters_and_inference_keep_nothing(omt):
    from omarchy_mac_torch import ffn
    m = ffn.GatedFeedForward(64, 128).to(omt.DEVICE)
    x = torch.randn(10, 64, device=omt.DEVICE)
    with torch.no_grad():
        assert m(x).grad_fn is None
    m.gate.requires_grad_(False)
    m(x).sum().backward()
    assert m.gate.grad is None and m.up.grad is not None and x.grad is None
    n = ffn.RMSNorm(64).to(omt.DEVICE)
    n.weight.requires_grad_(False)
    x.requires_grad_(True)
    n(x).sum().backward()
    assert n.weight.grad is None and x.grad is not None
    with pytest.raises(ValueError):
        ffn.glu(x, m.gate, m.up, checkpoint="int8")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_language_model_trains_and_is_served(omt, dtype):
    """Ten AdamW steps on sequences that follow a rule, beside the same model in plain torch on the CPU in float32: the
    losses stay within 2% (float32 with 8-bit checkpoints) or 5% (bfloat16 throughout), and fall. Then the 8-bit model's
    logits: each of the sublayers' four roundings to e4m3 is 2.6% rms of what it adds to the stream."""
    from omarchy_mac_torch import models
    torch.manual_seed(0)
    ref = models.mlp_lm(64, 128, 320, 2)
    dev = models.mlp_lm(64, 128, 320, 2)
    dev.load_state_dict(ref.state_dict())
    dev = dev.to(omt.DEVICE, dtype)
    opts = [torch.optim.AdamW(m.parameters(), lr=2e-3) for m in (ref, dev)]
    g = torch.Generator().manual_seed(1)
    losses = [[], []]
    for _ in range(10):
        tokens = torch.randint(64, (16, 24), generator=g)
        for i in range(4, 24):
            tokens[:, i] = (tokens[:, i - 1] + tokens[:, i - 4]) % 64
        for k, (m, opt) in enumerate(zip((ref, dev), opts)):
            t = tokens if k == 0 else tokens.to(omt.DEVICE)
            logits = plain_lm(m, t[:, :-1]) if k == 0 else m(t[:, :-1])
            loss = F.cross_entropy(logits.float().flatten(0, 1), t[:, 4:].flatten())
            opt.zero_grad()
            loss.backward()
            opt.step()
            losses[k].append(float(loss))
    bound = 0.02 if dtype == torch.float32 else 0.05
    assert all(abs(a - b) <= bound * a for a, b in zip(*losses)), losses
    assert losses[1][-1] < losses[1][0]
    served = dev.serve()
    with torch.no_grad():
        for length in (4, 5, 24):  # one position, two, many
            t = tokens[:, :length].to(omt.DEVICE)
            a, b = served(t).float().cpu(), dev(t).float().cpu()
            assert a.shape == (16, length - 3, 64) and rel(a, b) <= 4 * 2 * 0.026
    assert not any(k.startswith("omt::") for k in omt.FALLBACKS)


def test_operators_on_the_device_and_its_streams(omt):
    """torch.ops.omt on device tensors gives what it gives on torch.cuda tensors, on a side stream too."""
    ops = omt.hip_ops
    x, w = torch.randn(70, 200), 1 + 0.1 * torch.randn(200)
    want = ops.rms_norm_fp8(x.cuda(), w.cuda(), x.cuda())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.rms_norm_fp8(x.to(omt.DEVICE), w.to(omt.DEVICE), x.to(omt.DEVICE))
        host = [t.view(torch.uint8).cpu() if t.dtype == torch.float8_e4m3fn else t.cpu() for t in got]
    assert all(t.device.type == omt.DEVICE for t in got)
    for a, b in zip(host, want):
        assert torch.equal(a, b.view(torch.uint8).cpu() if b.dtype == torch.float8_e4m3fn else b.cpu())
    with pytest.raises(ValueError):
        ops.rms_norm(x.to(omt.DEVICE), w.cuda())
    with pytest.raises(TypeError):
        ops.rms_norm(x, w)


def test_compiled_model_keeps_the_operators(omt):
    from omarchy_mac_torch import ffn
    torch.manual_seed(5)
    m = ffn.FeedForward(64, 192, checkpoint="full").to(omt.DEVICE)
    x = torch.randn(20, 64, device=omt.DEVICE)
    want, _ = m(x)
    want.sum().backward()
    grads = [p.grad.cpu().clone() for p in m.parameters()]
    for p in m.parameters():
        p.grad = None
    got, _ = torch.compile(m, backend=omt.DEVICE)(x)
    got.sum().backward()
    assert rel(got, want.cpu()) <= 1e-5
    assert all(rel(p.grad, g) <= 1e-5 for p, g in zip(m.parameters(), grads))
