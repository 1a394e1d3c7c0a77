"""Both ends of a language model's training step on the omarchy_mac_torch device: autograd, the small language model trained on pairs
and on rewards with AdamW in 8 bits, against the same mathematics in plain torch on the CPU in float64."""

import math

import pytest
import torch
import torch.nn.functional as F

from test_gpu_ffn_device import plain_lm, rel
from test_gpu_lm import U, check_held, log_probs, some_logits, values, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def omt(cuda):
    import omarchy_mac_torch
    return omarchy_mac_torch


def test_embedding_gradient(omt):
    from omarchy_mac_torch import lm
    g = torch.Generator().manual_seed(0)
    w, t = torch.randn(50, 24, generator=g), torch.randint(50, (3, 70), generator=g)
    gy = torch.randn(3, 70, 24, generator=g)
    dev = w.to(omt.DEVICE).requires_grad_(True)
    y = lm.embedding(t.to(omt.DEVICE), dev, scale=0.5, padding_idx=-50)
    assert torch.equal(y.detach().cpu(), 0.5 * w[t])
    y.backward(gy.to(omt.DEVICE))
    ref = w.double().requires_grad_(True)
    (0.5 * F.embedding(t, ref, padding_idx=0)).backward(gy.double())
    assert rel(dev.grad, ref.grad) <= 2e-6 and not bool(dev.grad.cpu()[0].any())  # float32 sums of a few terms
    with torch.no_grad():
        assert lm.embedding(t.to(omt.DEVICE), dev).grad_fn is None


def test_embedding_module(omt):
    """The device's gradient is the host's; padding's row has none; the model's embedding is one."""
    from omarchy_mac_torch import lm, models
    host = lm.Embedding(30, 20, padding_idx=3, scale=2.5)
    dev = lm.Embedding(30, 20, padding_idx=3, scale=2.5)
    dev.load_state_dict(host.state_dict())
    dev = dev.to(omt.DEVICE)
    t = torch.randint(30, (4, 50))
    a, b = host(t), dev(t.to(omt.DEVICE))
    assert torch.equal(a.detach(), b.detach().cpu())
    gy = torch.randn(4, 50, 20)
    a.backward(gy)
    b.backward(gy.to(omt.DEVICE))
    assert rel(dev.weight.grad, host.weight.grad.double()) <= 2e-6 and not bool(dev.weight.grad.cpu()[3].any())
    m = models.mlp_lm(16, 32, 48, 1, embed_scale=3.0)
    assert isinstance(m.embed, lm.Embedding) and m.embed.scale == 3.0 and "scale=3.0" in repr(m)


def test_a_compiled_model_keeps_the_embedding(omt):
    from omarchy_mac_torch import models
    torch.manual_seed(6)
    m = models.mlp_lm(16, 32, 48, 1, checkpoint="full", embed_scale=3.0).to(omt.DEVICE)
    t = torch.randint(16, (3, 9)).to(omt.DEVICE)
    want = m(t)
    want.sum().backward()
    grads = [p.grad.cpu().clone() for p in m.parameters()]
    m.zero_grad()
    got = torch.compile(m, backend=omt.DEVICE)(t)
    got.sum().backward()
    assert rel(got, want.cpu()) <= 1e-5
    assert all(rel(p.grad, g) <= 1e-5 for p, g in zip(m.parameters(), grads))


@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_losses_hand_their_gradient_on(omt, scale):
    """Through what comes before them and with what comes after; against differences too."""
    from omarchy_mac_torch import lm
    g = torch.Generator().manual_seed(1)
    h, w = torch.randn(4, 6, 16, generator=g), torch.randn(40, 16, generator=g)
    labels = torch.randint(40, (4, 7), generator=g)
    labels[:, :2] = -100
    labels[3, 5:] = -100
    target = labels[:, 1:]
    ref, old, adv = -30 + torch.randn(4, generator=g), -5 + 0.1 * torch.randn(4, 6, generator=g), torch.randn(4, generator=g)

    def plain(logits):
        lp = torch.log_softmax(logits, -1).gather(2, target.clamp(min=0)[..., None])[..., 0] * (target != -100)
        gain = lp.sum(1) - ref.double()
        pref = -F.logsigmoid(0.1 * (gain[:2] - gain[2:])).mean()
        on = (target != -100).double()
        r, a = (lp - old.double()).exp(), adv.double()[:, None]
        pol = (-torch.minimum(r * a, r.clamp(0.8, 1.2) * a) * on).sum() / on.sum()
        return pref, pol, (lp * torch.arange(6)).sum()

    def ours(logits):
        t = target.to(omt.DEVICE)
        return (lm.preference_loss(logits, t, ref.to(omt.DEVICE))[0],
                lm.policy_loss(logits, t, old.to(omt.DEVICE), adv.to(omt.DEVICE))[0],
                (lm.token_logps(logits, t) * torch.arange(6, device=omt.DEVICE)).sum())

    for k in range(3):
        leaves = [[t.double().requires_grad_(True) for t in (h, w)], [t.to(omt.DEVICE).requires_grad_(True) for t in (h, w)]]
        a, b = plain(leaves[0][0] @ leaves[0][1].T)[k], ours(leaves[1][0] @ leaves[1][1].T)[k]
        assert abs(float(b) - float(a)) <= 2e-5 * max(1, abs(float(a)))
        (scale * a).backward()
        (scale * b).backward()
        for p, q in zip(leaves[1], leaves[0]):
            assert rel(p.grad, q.grad) <= 2e-5
        with torch.no_grad():  # along a direction, by differences of the device's losses: their float32 limits the step
            d = torch.randn(4, 6, 16, generator=g)
            step = 1e-2
            up, down = (ours((h + s * step * d).to(omt.DEVICE) @ w.to(omt.DEVICE).T)[k] for s in (1, -1))
            slope = float((leaves[0][0].grad * d.double()).sum()) / scale
            exact = [plain((h + s * step * d).double() @ w.double().T)[k] for s in (1, -1)]
            difference = float(exact[0] - exact[1]) / (2 * step)
            assert abs((float(up) - float(down)) / (2 * step) - difference) <= 2e-5 * max(1, abs(float(a))) / step
            assert abs(difference - slope) <= 0.05 * float(leaves[0][0].grad.norm()) / scale * float(d.norm())


def test_a_loss_of_a_view_keeps_the_rest_at_zero(omt):
    from omarchy_mac_torch import lm
    x = torch.randn(2, 5, 12).to(omt.DEVICE).requires_grad_(True)
    labels = torch.randint(12, (2, 4)).to(omt.DEVICE)
    loss, rewards = lm.preference_loss(x[:, :-1], labels, torch.zeros(2).to(omt.DEVICE))
    loss.backward()
    assert not rewards.requires_grad and not bool(x.grad[:, -1].cpu().any()) and bool(x.grad[:, :-1].cpu().any())


def reference_adamw(p, g, state, lr, betas, eps, decay):
    state["t"] = state.get("t", 0) + 1
    state["m"] = betas[0] * state.get("m", 0) + (1 - betas[0]) * g
    state["v"] = betas[1] * state.get("v", 0) + (1 - betas[1]) * g * g
    m, v = state["m"] / (1 - betas[0] ** state["t"]), state["v"] / (1 - betas[1] ** state["t"])
    return p - lr * decay * p - lr * m / (v.sqrt() + eps)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer(omt, bits):
    """Float32 parameters over several steps: states in 32 bits follow float64 to its rounding; in 8 bits, the first step too, and
    later ones to the states' rounding: m within 2^-4 and sqrt(v) within 2^-4 of the exact, each step's from what was held."""
    from omarchy_mac_torch import optim
    g = torch.Generator().manual_seed(2)
    shapes = [(33, 40), (7,), (256,)]
    start = [torch.randn(s, generator=g) for s in shapes]
    params = [torch.nn.Parameter(p.to(omt.DEVICE)) for p in start]
    opt = optim.AdamW(params, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.05, state_bits=bits)
    exact, states = [p.double() for p in start], [{} for _ in start]
    for k in range(4):
        grads = [torch.randn(s, generator=g) for s in shapes]
        for p, d in zip(params, grads):
            p.grad = d.to(omt.DEVICE)
        opt.step()
        before = exact
        exact = [reference_adamw(p, d.double(), s, 1e-2, (0.9, 0.99), 1e-8, 0.05) for p, d, s in zip(exact, grads, states)]
        for p, e, b in zip(params, exact, before):
            off = (p.detach().cpu().double() - e).abs()
            if bits == 32 or k == 0:
                # float32: of the parameter 3 roundings a step, of the update 16
                assert bool((off <= (k + 1) * 2.0 ** -24 * (4 * e.abs() + 4 * b.abs() + 16 * 1e-2 * 10)).all())
            else:  # a step's update is at most lr (1 - b1) / sqrt(1 - b2) over the corrections, here 2.8 lr
                assert bool((off <= k * 2.8e-2 * 3 * 2.0 ** -4 * 2).all())
    assert float(opt.state[params[0]]["step"]) == 4


def test_optimizer_resumes_from_its_state(omt):
    from omarchy_mac_torch import optim
    g = torch.Generator().manual_seed(3)
    start, grads = torch.randn(300, generator=g), [torch.randn(300, generator=g) for _ in range(4)]

    def made(p):
        p = torch.nn.Parameter(p.to(omt.DEVICE, torch.bfloat16))
        return p, optim.AdamW([p], lr=1e-2)

    def run(p, opt, ds):
        for d in ds:
            p.grad = d.to(omt.DEVICE, torch.bfloat16)
            opt.step()

    p, opt = made(start)
    run(p, opt, grads[:2])
    q, other = made(p.detach().cpu())
    other.load_state_dict(opt.state_dict())
    run(p, opt, grads[2:])
    run(q, other, grads[2:])
    assert torch.equal(p.detach().cpu(), q.detach().cpu())
    for name, t in opt.state[p].items():
        assert torch.equal(t.float().cpu(), other.state[q][name].float().cpu()), name


def sequences(g, n, length, vocab):
    t = torch.randint(vocab, (n, length), generator=g)
    for i in range(4, length):
        t[:, i] = (t[:, i - 1] + t[:, i - 4]) % vocab
    return t


@pytest.mark.parametrize("loss", ["preference", "policy"])
def test_language_model_is_tuned(omt, loss):
    """The operators together: embedding with a scale, the sublayers, the head, a loss on the logits, AdamW in 8 bits. The first
    step's loss and gradients against float64, and that the steps after it run."""
    from omarchy_mac_torch import lm, models, optim
    torch.manual_seed(0)
    ref = models.mlp_lm(64, 128, 320, 2, checkpoint="full", embed_scale=128 ** 0.5)
    dev = models.mlp_lm(64, 128, 320, 2, checkpoint="full", embed_scale=128 ** 0.5)
    dev.load_state_dict(ref.state_dict())
    ref, dev = ref.double(), dev.to(omt.DEVICE)
    g = torch.Generator().manual_seed(1)
    tokens = torch.cat([sequences(g, 4, 24, 64), torch.randint(64, (4, 24), generator=g)])
    labels = tokens[:, 4:].clone()
    labels[:, :5] = -100
    labels[2, 15:] = labels[6, 9:] = -100
    t, y = tokens.to(omt.DEVICE), labels.to(omt.DEVICE)
    with torch.no_grad():
        held = lm.token_logps(dev(t[:, :-1]), y)
    opt = optim.AdamW(dev.parameters(), lr=1e-3)
    adv = torch.tensor([1.0] * 4 + [-1.0] * 4)
    names = dict(ref.named_parameters())
    for k in range(4):
        logits = dev(t[:, :-1])
        if loss == "preference":
            out, rewards = lm.preference_loss(logits, y, held.sum(1), beta=0.5)
        else:
            out, kl, _ = lm.policy_loss(logits, y, held, adv.to(omt.DEVICE), reference=held, kl=0.1, reduction="sequence")
        opt.zero_grad()
        out.backward()
        if k == 0:
            plain = plain_lm(ref, tokens[:, :-1])
            lp = torch.log_softmax(plain, -1).gather(2, labels.clamp(min=0)[..., None])[..., 0] * (labels != -100)
            was = held.cpu().double()
            if loss == "preference":
                gain = lp.sum(1) - was.sum(1)
                want = -F.logsigmoid(0.5 * (gain[:4] - gain[4:])).mean()
            else:
                on = (labels != -100).double()
                r, more = (lp - was).exp(), was - lp
                each = -torch.minimum(r * adv.double()[:, None], r.clamp(0.8, 1.2) * adv.double()[:, None])
                want = (((each + 0.1 * (more.exp() - more - 1)) * on).sum(1) / on.sum(1)).mean()
            want.backward()
            assert abs(float(out) - float(want)) <= 1e-4
            for name, p in dev.named_parameters():
                # float32 matrix products of up to 320 terms, four sublayers deep: 2e-5 each, as the sublayers' own tests have
                assert rel(p.grad, names[name].grad) <= 1e-4, name
        opt.step()
        assert math.isfinite(float(out))
    assert all(bool(torch.isfinite(p.detach().cpu()).all()) for p in dev.parameters())
    assert not any(k.startswith("omt::") for k in omt.FALLBACKS)


def test_a_captured_training_step(omt):
    """Embedding, loss and optimizer of a step in one graph, replayed on new tokens with eager work between."""
    from omarchy_mac_torch import graphs, lm, optim
    torch.manual_seed(4)
    start = [torch.randn(50, 32), torch.randn(50, 32)]
    tokens = [torch.randint(50, (4, 9)) for _ in range(8)]

    def made():
        ps = [torch.nn.Parameter(p.to(omt.DEVICE)) for p in start]
        return ps, optim.AdamW(ps, lr=1e-2), torch.zeros(4, 9, dtype=torch.int64).to(omt.DEVICE)

    def step(ps, opt, t):
        logits = lm.embedding(t[:, :-1], ps[0], scale=2.0) @ ps[1].T
        loss, _ = lm.preference_loss(logits, t[:, 1:], torch.zeros(4, device=omt.DEVICE))
        for p in ps:
            p.grad = None
        loss.backward()
        opt.step()
        return loss.detach()

    ps, opt, t = made()
    t.copy_(tokens[0])
    replay, _ = graphs.graphed(lambda: step(ps, opt, t), warmup=2)
    qs, other, u = made()
    u.copy_(tokens[0])
    for _ in range(2):
        step(qs, other, u)
    for k in range(1, 8):
        t.copy_(tokens[k])
        got = replay()
        u.copy_(tokens[k])
        want = step(qs, other, u)
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), want.cpu()), k
        for p, q in zip(ps, qs):
            assert torch.equal(p.detach().cpu(), q.detach().cpu()), k
    replay.graph.release()


def test_operators_of_the_dispatcher(omt):
    """torch.ops.omt on device tensors gives what hip_ops gives on torch.cuda tensors."""
    ops = omt.hip_ops
    w, t, x, y = torch.randn(20, 16), torch.randint(20, (30,)), torch.randn(2, 5, 20), torch.randint(20, (2, 5))
    d = omt.DEVICE
    got = torch.ops.omt.embedding(t.to(d), w.to(d), 2.0)
    assert got.device.type == d and torch.equal(got.cpu(), ops.embedding(t.cuda(), w.cuda(), 2.0).cpu())
    got = torch.ops.omt.embedding_backward(w[t].to(d), t.to(d), 20, 1.0, -1)
    assert torch.equal(got.cpu(), ops.embedding_backward(w[t].cuda(), t.cuda(), 20).cpu())
    for a, b in zip(torch.ops.omt.preference_loss(x.to(d), y.to(d), w[:2, 0].to(d), 0.1, 0, 0.0, False, -100, True),
                    ops.preference_loss(x.cuda(), y.cuda(), w[:2, 0].cuda())):
        assert torch.equal(a.cpu(), b.cpu())
    for a, b in zip(torch.ops.omt.policy_loss(x.to(d), y.to(d), x[..., 0].to(d), w[:2, 0].to(d), None, 0.2, 0.2, 0.0, False, -100, True),
                    ops.policy_loss(x.cuda(), y.cuda(), x[..., 0].cuda(), w[:2, 0].cuda())):
        assert torch.equal(a.cpu(), b.cpu())
    p, q = w.to(d), w.cuda()
    torch.ops.omt.adamw_([p], [p * 1], [p * 0], [p * 0], [torch.ones((), device=d)], [], [], [], 0.1, None, 0.9, 0.99, 1e-8, 0.0, None,
                         None, False)
    ops.adamw([q], [q * 1], [q * 0], [q * 0], torch.ones((), device="cuda"), lr=0.1, betas=(0.9, 0.99), weight_decay=0.0)
    assert torch.equal(p.cpu(), q.cpu())
    with pytest.raises(ValueError):
        ops.embedding(t.to(d), w.cuda())


def test_log_probabilities_gradient_far_from_zero(omt):
    """Logits shifted by thousands: softmax does not change, and its gradient's error does not grow with the shift. p is off by the
    sum's error, by 3 u |lp| + 2 u of the exponential, 3 u where the rounded part of log sum exp is put back and 1 u of a product."""
    from omarchy_mac_torch import lm
    for shift in (0.0, 1000.0, -16384.0):
        x, labels = some_logits(3, 5, 2050, torch.float32, 7)
        x += shift
        _, lp, off = log_probs(x, labels)
        dev = x.to(omt.DEVICE).requires_grad_(True)
        g = torch.randn(3, 5, generator=torch.Generator().manual_seed(1))
        lm.token_logps(dev, labels.to(omt.DEVICE)).backward(g.to(omt.DEVICE))
        counted = (labels != -100)[..., None]
        onehot, p = torch.zeros_like(lp).scatter_(2, labels.clamp(min=0)[..., None], 1.0), lp.exp()
        want = torch.where(counted, g.double()[..., None] * (onehot - p), 0.0)
        bound = g.double().abs()[..., None] * (p * (off + U * (3 * lp.abs() + 6)) + 3 * U * (p + onehot)) + 2.0 ** -126
        within(dev.grad, want, torch.where(counted, bound, 0.0))


def test_embedding_module_takes_torchs_way(omt):
    """With what the operators lack, on the device too: other types and options, with torch's results."""
    from omarchy_mac_torch import lm
    w, t = torch.randn(9, 8), torch.randint(9, (4, 5))
    for dtype, options in ((torch.float64, {}), (torch.float16, {}), (torch.float32, dict(scale_grad_by_freq=True))):
        host = torch.nn.Embedding.from_pretrained(w.to(dtype), freeze=False, **options)
        dev = lm.Embedding.from_pretrained(w.to(dtype), freeze=False, scale=2.0, **options).to(omt.DEVICE)
        y = dev(t.to(omt.DEVICE))
        assert y.dtype == dtype and torch.equal(y.detach().cpu(), 2 * host(t).detach())
        y.sum().backward()
        (2 * host(t)).sum().backward()
        assert rel(dev.weight.grad, host.weight.grad.double()) <= 2e-6  # sums of twos, by the frequency in float32
    dev = lm.Embedding.from_pretrained(w, freeze=False, padding_idx=2, scale=2.0).to(omt.DEVICE)
    y = dev(t.to(omt.DEVICE))
    assert "_Embedding" in type(y.grad_fn).__name__ and torch.equal(y.detach().cpu(), 2 * w[t])


@pytest.mark.parametrize("padding_idx", [None, 3])
def test_embeddings_second_derivative_and_forward_mode(omt, padding_idx):
    """As nn.Embedding has them: the second derivative, and tangents, on the device against torch in float64 on the host."""
    from torch.autograd import forward_ad
    from omarchy_mac_torch import lm
    g = torch.Generator().manual_seed(0)
    w, v, t = torch.randn(20, 12, generator=g), torch.randn(20, 12, generator=g), torch.randint(20, (5, 9), generator=g)

    def second(e, w, v):
        w = w.detach().requires_grad_(True)
        first, = torch.autograd.grad((e(w) ** 3).sum(), w, create_graph=True)
        return torch.autograd.grad((first * v).sum(), w)[0]

    mine = lambda w: lm.embedding(t.to(omt.DEVICE), w, 1.5, padding_idx)  # noqa: E731
    want = second(lambda w: 1.5 * F.embedding(t, w, padding_idx), w.double(), v.double())
    assert rel(second(mine, w.to(omt.DEVICE), v.to(omt.DEVICE)), want) <= 4e-6  # two float32 sums of a few terms, one after the other
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(mine(forward_ad.make_dual(w.to(omt.DEVICE), v.to(omt.DEVICE))))
        assert torch.equal(y.primal.cpu(), 1.5 * w[t]) and torch.equal(y.tangent.cpu(), 1.5 * v[t])
    got = torch.func.vmap(mine)(torch.stack([w, v]).to(omt.DEVICE))
    assert torch.equal(got.cpu(), 1.5 * torch.stack([w[t], v[t]]))


def test_a_refused_step_leaves_the_optimizer_as_it_was(omt):
    """A rate on the host is refused; the same step with one on the device is the first."""
    from omarchy_mac_torch import optim
    start, grad = torch.randn(300), torch.randn(300)
    ps = [torch.nn.Parameter(start.to(omt.DEVICE)) for _ in range(2)]
    opts = [optim.AdamW([p], lr=torch.tensor(1e-2, device=device)) for p, device in zip(ps, ("cpu", omt.DEVICE))]
    for p in ps:
        p.grad = grad.to(omt.DEVICE)
    with pytest.raises(TypeError, match="lr"):
        opts[0].step()
    assert torch.equal(ps[0].detach().cpu(), start)
    opts[0].param_groups[0]["lr"] = opts[1].param_groups[0]["lr"]
    for opt in opts:
        opt.step()
    assert torch.equal(ps[0].detach().cpu(), ps[1].detach().cpu()) and not torch.equal(ps[0].detach().cpu(), start)
    for name, t in opts[0].state[ps[0]].items():
        assert torch.equal(t.float().cpu(), opts[1].state[ps[1]][name].float().cpu()), name


def test_optimizer_goes_on_where_torchs_stopped(omt):
    """Two steps of torch.optim.AdamW, then one of each from the same state: the parameter's three roundings a side and 16 of an
    update of up to 3 lr."""
    from omarchy_mac_torch import optim
    g = torch.Generator().manual_seed(6)
    start, grads = torch.randn(1000, generator=g), [torch.randn(1000, generator=g) for _ in range(3)]
    p, q = (torch.nn.Parameter(start.to(omt.DEVICE)) for _ in range(2))
    theirs = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    ours = optim.AdamW([q], state_bits=32)
    for k, grad in enumerate(grads):
        p.grad, q.grad = grad.to(omt.DEVICE), grad.to(omt.DEVICE)
        if k == 2:
            with torch.no_grad():
                q.copy_(p)
            ours.load_state_dict(theirs.state_dict())
            ours.step()
        theirs.step()
    got, want = q.detach().cpu().double(), p.detach().cpu().double()
    assert bool(((got - want).abs() <= U * (6 * start.abs() + 6 * want.abs() + 32 * 3e-2)).all())
    assert bool(((want - start.double()).abs().max() > 1e-2)) and float(ours.state[q]["step"]) == 3


@pytest.mark.parametrize("dtype,masters", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
def test_optimizer_in_8_bits_step_by_step(omt, dtype, masters):
    """Each step against float64 from the states that were held before it, with the bounds of one step."""
    from omarchy_mac_torch import optim
    g = torch.Generator().manual_seed(5)
    lr, (b1, b2), eps, decay = 1e-2, (0.9, 0.99), 1e-6, 0.05
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).to(omt.DEVICE)) for s in [(33, 40), (7,), (256,)]]
    opt = optim.AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay, state_bits=8, masters=masters)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else U
    for k in range(1, 5):
        before = []
        for p in params:
            s = opt.state[p]
            m, root = (values(s[n], s[n + "_scale"]) if s else torch.zeros(p.shape, dtype=torch.float64) for n in ("exp_avg", "exp_avg_sq"))
            before.append(((s["master"] if s and masters else p).detach().cpu().double(), m, root ** 2))
            p.grad = torch.randn(p.shape, generator=g).to(dtype).to(omt.DEVICE)
        opt.step()
        for p, (old, m, v) in zip(params, before):
            s, d = opt.state[p], p.grad.cpu().double()
            size, m, v = b1 * m.abs() + (1 - b1) * d.abs(), b1 * m + (1 - b1) * d, b2 * v + (1 - b2) * d * d
            over = lr / (1 - b1 ** k) / ((v / (1 - b2 ** k)).sqrt() + eps)
            want, off = old - lr * decay * old - over * m, 16 * U * over * size + 3 * U * old.abs()
            assert bool((over * m).abs().max() > 2e-3)  # what a step that did nothing would be off by
            if masters:
                within(s["master"], want, off)
                assert torch.equal(p.detach().cpu(), s["master"].cpu().to(dtype))
            else:
                within(p, want, off + half * want.abs() * (1 + 1e-3))
            check_held(s["exp_avg"], s["exp_avg_scale"], m)
            check_held(s["exp_avg_sq"], s["exp_avg_sq_scale"], v.sqrt(), root=True)
            assert float(s["step"]) == k
