"""Embedding, losses on logits and AdamW where rounding, weights of zero, shared memory and captured graphs decide, beside
test_gpu_lm.py, whose bounds and inputs these use. u = 2^-24, half a step of float32 relative to the value."""

import math

import pytest
import torch

from test_gpu_lm import BF16, F32, U, Case, gen, log_probs, rounding, some_logits, some_tokens, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


def level(sequences, length, vocab):
    """Rows of equal logits, whose sums are exact: each log-probability is -log(vocab) to float64's last places."""
    x = torch.full((sequences, length, vocab), 3.0)
    labels = torch.randint(vocab, (sequences, length), generator=gen(vocab))
    labels[:, 1::5] = -100
    return x, labels


# ---- the KL term ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("vocab", [40, 70001])
def test_a_kl_term_of_weight_zero_takes_no_part(ops, cuda, reduction, vocab):
    """Infinite terms that are only watched: a label that the reference bans, one that the policy bans."""
    x, labels = some_logits(4, 5, vocab, F32, 21, masked=0.0)
    x[1, 2, labels[1, 2]] = -math.inf
    x[3, 0, labels[3, 0]] = -math.inf
    ref, old = torch.full((4, 5), -3.0), torch.full((4, 5), -4.0)
    ref[0, 1] = ref[2, 4] = -math.inf
    adv = torch.tensor([1.0, 1.0, -2.0, -2.0])
    args = [t.cuda() for t in (x, labels, old, adv)]
    loss, none, logps, gx = ops.policy_loss(*args, reduction=reduction)
    got = ops.policy_loss(*args, reference=ref.cuda(), kl=0.0, reduction=reduction)
    assert math.isfinite(float(loss)) and float(none) == 0 and not math.isfinite(float(got[1]))
    assert torch.equal(got[0], loss) and torch.equal(got[2], logps) and torch.equal(got[3], gx) and not bool(gx.isnan().any())


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_the_kl_term_beside_the_reference(ops, cuda, reduction):
    """k = exp(m) - m - 1 is m^2 / 2 at small m: known to float32's rounding, and m's own, of a log-probability off by 2^-52."""
    x, labels = level(6, 7, 2)
    lp = torch.tensor(2.0, dtype=torch.float64).log().neg()
    ref = (lp + torch.linspace(-3e-6, 3e-6, 42, dtype=torch.float64).view(6, 7)).float()
    m = ref.double() - lp
    k, counted = m * m / 2 + m ** 3 / 6 + m ** 4 / 24, (labels != -100).double()
    share = counted / counted.sum() if reduction == "token" else counted / counted.sum(1, keepdim=True) / 6
    old, adv = lp.float().expand(6, 7), torch.zeros(6)
    loss, mean_k, _, gx = ops.policy_loss(x.cuda(), labels.cuda(), old.cuda(), adv.cuda(), reference=ref.cuda(), kl=0.5, reduction=reduction)
    want, off = (k * share).sum(), (m.abs() * share).sum() * 2.0 ** -51
    within(mean_k, want, 2 * U * want + off)
    within(loss, want / 2, 2 * U * want + off)
    c = -0.5 * torch.expm1(m) * share
    onehot = torch.zeros(6, 7, 2, dtype=torch.float64).scatter_(2, labels.clamp(min=0)[..., None], 1.0)
    within(gx, c[..., None] * (onehot - 0.5), (c.abs() * 4 * U + share * 2.0 ** -51)[..., None].expand(6, 7, 2))


# ---- sums of log-probabilities --------------------------------------------------------------------------------------

@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("vocab,length", [(2, 3), (2, 256), (2, 3001), (1000, 300), (40000, 40)])
@pytest.mark.parametrize("pairs", [1, 5])
def test_sequences_add_up_in_64_bits(ops, cuda, pairs, vocab, length, average):
    """A sequence's log-probability beside its reference: off by float64's rounding of its sum, not by float32's of each."""
    x, labels = level(2 * pairs, length, vocab)
    count = (labels != -100).sum(1).double()
    sums = -math.log(vocab) * (1 if average else count)
    reference = (sums + torch.zeros(2 * pairs)).float()
    _, rewards, _ = ops.preference_loss(x.cuda(), labels.cuda(), reference.cuda(), beta=1.0, average=average)
    want = sums - reference.double()
    within(rewards, want, 2 * U * want.abs() + (count + 4) * 2.0 ** -52 * reference.double().abs())


# ---- the gradient of log-probabilities ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [9, 2050, 33000, 70001])
def test_log_probabilities_by_lse_in_64_bits(ops, cuda, dtype, vocab):
    """The same log-probabilities; lse without float32's rounding, and a gradient without it: p is off by the sum's error, by
    3 u |lp| + 2 u of the exponential, 3 u where the rounded part of lse is put back and 1 u of a product."""
    x, labels = some_logits(2, 5, vocab, dtype, vocab)
    x = x + 2048  # (in bfloat16, in steps of 16)
    own, lp, off = log_probs(x, labels)
    logps, lse = ops.token_logps(x.cuda(), labels.cuda(), lse_dtype=torch.float64)
    short = ops.token_logps(x.cuda(), labels.cuda())
    assert lse.dtype == torch.float64 and torch.equal(logps, short[0]) and torch.equal(lse.float(), short[1])
    for got, want in zip(torch.ops.omt.token_logps(x.cuda(), labels.cuda(), -100), short):
        assert torch.equal(got, want)
    counted = labels != -100
    within(lse, torch.where(counted, torch.logsumexp(x.double(), -1), 0.0), torch.where(counted, off, 0.0))
    g = torch.randn(2, 5, generator=gen(1))
    gx = ops.token_logps_backward(g.cuda(), x.cuda(), labels.cuda(), lse)
    onehot, p = torch.zeros_like(lp).scatter_(2, labels.clamp(min=0)[..., None], 1.0), lp.exp()
    want = torch.where(counted[..., None], g.double()[..., None] * (onehot - p), 0.0)
    bound = g.double().abs()[..., None] * (p * (off + U * (3 * lp.abs() + 6)) + 3 * U * (p + onehot)) + 2.0 ** -126
    within(gx, want, torch.where(counted[..., None], bound * (1 + 2.0 ** -8) + rounding(dtype) * want.abs(), 0.0))
    with pytest.raises(ValueError):
        ops.token_logps(x.cuda(), labels.cuda(), lse_dtype=dtype if dtype == BF16 else torch.float16)
    with pytest.raises(TypeError):
        ops.token_logps_backward(g.cuda(), x.cuda(), labels.cuda(), lse.half())
    bad = labels.clone()
    bad[1, 2] = vocab
    gx = ops.token_logps_backward(g.cuda(), x.cuda(), bad.cuda(), lse)
    assert bool(gx[1, 2].isnan().all()) and not bool(gx[0].isnan().any())


# ---- tensors written in place ---------------------------------------------------------------------------------------

def test_scale_by_is_seen_by_autograd(ops, cuda):
    import omarchy_mac_torch as omt
    for scale in (ops.scale_by_, torch.ops.omt.scale_by_):
        for device in ("cuda", omt.DEVICE):
            x, two = torch.ones(5, device=device), torch.full((), 2.0, device=device)
            before = x._version
            scale(x, two)
            assert x._version == before + 1 and bool((x == 2).all())
        w = torch.ones(5, device=device, requires_grad=True)
        y = (w * x).sum()
        scale(x, two)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("at", [0, 1234567, -1])
def test_scale_by_one_of_the_elements(ops, cuda, at):
    x = torch.randn(5000001, generator=gen(3)).cuda()
    want = x * x[at].clone()
    assert torch.equal(ops.scale_by_(x, x[at]), want)


@pytest.mark.parametrize("masters", [False, True])
def test_adamw_refuses_shared_memory(ops, cuda, masters):
    """Tensors that are written by one thread and held by another: given twice, or overlapping by an element."""
    c = Case([(300,), (300,)], BF16, 8, masters)
    step, names = torch.ones((), device="cuda"), ("params", "grads", "m", "v", "ms", "vs") + ("masters",) * masters
    before = {name: [t.clone() for t in getattr(c, name)] for name in names}

    def call(**other):
        of = {name: other.get(name, getattr(c, name)) for name in names}
        ops.adamw(of["params"], of["grads"], of["m"], of["v"], step, of["ms"], of["vs"], of.get("masters"))

    def overlapping(like, apart):
        big = torch.zeros(2 * len(like), device="cuda").to(like.dtype)
        return [big[:len(like)], big[apart:apart + len(like)]]

    for name in names:
        t = getattr(c, name)
        if name != "grads":
            for wrong in ([t[0], t[0]], [t[1], t[1]], overlapping(t[0], 1), overlapping(t[0], len(t[0]) - 1), overlapping(t[0], 0)):
                with pytest.raises(ValueError, match="overlaps"):
                    call(**{name: wrong})
    for other in (dict(m=c.m, v=c.m), dict(ms=c.ms, vs=c.ms), dict(m=c.m, v=c.m[::-1]), dict(grads=c.params[::-1])):
        with pytest.raises(ValueError, match="overlaps"):
            call(**other)
    assert all(torch.equal(a.float(), b.float()) for name in names for a, b in zip(before[name], getattr(c, name)))


def test_adamw_of_shared_gradients_and_neighbours(ops, cuda):
    """One gradient of two parameters; parameters and states side by side in one buffer; a parameter that is its own gradient."""
    c, d = (Case([(300,), (300,)], F32, 32, False) for _ in range(2))
    step = torch.ones((), device="cuda")
    ops.adamw(c.params, [c.grads[0]] * 2, c.m, c.v, step)
    buffer = torch.cat(d.params + d.m + d.v)
    p, q, *held = buffer.split(300)
    ops.adamw([p, q], [d.grads[0].clone(), d.grads[0].clone()], held[:2], held[2:], step)
    assert torch.equal(buffer, torch.cat(c.params + c.m + c.v))
    c, d = (Case([(300,)], F32, 32, False) for _ in range(2))
    ops.adamw(c.params, [c.params[0].clone()], c.m, c.v, step)
    ops.adamw(d.params, d.params, d.m, d.v, step)
    assert torch.equal(c.params[0], d.params[0]) and torch.equal(c.v[0], d.v[0])


# ---- roundings ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,masters", [(F32, False), (BF16, False), (BF16, True)])
def test_adamw_in_32_bits_rounds_as_its_formula(ops, cuda, dtype, masters):
    """States of 32 bits: each operation of the formula rounded to float32 by itself, in its order, to the bit. (The root by way of
    float64, whose rounding to float32 is the root's own; torch's float32 root on the host is not rounded to nearest.)"""
    c = Case([(5000,), (33, 40)], dtype, 32, masters)
    lr, (b1, b2), eps, decay = 0.0078125, (0.875, 0.984375), 2.0 ** -20, 0.125  # (which float32 holds, and their powers)
    f = lambda v: torch.tensor(v, dtype=torch.float64).float()  # noqa: E731
    for count in (1, 2, 5):
        want = []
        for p, g, m, v in zip(c.masters if masters else c.params, c.grads, c.m, c.v):
            p, g, m, v = (t.cpu().float() for t in (p, g, m, v))
            m = f(b1) * m + f(1 - b1) * g
            v = f(b2) * v + f(1 - b2) * g * g
            p = p - f(lr * decay) * p
            want.append((p - f(lr / (1 - b1 ** count)) * m / (v.double().sqrt().float() / f((1 - b2 ** count) ** 0.5) + f(eps)), m, v))
        ops.adamw(c.params, c.grads, c.m, c.v, torch.tensor(float(count)).cuda(), None, None, c.masters if masters else None, lr=lr,
                  betas=(b1, b2), eps=eps, weight_decay=decay)
        for i, (p, m, v) in enumerate(want):
            assert torch.equal(c.m[i].cpu(), m) and torch.equal(c.v[i].cpu(), v)
            assert torch.equal(c.params[i].cpu(), p.to(dtype)) and (not masters or torch.equal(c.masters[i].cpu(), p))


# ---- captured graphs ------------------------------------------------------------------------------------------------

def way(name, ops, seed):
    """(inputs, the call on them): an operator in one of the ways that its sizes lead to."""
    g = gen(seed)
    kind, *size = name.split()
    size = [int(s) if s.isdigit() else s for s in size]
    if kind == "embedding":
        n, vocab, dim = size
        return [some_tokens(n, vocab, "skewed", seed).cuda(), torch.randn(vocab, dim, generator=g).cuda()], \
            lambda t, w: [ops.embedding(t, w, 2.0)]
    if kind == "gradient":
        n, vocab, dim = size
        return [torch.randn(n, dim, generator=g).cuda(), some_tokens(n, vocab, "skewed", seed).cuda()], \
            lambda a, t: [ops.embedding_backward(a, t, vocab, padding_idx=1)]
    if kind == "adamw":
        c = Case([(300,), (40, 50)], BF16 if size[0] == "bf16" else F32, size[1], size[2:] == ["masters"], seed)
        names = [name for name in ("params", "grads", "m", "v", "ms", "vs", "masters") if getattr(c, name)]

        def adamw(*ts):
            of = {name: [ts[2 * i].clone(), ts[2 * i + 1].clone()] for i, name in enumerate(names)}
            ops.adamw(of["params"], of["grads"], of["m"], of["v"], torch.full((), 3.0, device="cuda"), of.get("ms"), of.get("vs"),
                      of.get("masters") if c.has_masters else None)
            return [t.float() for name in names if name != "grads" for t in of[name]]

        return [t for name in names for t in getattr(c, name)], adamw
    n, length, vocab, *rest = size
    x, labels = some_logits(n, length, vocab, BF16, seed)
    x, labels, ref = x.cuda(), labels.cuda(), torch.randn(n, generator=g).cuda()
    old = torch.randn(n, length, generator=g).cuda() - 7
    if kind == "logps":
        return [x, labels], lambda x, y: list(ops.token_logps(x, y))
    if kind == "logps_gradient":
        return [old, x, labels, (old + 9).to(torch.float64 if rest[0] == "f64" else F32)], \
            lambda g, x, y, lse: [ops.token_logps_backward(g, x, y, lse)]
    if kind == "preference":
        return [x, labels, ref], lambda x, y, r: list(ops.preference_loss(x, y, r))
    return [x, labels, old, ref], lambda x, y, o, a: list(ops.policy_loss(x, y, o, a, reference=o * 0.99, kl=0.1, reduction=rest[0]))


WAYS = ["embedding 500 600 72", "gradient 500 600 72", "gradient 900 6000 200", "gradient 2000 600 72",
        "gradient 200 40000 520",                                                                             # few positions, four plans
        "gradient 1500 200000 16", "gradient 5000 6000 72", "gradient 3000 20000 520",                       # sorted by one workgroup; bins
        "gradient 9000 300 72", "gradient 9000 600 72", "gradient 3000 300000 16",                            # the sort, of 1, 2 and 3 digits
        "logps 4 50 700", "logps 2 3 70001", "logps_gradient 4 50 700 f32", "logps_gradient 4 50 700 f64", "preference 4 50 700", "preference 12 50 700",
        "preference 4 2500 33", "policy 4 50 700 token", "policy 4 50 700 sequence", "policy 7 1500 33 token", "policy 7 1500 33 sequence",
        "policy 30 3000 16 token", "policy 2 3 70001 token", "adamw f32 8", "adamw f32 32", "adamw bf16 8", "adamw bf16 32",
        "adamw bf16 8 masters", "adamw bf16 32 masters"]


@pytest.mark.parametrize("name", WAYS)
def test_a_replay_gives_the_calls_values(ops, cuda, name):
    """Two graphs of the same call, captured once, replayed in turn on new inputs with eager work between, each replay's values
    against the eager call's, which differ from the last replay's."""
    inputs, call = way(name, ops, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in inputs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*static)
        graphs.append((graph, static, out))
    last = None
    for seed in (2, 3, 4):
        for k, (graph, static, out) in enumerate(graphs):
            new, _ = way(name, ops, 10 * seed + k)
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            want = call(*new)
            for a, b in zip(out, want):
                assert a.dtype == b.dtype
                torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
            assert last is None or not any(torch.equal(a, b) for a, b in zip(want, last) if a.numel() > 1)
            last = [t.clone() for t in want]
