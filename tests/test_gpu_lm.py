"""Both ends of a language model's training step (embedding, losses on logits, AdamW) against their definitions in float64 on the
CPU, element by element.

Tolerances. u = 2^-24, half a step of float32 relative to the value; rounding to bfloat16 is off by 2^-8 at most. A sum of k terms in
float32, in any order, is off by at most k u times the sum of their magnitudes. exp(x - m) in float32: the difference is off by
u |x - m|, its product with log2(e) by 2 u |x - m| more (the constant's rounding and the product's), and the instruction by 2 u,
so a term is off by (3 d + 2) u of itself, d = m - x; over a row the terms' share of that is at most 3 ln(vocab) + 2 (the mean of d
under the softmax is at most ln(vocab)), and the sum's order adds at most its longest chain of additions, vocab / 64 + 32 up to 2048
columns and 200 beyond. log and what follows are float64; a log-probability is stored in float32."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
TYPES = [F32, BF16]


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


def rounding(dtype):
    return 2.0 ** -8 if dtype == BF16 else U


def within(got, want, bound):
    """|got - want| <= bound, element by element, with the same NaN and infinities."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), "NaN"
    far = ~((got - want).abs() <= bound) & ~want.isnan() & (got != want)
    assert not bool(far.any()), (int(far.sum()), got[far][:4], want[far][:4])


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- embedding ------------------------------------------------------------------------------------------------------

def some_tokens(n, vocab, how, seed):
    g = gen(seed)
    if how == "one":
        return torch.full((n,), vocab // 2, dtype=torch.int64)
    if how == "distinct":
        return torch.randperm(max(n, vocab), generator=g)[:n] % vocab
    if how == "skewed":
        return (vocab * torch.rand(n, generator=g, dtype=torch.float64) ** 6).long()
    return torch.randint(vocab, (n,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 3, 8, 64, 72, 100, 128, 129, 256, 513, 1024, 2056, 4100])
def test_embedding(ops, cuda, dtype, dim):
    g = gen(dim)
    w = torch.randn(77, dim, generator=g).to(dtype)
    for shape, kind in (((1,), torch.int64), ((0,), torch.int64), ((3, 5), torch.int32), ((2, 1, 131), torch.int64), ((), torch.int64)):
        t = torch.randint(77, shape, generator=g, dtype=kind)
        y = ops.embedding(t.cuda(), w.cuda())
        assert y.dtype == dtype and torch.equal(y.cpu(), w[t.long()])
        y = ops.embedding(t.cuda(), w.cuda(), scale=1.7)
        want = w[t.long()].double() * 1.7
        within(y, want, want.abs() * (rounding(dtype) + 2 * U) * (1 + U))


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_of_tokens_outside_the_vocabulary_and_strided_operands(ops, cuda, dtype):
    w = torch.randn(10, 2 * 24, generator=gen(0)).to(dtype)
    t = torch.tensor([3, -1, 9, 10, 1 << 40, -(1 << 40)])
    y = ops.embedding(t.cuda(), w.cuda()).cpu()
    assert torch.equal(y[[0, 2]], w[[3, 9]]) and bool(y[[1, 3, 4, 5]].isnan().all())
    every = torch.arange(20).cuda() % 10
    assert torch.equal(ops.embedding(every[1::3], w.cuda()[:, ::2]).cpu(), w[:, ::2][every.cpu()[1::3]])
    assert torch.equal(ops.embedding(every, w.cuda()[1:]).cpu()[every.cpu() < 9], w[1:][every.cpu()[every.cpu() < 9]])


def check_embedding_grad(ops, n, vocab, dim, dtype, tokens, scale=1.3, padding=None, seed=1):
    gy = torch.randn(n, dim, generator=gen(seed)).to(dtype)
    got = ops.embedding_backward(gy.cuda(), tokens.cuda(), vocab, scale=scale, padding_idx=padding)
    assert got.dtype == dtype and torch.equal(got, ops.embedding_backward(gy.cuda(), tokens.cuda(), vocab, scale, padding))
    valid = (tokens >= 0) & (tokens < vocab) & (tokens != (vocab if padding is None else padding % vocab))
    t, rows = tokens[valid].long(), gy[valid].double()
    want = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, t, rows)
    size = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, t, rows.abs())
    count = torch.bincount(t, minlength=vocab)[:, None]
    within(got, want * scale, abs(scale) * (count + 3) * U * size * (1 + 2.0 ** -8) + rounding(dtype) * abs(scale) * want.abs())


@pytest.mark.parametrize("how", ["one", "distinct", "skewed", "any"])
@pytest.mark.parametrize("n,vocab", [(1, 1), (15, 2), (16, 16), (17, 511), (64, 512), (1000, 513), (1024, 65), (256, 40000),
                                     (257, 40000), (1025, 300), (1024, 8000), (2048, 511), (1500, 30000), (2048, 40000), (2049, 512), (4097, 70000), (8192, 300),
                                     (8193, 300), (9000, 262143), (20000, 262144), (70001, 1000)])
def test_embedding_grad_sorts_any_tokens(ops, cuda, n, vocab, how):
    """Few in LDS, by rows of 8 and 64; in bins; over 8192 by many workgroups, of one digit, two and three."""
    check_embedding_grad(ops, n, vocab, 8, F32, some_tokens(n, vocab, how, n))


@pytest.mark.parametrize("how", ["one", "distinct", "skewed", "any"])
@pytest.mark.parametrize("n,vocab,dim", [(300, 40000, 520), (2048, 40000, 520), (2049, 40000, 520), (5000, 3000, 1032), (1500, 200000, 8),
                                         (3000, 200000, 8), (3000, 100, 512), (4096, 131072, 136), (8192, 131071, 9), (8192, 40000, 128),
                                         (4096, 16000, 1016), (3000, 512, 513), (3000, 511, 513),
                                         (4097, 700, 200), (2049, 1, 16)])
def test_embedding_grad_of_wide_rows_and_many(ops, cuda, n, vocab, dim, how):
    """Up to 2048 by one workgroup, and by many, where bins are not taken; bins of one row, 64 and 256, of both widths."""
    check_embedding_grad(ops, n, vocab, dim, BF16, some_tokens(n, vocab, how, n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 64, 65, 128, 136, 256, 300, 512, 1000, 2056])
def test_embedding_grad_of_any_width(ops, cuda, dtype, dim):
    check_embedding_grad(ops, 333, 50, dim, dtype, some_tokens(333, 50, "skewed", dim), padding=-50)
    check_embedding_grad(ops, 40, 1000, dim, dtype, some_tokens(40, 1000, "any", dim).int())
    check_embedding_grad(ops, 1333, 50, dim, dtype, some_tokens(1333, 50, "skewed", dim), padding=3)
    check_embedding_grad(ops, 2333, 70, dim, dtype, some_tokens(2333, 70, "skewed", dim))
    check_embedding_grad(ops, 150, 33000, dim, dtype, some_tokens(150, 33000, "skewed", dim))
    check_embedding_grad(ops, 700, 6000, dim, dtype, some_tokens(700, 6000, "skewed", dim))


@pytest.mark.parametrize("n", [100, 1500, 10000])
def test_embedding_grad_leaves_out_padding_and_unknown_tokens(ops, cuda, n):
    t = some_tokens(n, 60, "any", n)
    t[::7] = -1
    t[3::11] = 60
    t[5::13] = 1 << 33
    check_embedding_grad(ops, n, 60, 48, BF16, t, padding=5)
    t[:] = -100
    check_embedding_grad(ops, n, 60, 48, F32, t)
    gw = ops.embedding_backward(torch.ones(0, 8).cuda(), torch.ones(0, dtype=torch.int64).cuda(), 7)
    assert gw.shape == (7, 8) and not bool(gw.any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [(50, 30, 64), (1500, 40000, 520), (3000, 600, 64), (9000, 600, 64)])
def test_embedding_at_any_alignment(ops, cuda, dtype, n, vocab, dim):
    """The C entries on arrays that begin at their second element."""
    import ctypes
    from omarchy_mac_torch import _lib
    kind = _lib.OMT_DT_F32 if dtype == F32 else _lib.OMT_DT_BF16
    tokens = some_tokens(n, vocab, "skewed", 1).cuda()

    def inside(t):
        big = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        big[1:] = t.flatten()
        return big

    w, gy = torch.randn(vocab, dim, generator=gen(2)).to(dtype).cuda(), torch.randn(n, dim, generator=gen(3)).to(dtype).cuda()
    at = lambda t: ctypes.c_void_p(t.data_ptr() + t.element_size())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    y, bw = inside(gy * 0), inside(w)
    assert _lib.L.omt_embedding_fwd(kind, _lib.OMT_DT_I64, n, vocab, dim, ctypes.c_void_p(tokens.data_ptr()), at(bw), 2.0, at(y), stream) == 0
    assert torch.equal(y[1:].view(n, dim), ops.embedding(tokens, w, 2.0))
    gw, bgy = inside(w * math.nan), inside(gy)
    need = _lib.L.omt_embedding_bwd_workspace(n, vocab, dim)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    assert _lib.L.omt_embedding_bwd(kind, _lib.OMT_DT_I64, n, vocab, dim, at(bgy), ctypes.c_void_p(tokens.data_ptr()), -1, 2.0, at(gw),
                                    ctypes.c_void_p(ws.data_ptr()), need, stream) == 0
    assert torch.equal(gw[1:].view(vocab, dim), ops.embedding_backward(gy, tokens, vocab, 2.0)) and float(gw[0]) == 0


def test_embedding_past_32_bit_offsets(ops, cuda):
    vocab, dim = 270000, 8192  # 2.2e9 elements
    w = torch.zeros(vocab, dim, device="cuda", dtype=BF16)
    w[-1] = torch.arange(dim, device="cuda") % 256
    t = torch.tensor([vocab - 1, 0], device="cuda")
    y = ops.embedding(t, w)
    assert torch.equal(y[0], w[-1]) and not bool(y[1].any())
    del w
    gw = ops.embedding_backward(y + 1, t, vocab)
    assert torch.equal(gw[-1], y[0] + 1) and bool((gw[0] == 1).all()) and not bool(gw[1:-1].any())


# ---- losses on logits -----------------------------------------------------------------------------------------------

VOCABS = [1, 2, 9, 64, 250, 512, 520, 1000, 1024, 2048, 2050, 4096, 4104, 8192, 10000, 16384, 20001, 32768, 40000, 65536, 70001, 131072,
          131080, 140001]


def some_logits(sequences, length, vocab, dtype, seed, masked=0.3):
    g = gen(seed)
    x = (2 * torch.randn(sequences, length, vocab, generator=g)).to(dtype)
    labels = torch.randint(vocab, (sequences, length), generator=g)
    labels[torch.rand(sequences, length, generator=g) < masked] = -100
    return x, labels


def log_probs(x, labels):
    """In float64: log-probabilities of the labels that count (0 for the others), all log-probabilities, and how far the first may
    be off."""
    lp = torch.log_softmax(torch.where((labels != -100)[..., None], x.double(), 0.0), -1)
    own = torch.where(labels == -100, 0.0, lp.gather(2, labels.clamp(min=0)[..., None])[..., 0])
    v = x.shape[-1]
    return own, lp, U * (3 * math.log(v) + 4 + (v / 64 + 32 if v <= 2048 else 200))


def within_gradient(got, c, c_off, x, labels, off):
    """got against c (onehot - softmax) of the rows that count, c known to c_off; zeros elsewhere."""
    _, lp, _ = log_probs(x, labels)
    counted = (labels != -100)[..., None]
    onehot = torch.zeros_like(lp).scatter_(2, labels.clamp(min=0)[..., None], 1.0)
    p = lp.exp()
    want = torch.where(counted, c[..., None] * (onehot - p), 0.0)
    # p is off by the sum's error, float32's rounding of lse and the exponential's of x - lse; then the product's and the label's
    # subtraction's rounding
    lse = (x.double() - lp).abs()
    p_off = p * (off + U * (lse + 3 * lp.abs() + 3)) + 2.0 ** -126
    bound = c.abs()[..., None] * (p_off + 3 * U * (p + onehot)) + c_off[..., None] * (onehot + p) * (1 + 1e-3)
    within(got, want, torch.where(counted, bound * (1 + 2.0 ** -8) + rounding(got.dtype) * want.abs() + 2.0 ** -126, 0.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_token_logps(ops, cuda, dtype, vocab):
    x, labels = some_logits(2, 5, vocab, dtype, vocab)
    own, lp, off = log_probs(x, labels)
    logps, lse = ops.token_logps(x.cuda(), labels.cuda())
    assert logps.dtype == lse.dtype == F32
    within(logps, own, off + U * own.abs())
    want = torch.where(labels == -100, 0.0, torch.logsumexp(x.double(), -1))
    within(lse, want, torch.where(labels == -100, 0.0, off + U * want.abs()))
    g = torch.randn(2, 5, generator=gen(1))
    gx = ops.token_logps_backward(g.cuda(), x.cuda(), labels.cuda(), lse)
    assert gx.dtype == dtype
    within_gradient(gx, g.double(), torch.zeros(2, 5), x, labels, off)


def preference(lp, labels, reference, beta, kind, smoothing, average):
    """(loss, rewards, the loss's first and second derivative by d) in float64, of float64 log-probabilities."""
    count = (labels != -100).sum(1)
    gain = lp.sum(1) / (count.clamp(min=1) if average else 1) - reference.double()
    half = len(gain) // 2
    d = (gain[:half] - gain[half:]).detach().requires_grad_(True)
    sig = torch.nn.functional.logsigmoid
    each = {"sigmoid": lambda: -(1 - smoothing) * sig(beta * d) - smoothing * sig(-beta * d),
            "hinge": lambda: torch.relu(1 - beta * d), "ipo": lambda: (d - 0.5 / beta) ** 2}[kind]()
    slope, = torch.autograd.grad(each.sum(), d)
    return each.mean().detach(), beta * gain.detach(), slope, {"sigmoid": beta ** 2 / 4, "hinge": 0.0, "ipo": 2.0}[kind]


def check_preference(ops, x, labels, layout=lambda t: t, kind="sigmoid", smoothing=0.0, average=False, beta=0.2, fill=None, seed=0):
    n, length, _ = x.shape
    own, _, off = log_probs(x, labels)
    count = (labels != -100).sum(1)
    share = 1 / count.clamp(min=1).double() if average else torch.ones(n, dtype=torch.float64)
    reference = (own.sum(1) * share + torch.randn(n, generator=gen(seed))).float()
    loss, rewards, slope, curve = preference(own, labels, reference, beta, kind, smoothing, average)
    given = x.clone()
    if fill is not None:
        given[labels == -100] = fill
    got = ops.preference_loss(layout(given.cuda()), labels.cuda(), reference.cuda(), beta=beta, kind=kind, smoothing=smoothing,
                              average=average)
    assert got[0].shape == () and got[0].dtype == got[1].dtype == F32 and got[2].dtype == x.dtype
    # a sequence's sum: each log-probability's error and its rounding to float32
    off_sum = (count * off + U * own.abs().sum(1)) * share
    off_d = off_sum[:n // 2] + off_sum[n // 2:]
    within(got[1], rewards, beta * off_sum + 2 * U * rewards.abs())
    within(got[0], loss, ((slope.abs() + curve * off_d) * off_d).mean() + 2 * U * loss.abs())
    c = torch.cat([slope, -slope]) / (n // 2) * share
    c_off = torch.cat([curve * off_d] * 2) / (n // 2) * share + U * c.abs()
    within_gradient(got[2], c[:, None].expand(n, length), c_off[:, None].expand(n, length), x, labels, off)
    none = ops.preference_loss(layout(given.cuda()), labels.cuda(), reference.cuda(), beta=beta, kind=kind, smoothing=smoothing,
                               average=average, grad=False)
    assert none[2] is None and torch.equal(none[0], got[0]) and torch.equal(none[1], got[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_preference_loss(ops, cuda, dtype, vocab):
    check_preference(ops, *some_logits(4, 3, vocab, dtype, vocab))


@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.1, False), ("sigmoid", 1.0, True), ("hinge", 0.0, False),
                                                    ("hinge", 0.0, True), ("ipo", 0.0, False), ("ipo", 0.0, True)])
@pytest.mark.parametrize("length", [1, 2, 200, 300, 3001])
def test_preference_kinds(ops, cuda, kind, smoothing, average, length):
    check_preference(ops, *some_logits(6, length, 33, F32, length), kind=kind, smoothing=smoothing, average=average)


def test_a_pair_that_is_told_apart_for_certain(ops, cuda):
    """A rejected sequence that holds a banned token: no loss and no gradient without smoothing, in either way to a pair's loss."""
    for pairs, length in ((1, 3), (5, 3)):
        x, labels = some_logits(2 * pairs, length, 40, F32, 11, masked=0.0)
        for b in range(pairs, 2 * pairs):
            x[b, 1, labels[b, 1]] = -math.inf
        loss, rewards, gx = ops.preference_loss(x.cuda(), labels.cuda(), torch.zeros(2 * pairs).cuda())
        assert float(loss) == 0 and bool((rewards[pairs:] == -math.inf).all()) and not bool(gx.any())
        loss, _, _ = ops.preference_loss(x.cuda(), labels.cuda(), torch.zeros(2 * pairs).cuda(), smoothing=0.1)
        assert float(loss) == math.inf


def check_policy(ops, x, labels, layout=lambda t: t, reduction="token", kl=0.05, reference=True, each=False, clip=(0.2, 0.3), fill=None,
                 seed=0):
    n, length, _ = x.shape
    g = gen(seed)
    own, _, off = log_probs(x, labels)
    # ratios away from the clip's borders by more than their error
    log_ratio = 0.3 * torch.randn(n, length, generator=g, dtype=torch.float64)
    for border in (math.log(1 - clip[0]) if clip[0] < 1 else -1e9, math.log(1 + clip[1])):
        log_ratio = torch.where((log_ratio - border).abs() < 1e-3, border + 2e-3, log_ratio)
    old = (own - log_ratio).float()
    ref = (own + 0.3 * torch.randn(n, length, generator=g)).float() if reference else None
    adv = torch.randn((n, length) if each else (n,), generator=g)
    counted = (labels != -100).double()
    share = counted / counted.sum().clamp(min=1) if reduction == "token" else counted / counted.sum(1, keepdim=True).clamp(min=1) / n
    a = adv.double() if each else adv.double()[:, None].expand(n, length)
    r = (own - old.double()).exp()
    far = ((r > 1 + clip[1]) & (a > 0)) | ((r < 1 - clip[0]) & (a < 0))
    each_loss = torch.where(far, -a * r.clamp(1 - clip[0], 1 + clip[1]), -a * r)
    slope = torch.where(far, 0.0, -a * r)
    k, curve = torch.zeros_like(own), slope.abs()
    if reference:
        more = (ref.double() - own).exp()
        k = more - (ref.double() - own) - 1
        each_loss, slope, curve = each_loss + kl * k, slope + kl * (1 - more), curve + kl * more
    given = x.clone()
    if fill is not None:
        given[labels == -100] = fill
    args = [layout(given.cuda()), labels.cuda(), old.cuda(), adv.cuda()]
    options = dict(reference=ref.cuda() if reference else None, clip=clip, kl=kl, reduction=reduction)
    loss, mean_k, logps, gx = ops.policy_loss(*args, **options)
    assert loss.shape == mean_k.shape == () and logps.shape == (n, length) and gx.dtype == x.dtype
    within(logps, own, off + U * own.abs())
    want = (each_loss * share).sum()
    within(loss, want, ((slope.abs() + curve * off) * share).sum() * off + U * want.abs() + 1e-15)
    want = (k * share).sum()
    within(mean_k, want, (((more - 1).abs() + more * off) * share).sum() * off + U * want.abs() + 1e-15 if reference else 0.0)
    c = slope * share
    within_gradient(gx, c, curve * share * off * (1 + 1e-3) + U * c.abs(), x, torch.where(c == 0, -100, labels), off)
    none = ops.policy_loss(*args, **options, grad=False)
    assert none[3] is None and all(torch.equal(p, q) for p, q in zip(none[:3], (loss, mean_k, logps)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_policy_loss(ops, cuda, dtype, vocab):
    check_policy(ops, *some_logits(3, 4, vocab, dtype, vocab))


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("reference,kl", [(False, 0.0), (True, 0.0), (True, 0.1)])
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("length", [1, 300])
def test_policy_kinds(ops, cuda, reduction, reference, kl, each, length):
    check_policy(ops, *some_logits(5, length, 33, F32, length), reduction=reduction, reference=reference, kl=kl, each=each)


def test_empty_batches(ops, cuda):
    x, labels = torch.zeros(4, 0, 7).cuda(), torch.zeros(4, 0, dtype=torch.int64).cuda()
    none, ref = torch.zeros(4, 0).cuda(), torch.tensor([1.0, 2.0, 3.0, 4.0]).cuda()
    loss, rewards, gx = ops.preference_loss(x, labels, ref, beta=0.5)
    within(loss, torch.nn.functional.softplus(torch.tensor(-1.0).double()), 1e-7)
    within(rewards, torch.tensor([-0.5, -1.0, -1.5, -2.0]), 0.0)
    assert gx.shape == x.shape
    for reduction in ("token", "sequence"):
        loss, kl, logps, gx = ops.policy_loss(x, labels, none, ref, reduction=reduction)
        assert float(loss) == float(kl) == 0 and logps.shape == (4, 0) and gx.shape == x.shape
        loss, kl, logps, gx = ops.policy_loss(x.view(0, 4, 7), labels.view(0, 4), none.view(0, 4), ref[:0], reduction=reduction)
        assert float(loss) == float(kl) == 0 and gx.shape == (0, 4, 7)
    logps, lse = ops.token_logps(x, labels)
    assert logps.shape == (4, 0) and ops.token_logps_backward(logps, x, labels, lse).shape == x.shape


def test_policy_of_many_tokens(ops, cuda):
    """So many that the terms are summed, and the labels counted, in parts."""
    for reduction in ("token", "sequence"):
        check_policy(ops, *some_logits(7, 5001, 3, F32, 5), reduction=reduction)
    check_policy(ops, *some_logits(3, 40, 19, F32, 6), clip=(0.0, 0.0))
    check_policy(ops, *some_logits(3, 40, 19, F32, 6), clip=(2.0, 5.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [7, 256, 4096, 33000])
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, 3e38])
def test_rows_that_do_not_count_are_not_read(ops, cuda, dtype, vocab, fill):
    x, labels = some_logits(4, 6, vocab, dtype, 3)
    labels[1] = -100  # a whole sequence
    labels[0, 0] = 0
    check_preference(ops, x, labels, fill=fill)
    check_preference(ops, x, labels, fill=fill, kind="ipo", average=True)
    check_policy(ops, x, labels, fill=fill)
    check_policy(ops, x, labels, fill=fill, reduction="sequence")
    labels[:] = -100
    check_preference(ops, x, labels, fill=fill)
    check_policy(ops, x, labels, fill=fill)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [16, 100, 5000, 40000])
def test_logits_as_they_lie(ops, cuda, dtype, vocab):
    """Views: without the last position, of one position, transposed, expanded, of every other column."""
    x, labels = some_logits(4, 5, vocab, dtype, 9)

    def inside(t):  # as in a larger tensor, from an odd element on
        big = torch.full((6, 7, vocab + 3), math.nan, dtype=dtype, device="cuda")
        big[1:5, 2:7, 1:vocab + 1] = t
        return big[1:5, 2:7, 1:vocab + 1]

    layouts = [lambda t: torch.cat([t, t[:, :1]], 1)[:, :-1], lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), inside,
               lambda t: t.repeat_interleave(2, -1)[..., ::2]]
    for layout in layouts:
        check_preference(ops, x, labels, layout=layout)
        check_policy(ops, x, labels, layout=layout)
    x = x[:, :1].expand(4, 5, vocab)
    check_preference(ops, x.contiguous(), labels, layout=lambda t: t[:, :1].expand(4, 5, vocab))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [32, 4096, 40000])
def test_banned_tokens_and_labels_outside_the_vocabulary(ops, cuda, dtype, vocab):
    x, labels = some_logits(2, 3, vocab, dtype, 4, masked=0.0)
    labels[labels == 5] = 6
    x[..., 5] = -math.inf
    x[0, 1, : vocab // 2] = -math.inf
    labels[0, 1] = vocab - 1
    check_preference(ops, x, labels)
    check_policy(ops, x, labels)
    bad = labels.clone()
    bad[1, 2] = vocab
    old = torch.zeros(2, 3).cuda()
    loss, rewards, gx = ops.preference_loss(x.cuda(), bad.cuda(), old[:, 0])
    assert bool(loss.isnan()) and rewards.isnan().tolist() == [False, True]
    for label in (vocab, -1, 1 << 40):
        bad[1, 2] = label
        logps, lse = ops.token_logps(x.cuda(), bad.cuda())
        assert logps.isnan().sum() == 1 and bool(logps[1, 2].isnan())
        gx = ops.token_logps_backward(old + 1, x.cuda(), bad.cuda(), lse)
        assert bool(gx[1, 2].isnan().all()) and not bool(gx[0].isnan().any()) and not bool(gx[1, :2].isnan().any())
        loss, _, logps, gx = ops.policy_loss(x.cuda(), bad.cuda(), logps.nan_to_num(0.0), old[:, 0] + 1)
        assert bool(loss.isnan()) and logps.isnan().sum() == 1
        assert bool(gx[1, 2].isnan().all()) and not bool(gx[0].isnan().any()) and not bool(gx[1, :2].isnan().any())


def test_logits_past_32_bit_offsets(ops, cuda):
    length, vocab = 17000, 131072  # 2.2e9 elements
    x = torch.full((2, length, vocab), math.nan, device="cuda", dtype=BF16)
    labels = torch.full((2, length), -100)
    rows = [(0, 0), (0, length - 1), (1, 5), (1, length - 1)]
    small, own = some_logits(2, 2, vocab, BF16, 8, masked=0.0)
    for i, (b, t) in enumerate(rows):
        x[b, t] = small.flatten(0, 1)[i].cuda()
        labels[b, t] = own.flatten()[i]
    lp, _, off = log_probs(small, own)
    old = torch.zeros(2, length, device="cuda")
    for i, (b, t) in enumerate(rows):
        old[b, t] = lp.flatten()[i]
    loss, _, logps, gx = ops.policy_loss(x, labels.cuda(), old, torch.ones(2, device="cuda"))
    within(loss, torch.tensor(-1.0), 1e-5)
    picked = torch.stack([gx[b, t] for b, t in rows]).view(2, 2, vocab)
    within_gradient(picked, torch.full((2, 2), -0.25, dtype=torch.float64), torch.full((2, 2), 1e-5), small, own, off)
    assert int((gx != 0).any(-1).sum()) == 4
    del gx
    loss, rewards, gx = ops.preference_loss(x, labels.cuda(), torch.zeros(2, device="cuda"))
    within(rewards, 0.1 * lp.sum(1), 1e-4)
    assert int((gx != 0).any(-1).sum()) == 4


def test_scale_by(ops, cuda):
    for dtype in TYPES:
        for n in (0, 1, 9, 5000):
            x = torch.randn(n, generator=gen(n)).to(dtype).cuda()
            y = ops.scale_by_(x.clone(), torch.tensor(1.0).cuda())
            assert torch.equal(x, y)
            y = ops.scale_by_(x.clone(), torch.tensor([-2.0]).cuda())
            assert torch.equal(-2 * x, y)


# ---- AdamW ----------------------------------------------------------------------------------------------------------

def values(q, scale):
    """What a tensor held in 8 bits stands for, in float64."""
    flat = q.detach().cpu().reshape(-1)
    return (flat.double() * scale.detach().cpu().double().repeat_interleave(128)[:len(flat)]).view(q.shape)


def scales(t):
    flat = torch.nn.functional.pad(t.detach().abs().reshape(-1), (0, -t.numel() % 128)).view(-1, 128)
    return flat.amax(1).clamp(min=1e-30) / 448


def check_held(q, scale, want, root=False):
    """q, scale hold `want` (float64, known to 4 u): within half of e4m3's steps, and a root over zero never as zero."""
    s = scales(want)
    within(scale, s, 8 * U * s)
    over = want / s.repeat_interleave(128)[:want.numel()].view(want.shape)
    if root:
        over = torch.where(over > 0, over.clamp(min=2.0 ** -9), over)
        assert bool(((q.float().cpu() > 0) == (want > 0)).all())
    # (a value half way between two neighbours, to within its error, may go to either)
    within(q.float(), over, torch.maximum(over.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * (1 + 1e-3))


class Case:
    """Parameters with their states, and one step of them in float64."""

    def __init__(self, shapes, dtype, bits, masters, seed=0, first=False):
        g = gen(seed)
        self.dtype, self.bits, self.has_masters = dtype, bits, masters
        self.masters = [0.5 * torch.randn(s, generator=g) for s in shapes]
        self.params = [p.to(dtype) for p in self.masters]
        self.grads = [(torch.randn(s, generator=g) * torch.exp(2 * torch.randn(s, generator=g))).to(dtype) for s in shapes]
        self.m, self.v, self.ms, self.vs = [], [], [], []
        for s in shapes:
            m, v = 0.3 * torch.randn(s, generator=g), torch.exp(2 * torch.randn(s, generator=g))
            if first:
                m, v = m * 0, v * 0
            if bits == 8:
                sm, sv = scales(m), scales(v.sqrt())
                self.ms.append(sm.float())
                self.vs.append(sv.float())
                each = lambda t, sc: (t / sc.repeat_interleave(128)[:t.numel()].view(t.shape)).to(FP8)  # noqa: E731
                m, v = each(m, sm), each(v.sqrt(), sv)
            self.m.append(m)
            self.v.append(v)
        for name in ("masters", "params", "grads", "m", "v", "ms", "vs"):
            setattr(self, name, [t.cuda() for t in getattr(self, name)])

    def step(self, ops, count, lr=1e-2, betas=(0.9, 0.99), eps=1e-6, decay=0.1, maximize=False, scale=1.0, **options):
        """One step on the device, checked against float64 from the states before it."""
        at = self.masters if self.has_masters else self.params
        before = [(p.cpu().double(), g.cpu().double()) for p, g in zip(at, self.grads)]
        held = [(values(m, a), values(v, b) ** 2) for m, a, v, b in zip(self.m, self.ms, self.v, self.vs)] if self.bits == 8 else \
            [(m.cpu().double(), v.cpu().double()) for m, v in zip(self.m, self.v)]
        kept = [g.clone() for g in self.grads]
        ops.adamw(self.params, self.grads, self.m, self.v, torch.tensor(float(count)).cuda(), self.ms if self.bits == 8 else None,
                  self.vs if self.bits == 8 else None, self.masters if self.has_masters else None, lr=lr, betas=betas, eps=eps,
                  weight_decay=decay, maximize=maximize, grad_scale=torch.tensor(scale).cuda() if scale != 1.0 else None, **options)
        assert all(torch.equal(a, b) for a, b in zip(kept, self.grads))
        rate = float(lr)
        for i, ((p, g), (m, v)) in enumerate(zip(before, held)):
            g = (-g if maximize else g) / scale
            m = betas[0] * m + (1 - betas[0]) * g
            v = betas[1] * v + (1 - betas[1]) * g * g
            update = rate / (1 - betas[0] ** count) * m / ((v / (1 - betas[1] ** count)).sqrt() + eps)
            size = (betas[0] * held[i][0].abs() + (1 - betas[0]) * g.abs())
            off = rate / (1 - betas[0] ** count) * size / ((v / (1 - betas[1] ** count)).sqrt() + eps)
            want = p - rate * decay * p - update
            if self.has_masters:
                within(self.masters[i], want, 16 * U * off + 3 * U * p.abs())
                assert torch.equal(self.params[i], self.masters[i].to(BF16))
            else:
                within(self.params[i], want, 16 * U * off + 3 * U * p.abs() + rounding(self.dtype) * want.abs() * (1 + 1e-3))
            if self.bits == 8:
                s = scales(m)
                # (where b1 m and (1 - b1) g cancel, m is known to their size; the half step is far over it)
                check_held(self.m[i], self.ms[i], m)
                check_held(self.v[i], self.vs[i], v.sqrt(), root=True)
                assert s.shape == self.ms[i].shape
            else:
                within(self.m[i], m, 4 * U * size)
                within(self.v[i], v, 6 * U * v)


SHAPES = [(1,), (7,), (8,), (127,), (128,), (129,), (0,), (3, 43), (8191,), (8192,), (8193,), (50, 1000), (256, 512)]
KINDS = [(F32, 8, False), (F32, 32, False), (BF16, 8, False), (BF16, 32, False), (BF16, 8, True), (BF16, 32, True)]


@pytest.mark.parametrize("dtype,bits,masters", KINDS)
def test_adamw(ops, cuda, dtype, bits, masters):
    case = Case(SHAPES, dtype, bits, masters)
    for count in (1, 2, 1000):
        case.step(ops, count)
    case.step(ops, 3, maximize=True, scale=8.0, decay=0.0)
    case.step(ops, 4, lr=torch.tensor(2.0 ** -7).cuda(), betas=(0.0, 0.5))


@pytest.mark.parametrize("dtype,bits,masters", KINDS)
def test_adamw_from_nothing(ops, cuda, dtype, bits, masters):
    """The first steps of a run, from states of zeros, and gradients of zeros."""
    case = Case([(5, 100), (300,)], dtype, bits, masters, first=True)
    case.grads[1].zero_()
    before = case.params[1].clone()
    for count in (1, 2, 3):
        case.step(ops, count, decay=0.0)
    assert torch.equal(case.params[1], before)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_many_tensors(ops, cuda, bits):
    case = Case([(1 + i * 37 % 300,) for i in range(100)], F32, bits, False)
    case.step(ops, 2)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", TYPES)
def test_adamw_in_other_orders(ops, cuda, dtype, bits):
    """Tensors that begin at any element, filters in channels-last order, gradients in another order."""
    case = Case([(1001,), (6, 5, 3, 3), (40, 30)], dtype, bits, False)
    for name in ("params", "grads", "m", "v"):
        ts = getattr(case, name)
        big = torch.zeros(1010, device="cuda").to(ts[0].dtype)
        big[1:1002] = ts[0]
        ts[0] = big[1:1002]
        if name != "grads":
            ts[1] = ts[1].to(torch.float32).contiguous(memory_format=torch.channels_last).to(ts[1].dtype)
            assert not ts[1].is_contiguous()
    case.grads[2] = case.grads[2].t().contiguous().t()
    # (the definition above goes by the tensors' order, the blocks of 128 by the memory's: the filter is compared in its own)
    plain = Case([(1001,), (6, 3, 3, 5), (40, 30)], dtype, bits, False)
    for name in ("params", "grads", "m", "v", "ms", "vs"):
        for i, t in enumerate(getattr(case, name)):
            t = t.permute(0, 2, 3, 1) if t.dim() == 4 else t
            getattr(plain, name)[i] = t.contiguous().clone()
    for c in (case, plain):
        ops.adamw(c.params, c.grads, c.m, c.v, [torch.tensor(float(k), device="cuda") for k in (1, 2, 3)],
                  c.ms if bits == 8 else None, c.vs if bits == 8 else None)
    for name in ("params", "m", "v", "ms", "vs"):
        for a, b in zip(getattr(case, name), getattr(plain, name)):
            a = a.permute(0, 2, 3, 1) if a.dim() == 4 else a
            assert torch.equal(a.float(), b.float()), name


@pytest.mark.parametrize("dtype,bits,masters", KINDS)
def test_adamw_skips_a_step_with_infinities(ops, cuda, dtype, bits, masters):
    case = Case([(1000,)], dtype, bits, masters)
    names = ("params", "masters", "m", "v", "ms", "vs")
    before = {name: [t.clone() for t in getattr(case, name)] for name in names}
    ops.adamw(case.params, case.grads, case.m, case.v, torch.ones((), device="cuda"), case.ms or None, case.vs or None,
              case.masters if masters else None, found_inf=torch.ones((), device="cuda"))
    for name in names:
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(before[name], getattr(case, name)))


def test_adamw_keeps_a_nan_to_its_block(ops, cuda):
    case = Case([(1000,)], F32, 8, False)
    case.grads[0][300] = math.nan
    ops.adamw(case.params, case.grads, case.m, case.v, torch.ones((), device="cuda"), case.ms, case.vs)
    bad = values(case.m[0], case.ms[0]).isnan()
    assert bool(bad[256:384].all()) and int(bad.sum()) == 128
    assert case.params[0].isnan().nonzero().flatten().tolist() == [300]


def test_adamw_refuses(ops, cuda):
    c = Case([(300,), (20,)], BF16, 8, True)
    step = torch.ones((), device="cuda")

    def call(params=c.params, grads=c.grads, m=c.m, v=c.v, step=step, ms=c.ms, vs=c.vs, masters=c.masters, **options):
        ops.adamw(params, grads, m, v, step, ms, vs, masters, **options)

    before = [t.clone() for t in c.params]
    for error, options in ((ValueError, dict(params=[c.params[0]] * 2, grads=[c.grads[0]] * 2, m=[c.m[0]] * 2, v=[c.v[0]] * 2,
                                             ms=[c.ms[0]] * 2, vs=[c.vs[0]] * 2, masters=[c.masters[0]] * 2)),
                           (ValueError, dict(grads=c.grads[:1])), (ValueError, dict(ms=c.ms[:1])), (ValueError, dict(vs=None)),
                           (ValueError, dict(masters=c.masters[:1])), (ValueError, dict(ms=c.ms[::-1])),
                           (ValueError, dict(m=c.m[::-1])), (ValueError, dict(grads=c.grads[::-1])),
                           (TypeError, dict(m=[t.float() for t in c.m])), (TypeError, dict(grads=[t.float() for t in c.grads])),
                           (TypeError, dict(masters=c.params)), (TypeError, dict(ms=None, vs=None)),
                           (TypeError, dict(step=step.cpu())), (TypeError, dict(step=step.double())),
                           (ValueError, dict(step=torch.ones(2, device="cuda"))), (ValueError, dict(betas=(0.9, 1.0))),
                           (TypeError, dict(lr=torch.ones((), dtype=torch.float64, device="cuda"))),
                           (TypeError, dict(params=[t.float() for t in c.params])),
                           (TypeError, dict(params=[t.half() for t in c.params])),
                           (ValueError, dict(params=[torch.zeros(600, device="cuda", dtype=BF16)[::2], c.params[1]]))):
        with pytest.raises(error):
            call(**options)
    assert all(torch.equal(a, b) for a, b in zip(before, c.params))


def test_losses_refuse(ops, cuda):
    x, labels = some_logits(4, 3, 10, F32, 0)
    x, labels, ref, old = x.cuda(), labels.cuda(), torch.zeros(4).cuda(), torch.zeros(4, 3).cuda()
    for error, call in ((ValueError, lambda: ops.preference_loss(x[:3], labels[:3], ref[:3])),
                        (ValueError, lambda: ops.preference_loss(x[:0], labels[:0], ref[:0])),
                        (ValueError, lambda: ops.preference_loss(x, labels[:, :2], ref)),
                        (ValueError, lambda: ops.preference_loss(x, labels, ref[:2])),
                        (ValueError, lambda: ops.preference_loss(x, labels, ref, beta=0.0)),
                        (ValueError, lambda: ops.preference_loss(x, labels, ref, smoothing=2.0)),
                        (ValueError, lambda: ops.preference_loss(x, labels, ref, kind="ipo", smoothing=0.1)),
                        (TypeError, lambda: ops.preference_loss(x.half(), labels, ref)),
                        (TypeError, lambda: ops.preference_loss(x, labels.int(), ref)),
                        (TypeError, lambda: ops.preference_loss(x, labels, ref.double())),
                        (ValueError, lambda: ops.preference_loss(x[0], labels[0], ref)),
                        (TypeError, lambda: ops.preference_loss(x, labels.cpu(), ref)),
                        (ValueError, lambda: ops.policy_loss(x, labels, old[:, :2], ref)),
                        (ValueError, lambda: ops.policy_loss(x, labels, old, ref[:2])),
                        (ValueError, lambda: ops.policy_loss(x, labels, old, old[:, :1])),
                        (ValueError, lambda: ops.policy_loss(x, labels, old, ref, reference=ref)),
                        (ValueError, lambda: ops.policy_loss(x, labels, old, ref, clip=(-0.1, 0.2))),
                        (TypeError, lambda: ops.policy_loss(x, labels, old.to(BF16), ref)),
                        (ValueError, lambda: ops.token_logps_backward(ref, x, labels, old)),
                        (ValueError, lambda: ops.embedding_backward(x, labels[:, :2], 10)),
                        (ValueError, lambda: ops.embedding_backward(x, labels, 0)),
                        (TypeError, lambda: ops.embedding(old, x[0])), (ValueError, lambda: ops.embedding(labels, x)),
                        (ValueError, lambda: ops.scale_by_(x, ref)), (ValueError, lambda: ops.scale_by_(x[..., ::2], ref[0]))):
        with pytest.raises(error):
            call()


# ---- streams and graphs ---------------------------------------------------------------------------------------------

def every_operator(ops, seed, n=9000):
    """{name: (its inputs, the call on them)}: each operator with what it takes from the device."""
    g = gen(seed)
    x, labels = some_logits(4, 50, 700, BF16, seed)
    c = Case([(300,), (40, 50)], BF16, 8, True, seed)
    tokens, few = some_tokens(n, 600, "skewed", seed).cuda(), some_tokens(500, 600, "any", seed).cuda()
    gy, w = torch.randn(n, 72, generator=g).cuda(), torch.randn(600, 72, generator=g).cuda()
    x, labels, ref, old = x.cuda(), labels.cuda(), torch.randn(4, generator=g).cuda(), torch.randn(4, 50, generator=g).cuda() - 7

    def adamw(*ts):
        p, gr, m, v, ms, vs, k = ([a.clone(), b.clone()] for a, b in zip(ts[::2], ts[1::2]))
        ops.adamw(p, gr, m, v, torch.ones((), device="cuda"), ms, vs, k)
        return p + [t.float() for t in m + v] + ms + vs + k

    pairs = [t for name in ("params", "grads", "m", "v", "ms", "vs", "masters") for t in getattr(c, name)]
    return {"embedding": ([few, w], lambda t, w: [ops.embedding(t, w, 2.0)]),
            "embedding_backward": ([gy, tokens], lambda a, t: [ops.embedding_backward(a, t, 600)]),
            "embedding_backward_bins": ([gy[:5000].clone(), tokens[:5000].clone()], lambda a, t: [ops.embedding_backward(a, t, 6000)]),
            "embedding_backward_few": ([gy[:500].clone(), few], lambda a, t: [ops.embedding_backward(a, t, 600)]),
            "embedding_backward_small": ([gy[:1500].clone(), tokens[:1500].clone()], lambda a, t: [ops.embedding_backward(a, t, 200000)]),
            "token_logps": ([x, labels], lambda x, y: list(ops.token_logps(x, y))),
            "preference": ([x, labels, ref], lambda x, y, r: list(ops.preference_loss(x, y, r))),
            "policy": ([x, labels, old, ref], lambda x, y, o, a: list(ops.policy_loss(x, y, o, a, reference=o * 0.99, kl=0.1))),
            "adamw": (pairs, adamw)}


NAMES = ["embedding", "embedding_backward", "embedding_backward_few", "embedding_backward_bins", "embedding_backward_small", "token_logps", "preference", "policy", "adamw"]


@pytest.mark.parametrize("name", NAMES)
def test_replayed_graphs_give_what_the_calls_give(ops, cuda, name):
    """Captured once, replayed on new inputs with other work between; two graphs of the same call, replayed in turn."""
    inputs, call = every_operator(ops, 1)[name]
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
    for seed in (1, 2, 3):
        for k, (graph, static, out) in enumerate(graphs):
            new, _ = every_operator(ops, 10 * seed + k)[name]
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            want = call(*new)
            for a, b in zip(out, want):
                assert torch.equal(a.float(), b.float()) or bool((a.isnan() == b.isnan()).all())


@pytest.mark.parametrize("name", NAMES)
def test_side_streams_and_calls_at_once(ops, cuda, name):
    both = [every_operator(ops, seed)[name] for seed in (1, 2)]
    want = [call(*inputs) for inputs, call in both]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for k, (inputs, call) in enumerate(both):
            with torch.cuda.stream(streams[k]):
                got[k].append(call(*inputs))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
