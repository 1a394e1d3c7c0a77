"""Both ends of a language model's training step, as cases that can be timed and compared.

    embed       y[i] = scale * weight[tokens[i]]
    embed_grad  its gradient: each row of the weight's sums the gradients of the positions that hold its token
    preference  training on pairs: each sequence's log-probability under its labels against a reference's, a loss of the
                pair's difference (sigmoid, hinge or ipo), and the gradient of the logits
    policy      training on rewards: the clipped ratio of each token's probability to the one it was sampled with, times
                its advantage, with a KL term to a reference, and the gradient of the logits
    adamw       one AdamW step over all of a model's tensors, states in 8 bits or in 32

Logits are [sequences, length, vocabulary], labels of -100 are left out (the prompt, the padding). The preference loss
takes the chosen sequences in the first half and the rejected ones, in the same order, in the second. States in 8 bits:
e4m3 with a float32 scale for each block of 128 values of a tensor, scale = max(largest magnitude, 1e-30) / 448; the
second moment is held as its square root, and what is over zero is held as e4m3's smallest value at least. They are
returned as they are, with their scales.
"""

import functools
import math
import pathlib
import sys

import torch

own = False

BLOCK = 128
IGNORE = -100
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
FP8 = torch.float8_e4m3fn
FP8_SMALLEST = 2.0 ** -9
BETAS, EPS, LR, DECAY, STEP = (0.9, 0.999), 1e-8, 1e-4, 0.01, 1000


def _embed(name, kind, n, vocab, d, dtype, pad=False):
    return {"name": name, "kind": kind, "n": n, "vocab": vocab, "d": d, "dtype": dtype, "pad": pad}


def _pref(name, pairs, length, vocab, dtype, loss="sigmoid", smoothing=0.0, average=False):
    return {"name": name, "kind": "preference", "sequences": 2 * pairs, "length": length, "vocab": vocab, "dtype": dtype,
            "loss": loss, "smoothing": smoothing, "average": average}


def _policy(name, sequences, length, vocab, dtype, kl=0.04, reduction="token"):
    return {"name": name, "kind": "policy", "sequences": sequences, "length": length, "vocab": vocab, "dtype": dtype,
            "kl": kl, "reduction": reduction}


def _adamw(name, vocab, dim, hidden, depth, dtype, bits, masters=False):
    return {"name": name, "kind": "adamw", "vocab": vocab, "dim": dim, "hidden": hidden, "depth": depth, "dtype": dtype,
            "bits": bits, "masters": masters}


def listed():
    return [
        # a batch of sequences at serving, one new token each: the smallest call, where the launch counts
        _embed("embed_tokens", "embed", 64, 32768, 1024, "bf16"),
        # prompts, or a training batch's forward pass
        _embed("embed_prompts", "embed", 65536, 131072, 2048, "bf16"),
        # a model of bytes: few rows, each of them the sum of many positions; a ragged number of tokens
        _embed("embed_grad_bytes", "embed_grad", 8191, 256, 128, "f32", pad=True),
        # a large vocabulary: most of its rows get nothing, some get thousands of positions
        _embed("embed_grad", "embed_grad", 32768, 131072, 2048, "bf16"),
        # a batch of pairs for a model of bytes: launches count
        _pref("preference_bytes", 2, 63, 256, "f32"),
        # training in 32 bits, a vocabulary of an odd size, so that rows lie on 4 bytes only
        _pref("preference_f32_odd", 3, 301, 50021, "f32", loss="ipo", average=True),
        # training in 16 bits
        _pref("preference_bf16", 8, 512, 32768, "bf16", smoothing=0.1),
        # a group of short samples for a model of bytes, odd lengths
        _policy("policy_bytes", 8, 61, 256, "f32", reduction="sequence"),
        # a group of samples with a large vocabulary, the largest step on logits
        _policy("policy_bf16", 16, 512, 131072, "bf16"),
        # the optimizer step of this repository's small language model, float32
        _adamw("adamw8_small", 256, 512, 1408, 4, "f32", 8),
        # tensors of odd sizes in 16 bits, states in 32
        _adamw("adamw32_odd", 257, 100, 273, 2, "bf16", 32),
        # a large model in 16 bits with master weights in 32
        _adamw("adamw8_bf16", 32768, 4096, 8192, 3, "bf16", 8, masters=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    step = rng.choice([1, 8, 64, 128, 256])  # most models use round widths
    return w if w < step else w // step * step


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "preference", "preference", "policy", "policy", "adamw", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if kind.startswith("embed"):
        n, vocab, d = _log(rng, 1, 65536), _width(rng, 64, 131072), _width(rng, 16, 4096)
        d = min(d, (1 << 28) // max(n, vocab) // SIZE[dtype] * 2)
        return {"kind": kind, "n": n, "vocab": vocab, "d": d, "dtype": dtype, "pad": rng.random() < 0.3}
    if kind == "adamw":
        return {"kind": kind, "vocab": _width(rng, 64, 32768), "dim": 4 * _width(rng, 16, 1024), "hidden": _width(rng, 64, 8192),
                "depth": rng.randint(1, 3), "dtype": dtype, "bits": rng.choice([8, 8, 32]),
                "masters": dtype == "bf16" and rng.random() < 0.5}
    case = {"kind": kind, "sequences": _log(rng, 1, 8) * 2, "length": _log(rng, 1, 512), "vocab": _width(rng, 64, 131072),
            "dtype": dtype}
    if dtype == "f32" and case["length"] > 256:
        case["length"] //= 2
    if kind == "preference":
        loss = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        return case | {"loss": loss, "smoothing": rng.choice([0.0, 0.1]) if loss == "sigmoid" else 0.0,
                       "average": loss == "ipo" or rng.random() < 0.3}
    return case | {"kl": rng.choice([0.0, 0.04, 0.1]), "reduction": rng.choice(["token", "sequence"])}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _spans(case):
    """[(first, end)] of each sequence's unmasked labels: prompts of up to a quarter of the length, the same for both
    sequences of a pair, and ends in its second half."""
    n, length = case["sequences"], case["length"]
    pairs = n // 2 if case["kind"] == "preference" else n
    at = [int(length * 0.25 * (0.618034 * (b % pairs + 1) % 1)) for b in range(n)]
    return [(a, max(a + 1, math.ceil(length * (0.5 + 0.5 * (0.754878 * (b + 1) % 1))))) for b, a in enumerate(at)]


@functools.lru_cache(maxsize=8)
def _zipf(vocab):
    """The probabilities of a vocabulary's tokens: by rank, as text has them."""
    p = 1 / (torch.arange(vocab, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _quantize(t):
    """(e4m3 values, scales) of a flat tensor of 32 bits whose size is a multiple of 128."""
    b = t.unflatten(0, (-1, BLOCK))
    s = b.abs().amax(-1).clamp(min=1e-30) / 448
    return (b * (1 / s)[:, None]).flatten().to(FP8), s


def _quantize_root(t):
    """The same of a second moment's root: what is over zero stays over it."""
    b = t.unflatten(0, (-1, BLOCK))
    s = b.amax(-1).clamp(min=1e-30) / 448
    q = b * (1 / s)[:, None]
    return torch.where(b > 0, q.clamp(min=FP8_SMALLEST), q).flatten().to(FP8), s


def _shapes(case):
    """The tensors of a model of feed-forward sublayers on the embeddings of the last four tokens."""
    vocab, dim, hidden = case["vocab"], case["dim"], case["hidden"]
    block = [(dim,), (hidden, dim), (hidden, dim), (dim, hidden)]
    return [(vocab, dim // 4)] + case["depth"] * block + [(dim,), (vocab, dim)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPE[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if kind in ("embed", "embed_grad"):
        n, vocab, d = case["n"], case["vocab"], case["d"]
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        tokens = torch.searchsorted(_zipf(vocab).to("cuda").cumsum(0), u).clamp(max=vocab - 1)
        if case["pad"]:  # padding at the end of a batch's sequences
            tokens[n - n // 10:] = 0
        if kind == "embed":
            return case | {"tokens": tokens, "weight": randn(vocab, d).to(dtype), "scale": d ** 0.5}
        return case | {"tokens": tokens, "gy": (randn(n, d) / n).to(dtype), "scale": d ** 0.5,
                       "padding": 0 if case["pad"] else None}
    if kind == "adamw":
        return case | _prepare_adamw(case, randn)
    n, length, vocab = case["sequences"], case["length"], case["vocab"]
    spans = torch.tensor(_spans(case), device="cuda")
    at = torch.arange(length, device="cuda")
    kept = (at >= spans[:, :1]) & (at < spans[:, 1:])
    labels = torch.randint(vocab, (n, length), device="cuda", generator=g)
    logits = torch.empty(n, length, vocab, device="cuda", dtype=dtype)
    logps = torch.empty(n, length, device="cuda", dtype=torch.float64)
    for b in range(n):  # one sequence at a time: the logits in 32 bits are twice those kept
        x = 2 * randn(length, vocab)
        x.scatter_(1, labels[b][:, None], 8 + 2 * randn(length, 1))  # labels that a trained model finds likely
        logits[b] = x.to(dtype)
        x = logits[b].float()
        logps[b] = (x.gather(1, labels[b][:, None])[:, 0] - torch.logsumexp(x, -1)).double()
    labels = torch.where(kept, labels, IGNORE)
    state = {"logits": logits, "labels": labels}
    if kind == "preference":
        # a policy that has moved from the reference: what was chosen likelier, what was rejected less
        sums = (logps * kept).sum(1) / (kept.sum(1) if case["average"] else 1)
        moved = (1 + 2 * randn(n).abs()) * torch.where(torch.arange(n, device="cuda") < n // 2, 1, -1)
        return case | state | {"reference": (sums - moved).float(), "beta": 0.1}
    state |= {"old": (logps + 0.15 * randn(n, length)).float(), "advantages": randn(n)}
    return case | state | {"reference": (logps + 0.3 * randn(n, length)).float() if case["kl"] else None, "clip": (0.2, 0.28)}


def _prepare_adamw(case, randn):
    # all tensors of one kind in one buffer, each at a multiple of 128
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for size in sizes:
        starts.append(total)
        total += -(-size // BLOCK) * BLOCK
    used = torch.zeros(total, device="cuda", dtype=torch.bool)
    for at, size in zip(starts, sizes):
        used[at:at + size] = True
    dtype, bits = DTYPE[case["dtype"]], case["bits"]

    def views(flat):
        return [flat[at:at + size].view(shape) for at, size, shape in zip(starts, sizes, shapes)]

    def blocks(flat):
        return [flat[at // BLOCK:-(-(at + size) // BLOCK)] for at, size in zip(starts, sizes)]

    spread = 1e-3 * torch.exp(randn(total))  # gradients differ in size from weight to weight
    param = torch.where(used, 0.02 * randn(total), 0.0)
    grad = torch.where(used, spread * randn(total), 0.0).to(dtype)
    m, root = torch.where(used, 0.2 * spread * randn(total), 0.0), torch.where(used, spread, 0.0)
    flat = {"param": param.to(dtype), "grad": grad}
    if case["masters"]:
        flat["master"] = param
    if bits == 8:
        (flat["exp_avg"], flat["exp_avg_scale"]), (flat["exp_avg_sq"], flat["exp_avg_sq_scale"]) = _quantize(m), _quantize_root(root)
    else:
        flat["exp_avg"], flat["exp_avg_sq"] = m, root.square()
    return {"flat": flat, "tensors": {k: (blocks if k.endswith("scale") else views)(t) for k, t in flat.items()},
            "step": torch.full((), float(STEP), device="cuda")}


# ---- the plain form -------------------------------------------------------------------------------------------------

def _values(q, s):
    """What a flat tensor held in 8 bits stands for, in 32."""
    return (q.float().unflatten(0, (-1, BLOCK)) * s[:, None]).flatten()


def _plain_embed(s):
    dtype = DTYPE[s["dtype"]]
    if s["kind"] == "embed":
        return {"y": (s["weight"][s["tokens"]].float() * s["scale"]).to(dtype)}
    # sums over thousands of positions: in 64 bits
    gw = torch.zeros(s["vocab"], s["d"], device="cuda", dtype=torch.float64)
    gw.index_add_(0, s["tokens"], s["gy"].double())
    if s["padding"] is not None:
        gw[s["padding"]] = 0
    return {"gweight": (gw * s["scale"]).to(dtype)}


def _plain_rows(s):
    """Of the rows whose labels count: where they are, their labels, exp(x - the largest), its sums, and the labels'
    log-probabilities (in 64 bits: they are added up, and compared with others near to them)."""
    labels = s["labels"].flatten()
    rows = (labels != IGNORE).nonzero()[:, 0]
    x, label = s["logits"].flatten(0, 1)[rows].float(), labels[rows][:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lp = x.gather(1, label).double() - top.double() - total.double().log()
    return rows, label, e, total, lp[:, 0]


def _plain_grad(s, rows, label, e, total, c):
    """The logits' gradient from c, the gradient of each of the rows' log-probabilities."""
    c = c.float()[:, None]
    g = e * (-c / total)
    g.scatter_add_(1, label, c)
    out = torch.zeros_like(s["logits"])
    out.view(-1, s["vocab"])[rows] = g.to(out.dtype)
    return out


def _plain_preference(s):
    n, beta, smooth = s["sequences"], s["beta"], s["smoothing"]
    rows, label, e, total, lp = _plain_rows(s)
    seq = rows // s["length"]
    count = torch.zeros(n, device="cuda", dtype=torch.float64).index_add_(0, seq, torch.ones_like(lp))
    share = 1 / count.clamp(min=1) if s["average"] else torch.ones_like(count)
    ratio = torch.zeros_like(count).index_add_(0, seq, lp) * share - s["reference"].double()
    d = ratio[:n // 2] - ratio[n // 2:]
    if s["loss"] == "sigmoid":
        loss = (1 - smooth) * torch.log1p(torch.exp(-beta * d)) + smooth * torch.log1p(torch.exp(beta * d))
        slope = beta * (smooth - 1 / (1 + torch.exp(beta * d)))
    elif s["loss"] == "hinge":
        loss, slope = (1 - beta * d).clamp(min=0), torch.where(beta * d < 1, -beta, 0.0)
    else:
        loss, slope = (d - 0.5 / beta).square(), 2 * (d - 0.5 / beta)
    c = torch.cat([slope, -slope]) / (n // 2) * share
    return {"loss": loss.mean().float(), "rewards": (beta * ratio).float(), "glogits": _plain_grad(s, rows, label, e, total, c[seq])}


def _plain_policy(s):
    n = s["sequences"]
    rows, label, e, total, lp = _plain_rows(s)
    seq = rows // s["length"]
    count = torch.zeros(n, device="cuda", dtype=torch.float64).index_add_(0, seq, torch.ones_like(lp))
    share = 1 / (count * n) if s["reduction"] == "sequence" else torch.ones_like(count) / count.sum()
    a, ratio = s["advantages"].double()[seq], torch.exp(lp - s["old"].flatten().double()[rows])
    bounded = ratio.clamp(1 - s["clip"][0], 1 + s["clip"][1])
    loss, c = -torch.minimum(ratio * a, bounded * a), torch.where(ratio * a <= bounded * a, -ratio * a, 0.0)
    kl = torch.zeros_like(lp)
    if s["reference"] is not None:
        more = s["reference"].flatten().double()[rows] - lp
        kl = torch.exp(more) - more - 1
        loss, c = loss + s["kl"] * kl, c + s["kl"] * (1 - torch.exp(more))
    logps = torch.zeros(n * s["length"], device="cuda", dtype=torch.float64).index_copy_(0, rows, lp)
    return {"loss": (loss * share[seq]).sum().float(), "kl": (kl * share[seq]).sum().float(),
            "logps": logps.view(n, -1).float(), "glogits": _plain_grad(s, rows, label, e, total, c * share[seq])}


def _plain_adamw(s):
    f, (b1, b2) = s["flat"], BETAS
    p, g = f["master" if s["masters"] else "param"].float(), f["grad"].float()
    if s["bits"] == 8:
        m, v = _values(f["exp_avg"], f["exp_avg_scale"]), _values(f["exp_avg_sq"], f["exp_avg_sq_scale"]).square()
    else:
        m, v = f["exp_avg"], f["exp_avg_sq"]
    step = s["step"].double()
    rate, root = (LR / (1 - b1 ** step)).float(), (1 - b2 ** step).sqrt().float()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p - LR * DECAY * p
    p = p - rate * m / (v.sqrt() / root + EPS)
    if s["masters"]:
        f["master"].copy_(p)
    f["param"].copy_(p)
    if s["bits"] == 8:
        for name, (q, scale) in (("exp_avg", _quantize(m)), ("exp_avg_sq", _quantize_root(v.sqrt()))):
            f[name].copy_(q)
            f[name + "_scale"].copy_(scale)
    else:
        f["exp_avg"].copy_(m)
        f["exp_avg_sq"].copy_(v)
    return _updated(f)


def _updated(flat):
    return {name: t for name, t in flat.items() if name != "grad"}


_PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed, "preference": _plain_preference, "policy": _plain_policy,
          "adamw": _plain_adamw}


# ---- the framework's operators --------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)  # as a program imports it: once
def _hip_ops():
    package = str(pathlib.Path(__file__).resolve().parent.parent / "omarchy-mac-torch_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from omarchy_mac_torch import hip_ops
    return hip_ops


def _own(s):
    ops, kind = _hip_ops(), s["kind"]
    if kind == "embed":
        return {"y": ops.embedding(s["tokens"], s["weight"], scale=s["scale"])}
    if kind == "embed_grad":
        return {"gweight": ops.embedding_backward(s["gy"], s["tokens"], s["vocab"], scale=s["scale"], padding_idx=s["padding"])}
    if kind == "preference":
        loss, rewards, glogits = ops.preference_loss(s["logits"], s["labels"], s["reference"], beta=s["beta"], kind=s["loss"],
                                                     smoothing=s["smoothing"], average=s["average"])
        return {"loss": loss, "rewards": rewards, "glogits": glogits}
    if kind == "policy":
        loss, kl, logps, glogits = ops.policy_loss(s["logits"], s["labels"], s["old"], s["advantages"], reference=s["reference"],
                                                   clip=s["clip"], kl=s["kl"], reduction=s["reduction"])
        return {"loss": loss, "kl": kl, "logps": logps, "glogits": glogits}
    t = s["tensors"]
    ops.adamw(t["param"], t["grad"], t["exp_avg"], t["exp_avg_sq"], s["step"], exp_avg_scales=t.get("exp_avg_scale"),
              exp_avg_sq_scales=t.get("exp_avg_sq_scale"), masters=t.get("master"), lr=LR, betas=BETAS, eps=EPS,
              weight_decay=DECAY)
    return _updated(s["flat"])


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ---- the work that no form can do without ---------------------------------------------------------------------------

def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("embed", "embed_grad"):
        n, vocab, d = case["n"], case["vocab"], case["d"]
        if kind == "embed_grad":
            return {"bytes": 8 * n + (n + vocab) * d * e, "flops": n * d}
        read = n - n // 10 if case["pad"] else n
        distinct = float((1 - (1 - _zipf(vocab)) ** read).sum())  # as many rows as are expected to occur
        return {"bytes": 8 * n + (distinct + n) * d * e, "flops": n * d}
    if kind == "adamw":
        count = sum(math.prod(s) for s in _shapes(case))
        blocks = sum(-(-math.prod(s) // BLOCK) for s in _shapes(case))
        state = 2 * (2 * count + 2 * 4 * blocks if case["bits"] == 8 else 8 * count)  # both states, read and written
        return {"bytes": state + count * (e + (8 + e if case["masters"] else 2 * e)), "flops": 20 * count}
    n, length, vocab = case["sequences"], case["length"], case["vocab"]
    rows = sum(end - first for first, end in _spans(case))
    beside = 8 * n * length + (12 * n * length if kind == "policy" else 8 * n)
    return {"bytes": (rows + n * length) * vocab * e + beside, "flops": 8 * rows * vocab}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_adamw(s):
    f, (b1, b2) = {name: t.double() for name, t in s["flat"].items()}, BETAS
    if s["bits"] == 8:
        m = (f["exp_avg"].view(-1, BLOCK) * f["exp_avg_scale"][:, None]).flatten()
        v = ((f["exp_avg_sq"].view(-1, BLOCK) * f["exp_avg_sq_scale"][:, None]) ** 2).flatten()
    else:
        m, v = f["exp_avg"], f["exp_avg_sq"]
    m, v = torch.lerp(f["grad"], m, b1), torch.lerp(f["grad"] ** 2, v, b2)
    old = f.get("master", f["param"])
    new = old * (1 - LR * DECAY) - LR * (m / (1 - b1 ** STEP)) / ((v / (1 - b2 ** STEP)) ** 0.5 + EPS)
    out = {"param": new, "exp_avg": m, "exp_avg_sq": v}
    if s["masters"]:
        out["master"] = new
    if s["bits"] == 8:  # over the scale, not rounded
        for name, t in (("exp_avg", m), ("exp_avg_sq", v ** 0.5)):
            rows = t.view(-1, BLOCK)
            scale = rows.abs().max(1).values.clamp(min=1e-30) / 448
            out[name], out[name + "_scale"] = (rows / scale[:, None]).flatten(), scale
    return out


def exact(case, seed):
    """From the definitions in 64 bits. A value held in 8 bits has its value over the scale in its place, not rounded."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        return {"y": torch.nn.functional.one_hot(s["tokens"], case["vocab"]).double() @ (s["weight"].double() * s["scale"])} \
            if case["n"] * case["vocab"] < 1 << 26 else {"y": s["weight"].double().mul_(s["scale"]).index_select(0, s["tokens"])}
    if kind == "embed_grad":
        order = torch.argsort(s["tokens"], stable=True)
        sums = s["gy"].double()[order].cumsum(0)  # a token's sum is the difference of two of the running sums
        ends = torch.searchsorted(s["tokens"][order], torch.arange(case["vocab"], device="cuda"), right=True)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])
        gw = sums[ends].diff(dim=0, prepend=sums[:1]) * s["scale"]
        if s["padding"] is not None:
            gw[s["padding"]] = 0
        return {"gweight": gw}
    if kind == "adamw":
        return _exact_adamw(s)
    n, length = s["labels"].shape
    counted = s["labels"] >= 0
    label = s["labels"].clamp(min=0)
    probs = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    for b in range(n):
        torch.softmax(s["logits"][b].double(), -1, out=probs[b])
    # the loss of the log-probabilities by the definition, differentiated by torch, on the host
    lp = probs.gather(2, label[..., None])[..., 0].log().cpu().requires_grad_()
    on, tokens = counted.cpu().double(), counted.sum(1).cpu().double()
    if kind == "preference":
        means = tokens.clamp(min=1) if case["average"] else 1.0
        gain = (lp * on).sum(1) / means - s["reference"].double().cpu()
        d = gain[:n // 2] - gain[n // 2:]
        sig = torch.nn.functional.logsigmoid
        each = {"sigmoid": lambda: -(1 - case["smoothing"]) * sig(s["beta"] * d) - case["smoothing"] * sig(-s["beta"] * d),
                "hinge": lambda: torch.relu(1 - s["beta"] * d), "ipo": lambda: (d - 1 / (2 * s["beta"])) ** 2}[case["loss"]]()
        loss = each.mean()
        out = {"rewards": s["beta"] * gain.detach()}
    else:
        r, a = torch.exp(lp - s["old"].double().cpu()), s["advantages"].double().cpu()[:, None]
        lo, hi = s["clip"]
        far = (r > 1 + hi) & (a > 0) | (r < 1 - lo) & (a < 0)
        each = -a * torch.where(far, torch.where(a > 0, 1 + hi, 1 - lo), r)
        kl = torch.zeros_like(lp)
        if s["reference"] is not None:
            kl = torch.expm1(s["reference"].double().cpu() - lp) - (s["reference"].double().cpu() - lp)
        mean = (lambda t: ((t * on).sum(1) / tokens).mean()) if case["reduction"] == "sequence" else \
            (lambda t: (t * on).sum() / tokens.sum())
        loss = mean(each + case["kl"] * kl)
        out = {"kl": mean(kl).detach(), "logps": (lp * on).detach()}
    c, = torch.autograd.grad(loss, lp)
    c = (c * on).to("cuda")
    glogits = probs.mul_(-c[..., None])
    glogits.scatter_add_(2, label[..., None], c[..., None])
    return out | {"loss": loss.detach(), "glogits": glogits}
