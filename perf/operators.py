"""The feed-forward sublayer of a language model, as cases that can be timed and compared.

The sublayer adds its input to the residual stream, takes the stream's root-mean-square norm, and runs a gated
feed-forward block on it. Kinds of cases:

    norm    training: h = x + residual and y = rms_norm(h) * weight, then both gradients
    norm8   serving: the same sum, and the norm in 8-bit floating point (e4m3) with a scale for each block of 128
    mm8     serving: a matrix product of 8-bit operands, scales by 1 x 128 (activations) and 128 x 128 (weights)
    glu8    serving: act(x Wg^T) * (x Wu^T) of 8-bit operands, its result in 8 bits
    glu     act(x Wg^T) * (x Wu^T) in 32 or 16 bits; for training with what the backward pass needs kept in 8 bits
    glu_bwd its backward pass from those 8-bit checkpoints

A block's scale is its largest magnitude / 448 (1e-30 at least), or, for the checkpoint of x, the next power of two
from there on, so that the values it stands for are exact in bfloat16. Tensors held in 8 bits are returned as they are,
with their scales.
"""

import math
import pathlib
import sys

import torch

own = False

BLOCK = 128
EPS = 1e-6
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
FP8 = torch.float8_e4m3fn


def _norm8(name, m, d, dtype):
    return {"name": name, "kind": "norm8", "m": m, "d": d, "dtype": dtype}


def _norm(name, m, d, dtype):
    return {"name": name, "kind": "norm", "m": m, "d": d, "dtype": dtype}


def _mm8(name, m, n, k, dtype):
    return {"name": name, "kind": "mm8", "m": m, "n": n, "k": k, "dtype": dtype}


def _glu(name, kind, m, k, f, dtype, act="silu", train=True):
    return {"name": name, "kind": kind, "m": m, "k": k, "f": f, "dtype": dtype, "act": act, "train": train}


def listed():
    return [
        # one new token at serving: the smallest call, where the launch counts
        _norm8("norm8_token", 1, 4096, "bf16"),
        # a batch of prompts at serving
        _norm8("norm8_prompt", 8192, 4096, "bf16"),
        # training in 32 bits, a stream of a width of its own and a ragged number of tokens
        _norm("norm_f32_ragged", 3001, 1000, "f32"),
        # training in 16 bits, a large batch of tokens
        _norm("norm_bf16", 8192, 4096, "bf16"),
        # the down projection of one token: the weights are read for a single row
        _mm8("mm8_token", 1, 4096, 8192, "bf16"),
        # the down projection of a prompt
        _mm8("mm8_prompt", 4096, 4096, 8192, "bf16"),
        # a batch of sequences, one new token each
        _glu("glu8_tokens", "glu8", 16, 4096, 8192, "f32"),
        # a prompt through a block of odd sizes: no dimension a multiple of a tile, rows not aligned to 16 bytes
        _glu("glu8_ragged", "glu8", 777, 1928, 2504, "f32", act="gelu"),
        # training in 32 bits
        _glu("glu_f32", "glu", 4096, 1024, 4096, "f32"),
        # training in 16 bits, the largest step
        _glu("glu_bf16", "glu", 8192, 4096, 8192, "bf16"),
        # the backward pass in 32 bits at sizes that no tile divides
        _glu("glu_bwd_f32_ragged", "glu_bwd", 2049, 1000, 2730, "f32", act="gelu"),
        # the backward pass of the largest step
        _glu("glu_bwd_bf16", "glu_bwd", 8192, 4096, 8192, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    step = rng.choice([1, 8, 64, 128, 256])  # most models use round widths
    return w if w < step else w // step * step


def draw(rng):
    kind = rng.choice(["norm", "norm8", "mm8", "mm8", "glu8", "glu", "glu", "glu_bwd"])
    dtype = rng.choice(["f32", "bf16"])
    m = _log(rng, 1, 8192)
    if kind in ("norm", "norm8"):
        return {"kind": kind, "m": m, "d": _width(rng, 64, 4096), "dtype": dtype}
    if kind == "mm8":
        return {"kind": kind, "m": m, "n": _width(rng, 64, 8192), "k": _width(rng, 64, 8192), "dtype": dtype}
    case = {"kind": kind, "m": m, "k": _width(rng, 64, 4096), "f": _width(rng, 64, 8192), "dtype": dtype,
            "act": rng.choice(["silu", "gelu", "relu"]), "train": kind != "glu" or rng.random() < 0.6}
    if kind == "glu8":
        case["dtype"] = "f32"
    if dtype == "f32" and m > 4096:  # a product in 32 bits takes several times as long
        case["m"] = m // 2
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _pad_blocks(t):
    d = t.shape[-1]
    return torch.nn.functional.pad(t, (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))


def _quantize(t, pow2=False):
    """(e4m3 values, scales) of a tensor of 32 bits, by blocks of 128 along its last dimension."""
    b = _pad_blocks(t)
    s = b.abs().amax(-1).clamp(min=1e-30) / 448
    if pow2:
        frac, exp = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), exp - (frac == 0.5).to(exp.dtype))
    return (b / s[..., None]).flatten(-2)[..., :t.shape[-1]].to(FP8), s


def _quantize_weight(w):
    """(e4m3 values, scales) of a matrix, by blocks of 128 x 128."""
    n, k = w.shape
    b = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    b = b.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))
    s = b.abs().amax((1, 3)).clamp(min=1e-30) / 448
    q = (b / s[:, None, :, None]).flatten(2).flatten(0, 1)[:n, :k]
    return q.to(FP8).contiguous(), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, m, dtype = case["kind"], case["m"], DTYPE[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if kind in ("norm", "norm8"):
        d = case["d"]
        # a stream whose channels differ in size, and tokens too, as layers add to it
        stream = randn(m, d) * torch.exp(0.5 * randn(d)) * torch.exp(0.3 * randn(m, 1))
        state = {"x": randn(m, d).to(dtype), "residual": (2 * stream).to(dtype),
                 "weight": (1 + 0.2 * randn(d)).to(dtype)}
        if kind == "norm":
            state |= {"gy": (randn(m, d) / m).to(dtype), "gh": (randn(m, d) / m).to(dtype)}
        return case | state
    if kind == "mm8":
        n, k = case["n"], case["k"]
        a, sa = _quantize(randn(m, k) * torch.exp(0.3 * randn(m, 1)))
        b, sb = _quantize_weight(randn(n, k) * k ** -0.5)
        return case | {"a": a.contiguous(), "sa": sa, "b": b, "sb": sb}
    k, f = case["k"], case["f"]
    x = randn(m, k) * torch.exp(0.2 * randn(k))
    if kind == "glu_bwd":  # what the forward pass kept: x and both projections in 8 bits
        kept = _quantize(x.to(dtype).float(), pow2=True) + _quantize(randn(m, f)) + _quantize(randn(m, f))
    wg, wu = randn(f, k) * k ** -0.5, randn(f, k) * k ** -0.5
    if kind == "glu8":
        (xq, sx), (gq, sg), (uq, su) = _quantize(x), _quantize_weight(wg), _quantize_weight(wu)
        return case | {"x": xq.contiguous(), "sx": sx, "wg": gq, "sg": sg, "wu": uq, "su": su}
    if kind == "glu":
        return case | {"x": x.to(dtype), "wg": wg.to(dtype), "wu": wu.to(dtype)}
    return case | {"kept": [t.contiguous() for t in kept], "gh": (randn(m, f) / m).to(dtype), "wg": wg.to(dtype),
                   "wu": wu.to(dtype)}


# ---- the plain form -------------------------------------------------------------------------------------------------

def _values(q, s):
    """What a tensor held in 8 bits stands for, in 32."""
    return q.float() * s.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def _weight_values(q, s):
    return _values(q, s.repeat_interleave(BLOCK, 0)[:q.shape[0]])


def _act(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "gelu":
        return g * 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g.clamp(min=0)


def _act_grad(g, act):
    if act == "silu":
        p = torch.sigmoid(g)
        return p * (1 + g * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return (g > 0).to(g.dtype)


def _plain(s):
    kind, dtype = s["kind"], DTYPE[s["dtype"]]
    if kind in ("norm", "norm8"):
        h = (s["x"].float() + s["residual"].float()).to(dtype)  # the stream is handed on in its own type, and so normed
        hf, w = h.float(), s["weight"].float()
        r = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
        if kind == "norm8":
            q, scale = _quantize(hf * r * w)
            return {"q": q, "scale": scale, "h": h}
        gy, gh = s["gy"].float(), s["gh"].float()
        n, gn = hf * r, gy * w
        gx = gh + r * (gn - n * (gn * n).mean(-1, keepdim=True))
        return {"y": (n * w).to(dtype), "h": h, "gx": gx.to(dtype), "gweight": (gy * n).sum(0).to(dtype)}
    if kind == "mm8":
        return (_values(s["a"], s["sa"]) @ _weight_values(s["b"], s["sb"]).T).to(dtype)
    if kind == "glu8":
        x = _values(s["x"], s["sx"])
        g, u = x @ _weight_values(s["wg"], s["sg"]).T, x @ _weight_values(s["wu"], s["su"]).T
        q, scale = _quantize(_act(g, s["act"]) * u)
        return {"q": q, "scale": scale}
    wg, wu = s["wg"].float(), s["wu"].float()
    if kind == "glu":
        x = s["x"].float()
        g, u = x @ wg.T, x @ wu.T
        h = (_act(g, s["act"]) * u).to(dtype)
        if not s["train"]:
            return {"h": h}
        kept = _quantize(x, pow2=True) + _quantize(g) + _quantize(u)
        return {"h": h, "kept": list(kept)}
    xq, sx, gq, sg, uq, su = s["kept"]
    x, g, u, gh = _values(xq, sx), _values(gq, sg), _values(uq, su), s["gh"].float()
    gg, gu = gh * u * _act_grad(g, s["act"]), gh * _act(g, s["act"])
    return {"gx": (gg @ wg + gu @ wu).to(dtype), "gwg": (gg.T @ x).to(dtype), "gwu": (gu.T @ x).to(dtype)}


# ---- the framework's operators --------------------------------------------------------------------------------------

def _hip_ops():
    package = str(pathlib.Path(__file__).resolve().parent.parent / "omarchy-mac-torch_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from omarchy_mac_torch import hip_ops
    return hip_ops


def _own(s):
    ops, kind = _hip_ops(), s["kind"]
    if kind == "norm8":
        q, scale, h = ops.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return {"q": q, "scale": scale, "h": h}
    if kind == "norm":
        y, h, rstd = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        gx, gweight = ops.rms_norm_backward(s["gy"], h, s["weight"], rstd, gh=s["gh"])
        return {"y": y, "h": h, "gx": gx, "gweight": gweight}
    if kind == "mm8":
        return ops.matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], dtype=DTYPE[s["dtype"]])
    if kind == "glu8":
        q, scale = ops.glu_fp8(s["x"], s["sx"], s["wg"], s["sg"], s["wu"], s["su"], act=s["act"])
        return {"q": q, "scale": scale}
    if kind == "glu":
        h, kept = ops.glu(s["x"], s["wg"], s["wu"], act=s["act"], checkpoint="fp8" if s["train"] else None)
        return {"h": h, "kept": list(kept)} if s["train"] else {"h": h}
    gx, gwg, gwu = ops.glu_backward(s["gh"], s["kept"], s["wg"], s["wu"], act=s["act"])
    return {"gx": gx, "gwg": gwg, "gwu": gwu}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the work that no form can do without ---------------------------------------------------------------------------

def _held8(rows, cols):
    return rows * cols + 4 * rows * math.ceil(cols / BLOCK)


def _weight8(rows, cols):
    return rows * cols + 4 * math.ceil(rows / BLOCK) * math.ceil(cols / BLOCK)


def work(case):
    kind, m, e = case["kind"], case["m"], SIZE[case["dtype"]]
    if kind == "norm8":
        d = case["d"]
        return {"bytes": 3 * m * d * e + d * e + _held8(m, d), "flops": 8 * m * d}
    if kind == "norm":
        d = case["d"]
        return {"bytes": 7 * m * d * e + 2 * d * e, "flops": 16 * m * d}
    if kind == "mm8":
        n, k = case["n"], case["k"]
        return {"bytes": _held8(m, k) + _weight8(n, k) + m * n * e, "flops": 2 * m * n * k}
    k, f = case["k"], case["f"]
    if kind == "glu8":
        return {"bytes": _held8(m, k) + 2 * _weight8(f, k) + _held8(m, f), "flops": 4 * m * k * f}
    kept = _held8(m, k) + 2 * _held8(m, f)
    if kind == "glu":
        return {"bytes": (m * k + 2 * f * k + m * f) * e + (kept if case["train"] else 0), "flops": 4 * m * k * f}
    return {"bytes": kept + (m * f + m * k + 4 * f * k) * e, "flops": 8 * m * k * f}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _scales64(v, pow2=False):
    """The scale of each block of 128 along the last dimension, from its largest magnitude."""
    n = -(-v.shape[-1] // BLOCK)
    big = torch.zeros(*v.shape[:-1], n, dtype=torch.float64, device=v.device)
    for i in range(n):
        big[..., i] = v[..., BLOCK * i:BLOCK * (i + 1)].abs().max(-1).values
    s = torch.maximum(big, torch.full_like(big, 1e-30)) / 448
    if not pow2:
        return s
    e = torch.log2(s)
    near = e.round()  # a power of two itself, whatever the logarithm's last bit
    return 2.0 ** torch.where((e - near).abs() < 1e-12, near, e.ceil())


def _spread(s, cols):
    return s[..., torch.arange(cols, device=s.device) // BLOCK]


def _in8(v, pow2=False):
    """What 8 bits and a scale stand for, before the values are rounded: v / scale, and the scale."""
    s = _scales64(v, pow2)
    return [v / _spread(s, v.shape[-1]), s]


def _phi(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return x * torch.special.ndtr(x)
    return torch.where(x > 0, x, torch.zeros_like(x))


def _dphi(x, act):
    if act == "silu":
        e = torch.exp(-x)
        return (1 + e + x * e) / (1 + e) ** 2
    if act == "gelu":
        return torch.special.ndtr(x) + x * torch.exp(-x * x / 2) / (2 * math.pi) ** 0.5
    return torch.where(x > 0, torch.ones_like(x), torch.zeros_like(x))


def exact(case, seed):
    """From the definitions in 64 bits. A value held in 8 bits has its value over the scale in its place, not rounded."""
    s = prepare(case, seed)
    d = {name: t.double() for name, t in s.items() if isinstance(t, torch.Tensor)}
    kind = case["kind"]
    if kind in ("norm", "norm8"):
        total = d["x"] + d["residual"]
        h = total.to(DTYPE[case["dtype"]]).double()
        rms = torch.sqrt((h * h).sum(-1) / h.shape[-1] + EPS)[:, None]
        y = h / rms * d["weight"]
        if kind == "norm8":
            q, scale = _in8(y)
            return {"q": q, "scale": scale, "h": total}
        # d y_j / d h_i = w_j (delta_ij / rms - h_i h_j / (D rms^3))
        inner = (d["gy"] * d["weight"] * h).sum(-1, keepdim=True)
        gx = d["gh"] + d["gy"] * d["weight"] / rms - h * inner / (h.shape[-1] * rms ** 3)
        return {"y": y, "h": total, "gx": gx, "gweight": (d["gy"] * h / rms).sum(0)}
    if kind == "mm8":
        rows = torch.arange(case["n"], device="cuda") // BLOCK
        return (d["a"] * _spread(d["sa"], case["k"])) @ (d["b"] * _spread(d["sb"], case["k"])[rows]).T
    if kind == "glu8":
        rows = torch.arange(case["f"], device="cuda") // BLOCK
        x = d["x"] * _spread(d["sx"], case["k"])
        g = x @ (d["wg"] * _spread(d["sg"], case["k"])[rows]).T
        u = x @ (d["wu"] * _spread(d["su"], case["k"])[rows]).T
        q, scale = _in8(_phi(g, case["act"]) * u)
        return {"q": q, "scale": scale}
    if kind == "glu":
        g, u = d["x"] @ d["wg"].T, d["x"] @ d["wu"].T
        h = _phi(g, case["act"]) * u
        return {"h": h, "kept": _in8(d["x"], pow2=True) + _in8(g) + _in8(u)} if case["train"] else {"h": h}
    x, g, u = (q.double() * _spread(scale.double(), q.shape[-1]) for q, scale in zip(s["kept"][::2], s["kept"][1::2]))
    gu = d["gh"] * _phi(g, case["act"])
    gg = d["gh"] * _dphi(g, case["act"]) * u
    return {"gx": gg @ d["wg"] + gu @ d["wu"], "gwg": gg.T @ x, "gwu": gu.T @ x}
