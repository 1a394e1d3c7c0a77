"""The feed-forward sublayer's operators (norm with the residual's addition, 8-bit quantization and matrix products, the
gated block with its 8-bit checkpoints and its backward) against their definitions in float64 on the CPU.

Tolerances, relative 2-norm: a sum of k terms in float32 is within (8 + 2 sqrt(k)) 2^-24 of its value relative to the
sum's own size for terms of random signs, twice that where both operands are first split into two 11-bit halves; a
result rounded to bfloat16 (8 bits) adds 2^-8 at most, an operand rounded to bfloat16 another. An e4m3 value is within 2^-4 of
what it stands for, or within half of e4m3's smallest step, 2^-10, times the scale; a value that lies between two
neighbours to within float32's error may go to either."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


def rnd(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def rel(got, want):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    return float((got - want).norm() / want.norm().clamp(min=1e-300))


def tol(k, dtype, rounded=0):
    return (16 + 4 * math.sqrt(k)) * 2 ** -24 + ((1 + rounded) * 2 ** -8 if dtype == BF16 else 0)


def spread(s, cols):
    return s.repeat_interleave(BLOCK, -1)[..., :cols]


def values(q, s):
    return q.float().cpu().double() * spread(s.cpu().double(), q.shape[-1])


def weight_values(q, s):
    return values(q, s.cpu().repeat_interleave(BLOCK, 0)[:q.shape[0]])


def scales_of(v):
    pad = torch.nn.functional.pad(v.abs(), (0, -v.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    return pad.amax(-1).clamp(min=1e-30) / 448


def check_fp8(q, s, want, slack=2e-5, exact_scale=None):
    """q, s stand for `want` (float64, itself known to `slack` of its row's size)."""
    scale = scales_of(want) if exact_scale is None else exact_scale
    assert q.dtype == FP8 and s.dtype == F32 and s.shape == scale.shape
    top = want.abs().amax(-1, keepdim=True)
    assert bool(((s.double().cpu() - scale).abs() <= slack * torch.maximum(scale, top / 448)).all())
    sc = spread(s.double().cpu(), want.shape[-1])
    off = (values(q, s) - want).abs()
    assert bool((off <= torch.maximum(want.abs() * 2 ** -4, sc * 2 ** -10) * (1 + 1e-4) + slack * top).all())


def to(t, dtype, cuda):
    return t.to(dtype).to(cuda)


ACT = {"silu": lambda g: g * torch.sigmoid(g), "gelu": lambda g: g * torch.special.ndtr(g), "relu": torch.relu}


def act_grad(g, act):
    g = g.clone().requires_grad_(True)
    ACT[act](g).sum().backward()
    return g.grad


# ---- the norm -------------------------------------------------------------------------------------------------------

DIMS = [1, 7, 8, 128, 129, 512, 520, 1000, 1025, 2048, 2056, 4099, 8192, 8200, 16384, 16390, 32768]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rms_norm_forward_and_backward(ops, cuda, dim, dtype):
    rows, eps = (5, 1e-6) if dim > 4 else (70, 1e-5)
    x, res, gy, gh = (rnd((rows, dim), s) for s in (1, 2, 3, 4))
    x, res, gy, gh = (t.to(dtype) for t in (x * torch.exp(rnd((rows, 1), 9)), 2 * res, gy, gh))
    w32 = (1 + 0.2 * rnd((dim,), 5)).to(F32)
    for weight, residual in ((w32.to(dtype), res), (w32, None)):
        h = (x.float() + residual.float()).to(dtype).double() if residual is not None else x.double()
        wd, gyd, ghd = weight.double(), gy.double(), gh.double()
        r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
        dx = lambda t: None if t is None else t.to(cuda)  # noqa: E731
        y, hk, rstd = ops.rms_norm(dx(x), dx(weight), dx(residual), eps)
        assert y.dtype == dtype and hk.dtype == dtype and rel(y, h * r * wd) <= tol(dim, dtype)
        assert torch.equal(hk.cpu().double(), h) and rel(rstd, r[:, 0]) <= tol(dim, F32)
        q, s, hk8 = ops.rms_norm_fp8(dx(x), dx(weight), dx(residual), eps)
        assert torch.equal(hk8, hk)
        check_fp8(q, s, h * r * wd)
        n, g = h * r, gyd * wd
        for use_gh in (True, False):
            want = r * (g - n * (g * n).mean(-1, keepdim=True)) + (ghd if use_gh else 0)
            gx, gw = ops.rms_norm_backward(dx(gy), hk, dx(weight), rstd, gh=dx(gh) if use_gh else None)
            # dim 1: the two terms cancel; the error is float32's of each
            size = r * g.abs() + (ghd.abs() if use_gh else 0)
            assert float((gx.double().cpu() - want).norm() / size.norm()) <= tol(dim, dtype)
            assert gw.dtype == weight.dtype and rel(gw, (gyd * n).sum(0)) <= tol(rows, weight.dtype) + 1e-6
        again = ops.rms_norm_backward(dx(gy), hk, dx(weight), rstd, gh=dx(gh))
        first = ops.rms_norm_backward(dx(gy), hk, dx(weight), rstd, gh=dx(gh))
        assert all(torch.equal(a, b) for a, b in zip(again, first))


@pytest.mark.parametrize("rows,dim", [(4097, 96), (3001, 1000), (1500, 4104)])
def test_rms_norm_weight_gradient_over_many_rows(ops, cuda, rows, dim):
    h, gy = rnd((rows, dim), 1).float(), rnd((rows, dim), 2).float()
    w = torch.ones(dim)
    y, _, rstd = ops.rms_norm(h.to(cuda), w.to(cuda))
    _, gw = ops.rms_norm_backward(gy.to(cuda), h.to(cuda), w.to(cuda), rstd)
    n = h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-6)
    assert rel(gw, (gy.double() * n).sum(0)) <= tol(rows, F32)
    assert rel(y, n) <= tol(dim, F32)


def test_rms_norm_gradient_against_differences(ops, cuda):
    """<gradient, d> against (L(x + t d) - L(x - t d)) / 2t, L = <y, c> + <h, e>: the difference is within t^2 of the
    derivative relative to the terms' size, and float32 adds 2^-22 / t."""
    rows, dim, t = 6, 200, 2 ** -7
    x, d, c, e = (rnd((rows, dim), s).float() for s in (1, 2, 3, 4))
    w, dw = (1 + 0.1 * rnd((dim,), 5)).float(), rnd((dim,), 6).float()
    dx = lambda v: v.to(cuda)  # noqa: E731
    zero = torch.zeros_like(x)

    def loss(xv, wv):
        y, h, _ = ops.rms_norm(dx(xv), dx(wv), dx(zero))
        return float((y.double().cpu() * c.double()).sum() + (h.double().cpu() * e.double()).sum())

    _, h, rstd = ops.rms_norm(dx(x), dx(w), dx(zero))
    gx, gw = ops.rms_norm_backward(dx(c), h, dx(w), rstd, gh=dx(e))
    size = math.sqrt(rows * dim)
    for got, diff in ((float((gx.cpu() * d).sum()), (loss(x + t * d, w) - loss(x - t * d, w)) / (2 * t)),
                      (float((gw.cpu() * dw).sum()), (loss(x, w + t * dw) - loss(x, w - t * dw)) / (2 * t))):
        assert abs(got - diff) <= 10 * size * (t * t + 2 ** -22 / t)


def test_rms_norm_keeps_a_row_to_itself(ops, cuda):
    """NaN and infinities reach their own row alone; a row of zeros gives zeros."""
    x = rnd((6, 300), 1).float()
    x[1, 5], x[3, 299], x[4] = float("nan"), float("inf"), 0
    w = torch.ones(300)
    y, _, _ = ops.rms_norm(x.to(cuda), w.to(cuda))
    q, s, _ = ops.rms_norm_fp8(x.to(cuda), w.to(cuda))
    y, v = y.cpu(), values(q, s)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().any()) and bool((y[4] == 0).all()) and bool((v[4] == 0).all())
    for i in (0, 2, 5):
        assert bool(y[i].isfinite().all()) and bool(v[i].isfinite().all())
    assert bool(v[1].isnan().all())


# ---- 8 bits -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (2, 5, 128), (70, 129), (33, 1000), (9, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_fp8(ops, cuda, shape, dtype):
    x = (rnd(shape, 1) * torch.exp(2 * rnd((*shape[:-1], 1), 2))).to(dtype)
    q, s = ops.quantize_fp8(x.to(cuda))
    check_fp8(q, s, x.double(), slack=2 ** -22)
    q, s = ops.quantize_fp8(x.to(cuda), pow2=True)
    t = scales_of(x.double())
    frac, exp = torch.frexp(t)
    check_fp8(q, s, x.double(), slack=0, exact_scale=torch.ldexp(torch.ones_like(t), exp - (frac == 0.5).long()))
    # rounded to nearest even, as torch rounds
    assert torch.equal(q.cpu().float(), (x.float() / spread(s.cpu(), shape[-1])).to(FP8).float())


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 300), (257, 136)])
def test_quantize_fp8_weight(ops, cuda, shape):
    w = rnd(shape, 3).float()
    q, s = ops.quantize_fp8_weight(w.to(cuda))
    n, k = shape
    pad = torch.nn.functional.pad(w.double().abs(), (0, -k % BLOCK, 0, -n % BLOCK))
    want = pad.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK)).amax((1, 3)) / 448
    assert torch.allclose(s.cpu().double(), want, rtol=2 ** -22, atol=0)
    off = (weight_values(q, s) - w.double()).abs()
    step = s.cpu().double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k] * 2 ** -10
    assert bool((off <= torch.maximum(w.double().abs() * 2 ** -4, step) * (1 + 1e-5)).all())


def test_quantize_fp8_of_zeros_extremes_and_what_is_not_finite(ops, cuda):
    x = torch.ones(6, 256)
    x[0] = 0
    x[1, 3], x[2, 200], x[3, 0] = float("nan"), -float("inf"), 3e38
    x[4] = 1e-38
    x[5, :128] = 448 * 2.0 ** torch.arange(128).sub(100)
    for pow2 in (False, True):
        q, s = ops.quantize_fp8(x.to(cuda), pow2=pow2)
        v, s = values(q, s), s.cpu()
        assert bool((v[0] == 0).all()) and bool((s[0] > 0).all()) and bool(s[0].isfinite().all())
        assert bool(v[1, :128].isnan().all()) and bool((v[1, 128:] - 1).abs().le(2 ** -4).all())
        assert bool(v[2, 128:].isnan().all()) and bool((v[2, :128] - 1).abs().le(2 ** -4).all())
        assert bool(v[3].isfinite().all()) and abs(float(v[3, 0]) / 3e38 - 1) <= 2 ** -4
        assert bool((v[4].abs() <= 1e-32).all())
        top = float(x[5, :128].max())
        assert float(s[5, 0]) == top / 448 and float(v[5, 127]) == top


# ---- products of 8-bit operands ------------------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 5, 128), (2, 256, 16), (16, 256, 128), (17, 257, 129), (64, 300, 1000), (65, 129, 144),
         (130, 513, 2056), (3, 2, 8192), (257, 260, 384), (300, 1000, 2048), (1, 4096, 2048)]


def fp8_operands(m, n, k, seed, cuda):
    from omarchy_mac_torch import hip_ops
    a = (rnd((m, k), seed) * torch.exp(rnd((m, 1), seed + 1))).float().to(cuda)
    b = (rnd((n, k), seed + 2) * k ** -0.5).float().to(cuda)
    return hip_ops.quantize_fp8(a) + hip_ops.quantize_fp8_weight(b)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul_fp8(ops, cuda, m, n, k):
    a, sa, b, sb = fp8_operands(m, n, k, 10, cuda)
    want = values(a, sa) @ weight_values(b, sb).T
    for dtype in (F32, BF16):
        got = ops.matmul_fp8(a, sa, b, sb, dtype=dtype)
        assert got.dtype == dtype and rel(got, want) <= tol(k, dtype)
        assert torch.equal(got, ops.matmul_fp8(a, sa, b, sb, dtype=dtype))


def test_matmul_fp8_leading_dimensions_strides_and_offsets(ops, cuda):
    a, sa, b, sb = fp8_operands(24, 200, 272, 20, cuda)
    want = ops.matmul_fp8(a, sa, b, sb, dtype=F32)
    got = ops.matmul_fp8(a.view(2, 3, 4, 272), sa.view(2, 3, 4, 3), b, sb, dtype=F32)
    assert torch.equal(got.view(24, 200), want)
    wide = torch.zeros(24, 300, device=cuda, dtype=torch.uint8)
    wide[:, 5:277] = a.view(torch.uint8)  # rows of another stride, off 16 bytes
    assert torch.equal(ops.matmul_fp8(wide[:, 5:277].view(FP8), sa, b, sb, dtype=F32), want)
    flat = torch.zeros(200 * 272 + 3, device=cuda, dtype=torch.uint8)
    flat[3:] = b.view(torch.uint8).reshape(-1)
    assert torch.equal(ops.matmul_fp8(a, sa, flat[3:].view(FP8).view(200, 272), sb, dtype=F32), want)
    assert ops.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 200)


def test_matmul_fp8_what_is_not_finite_stays_in_its_row(ops, cuda):
    a, sa, b, sb = fp8_operands(70, 140, 300, 30, cuda)
    sa[3, 1], sa[69, 2] = float("nan"), float("inf")
    got = ops.matmul_fp8(a, sa, b, sb, dtype=F32).cpu()
    bad = torch.zeros(70, dtype=torch.bool)
    bad[3] = bad[69] = True
    assert bool((~got[bad].isfinite()).all()) and bool(got[~bad].isfinite().all())


# ---- the gated block ---------------------------------------------------------------------------------------------------------

GLU_SIZES = [(1, 1, 1), (1, 512, 256), (3, 7, 5), (16, 64, 128), (17, 65, 129), (64, 100, 300), (70, 136, 384),
             (129, 1000, 130), (260, 512, 700), (2, 2048, 1030), (520, 320, 513)]


def glu_operands(m, k, f, dtype, seed=40):
    x = (rnd((m, k), seed) * torch.exp(0.3 * rnd((k,), seed + 1))).to(dtype)
    wg, wu = ((rnd((f, k), seed + 2 + i) * k ** -0.5).to(dtype) for i in range(2))
    return x, wg, wu


@pytest.mark.parametrize("m,k,f", GLU_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_glu_forward(ops, cuda, m, k, f, dtype):
    x, wg, wu = glu_operands(m, k, f, dtype)
    act = ["silu", "gelu", "relu"][(m + k + f) % 3]
    g, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    want = ACT[act](g) * u
    d = [t.to(cuda) for t in (x, wg, wu)]
    h, none = ops.glu(*d, act=act)
    assert none is None and h.dtype == dtype and rel(h, want) <= 2 * tol(k, dtype)
    h8, kept = ops.glu(*d, act=act, checkpoint="fp8")
    assert torch.equal(h8, h)
    q, s = ops.quantize_fp8(d[0], pow2=True)
    assert torch.equal(kept[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(kept[1], s)
    check_fp8(kept[2], kept[3], g)
    check_fp8(kept[4], kept[5], u)
    hf, full = ops.glu(*d, act=act, checkpoint="full")
    assert torch.equal(hf, h) and full[0] is d[0]
    assert rel(full[2], g) <= tol(k, dtype) and rel(full[4], u) <= tol(k, dtype)


@pytest.mark.parametrize("m,k,f", GLU_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("checkpoint", ["fp8", "full"])
def test_glu_backward(ops, cuda, m, k, f, dtype, checkpoint):
    x, wg, wu = glu_operands(m, k, f, dtype)
    act = ["silu", "gelu", "relu"][(m + k + f) % 3]
    gh = rnd((m, f), 50).to(dtype)
    d = [t.to(cuda) for t in (x, wg, wu)]
    _, kept = ops.glu(*d, act=act, checkpoint=checkpoint)
    if checkpoint == "fp8":
        xv, g, u = (values(kept[i], kept[i + 1]) for i in (0, 2, 4))
    else:
        xv, g, u = (kept[i].double().cpu() for i in (0, 2, 4))
    dg, du = gh.double() * u * act_grad(g, act), gh.double() * ACT[act](g)
    got = ops.glu_backward(gh.to(cuda), kept, d[1], d[2], act=act)
    want = (dg @ wg.double() + du @ wu.double(), dg.T @ xv, du.T @ xv)
    for a, b, terms in zip(got, want, (2 * f, m, m)):
        # the operands dg and du are rounded to bfloat16 where that is the type
        assert a.dtype == dtype and rel(a, b) <= 2 * tol(terms, dtype, rounded=1)
    only_x = ops.glu_backward(gh.to(cuda), kept, d[1], d[2], act=act, weight_grad=False)
    only_w = ops.glu_backward(gh.to(cuda), kept, d[1], d[2], act=act, input_grad=False)
    assert only_x[1] is None and only_w[0] is None
    assert torch.equal(only_x[0], got[0]) and all(torch.equal(a, b) for a, b in zip(only_w[1:], got[1:]))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_glu_gradient_against_differences(ops, cuda, act):
    """As for the norm: L = <h, c>, along random directions of x and of both weights."""
    m, k, f, t = 9, 40, 70, 2 ** -8
    x, wg, wu = glu_operands(m, k, f, F32)
    c = rnd((m, f), 60).float()
    dirs = [rnd(v.shape, 61 + i, scale=float(v.std())).float() for i, v in enumerate((x, wg, wu))]

    def loss(*v):
        return float((ops.glu(*[a.to(cuda) for a in v], act=act)[0].double().cpu() * c.double()).sum())

    d = [v.to(cuda) for v in (x, wg, wu)]
    _, kept = ops.glu(*d, act=act, checkpoint="full")
    grads = ops.glu_backward(c.to(cuda), kept, d[1], d[2], act=act)
    size = math.sqrt(m * f)
    for i, grad in enumerate(grads):
        v = [x, wg, wu]
        up, down = list(v), list(v)
        up[i], down[i] = v[i] + t * dirs[i], v[i] - t * dirs[i]
        diff = (loss(*up) - loss(*down)) / (2 * t)
        assert abs(float((grad.cpu().double() * dirs[i].double()).sum()) - diff) <= 20 * size * (t * t + 2 ** -22 / t)


@pytest.mark.parametrize("m,k,f", GLU_SIZES)
def test_glu_fp8(ops, cuda, m, k, f):
    x, wg, wu = (t.to(cuda) for t in glu_operands(m, k, f, F32))
    act = ["silu", "gelu", "relu"][(m + k + f) % 3]
    (xq, xs), (gq, gs), (uq, us) = ops.quantize_fp8(x), ops.quantize_fp8_weight(wg), ops.quantize_fp8_weight(wu)
    xv = values(xq, xs)
    want = ACT[act](xv @ weight_values(gq, gs).T) * (xv @ weight_values(uq, us).T)
    q, s = ops.glu_fp8(xq, xs, gq, gs, uq, us, act=act)
    check_fp8(q, s, want)


def test_glu_empty_and_what_is_not_finite(ops, cuda):
    x, wg, wu = (t.to(cuda) for t in glu_operands(20, 96, 130, F32))
    x[3, 7], x[11, 0] = float("nan"), float("inf")
    h, kept = ops.glu(x, wg, wu, checkpoint="fp8")
    bad = torch.zeros(20, dtype=torch.bool)
    bad[3] = bad[11] = True
    assert bool((~h.cpu()[bad].isfinite()).any(-1).all()) and bool(h.cpu()[3].isnan().all())
    assert bool(h.cpu()[~bad].isfinite().all()) and bool(values(kept[2], kept[3])[~bad].isfinite().all())
    empty, kept = ops.glu(x[:0], wg, wu, checkpoint="fp8")
    assert empty.shape == (0, 130)
    gx, gwg, gwu = ops.glu_backward(empty, kept, wg, wu)
    assert gx.shape == (0, 96) and bool((gwg == 0).all()) and bool((gwu == 0).all())


# ---- streams, graphs, refusals ---------------------------------------------------------------------------------------------------

def sublayer(ops, x, res, w, wg, wu, gh):
    y, h, rstd = ops.rms_norm(x, w, res)
    a, kept = ops.glu(y, wg, wu, checkpoint="fp8")
    gy, gwg, gwu = ops.glu_backward(gh, kept, wg, wu)
    return (h, a, gwg, gwu) + ops.rms_norm_backward(gy, h, w, rstd, gh=x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_on_another_stream_and_in_a_graph(ops, cuda, dtype):
    m, k, f = 130, 192, 260
    x, wg, wu = (t.to(cuda) for t in glu_operands(m, k, f, dtype))
    res, gh, w = to(rnd((m, k), 70), dtype, cuda), to(rnd((m, f), 71), dtype, cuda), to(1 + 0.1 * rnd((k,), 72), dtype, cuda)
    args = (x, res, w, wg, wu, gh)
    want = sublayer(ops, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sublayer(ops, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sublayer(ops, *args)
    for i in range(4):
        x.mul_(0.5).add_(i)
        want = sublayer(ops, *args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals(ops, cuda):
    x, w = torch.ones(4, 256, device=cuda), torch.ones(256, device=cuda)
    q, s = ops.quantize_fp8(x)
    wq, ws = ops.quantize_fp8_weight(x)
    from omarchy_mac_torch._lib import Unsupported
    for error, call in [
            (TypeError, lambda: ops.rms_norm(x.half(), w)), (TypeError, lambda: ops.rms_norm(x.cpu(), w)),
            (TypeError, lambda: ops.rms_norm(x, w.bfloat16())), (ValueError, lambda: ops.rms_norm(x, w[:8])),
            (ValueError, lambda: ops.rms_norm(x, w, x[:2])), (TypeError, lambda: ops.rms_norm(x, w, x.bfloat16())),
            (Unsupported, lambda: ops.rms_norm(torch.ones(1, 32769, device=cuda), torch.ones(32769, device=cuda))),
            (ValueError, lambda: ops.rms_norm_backward(x, x, w, torch.ones(3, device=cuda))),
            (TypeError, lambda: ops.quantize_fp8(x.long())), (ValueError, lambda: ops.quantize_fp8_weight(w)),
            (ValueError, lambda: ops.quantize_fp8(x[:, :0])),
            (TypeError, lambda: ops.matmul_fp8(x, s, wq, ws)), (ValueError, lambda: ops.matmul_fp8(q, s[:, :1], wq, ws)),
            (ValueError, lambda: ops.matmul_fp8(q[:, :128], s[:, :1], wq, ws)),
            (TypeError, lambda: ops.matmul_fp8(q, s, wq, ws, dtype=torch.float16)),
            (TypeError, lambda: ops.matmul_fp8(q, s.double(), wq, ws)),
            (ValueError, lambda: ops.glu(x, x, x, act="tanh")), (ValueError, lambda: ops.glu(x, x, x, checkpoint="int8")),
            (TypeError, lambda: ops.glu(x, x.bfloat16(), x.bfloat16())), (ValueError, lambda: ops.glu(x, x, x[:2])),
            (ValueError, lambda: ops.glu(x, x[:, :8], x[:, :8])),
            (ValueError, lambda: ops.glu_fp8(q, s, wq, ws, wq[:2], ws)),
            (ValueError, lambda: ops.glu_backward(x, (x, None, x, None), x, x)),
            (ValueError, lambda: ops.glu_backward(x, (x, None, x[:2], None, x, None), x[:, :8], x[:, :8]))]:
        with pytest.raises(error):
            call()


# ---- every tile, in every mode, a workgroup's own and shared --------------------------------------------------------------------

# (operator, type, m, k, n): the smallest of 60000 random sizes for each combination of operator, mode, rows of a tile, and
# whether tiles are shared
PLANS = [
    (0, 0, 1, 8, 8), (0, 0, 1, 671, 8), (0, 0, 4554, 9, 545), (0, 0, 2066, 2013, 10), (0, 0, 3633, 8, 1575),
    (0, 0, 98, 4432, 3839), (0, 0, 3585, 9, 2183), (0, 0, 2288, 8, 4386), (0, 0, 4768, 8, 2625),
    (0, 0, 3750, 8, 4064), (0, 2, 1, 8, 8), (0, 2, 1, 815, 8), (0, 2, 4554, 9, 545), (0, 2, 1305, 3498, 10),
    (0, 2, 3633, 8, 1575), (0, 2, 98, 4432, 3839), (0, 2, 3585, 9, 2183), (0, 2, 2288, 8, 4386),
    (0, 2, 4768, 8, 2625), (0, 2, 3750, 8, 4064), (1, 0, 1, 8, 8), (1, 0, 1, 214, 8), (1, 0, 1051, 8, 3638),
    (1, 0, 2471, 1902, 13), (1, 0, 3340, 8, 531), (1, 0, 1321, 3808, 8), (1, 0, 3701, 8, 807),
    (1, 0, 128, 3787, 1556), (1, 0, 1259, 8, 3298), (1, 0, 136, 4177, 2176), (1, 0, 1155, 8, 4148),
    (1, 0, 1930, 8, 3105), (1, 0, 4447, 8, 1541), (1, 2, 1, 8, 8), (1, 2, 1, 458, 8), (1, 2, 36, 4438, 3102),
    (1, 2, 1499, 793, 8), (1, 2, 1478, 1780, 8), (1, 2, 3701, 8, 807), (1, 2, 97, 2625, 1875), (1, 2, 1051, 8, 3638),
    (1, 2, 136, 4468, 3931), (1, 2, 1155, 8, 4148), (1, 2, 1930, 8, 3105), (1, 2, 4447, 8, 1541),
    (1, 0, 1998, 818, 273), (1, 0, 4868, 397, 157), (1, 0, 1951, 1569, 134), (1, 0, 4555, 172, 692),
    (1, 0, 889, 1380, 1058), (1, 0, 4999, 100, 787), (1, 0, 298, 3787, 2332), (1, 0, 3260, 37, 3238),
    (1, 0, 3207, 3637, 579), (1, 0, 4248, 37, 3077), (1, 0, 399, 3799, 3971), (1, 0, 4378, 82, 1611),
    (1, 0, 3235, 1282, 2498), (2, 0, 1, 8, 8), (2, 0, 1, 671, 8), (2, 0, 49, 4425, 3900), (2, 0, 4103, 8, 307),
    (2, 0, 2066, 2013, 10), (2, 0, 3701, 8, 807), (2, 0, 114, 3076, 2107), (2, 0, 1051, 8, 3638),
    (2, 0, 135, 3192, 4078), (2, 0, 1155, 8, 4148), (2, 0, 4162, 4278, 4477), (2, 0, 1930, 8, 3105),
    (2, 0, 4447, 8, 1541), (2, 0, 3262, 3383, 2508), (3, 2, 1, 8, 8), (3, 2, 1, 8, 208), (3, 2, 18, 3773, 4459),
    (3, 2, 1510, 8, 387), (3, 2, 953, 8, 1575), (3, 2, 2576, 2347, 8), (3, 2, 97, 3299, 1306), (3, 2, 3754, 2109, 8),
    (3, 2, 3395, 2890, 8), (3, 2, 4174, 3019, 9), (3, 2, 3410, 4243, 8), (3, 0, 1, 8, 8), (3, 0, 1, 8, 69),
    (3, 0, 49, 3468, 4071), (3, 0, 4303, 297, 9), (3, 0, 3813, 8, 454), (3, 0, 2576, 2347, 8), (3, 0, 4086, 10, 3050),
    (3, 0, 3754, 2109, 8), (3, 0, 130, 2783, 3447), (3, 0, 3395, 2890, 8), (3, 0, 922, 2558, 2849),
    (3, 0, 4174, 3019, 9), (3, 0, 1771, 3731, 4167), (3, 0, 3410, 4243, 8), (3, 0, 3723, 4440, 2094), (4, 2, 1, 8, 8),
    (4, 2, 449, 8, 8), (4, 2, 1, 277, 4445), (4, 2, 3289, 8, 426), (4, 2, 1, 544, 4245), (4, 2, 4783, 1960, 49),
    (4, 2, 1, 1046, 3455), (4, 2, 4553, 2744, 3823), (4, 2, 1, 1373, 3436), (4, 2, 1, 1422, 4103),
    (4, 2, 1, 1648, 4162), (4, 0, 1, 8, 8), (4, 0, 214, 8, 11), (4, 0, 1, 277, 4445), (4, 0, 2454, 8, 747),
    (4, 0, 1, 544, 4245), (4, 0, 4022, 8, 2665), (4, 0, 1, 1046, 3455), (4, 0, 4926, 4362, 156),
    (4, 0, 1, 1373, 3436), (4, 0, 4869, 2892, 644), (4, 0, 1, 1422, 4103), (4, 0, 3449, 1613, 4089),
    (4, 0, 1, 1648, 4162), (4, 0, 3920, 4310, 2409),
]
# the same for the bfloat16 gradients whose products run across the reduction (k and n multiples of 8)
ACROSS = [
    (3, 2, 1, 8, 8), (3, 2, 1, 8, 200), (3, 2, 17, 4296, 4184), (3, 2, 4230, 8, 144), (3, 2, 1034, 8, 1008),
    (3, 2, 3096, 1800, 8), (3, 2, 113, 1112, 2920), (3, 2, 4974, 1592, 8), (3, 2, 3136, 3120, 8), (3, 2, 4500, 2696, 8),
    (3, 2, 4292, 3192, 8), (3, 2, 4783, 3504, 3008), (4, 2, 449, 8, 8), (4, 2, 1, 864, 4176), (4, 2, 1739, 2496, 3296),
    (4, 2, 65, 264, 72), (3, 2, 200, 264, 72), (4, 2, 4096, 128, 512),
]
# 8-bit products of few rows: rows and weights that fill a workgroup or not, the reduction in whole blocks, ending inside one,
# on no word, shorter than the waves; and their neighbours that go to the tiles
FEW = [(0, d, *s) for d in (0, 2) for s in (
    (1, 4, 1), (1, 128, 16), (3, 132, 17), (16, 8192, 15), (15, 2052, 4097), (5, 130, 300), (16, 257, 128), (1, 8192, 8192),
    (16, 1000, 8209), (7, 129, 8200), (17, 64, 31), (32, 4096, 100), (30, 515, 4096), (33, 2048, 129), (64, 1924, 33),
    (50, 1023, 257), (16, 8196, 64), (32, 4100, 64), (64, 2052, 64), (17, 128, 4100))]


@pytest.mark.parametrize("op,dtype,m,k,n", PLANS + ACROSS + FEW)
def test_every_tile(ops, cuda, op, dtype, m, k, n):
    import ctypes
    from omarchy_mac_torch import _lib
    v = [ctypes.c_int() for _ in range(3)]
    assert _lib.L.omt_ffn_plan(op, dtype, m, k, n, *v) == 0
    print("plan", [x.value for x in v], flush=True)
    t = F32 if dtype == 0 else BF16
    g = torch.Generator(device=cuda).manual_seed(m + k + n)

    def new(*shape):
        return torch.randn(*shape, device=cuda, generator=g)

    def near(got, want, bound):
        assert float((got.double() - want).norm() / want.norm()) <= bound

    def wide(q, s):
        return q.double() * s.double().repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]

    def wide_weight(q, s):
        return wide(q, s.repeat_interleave(BLOCK, 0)[:q.shape[0]])

    if op == 0:
        a, b = ops.quantize_fp8(new(m, k)), ops.quantize_fp8_weight(new(n, k))
        near(ops.matmul_fp8(*a, *b, dtype=t), wide(*a) @ wide_weight(*b).T, tol(k, t))
        return
    x, wg, wu = new(m, k).to(t), (new(n, k) * k ** -0.5).to(t), (new(n, k) * k ** -0.5).to(t)
    if op == 2:
        a, b, c = ops.quantize_fp8(x), ops.quantize_fp8_weight(wg), ops.quantize_fp8_weight(wu)
        p, q = wide(*a) @ wide_weight(*b).T, wide(*a) @ wide_weight(*c).T
        check_fp8(*ops.glu_fp8(*a, *b, *c), (p * torch.sigmoid(p) * q).cpu())
        return
    if op == 1:
        p, q = x.double() @ wg.double().T, x.double() @ wu.double().T
        h, kept = ops.glu(x, wg, wu, checkpoint="fp8")
        near(h, p * torch.sigmoid(p) * q, 2 * tol(k, t))
        check_fp8(kept[2], kept[3], p.cpu())
        check_fp8(kept[4], kept[5], q.cpu())
        return
    p, q, gh = new(m, n).to(t), new(m, n).to(t), new(m, n).to(t)
    s = torch.sigmoid(p.double())
    dg, du = gh.double() * q.double() * s * (1 + p.double() * (1 - s)), gh.double() * p.double() * s
    got = ops.glu_backward(gh, (x, None, p, None, q, None), wg, wu, input_grad=op == 3, weight_grad=op == 4)
    if op == 3:
        near(got[0], dg @ wg.double() + du @ wu.double(), 2 * tol(2 * n, t, rounded=1))
    else:
        near(got[1], dg.T @ x.double(), 2 * tol(m, t, rounded=1))
        near(got[2], du.T @ x.double(), 2 * tol(m, t, rounded=1))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_glu_infinities_and_nan_at_training_sizes(ops, cuda, dtype):
    """An infinity or NaN of x, at sizes where float32 runs as halves: its own row of h, and no other, and infinities of
    the sign that float32 gives where the activation passes them."""
    m, k, f = 1647, 871, 407
    x, wg, wu = (t.to(cuda) for t in glu_operands(m, k, f, dtype))
    x[5, 3], x[600, 870], x[1646, 0] = float("inf"), float("nan"), -float("inf")
    h, kept = ops.glu(x, wg, wu, act="relu", checkpoint="full")
    bad = torch.zeros(m, dtype=torch.bool, device=cuda)
    bad[[5, 600, 1646]] = True
    assert bool(h[~bad].isfinite().all()) and bool(h[600].isnan().all())
    for row, col in ((5, 3), (1646, 0)):
        for got, w in ((kept[2], wg), (kept[4], wu)):
            assert torch.equal(got[row].float(), (x[row, col].float() * w[:, col].float()).sign() * float("inf"))
    gh = torch.ones_like(h)
    gx, gwg, gwu = ops.glu_backward(gh, kept, wg, wu, act="relu")
    assert bool(gx[~bad].isfinite().all()) and not bool(gx[600].isfinite().any())
