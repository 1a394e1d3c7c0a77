"""The feed-forward operators where they can go wrong: infinities and NaN in each form of the products, sums whose terms
cancel, every row and column of a gradient by itself, scales to the bit, long and wide norms. Oracles in float64, on the CPU
or the GPU; tolerances are derived beside each test."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128
F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


def rnd(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def mode_of(op, dtype, m, k, n):
    import ctypes
    from omarchy_mac_torch import _lib
    v = [ctypes.c_int() for _ in range(3)]
    assert _lib.L.omt_ffn_plan(op, dtype, m, k, n, *v) == 0
    return v[0].value


def same_kind(got, want):
    """Both +inf, both -inf, both NaN, or both finite, element by element."""
    got, want = got.double().cpu(), want.double().cpu()
    return (torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf())
            and torch.equal(got.isneginf(), want.isneginf()))


def products(x, w):
    """x w^T, one rounding to each product, as IEEE has infinities and NaN."""
    return torch.stack([(x.double()[:, None, :] * r.double()).sum(-1) for r in w.split(1)], 1)[..., 0]


# ---- what is not finite ------------------------------------------------------------------------------------------------

def test_glu_infinities_of_both_operands(ops, cuda):
    """float32 as float16 halves: infinities of x and of the weights in one group of 32 (at one place, at two), of both
    signs, beside zeros and beside values far below their group's largest: as float32 has them, one by one."""
    m, k, f = 1647, 871, 407
    assert mode_of(1, 0, m, k, f) == 4
    x, wg, wu = rnd((m, k), 1).float(), rnd((f, k), 2, k ** -0.5).float(), rnd((f, k), 3, k ** -0.5).float()
    x[5, 3], x[6, 3], x[6, 9] = INF, INF, INF       # one; two, whose signs the weight decides
    x[7, 3], x[7, 9] = INF, -INF
    x[8, 40], x[9, 870] = -INF, INF                 # another group; the last element
    x[10, 3], x[10, 5] = INF, NAN
    x[11, 7] = 0
    wg[2, 7], wg[3, 3], wg[4, 3] = -INF, INF, -INF  # elsewhere in x's group; at its own place
    wg[5, 3], wg[5, 40] = 0, 1e-30
    wg[6, 3], wg[6, 9], wg[7, 870] = -0.0, 1e-38, NAN
    wu[2, 3], wu[2, 7], wu[3] = INF, -INF, 0
    rows, cols = torch.tensor([4, 5, 6, 7, 8, 9, 10, 11, 12, 1646]), torch.arange(12)
    h, kept = ops.glu(x.to(cuda), wg.to(cuda), wu.to(cuda), act="relu", checkpoint="full")
    for got, w in ((kept[2], wg), (kept[4], wu)):
        got = got.cpu()
        assert same_kind(got[rows][:, cols], products(x[rows], w[cols]))
        plain = torch.ones(m, dtype=torch.bool)
        plain[5:11] = False
        finite = w.isfinite().all(1)
        assert bool(got[plain][:, finite].isfinite().all()) and not bool(got[5:11].isfinite().any())


def test_glu_backward_infinities_of_the_weights(ops, cuda):
    """gx = dg Wg + du Wu with an infinity in a weight: by the sign of dg, NaN where dg is 0."""
    m, k, f = 1647, 871, 407
    assert mode_of(3, 0, m, k, f) == 4 and mode_of(4, 0, m, k, f) == 4
    x, g, u, gh = (rnd(s, i).float() for i, s in enumerate(((m, k), (m, f), (m, f), (m, f))))
    wg, wu = rnd((f, k), 7, k ** -0.5).float(), rnd((f, k), 8, k ** -0.5).float()
    wg[9, 7], wu[40, 8] = INF, -INF
    gh[3] = 0
    gx, gwg, gwu = ops.glu_backward(gh.to(cuda), (x.to(cuda), None, g.to(cuda), None, u.to(cuda), None), wg.to(cuda),
                                    wu.to(cuda), act="relu")
    dg, du = gh.double() * u.double() * (g > 0), gh.double() * g.double().clamp(min=0)
    assert same_kind(gx[:, 7], dg[:, 9] * INF) and same_kind(gx[:, 8], du[:, 40] * -INF)
    gx[:, 7:9] = 0
    assert bool(gx.isfinite().all()) and bool(gwg.isfinite().all()) and bool(gwu.isfinite().all())


# few rows (16, 32 and 64 of them), tiles, a reduction that ends inside a block
@pytest.mark.parametrize("m,n,k", [(2, 140, 300), (16, 200, 512), (30, 140, 384), (64, 257, 300), (70, 140, 300), (300, 260, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_matmul_fp8_blocks_that_stand_for_nan(ops, cuda, m, n, k, dtype):
    """An infinity or NaN before quantization makes its block NaN throughout: of x its row of the result, of the weight the
    columns of its 128 rows. Every form, both result types."""
    x, w = rnd((m, k), 1).float(), rnd((n, k), 2).float()
    x[1, 5], x[m - 1, k - 1] = INF, NAN
    a, b = ops.quantize_fp8(x.to(cuda)), ops.quantize_fp8_weight(w.to(cuda))
    got = ops.matmul_fp8(*a, *b, dtype=dtype).cpu()
    rows = torch.zeros(m, dtype=torch.bool)
    rows[[1, m - 1]] = True
    assert bool(got[rows].isnan().all()) and bool(got[~rows].isfinite().all())
    for bad in (-INF, NAN):
        w[n - 1, k - 1] = bad
        c = ops.quantize_fp8_weight(w.to(cuda))
        got = ops.matmul_fp8(*a, *c, dtype=dtype).cpu()
        cols = torch.arange(n) // BLOCK == (n - 1) // BLOCK
        assert bool(got[:, cols].isnan().all()) and bool(got[~rows][:, ~cols].isfinite().all())


# ---- sums that cancel ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 16, 40, 80, 300])
def test_matmul_fp8_terms_that_cancel(ops, cuda, m):
    """Large products that cancel beside small ones, in every block. A float32 result has float32's sums. A bfloat16 one may lose
    what is under 2^-13 of the largest of eight consecutive products: at most 7 such parts to eight products, each 2^-13 of the
    largest, and 2^-8 of the result."""
    n, k = 256, 512
    a, b = rnd((m, k), 1, 2.0), rnd((n, k), 2, 2.0)
    for block in range(0, k, 128):
        a[:, block + 3], a[:, block + 5], a[:, block + 9] = 448, -448, 384  # within eight, and over two eights
        a[:, block + 90] = -384
        b[:, [block + 3, block + 5]] = 256
        b[:, [block + 9, block + 90]] = 448
    a, b = a.to(FP8).to(cuda), b.to(FP8).to(cuda)
    sa, sb = torch.ones(m, k // BLOCK, device=cuda), torch.ones(n // BLOCK, k // BLOCK, device=cuda)
    terms = a.double()[:, None] * b.double()
    want = terms.sum(-1)
    exact = ops.matmul_fp8(a, sa, b, sb, dtype=F32).double()
    assert bool(((exact - want).abs() <= (16 + 4 * k ** 0.5) * 2 ** -24 * terms.norm(dim=-1)).all())
    got = ops.matmul_fp8(a, sa, b, sb, dtype=BF16).double()
    lost = 7 * 2 ** -13 * terms.abs().unflatten(-1, (-1, 8)).amax(-1).sum(-1)
    assert bool(((got - want).abs() <= 2 ** -8 * want.abs() + lost + (16 + 4 * k ** 0.5) * 2 ** -24 * terms.norm(dim=-1)).all())


# ---- very many rows ------------------------------------------------------------------------------------------------------

def test_glu_of_more_rows_than_a_grid_dimension_holds(ops, cuda):
    """2^29 rows, as halves: laid out 32 to a workgroup of 256 they are 2^32 threads. Products of small whole numbers, exact."""
    m = 2 ** 29 + 40
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 160 GB of GPU memory")
    assert mode_of(1, 0, m, 1, 1) == 4
    x = (torch.arange(m, device=cuda, dtype=torch.int32) % 61).to(F32).view(m, 1)
    h, _ = ops.glu(x, torch.full((1, 1), 2.0, device=cuda), torch.full((1, 1), 3.0, device=cuda), act="relu")
    assert torch.equal(h, x.square_().mul_(6))
    del h, x
    torch.cuda.empty_cache()


# ---- scales ------------------------------------------------------------------------------------------------------------

# float32 instructions and halves, tiles a workgroup's own and shared (the second, fourth and sixth)
@pytest.mark.parametrize("m,k,f", [(16, 64, 128), (1, 512, 700), (4868, 397, 157), (1951, 1569, 134), (4096, 256, 1024),
                                   (889, 1380, 1058)])
def test_glu_checkpoints_to_the_bit(ops, cuda, m, k, f):
    """A block's scale is float32's max(largest magnitude, 1e-30) / 448, and its values float32's product with 1 / scale rounded
    to e4m3, of the same projections that the whole checkpoints give."""
    x, wg, wu = (t.float().to(cuda) for t in (rnd((m, k), 1), rnd((f, k), 2, k ** -0.5), rnd((f, k), 3, k ** -0.5)))
    _, full = ops.glu(x, wg, wu, checkpoint="full")
    _, kept = ops.glu(x, wg, wu, checkpoint="fp8")
    for i in (2, 4):
        t = full[i].cpu()
        blocks = torch.nn.functional.pad(t, (0, -f % BLOCK)).unflatten(-1, (-1, BLOCK))
        scale = blocks.abs().amax(-1).clamp(min=1e-30) / 448
        assert torch.equal(kept[i + 1].cpu(), scale)
        q = (blocks * (1 / scale)[..., None]).flatten(-2)[:, :f].to(FP8)
        assert torch.equal(kept[i].cpu().view(torch.uint8), q.contiguous().view(torch.uint8))


# ---- norms ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,dim", [(2 ** 26 + 5, 8), (2 ** 23 + 3, 8), (2 ** 21 + 2, 2056)])
def test_rms_norm_of_more_rows_than_a_grid_dimension_holds(ops, cuda, rows, dim):
    """A workgroup to four short rows or to one long one: 2^24 of them of 256 threads pass a dimension's 2^32 threads. Rows
    differ in size, so that each shows whose statistics it has. bfloat16: 2^-8 for the result's rounding, and as much again
    for float32's sums, far below it."""
    x = torch.ones(rows, dim, device=cuda, dtype=BF16)
    x[:, 0] = (torch.arange(rows, device=cuda) % 97).to(BF16)
    w = torch.ones(dim, device=cuda, dtype=BF16)
    y, _, rstd = ops.rms_norm(x, w)
    want = torch.rsqrt(((torch.arange(rows, device=cuda) % 97).double().square() + dim - 1) / dim + 1e-6)
    assert float((rstd.double() / want - 1).abs().max()) <= (8 + dim) * 2 ** -24
    assert float((y[:, 1].double() / want - 1).abs().max()) <= 2 ** -7
    q, scale, _ = ops.rms_norm_fp8(x, w)
    top = torch.maximum(torch.arange(rows, device=cuda) % 97, torch.ones((), device=cuda)).double() * want
    assert float((scale[:, 0].double() * 448 / top - 1).abs().max()) <= (16 + dim) * 2 ** -24


@pytest.mark.parametrize("dim", [16400, 24577, 32766, 32768])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rms_norm_backward_of_wide_rows(ops, cuda, dim, dtype):
    """More rows than workgroups, so that each sums the weight's gradient over some. Per row and per column: float32's sums of
    `dim` or `rows` terms, (8 + 2 sqrt(n)) 2^-24 of the terms' norm for random signs, twice for the two terms of gx, and for
    bfloat16 results 2^-8."""
    rows = 700
    g = torch.Generator(device=cuda).manual_seed(dim)
    h, gy, gh = (torch.randn(rows, dim, device=cuda, generator=g).to(dtype) for _ in range(3))
    w = (1 + 0.2 * torch.randn(dim, device=cuda, generator=g)).to(dtype)
    _, _, rstd = ops.rms_norm(h, w)
    hd, gyd, r = h.double(), gy.double(), torch.rsqrt(h.double().square().mean(-1, keepdim=True) + 1e-6)
    n, t = hd * r, gyd * w.double()
    want = r * (t - n * (t * n).mean(-1, keepdim=True))
    rounded = 2 ** -8 if dtype == BF16 else 0
    for use_gh in (True, False):
        gx, gw = ops.rms_norm_backward(gy, h, w, rstd, gh=gh if use_gh else None)
        v = want + gh.double() if use_gh else want
        assert bool(((gx.double() - v).norm(dim=1) <= (2 * (8 + 2 * dim ** 0.5) * 2 ** -24 + rounded) * v.norm(dim=1)).all())
        off = (gw.double() - (gyd * n).sum(0)).abs()
        assert bool((off <= 4 * (8 + 2 * rows ** 0.5) * 2 ** -24 * (gyd * n).norm(dim=0) + rounded * gw.double().abs()).all())
        alone, none = ops.rms_norm_backward(gy, h, w, rstd, gh=gh if use_gh else None, weight_grad=False)
        assert none is None and torch.equal(alone, gx)
