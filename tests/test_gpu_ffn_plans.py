"""Tiles of the feed-forward products that tests/test_gpu_ffn.py's sizes do not lead to, and every row and column of a result by
itself, so that one left out, or taken for another, shows whatever the others' size.

With s the norm of an element's terms (s^2 the sum of their squares), float32's sum of k terms of random signs is within
(16 + 4 sqrt(k)) 2^-24 s. Rows may have one element, and there are up to a million: 5.5 standard deviations of the element,
5.5 s, bound what a result's rounding to bfloat16 is relative to, 2^-8 of it; terms each off by up to 2^-8 of their size,
evenly spread, sum up to an error of 2^-8 / sqrt(3) s, 5.5 of which are 3.2 2^-8 s. The 8-bit matrix instructions drop what is under
2^-13 of the largest of 32 products, within 3 s of an element's terms."""

import pytest
import torch

import test_gpu_ffn as base
from test_gpu_ffn import BF16, F32, check_fp8

pytestmark = pytest.mark.gpu
BLOCK = 128


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


# (operator, type, m, k, n): the cheapest of 400000 random sizes for each combination of operator, mode, rows of a tile, whether
# tiles are shared, and whether the reduction runs across the operands' rows, that no size of tests/test_gpu_ffn.py leads to
MORE = [
    (0, 0, 5611, 2, 549), (0, 0, 672, 7237, 1), (0, 0, 102, 3380, 4670), (0, 0, 2968, 4725, 6748), (0, 0, 4738, 5476, 5276),
    (0, 2, 195, 5624, 6856), (0, 2, 6568, 6768, 2504), (1, 0, 1469, 3168, 8), (1, 0, 205, 4673, 5628),
    (1, 2, 5988, 4942, 4799), (1, 2, 7350, 5581, 1128), (1, 0, 900, 1216, 280), (1, 0, 495, 1704, 520),
    (1, 0, 443, 8166, 1976), (1, 0, 1516, 2574, 5457), (2, 0, 5748, 1, 277), (2, 0, 287, 3472, 520),
    (2, 0, 4032, 5648, 5416), (3, 2, 1, 1, 1), (3, 2, 1, 1, 225), (3, 2, 2635, 1103, 6694), (3, 2, 313, 5984, 5232),
    (3, 2, 5552, 3029, 4100), (4, 2, 1, 1, 1), (4, 2, 475, 1, 1), (4, 2, 4043, 6162, 31), (4, 2, 6818, 5531, 5980),
    (4, 0, 5043, 464, 256), (4, 0, 3267, 840, 440), (4, 0, 5664, 6614, 1262),
]
# the longest products of tests/test_gpu_ffn.py's list, where one row of thousands is little beside the whole
LONG = [(0, 2, 4768, 8, 2625), (1, 2, 4447, 8, 1541), (1, 0, 4999, 100, 787), (3, 2, 4974, 1592, 8), (3, 2, 4500, 2696, 8),
        (3, 2, 4783, 3504, 3008), (3, 0, 4174, 3019, 9), (4, 2, 4783, 1960, 49), (4, 2, 4096, 128, 512), (4, 0, 4869, 2892, 644)]


def wide(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def wide_weight(q, s):
    return wide(q, s.repeat_interleave(BLOCK, 0)[:q.shape[0]])


def check_lines(got, want, size, bound):
    """Every row's and every column's error, 2-norm, within `bound` of `size`'s."""
    off = got.double() - want
    for dim in (0, 1):
        assert bool((off.norm(dim=dim) <= bound * size.norm(dim=dim) + 1e-300).all())


def sums(k):
    return (16 + 4 * k ** 0.5) * 2 ** -24


@pytest.mark.parametrize("op,dtype,m,k,n", MORE + LONG)
def test_every_row_and_column(ops, cuda, op, dtype, m, k, n):
    t = F32 if dtype == 0 else BF16
    rounded = 5.5 * 2 ** -8 if t == BF16 else 0
    g = torch.Generator(device=cuda).manual_seed(m + k + n)

    def new(*shape):
        return torch.randn(*shape, device=cuda, generator=g)

    if op == 0:
        a, b = ops.quantize_fp8(new(m, k)), ops.quantize_fp8_weight(new(n, k))
        av, bv = wide(*a), wide_weight(*b)
        size = (av.square() @ bv.square().T).sqrt()
        check_lines(ops.matmul_fp8(*a, *b, dtype=t), av @ bv.T, size,
                    sums(k) + (rounded + 3 * 2 ** -13 if t == BF16 else 0))
        return
    x, wg, wu = new(m, k).to(t), (new(n, k) * k ** -0.5).to(t), (new(n, k) * k ** -0.5).to(t)
    if op == 2:
        a, b, c = ops.quantize_fp8(x), ops.quantize_fp8_weight(wg), ops.quantize_fp8_weight(wu)
        p, q = wide(*a) @ wide_weight(*b).T, wide(*a) @ wide_weight(*c).T
        check_fp8(*ops.glu_fp8(*a, *b, *c), (p * torch.sigmoid(p) * q).cpu())
        return
    xd, gd, ud = x.double(), wg.double(), wu.double()
    if op == 1:
        p, q = xd @ gd.T, xd @ ud.T
        sp, sq = (xd.square() @ gd.square().T).sqrt(), (xd.square() @ ud.square().T).sqrt()
        h, kept = ops.glu(x, wg, wu, checkpoint="fp8")
        act, want = p * torch.sigmoid(p), p * torch.sigmoid(p) * q
        # silu's slope is at most 1.1; the exponential instruction is within 2^-20 of act, and a result's rounding of itself
        size = sums(k) * 2 * (1.1 * q.abs() * sp + act.abs() * sq) + (2 ** -20 + (2 ** -8 if t == BF16 else 0)) * want.abs()
        check_lines(h, want, size, 1)
        check_fp8(kept[2], kept[3], p.cpu())
        check_fp8(kept[4], kept[5], q.cpu())
        return
    p, q, gh = new(m, n).to(t), new(m, n).to(t), new(m, n).to(t)
    s = torch.sigmoid(p.double())
    dg, du = gh.double() * q.double() * s * (1 + p.double() * (1 - s)), gh.double() * p.double() * s
    got = ops.glu_backward(gh, (x, None, p, None, q, None), wg, wu, input_grad=op == 3, weight_grad=op == 4)
    # dg and du are off by the exponential instruction's 2^-20, and are rounded to bfloat16 where that is the type
    bound = 2 ** -19 + rounded + (3.2 * 2 ** -8 if t == BF16 else 0)
    if op == 3:
        size = (dg.square() @ gd.square() + du.square() @ ud.square()).sqrt()
        check_lines(got[0], dg @ gd + du @ ud, size, 2 * sums(2 * n) + bound)
    else:
        for got, d in ((got[1], dg), (got[2], du)):
            check_lines(got, d.T @ xd, (d.square().T @ xd.square()).sqrt(), 2 * sums(m) + bound)


def test_a_row_left_out_shows(cuda):
    """The check by itself, on the largest of the bfloat16 gradients: a row of zeros in a result rounded as the operator
    rounds it passes the whole result's norm, and not the row's."""
    m, k, n = 4783, 3504, 3008
    g = torch.Generator(device=cuda).manual_seed(1)
    a, b = (torch.randn(*s, device=cuda, generator=g, dtype=torch.float64) for s in ((m, n), (k, n)))
    want, size = a @ b.T, (a.square() @ b.square().T).sqrt()
    got = want.to(BF16)
    check_lines(got, want, size, 8.7 * 2 ** -8)
    got[17] = 0
    assert base.rel(got, want.cpu()) <= 2 * base.tol(2 * n, BF16, rounded=1)
    with pytest.raises(AssertionError):
        check_lines(got, want, size, 8.7 * 2 ** -8)
