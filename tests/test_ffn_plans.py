"""Which tiles and shares the feed-forward products take, and which addresses and sizes, without a GPU."""

import ctypes

import pytest
import torch

F32, BF16 = 0, 2
OPS = range(5)


@pytest.fixture(scope="module")
def plan():
    from omarchy_mac_torch import _lib

    def plan(op, dtype, m, k, n):
        v = [ctypes.c_int() for _ in range(3)]
        assert _lib.L.omt_ffn_plan(op, dtype, m, k, n, *v) == _lib.OMT_OK
        return tuple(x.value for x in v)

    return plan


def random_sizes(seed, count, low=8, octaves=9):
    """(m, k, n), each spread over its logarithm from `low` on; k and n of every second one are multiples of 8."""
    g = torch.Generator().manual_seed(seed)
    for i in range(count):
        size = [int(low * 2 ** (float(torch.rand((), generator=g)) * octaves)) for _ in range(3)]
        if i % 2:
            size[1:] = [max(8, v // 8 * 8) for v in size[1:]]
        yield tuple(size)


def test_sharers_run_at_once(plan):
    """No more workgroups share tiles than run at once on the 256 CUs: two to a CU where its 160 KB of LDS hold the two stages
    of both, which are rows of 128 bytes of x and of 256 rows of a weight, and for the modes with scales (e4m3, widened,
    halves) a scale to each."""
    sizes = [(36, 4832, 4976), (34, 4088, 8072), (40, 4096, 4096), (64, 8192, 4096), *random_sizes(3, 400)]
    for size in sizes:
        for op in OPS:
            for dtype in (F32, BF16):
                mode, rows, sharers = plan(op, dtype, *size)
                if mode == 5:
                    continue
                stage = (rows + 256) * 128 + ((rows + 63) // 64 * 64 + 256) * 4 * (mode in (2, 3, 4))
                at_once = 512 if rows <= 64 and 2 * 2 * stage <= 160 * 1024 else 256
                assert sharers <= at_once, (op, dtype, size, mode, rows, sharers)


def test_every_combination_that_random_sizes_lead_to_is_run(plan):
    """Operator, mode, rows of a tile, shared or not, and which way the reduction runs: each that random sizes up to 8192 lead
    to is among those of the sizes that the GPU tests run."""
    import test_gpu_ffn
    import test_gpu_ffn_plans

    def kind(op, dtype, m, k, n):
        mode, rows, sharers = plan(op, dtype, m, k, n)
        return op, mode, rows, sharers > 0, op in (3, 4) and dtype == BF16 and k % 8 == 0 and n % 8 == 0

    tested = {kind(*p) for p in test_gpu_ffn.PLANS + test_gpu_ffn.ACROSS + test_gpu_ffn.FEW + test_gpu_ffn_plans.MORE}
    met = {kind(op, dtype, *size) for size in random_sizes(1, 4000, 1, 13) for op in OPS for dtype in (F32, BF16)}
    assert len(met) > 100 and met <= tested, sorted(met - tested)


def test_alignment_and_sizes_as_the_header_has_them():
    """Every address that the header wants on 16 bytes is refused off them before anything runs, and every size past its limits."""
    from omarchy_mac_torch import _lib
    L, on, off = _lib.L, 4096, 4100
    big = 1 << 40  # of workspace

    def refused(entry, sizes, pointers, tail, aligned):
        for i in aligned:
            args = [ctypes.c_void_p(off if j == i else on) for j in range(len(pointers))]
            assert entry(*sizes, *args, *tail) == _lib.OMT_INVALID, (entry.__name__, pointers[i])

    def product(a, a_scale, b, b_scale, c, ws):
        return L.omt_matmul_fp8(8, 16, 33, a, a_scale, b, b_scale, F32, c, ws, big, None)

    product.__name__ = "omt_matmul_fp8"
    refused(product, (), ["a", "a_scale", "b", "b_scale", "c", "workspace"], (), [0, 2, 4, 5])
    names = ["x", "w_gate", "w_up", "h", "x_q", "x_scale", "g", "g_scale", "u", "u_scale", "workspace"]
    refused(L.omt_glu_fwd, (BF16, 8, 33, 16, 0, 1), names, (big, None), [0, 1, 2, 3, 6, 8, 10])
    names = ["gh", "x", "x_scale", "g", "g_scale", "u", "u_scale", "w_gate", "w_up", "gx", "gw_gate", "gw_up", "workspace"]
    refused(L.omt_glu_bwd, (BF16, 8, 32, 16, 0, 1), names, (big, None), [1, 7, 8, 9, 10, 11, 12])
    names = ["x", "x_scale", "w_gate", "gate_scale", "w_up", "up_scale", "h_q", "h_scale", "workspace"]
    refused(L.omt_glu_fp8, (8, 33, 16, 0), names, (big, None), [0, 2, 4, 6, 8])

    p = ctypes.c_void_p(on)
    over = (1 << 30) + 1, (1 << 20) + 1
    for m, n, k in ((over[0], 8, 8), (8, over[1], 8), (8, 8, over[1])):
        assert L.omt_matmul_fp8(m, n, k, p, p, p, p, F32, p, p, big, None) == _lib.OMT_UNSUPPORTED
        assert L.omt_glu_fwd(F32, m, k, n, 0, 0, *[p] * 11, big, None) == _lib.OMT_UNSUPPORTED
        assert L.omt_glu_fp8(m, k, n, 0, *[p] * 9, big, None) == _lib.OMT_UNSUPPORTED
    for m, n in (((1 << 20) + 1, 8), (8, (1 << 18) + 1)):
        assert L.omt_glu_bwd(F32, m, 8, n, 0, 1, *[p] * 13, big, None) == _lib.OMT_UNSUPPORTED


def test_products_of_more_tiles_than_a_launch_holds():
    """2^23 tiles of 512 threads are 2^32: refused, where a launch would run a part of them with no error."""
    from omarchy_mac_torch import _lib
    p = ctypes.c_void_p(4096)
    for f in (256, 1 << 20):  # the latter are 2^35
        assert _lib.L.omt_glu_fp8(1 << 30, 64, f, 0, *[p] * 9, 1 << 40, None) == _lib.OMT_UNSUPPORTED
