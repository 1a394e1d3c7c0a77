"""Which tiles and shares the feed-forward products take, without a GPU."""

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
