"""The feed-forward operators' host side, without a GPU: argument statuses of every entry point, workspaces, plans."""

import ctypes

import pytest
import torch

F32, BF16 = 0, 2


@pytest.fixture(scope="module")
def lib():
    from omarchy_mac_torch import _lib
    return _lib


def plan(lib, op, dtype, m, k, n):
    v = [ctypes.c_int() for _ in range(3)]
    assert lib.L.omt_ffn_plan(op, dtype, m, k, n, *v) == lib.OMT_OK
    return tuple(x.value for x in v)


def test_statuses(lib):
    L, p = lib.L, ctypes.c_void_p(4096)
    odd = ctypes.c_void_p(4098)
    bad, no = lib.OMT_INVALID, lib.OMT_UNSUPPORTED
    f = L.omt_rms_norm_fwd
    assert f(1, 0, 4, 8, p, None, p, 1e-6, p, None, None, None, None, None) == bad          # int64
    assert f(F32, BF16, 4, 8, p, None, p, 1e-6, p, None, None, None, None, None) == bad     # a weight of another type
    assert f(F32, F32, -1, 8, p, None, p, 1e-6, p, None, None, None, None, None) == bad
    assert f(F32, F32, 4, 0, p, None, p, 1e-6, p, None, None, None, None, None) == bad
    assert f(F32, F32, 4, 32769, p, None, p, 1e-6, p, None, None, None, None, None) == no
    assert f(F32, F32, 4, 8, p, None, p, 1e-6, None, None, None, None, None, None) == bad   # no output
    assert f(F32, F32, 4, 8, p, p, p, 1e-6, p, None, None, None, None, None) == bad         # a sum with nowhere to go
    assert f(F32, F32, 4, 8, p, None, p, 1e-6, None, None, None, p, None, None) == bad      # values without scales
    assert f(F32, F32, 0, 8, None, None, None, 1e-6, None, None, None, None, None, None) == lib.OMT_OK
    b = L.omt_rms_norm_bwd
    assert b(F32, F32, 4, 8, p, None, p, p, p, p, p, None, 0, None) == bad                  # no workspace
    assert b(F32, F32, 4, 8, p, None, p, p, None, p, None, None, 0, None) == bad
    assert b(F32, F32, 0, 8, None, None, None, p, None, None, None, None, 0, None) == lib.OMT_OK
    assert L.omt_quantize_fp8(1, 4, 8, p, 0, p, p, None) == bad
    assert L.omt_quantize_fp8(F32, 4, 0, p, 0, p, p, None) == bad
    assert L.omt_quantize_fp8(F32, 4, 8, p, 0, p, None, None) == bad
    assert L.omt_quantize_fp8(F32, 0, 8, None, 0, None, None, None) == lib.OMT_OK
    assert L.omt_quantize_fp8_weight(F32, 0, 8, p, p, p, None) == bad
    assert L.omt_quantize_fp8_weight(F32, 8, 8, None, p, p, None) == bad
    mm = L.omt_matmul_fp8
    assert mm(4, 8, 16, p, p, p, p, 1, p, None, 0, None) == bad
    assert mm(4, 0, 16, p, p, p, p, F32, p, None, 0, None) == bad
    assert mm(4, 8, 16, p, p, p, None, F32, p, None, 0, None) == bad
    assert mm(4, 8, 16, odd, p, p, p, F32, p, None, 0, None) == bad
    assert mm(4, 8, 1 << 21, p, p, p, p, F32, p, None, 0, None) == no
    assert mm(4, 8, 17, p, p, p, p, F32, p, None, 0, None) == bad                           # rows to copy, no workspace
    assert mm(0, 8, 16, None, None, None, None, F32, None, None, 0, None) == lib.OMT_OK
    g = L.omt_glu_fwd
    one = [p] * 3 + [p] + [None] * 6
    assert g(1, 4, 16, 8, 0, 0, *one, None, 0, None) == bad
    assert g(F32, 4, 16, 8, 3, 0, *one, None, 0, None) == bad
    assert g(F32, 4, 16, 8, 0, 3, *one, None, 0, None) == bad
    assert g(F32, 4, 16, 8, 0, 1, *one, None, 0, None) == bad                               # nowhere to keep
    assert g(F32, 4, 16, 8, 0, 0, odd, *one[1:], None, 0, None) == bad
    assert g(F32, 0, 16, 8, 0, 0, *[None] * 10, None, 0, None) == lib.OMT_OK
    w = L.omt_glu_bwd
    args = [p, p, None, p, None, p, None, p, p, p, p, p]
    assert w(F32, 4, 16, 8, 0, 0, *args, p, 1 << 30, None) == bad                           # nothing was kept
    assert w(F32, 4, 16, 8, 0, 1, *args, p, 1 << 30, None) == bad                           # 8 bits without scales
    assert w(F32, 4, 16, 8, 0, 2, *args, p, 16, None) == bad                                # a small workspace
    assert w(F32, 4, 16, 8, 0, 2, *args[:-1], None, p, 1 << 30, None) == bad                # one weight's gradient alone
    assert w(F32, 1 << 21, 16, 8, 0, 2, *args, p, 1 << 30, None) == no
    h = L.omt_glu_fp8
    assert h(4, 16, 8, 7, *[p] * 8, None, 0, None) == bad
    assert h(4, 16, 8, 0, *[p] * 7, None, None, 0, None) == bad
    assert h(0, 16, 8, 0, *[None] * 8, None, 0, None) == lib.OMT_OK
    v = [ctypes.c_int() for _ in range(3)]
    assert L.omt_ffn_plan(9, F32, 4, 16, 8, *v) == bad and L.omt_ffn_plan(0, F32, 0, 16, 8, *v) == bad


def test_workspaces_cover_what_they_say(lib):
    L = lib.L
    assert L.omt_rms_norm_bwd_workspace(0, 8) > 0 and L.omt_rms_norm_bwd_workspace(5, 40000) == 0
    # in place, one slice: nothing
    assert L.omt_glu_fp8_workspace(4096, 4096, 4096) == 0 and L.omt_matmul_fp8_workspace(4096, 4096, 4096, BF16) == 0
    # rows of an odd number of bytes are copied
    assert L.omt_matmul_fp8_workspace(4096, 4096, 4097, BF16) >= 2 * 4096 * 4112
    # shared tiles: each workgroup's sums of two
    _, rows, sharers = plan(lib, lib.OMT_FFN_MATMUL_FP8, BF16, 17, 8192, 4096)
    assert sharers > 16 and L.omt_matmul_fp8_workspace(17, 4096, 8192, BF16) >= sharers * 2 * rows * 256 * 4
    # the backward: dg and du twice, the weights and x transposed
    m, k, f = 300, 200, 500
    for dtype, e in ((F32, 4), (BF16, 2)):
        assert L.omt_glu_bwd_workspace(dtype, m, k + 1, f) >= e * (2 * m * 512 + 2 * f * 320 + 2 * k * 512 + k * 320)
    # bfloat16 rows on 16 bytes: dg and du once, and x widened
    assert L.omt_glu_bwd_workspace(BF16, 320, 200, 504) >= 2 * (2 * 320 * 512 + 320 * 200)
    assert L.omt_glu_bwd_workspace(BF16, 320, 200, 504) < L.omt_glu_bwd_workspace(BF16, 320, 204, 504)
    assert L.omt_glu_fwd_workspace(3, 4, 16, 8) == 0


def test_plans_are_within_the_kernels_limits(lib):
    g = torch.Generator().manual_seed(0)
    for _ in range(3000):
        m, k, n = (int(2 ** (float(torch.rand((), generator=g)) * 13)) for _ in range(3))
        for op in range(5):
            for dtype in (F32, BF16):
                mode, rows, sharers = plan(lib, op, dtype, m, k, n)
                if mode == 5:  # few rows: all of them at once, nothing shared
                    assert op == lib.OMT_FFN_MATMUL_FP8 and m <= rows <= 64 and sharers == 0 and rows * k <= 16 * 8192
                    assert k % 4 or lib.L.omt_matmul_fp8_workspace(m, n, k, dtype) == 0
                    continue
                assert rows in (16, 64, 96, 128, 160, 192, 224, 256) and mode in range(5)
                assert 0 <= sharers <= (256 if rows > 64 else 512)
                if op != lib.OMT_FFN_GLU_GW:  # (of the weights' gradients in bfloat16 the tiles have 128 rows or 256)
                    assert rows <= 16 or rows // 4 < m


def test_the_tested_sizes_reach_the_tiles(lib):
    """Three quarters at least of the combinations (operator, mode, rows of a tile, shared or not) that random sizes lead to
    are among those of the sizes that the GPU tests run."""
    import test_gpu_ffn
    def kind(op, *size):
        mode, rows, sharers = plan(lib, op, *size)
        return op, mode, rows, sharers > 0
    tested = {kind(*p) for p in test_gpu_ffn.PLANS + test_gpu_ffn.FEW}
    g = torch.Generator().manual_seed(1)
    met = {kind(op, dtype, *(int(8 * 2 ** (float(torch.rand((), generator=g)) * 9)) for _ in range(3)))
           for _ in range(1000) for op in range(5) for dtype in (F32, BF16)}
    assert len(met & tested) >= 0.75 * len(met), sorted(met - tested)


def test_operators_refuse_cpu_tensors():
    from omarchy_mac_torch import hip_ops
    x = torch.ones(4, 8)
    for call in (lambda: hip_ops.rms_norm(x, x[0]), lambda: hip_ops.quantize_fp8(x), lambda: hip_ops.glu(x, x, x)):
        with pytest.raises(TypeError, match="HIP device"):
            call()
