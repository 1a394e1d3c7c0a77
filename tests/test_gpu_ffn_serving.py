"""A served feed-forward sublayer on the omarchy_mac_torch device after a change of type, and under the compile backend."""

import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def omt(cuda):
    import omarchy_mac_torch
    return omarchy_mac_torch


def test_a_served_sublayer_after_a_change_of_type(omt):
    from omarchy_mac_torch import ffn
    torch.manual_seed(2)
    served = ffn.FeedForward(96, 260).to(omt.DEVICE).serve()
    x, r = torch.randn(5, 96, device=omt.DEVICE), torch.randn(5, 96, device=omt.DEVICE)
    want = served(x, r)
    same = served.to(torch.bfloat16).to(omt.DEVICE, torch.float32)(x, r)
    # the norm's weight is ones: exact in bfloat16
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, same))
    y, h = served.to(torch.bfloat16)(x.bfloat16(), r.bfloat16())
    assert y.dtype == h.dtype == torch.bfloat16
    # four roundings to 3 bits, 2.6% rms each, and bfloat16's
    assert float((y.float() - want[0]).cpu().norm() / want[0].cpu().norm()) <= 4 * 2 * 0.026


def test_a_served_sublayer_under_the_compile_backend(omt):
    from omarchy_mac_torch import ffn
    torch.manual_seed(2)
    served = ffn.FeedForward(96, 260).to(omt.DEVICE).serve()
    x, r = torch.randn(5, 96, device=omt.DEVICE), torch.randn(5, 96, device=omt.DEVICE)
    want = served(x, r)
    with warnings.catch_warnings():  # a compiler that tries to trace the operators says that it cannot
        warnings.filterwarnings("error", message="Dynamo does not know how to trace")
        got = torch.compile(served, backend=omt.DEVICE)(x, r)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, got))
