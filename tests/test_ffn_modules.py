"""The feed-forward modules' host side, without a GPU: the operators are replaced by recorders of how they are called."""

import pytest
import torch


@pytest.fixture
def glu_calls(monkeypatch):
    """The checkpoint that each call of hip_ops.glu asks for; the results are plain torch's."""
    from omarchy_mac_torch import hip_ops
    calls = []

    def glu(x, w_gate, w_up, act="silu", checkpoint=None):
        calls.append(checkpoint)
        g, u = x @ w_gate.T, x @ w_up.T
        return torch.nn.functional.silu(g) * u, None if checkpoint is None else (x, None, g, None, u, None)

    monkeypatch.setattr(hip_ops, "glu", glu)
    return calls


@pytest.mark.parametrize("checkpoint", ["fp8", "full"])
def test_nothing_is_kept_where_no_gradient_can_be_asked_for(glu_calls, checkpoint):
    from omarchy_mac_torch import ffn
    m = ffn.GatedFeedForward(16, 32, checkpoint=checkpoint)
    x = torch.randn(3, 16)
    with torch.no_grad():
        m(x)
    with torch.inference_mode():
        m(x)
    assert glu_calls == [None, None]
    m(x)
    m(x.requires_grad_(True))
    assert glu_calls[2:] == [checkpoint, checkpoint]
    for p in m.parameters():
        p.requires_grad_(False)
    m(x)
    assert glu_calls[4:] == [checkpoint]
    m(x.detach())
    m.down.weight.requires_grad_(True)
    m(x.detach())
    assert glu_calls[5:] == [None, None]
