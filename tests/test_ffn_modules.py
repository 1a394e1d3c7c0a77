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


@pytest.fixture
def quantized(monkeypatch):
    """hip_ops.quantize_fp8_weight by plain torch."""
    from omarchy_mac_torch import hip_ops

    def quantize(w):
        n, k = w.shape
        b = torch.nn.functional.pad(w.float(), (0, -k % 128, 0, -n % 128)).unflatten(1, (-1, 128)).unflatten(0, (-1, 128))
        s = b.abs().amax((1, 3)).clamp(min=1e-30) / 448
        return (b / s[:, None, :, None]).flatten(2).flatten(0, 1)[:n, :k].contiguous().to(torch.float8_e4m3fn), s

    monkeypatch.setattr(hip_ops, "quantize_fp8_weight", quantize)


def test_serving_leaves_the_model_as_it_is(quantized):
    from omarchy_mac_torch import models
    lm = models.mlp_lm(32, 64, 96, 2).train()
    served = lm.serve()
    assert not any(m.training for m in served.modules())
    assert all(m.training for m in lm.modules()) and all(p.requires_grad for p in lm.parameters())
    assert isinstance(served, models.MlpLM) and served.context == lm.context
    before = [v.clone() for v in served.state_dict().values()]
    own = {v.data_ptr() for v in lm.state_dict().values()}
    assert not any(v.data_ptr() in own for v in served.state_dict().values())
    with torch.no_grad():
        for p in lm.parameters():
            p.add_(1)
    after = served.state_dict().values()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, after))


def test_a_served_sublayer_keeps_its_8_bit_types(quantized):
    from omarchy_mac_torch import ffn
    served = ffn.FeedForward(64, 96).serve()
    kept = {k: v.clone() for k, v in served.state_dict().items() if k != "weight"}
    for change in (lambda: served.to(torch.bfloat16), served.float, served.half, lambda: served.to("cpu", torch.float64)):
        change()
        for name, v in kept.items():
            now = getattr(served, name)
            assert now.dtype == v.dtype and torch.equal(now.view(torch.uint8), v.view(torch.uint8))
    assert served.weight.dtype == torch.float64
    assert all(b.device.type == "meta" for b in served.to("meta", torch.bfloat16).buffers())
    assert all(getattr(served, name).dtype == v.dtype for name, v in kept.items())
