"""Losses on logits where weights of zero decide, beside test_gpu_lm.py, whose inputs these use."""

import math

import pytest
import torch

from test_gpu_lm import F32, some_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    from omarchy_mac_torch import hip_ops
    return hip_ops


# ---- the KL term ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("vocab", [40, 70001])
def test_a_kl_term_of_weight_zero_takes_no_part(ops, cuda, reduction, vocab):
    """Infinite terms that are only watched: a label that the reference bans, one that the policy bans."""
    x, labels = some_logits(4, 5, vocab, F32, 21, masked=0.0)
    x[1, 2, labels[1, 2]] = -math.inf
    x[3, 0, labels[3, 0]] = -math.inf
    ref, old = torch.full((4, 5), -3.0), torch.full((4, 5), -4.0)
    ref[0, 1] = ref[2, 4] = -math.inf
    adv = torch.tensor([1.0, 1.0, -2.0, -2.0])
    args = [t.cuda() for t in (x, labels, old, adv)]
    loss, none, logps, gx = ops.policy_loss(*args, reduction=reduction)
    got = ops.policy_loss(*args, reference=ref.cuda(), kl=0.0, reduction=reduction)
    assert math.isfinite(float(loss)) and float(none) == 0 and not math.isfinite(float(got[1]))
    assert torch.equal(got[0], loss) and torch.equal(got[2], logps) and torch.equal(got[3], gx) and not bool(gx.isnan().any())
