"""Preference and policy tuning at the limits of the numbers: NaN in kept tokens, probabilities of zero, norms beyond fp32."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# one block, a block per part of a row, a warp per row
POLICY_SIZES = [(3, 5), (300, 100), (2048, 33)]


@pytest.mark.parametrize("batch,seq", POLICY_SIZES)
@pytest.mark.parametrize("where", ["logprobs", "old_logprobs"])
@pytest.mark.parametrize("masked", [False, True])
def test_policy_loss_keeps_a_nan_beside_an_advantage_of_zero(native_library, batch, seq, where, masked):
    """NaN times zero is NaN in loss and gradient; an infinite ratio times zero is zero, and so is what the mask leaves out."""
    from molt_b200.kernels import clipped_policy_loss

    given = {"logprobs": torch.full((batch, seq), -1.0, device="cuda"), "old_logprobs": torch.full((batch, seq), -1.5, device="cuda")}
    mask = torch.ones(batch, seq, dtype=torch.bool, device="cuda")
    mask[0, 0] = not masked
    given[where][0, 0] = float("nan")
    given["logprobs"][1, 1] = 400.0                       # a ratio of infinity
    leaf = given["logprobs"].requires_grad_()
    for reduction in ("token", "sequence"):
        got = clipped_policy_loss(leaf, given["old_logprobs"], torch.zeros(batch, device="cuda"), mask, reduction=reduction)
        (grad,) = torch.autograd.grad(got.loss, leaf)
        assert math.isnan(float(got.loss)) != masked and math.isnan(float(grad[0, 0])) != masked
        grad[0, 0] = 0.0
        assert not bool(grad.any())
        if masked:
            assert float(got.loss) == 0.0
        assert float(got.clip_fraction) == 0.0
