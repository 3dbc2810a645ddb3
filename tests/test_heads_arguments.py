"""What the head operators' Python calls refuse by themselves, each by its own message: on the host every
one of these calls would be refused for its device too, which says nothing about the check before it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from shipinfer_b200 import ConfigurationError, ValidationError, _heads
from shipinfer_b200.logprobs import token_logprobs_device
from shipinfer_b200.routing import combine_experts_device, plan_experts_device, route_experts_device


@pytest.mark.parametrize("value", [2.7, "3", None, float("nan"), float("inf"), np.float32(1.5)])
def test_counts_that_are_not_whole_numbers(value):
    x, ids = torch.zeros(3, 40), torch.zeros((3, 2), dtype=torch.int32)
    for call, name in (
        (lambda: token_logprobs_device(x, top=value), "top"),
        (lambda: route_experts_device(x, top_k=value), "top_k"),
        (lambda: route_experts_device(x, top_k=2, groups=value), "groups"),
        (lambda: route_experts_device(x, top_k=2, top_groups=value), "top_groups"),
        (lambda: plan_experts_device(ids, value), "experts"),
    ):
        with pytest.raises(ValidationError, match=f"^{name} must be a whole number"):
            call()


def test_whole_numbers_of_any_kind():
    assert [_heads.small(v, "n") for v in (3, 3.0, True, np.int64(3), np.float32(3), torch.tensor(3))] == [3, 3, 1, 3, 3, 3]
    with pytest.raises(ConfigurationError, match="does not fit"):
        _heads.small(1 << 31, "n")
    assert _heads.small(-(1 << 31), "n") == -(1 << 31)


def test_gradients_and_tangents():
    """Scores, weights and biases that carry a gradient or a forward-mode tangent: the results would lose it."""
    x, w, slots = torch.zeros(3, 40), torch.zeros(3, 2), torch.zeros((3, 2), dtype=torch.int32)
    bias = torch.zeros(40)

    def calls(carries):
        return [
            (lambda: token_logprobs_device(carries(x)), "logits"),
            (lambda: token_logprobs_device(x, entropy=carries(torch.zeros(3))), "entropy"),
            (lambda: route_experts_device(carries(x), top_k=2), "logits"),
            (lambda: route_experts_device(x, top_k=2, bias=carries(bias)), "bias"),
            (lambda: combine_experts_device(carries(x), w, slots), "rows"),
            (lambda: combine_experts_device(x, carries(w), slots), "weights"),
        ]

    def refused(carries):
        for call, name in calls(carries):
            with pytest.raises(ValidationError, match=f"^{name} asks for a gradient"):
                call()

    def passed_over(carries):  # to the next check, the device's
        for call, _ in calls(carries):
            with pytest.raises(ValidationError, match="must be CUDA tensors"):
                call()

    refused(lambda t: t.clone().requires_grad_())
    with torch.no_grad():
        passed_over(lambda t: t.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        refused(lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        passed_over(lambda t: torch.autograd.forward_ad.unpack_dual(
            torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))).primal)
        passed_over(lambda t: t)
    passed_over(lambda t: t)
