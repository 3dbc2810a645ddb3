"""What the head operators' Python calls refuse by themselves, each by its own message: on the host every
one of these calls would be refused for its device too, which says nothing about the check before it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from shipinfer_b200 import ConfigurationError, ValidationError, _heads, _native
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


def test_result_tensors():
    """check_dense is all that stands between a result that is too small, or not dense, and a write past it."""
    shape = (3, 4)
    good = torch.zeros(shape)
    _heads.check_dense(good, "out", torch.float32, shape)
    _heads.check_dense(torch.zeros((0, 4)), "out", torch.float32, (0, 4))
    _heads.check_dense(torch.zeros((5, 4))[1:4], "out", torch.float32, shape)
    for bad in (torch.zeros((3, 3)), torch.zeros((2, 4)), torch.zeros(12), torch.zeros((3, 4, 1)), torch.zeros((4, 3)).t(),
                torch.zeros((3, 8))[:, ::2], torch.zeros((3, 5))[:, :4], torch.zeros((1, 4)).expand(3, 4),
                good.double(), good.half(), good.int()):
        with pytest.raises(ValidationError, match="^out must be a contiguous float32"):
            _heads.check_dense(bad, "out", torch.float32, shape)


def test_matrices_and_types():
    assert _heads.check_matrix(torch.zeros((3, 8))[:, :5], "rows") == (3, 5)
    assert _heads.check_matrix(torch.zeros((1, 5)).expand(3, 5), "rows") == (3, 5)
    assert _heads.check_matrix(torch.zeros((3, 8))[:, ::8], "rows") == (3, 1)
    for bad in (torch.zeros(3), torch.zeros((1, 2, 3)), torch.zeros(())):
        with pytest.raises(ValidationError, match="^rows must have two dimensions"):
            _heads.check_matrix(bad, "rows")
    for bad in (torch.zeros((5, 3)).t(), torch.zeros((3, 8))[:, ::2], torch.zeros((3, 1)).expand(3, 5)):
        with pytest.raises(ValidationError, match="^rows: the values of a row must be adjacent"):
            _heads.check_matrix(bad, "rows")
    with pytest.raises(ConfigurationError, match="do not fit"):
        _heads.check_matrix(torch.zeros((1, 1)).expand(1, 1 << 31), "rows")
    codes = [_heads.element_code(torch.zeros(1, dtype=t), "x") for t in (torch.float32, torch.float16, torch.bfloat16)]
    assert codes == [0, 1, 2]
    for t in (torch.float64, torch.int32, torch.bool, torch.float8_e4m3fn, torch.complex64):
        with pytest.raises(ValidationError, match="^x must be float32, float16 or bfloat16"):
            _heads.element_code(torch.zeros(1, dtype=t), "x")


X, T, IDS, W = torch.zeros(3, 40), torch.zeros(3, dtype=torch.int64), torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, 2)
I32, I64 = torch.int32, torch.int64


@pytest.mark.parametrize(("call", "text"), [
    (lambda: token_logprobs_device(X[0]), "logits must have two dimensions"),
    (lambda: token_logprobs_device(X.double()), "logits must be float32"),
    (lambda: token_logprobs_device(torch.zeros(40, 3).t()), "logits: the values of a row must be adjacent"),
    (lambda: token_logprobs_device(X, T[:2]), r"tokens must be \[3\]"),
    (lambda: token_logprobs_device(X, T.view(1, 3, 1)), r"tokens must be \[3\]"),
    (lambda: token_logprobs_device(X, T.int()), "tokens must be a contiguous int64"),
    (lambda: token_logprobs_device(X, torch.zeros((2, 3), dtype=I64).t()), "tokens must be a contiguous int64"),
    (lambda: token_logprobs_device(X, allowed=torch.ones(40, dtype=torch.bool)), "allowed must be int32 bits"),
    (lambda: token_logprobs_device(X, allowed=torch.zeros(1, dtype=I32)), "allowed must be int32 bits"),
    (lambda: token_logprobs_device(X, allowed=torch.zeros((2, 2), dtype=I32)), "allowed must be int32 bits"),
    (lambda: token_logprobs_device(X, allowed=torch.zeros((2, 3), dtype=I32).t()), "allowed must be int32 bits"),
    (lambda: token_logprobs_device(X, allowed=torch.zeros((3, 1, 2), dtype=I32)), "allowed must be int32 bits"),
    (lambda: token_logprobs_device(X, T, logprobs=torch.zeros(3, 1)), "logprobs must be a contiguous float32"),
    (lambda: token_logprobs_device(X, logprobs=torch.zeros(3)), "logprobs must be a contiguous float32"),
    (lambda: token_logprobs_device(X, entropy=torch.zeros(2)), "entropy must be a contiguous float32"),
    (lambda: token_logprobs_device(X, top=2, top_ids=torch.zeros((3, 2), dtype=I32)), "top_ids must be a contiguous int64"),
    (lambda: token_logprobs_device(X, top=2, top_ids=torch.zeros((3, 1), dtype=I64)), "top_ids must be a contiguous int64"),
    (lambda: token_logprobs_device(X, top=2, top_logprobs=torch.zeros((2, 3)).t()), "top_logprobs must be a contiguous"),
    (lambda: token_logprobs_device(X, top=2, top_logprobs=torch.zeros((2, 2))), "top_logprobs must be a contiguous"),
    (lambda: route_experts_device(X[0], top_k=2), "logits must have two dimensions"),
    (lambda: route_experts_device(X.int(), top_k=2), "logits must be float32"),
    (lambda: route_experts_device(X, top_k=2, scores="linear"), "scores must be"),
    (lambda: route_experts_device(X, top_k=2, group_score="sum"), "group_score must be"),
    (lambda: route_experts_device(X, top_k=2, bias=torch.zeros(39)), "bias must be a contiguous float32"),
    (lambda: route_experts_device(X, top_k=2, bias=torch.zeros(40).half()), "bias must be a contiguous float32"),
    (lambda: route_experts_device(X, top_k=2, weights=torch.zeros(3, 1)), "weights must be a contiguous float32"),
    (lambda: route_experts_device(X, top_k=2, ids=torch.zeros((3, 2), dtype=I64)), "ids must be a contiguous int32"),
    (lambda: route_experts_device(X, top_k=2, ids=torch.zeros((2, 2), dtype=I32)), "ids must be a contiguous int32"),
    (lambda: plan_experts_device(IDS.view(-1), 4), r"ids must be int32 \[rows, k\]"),
    (lambda: plan_experts_device(IDS.long(), 4), "ids must be a contiguous int32"),
    (lambda: plan_experts_device(torch.zeros((2, 3), dtype=I32).t(), 4), "ids must be a contiguous int32"),
    (lambda: plan_experts_device(IDS, 4, order=torch.zeros(5, dtype=I32)), "order must be a contiguous int32"),
    (lambda: plan_experts_device(IDS, 4, slots=torch.zeros((2, 3), dtype=I32)), "slots must be a contiguous int32"),
    (lambda: plan_experts_device(IDS, 4, offsets=torch.zeros(4, dtype=I32)), "offsets must be a contiguous int32"),
    (lambda: combine_experts_device(X[0], W, IDS), "rows must have two dimensions"),
    (lambda: combine_experts_device(X.double(), W, IDS), "rows must be float32"),
    (lambda: combine_experts_device(X, W, IDS.view(-1)), r"slots must be int32 \[rows, k\]"),
    (lambda: combine_experts_device(X, W, IDS.long()), "slots must be a contiguous int32"),
    (lambda: combine_experts_device(X, W[:2], IDS), "weights must be a contiguous float32"),
    (lambda: combine_experts_device(X, W.half(), IDS), "weights must be a contiguous float32"),
    (lambda: combine_experts_device(X, W, IDS, out=torch.zeros(2, 40)), "out must be a contiguous float32"),
    (lambda: combine_experts_device(X, W, IDS, out=torch.zeros(3, 40).half()), "out must be a contiguous float32"),
    # and nothing before the device's check refuses what is right
    (lambda: token_logprobs_device(X, T, top=2, allowed=torch.zeros((3, 4), dtype=I32), logprobs=torch.zeros(3),
                                   entropy=torch.zeros(3), top_logprobs=torch.zeros(3, 2),
                                   top_ids=torch.zeros((3, 2), dtype=I64)), "must be CUDA tensors"),
    (lambda: route_experts_device(X, top_k=2, bias=torch.zeros(40), weights=W, ids=IDS), "must be CUDA tensors"),
    (lambda: plan_experts_device(IDS, 4, order=torch.zeros(6, dtype=I32), slots=IDS, offsets=torch.zeros(5, dtype=I32)),
     "must be CUDA tensors"),
    (lambda: combine_experts_device(X, W, IDS, out=torch.zeros(3, 40)), "must be CUDA tensors"),
])
def test_each_refusal_by_its_own_check(call, text):
    with pytest.raises(ValidationError, match=text):
        call()


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan"), 1e39])
def test_scales_that_are_not_finite(scale):
    """Times such a scale, the weight 0 of an expert that is not there would be NaN."""
    lib = _native.lib()
    code = lib.shipk_route_experts(None, 0, 0, 8, 8, None, 2, 0, 1, 1, 0, 1, scale, None, None, None)
    assert code == _native.EINVAL and "scale" in _native.last_error()
    for fine in (0.0, -2.5, 3.4e38):
        assert lib.shipk_route_experts(None, 0, 0, 8, 8, None, 2, 0, 1, 1, 0, 1, fine, None, None, None) == 0
