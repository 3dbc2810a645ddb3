"""The head operators without a GPU: refusals of the C ABI and of the Python calls before a device
is touched, the mask packing, and the 64-bit definitions on known answers."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _heads
from shipinfer_b200 import ConfigurationError, ValidationError, _native
from shipinfer_b200.logprobs import pack_allowed, token_logprobs_device
from shipinfer_b200.routing import combine_experts_device, plan_experts_device, route_experts_device

EINVAL, ERANGE = _native.EINVAL, _native.ERANGE


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def logprobs(lib, *, dtype=0, rows=2, vocab=10, stride=10, n=1, astride=0, temperature=1.0, top=3):
    return lib.shipk_token_logprobs(None, dtype, rows, vocab, stride, None, n, None, astride, temperature, top,
                                    None, None, None, None, None)


@pytest.mark.parametrize(("change", "code", "text"), [
    ({"dtype": 3}, EINVAL, "none of F32"), ({"rows": -1}, EINVAL, "negative"), ({"n": -1}, EINVAL, "negative"),
    ({"top": -1}, EINVAL, "negative"), ({"vocab": 0}, EINVAL, "empty"), ({"stride": -4}, EINVAL, "stride"),
    ({"astride": -1}, EINVAL, "stride"), ({"top": 11}, EINVAL, "above the vocabulary"),
    ({"vocab": 100, "top": 65}, ERANGE, "above 64"), ({"vocab": (1 << 30) + 1}, ERANGE, "2^30"),
    ({"temperature": 0.0}, EINVAL, "temperature"), ({"temperature": float("nan")}, EINVAL, "temperature"),
    ({"temperature": 1e7}, EINVAL, "temperature"), ({"temperature": -1.0}, EINVAL, "temperature"),
    ({}, EINVAL, "logits is null"),
])
def test_logprobs_refusals(lib, change, code, text):
    assert logprobs(lib, **change) == code and text in _native.last_error()


def test_no_rows_are_no_error(lib):
    assert logprobs(lib, rows=0) == 0
    assert route(lib, rows=0) == 0
    assert lib.shipk_combine_experts(None, 0, 0, 4, None, None, 0, 2, 4, None, None) == 0
    assert lib.shipk_combine_experts(None, 0, 0, 0, None, None, 3, 2, 0, None, None) == 0


def route(lib, *, dtype=0, rows=2, experts=8, stride=8, k=2, scores=0, groups=1, top_groups=1, group_score=0):
    return lib.shipk_route_experts(None, dtype, rows, experts, stride, None, k, scores, groups, top_groups,
                                   group_score, 1, 1.0, None, None, None)


@pytest.mark.parametrize(("change", "code", "text"), [
    ({"dtype": -1}, EINVAL, "none of F32"), ({"rows": -1}, EINVAL, "negative"), ({"experts": 0}, EINVAL, "top_k"),
    ({"k": 0}, EINVAL, "top_k"), ({"k": 9}, EINVAL, "top_k"), ({"experts": 1025, "stride": 1025}, ERANGE, "1024"),
    ({"experts": 64, "k": 33}, ERANGE, "above 32"), ({"groups": 3}, EINVAL, "do not divide"),
    ({"groups": 0}, EINVAL, "do not divide"), ({"experts": 64, "groups": 64}, ERANGE, "above 32"),
    ({"groups": 4, "top_groups": 5}, EINVAL, "top_groups"), ({"groups": 4, "top_groups": 0}, EINVAL, "top_groups"),
    ({"scores": 2}, EINVAL, "neither softmax nor sigmoid"), ({"group_score": 2}, EINVAL, "neither max nor top2"),
    ({"stride": -1}, EINVAL, "row_stride"), ({}, EINVAL, "logits is null"),
])
def test_route_refusals(lib, change, code, text):
    assert route(lib, **change) == code and text in _native.last_error()


def test_plan_and_combine_refusals(lib):
    def plan(rows, k, experts):
        return lib.shipk_plan_experts(None, rows, k, experts, None, None, None, None)

    assert plan(-1, 2, 8) == EINVAL and plan(2, 0, 8) == EINVAL and plan(2, 2, 0) == EINVAL
    assert plan(2, 2, 1025) == ERANGE and "1024" in _native.last_error()
    assert plan(1 << 30, 2, 8) == ERANGE and "2^31" in _native.last_error()
    assert plan(2, 2, 8) == EINVAL and "offsets is null" in _native.last_error()

    def combine(dtype=0, n=4, stride=4, rows=2, k=2, width=4):
        return lib.shipk_combine_experts(None, dtype, n, stride, None, None, rows, k, width, None, None)

    assert combine(dtype=9) == EINVAL and "none of F32" in _native.last_error()
    for bad in ({"n": -1}, {"rows": -1}, {"k": 0}, {"width": -1}, {"stride": -1}):
        assert combine(**bad) == EINVAL
    assert combine() == EINVAL and "in is null" in _native.last_error()


def test_python_refusals():
    x, t = torch.zeros(3, 40), torch.zeros(3, dtype=torch.int64)
    bad = [
        lambda: token_logprobs_device(torch.zeros(3, 4, 5)),
        lambda: token_logprobs_device(x.double()),
        lambda: token_logprobs_device(x.t()),
        lambda: token_logprobs_device(x, t[:2]),
        lambda: token_logprobs_device(x, t.int()),
        lambda: token_logprobs_device(x, t, allowed=torch.ones(40, dtype=torch.bool)),
        lambda: token_logprobs_device(x, t, allowed=torch.zeros(1, dtype=torch.int32)),
        lambda: token_logprobs_device(x, t, allowed=torch.zeros((2, 2), dtype=torch.int32)),
        lambda: token_logprobs_device(x, t, entropy=torch.zeros(2)),
        lambda: token_logprobs_device(x, t, top=2, top_ids=torch.zeros((3, 2), dtype=torch.int32)),
        lambda: token_logprobs_device(x, t, top=2, top_logprobs=torch.zeros((2, 3)).t()),
        lambda: token_logprobs_device(x.clone().requires_grad_()),
        lambda: token_logprobs_device(x, t),  # host memory
        lambda: route_experts_device(x, top_k=2, scores="linear"),
        lambda: route_experts_device(x, top_k=2, group_score="sum"),
        lambda: route_experts_device(x, top_k=2, bias=torch.zeros(39)),
        lambda: route_experts_device(x, top_k=2, ids=torch.zeros((3, 2), dtype=torch.int64)),
        lambda: route_experts_device(x, top_k=2),
        lambda: plan_experts_device(torch.zeros(3, dtype=torch.int32), 4),
        lambda: plan_experts_device(torch.zeros((3, 2)), 4),
        lambda: plan_experts_device(torch.zeros((3, 2), dtype=torch.int32), 4, offsets=torch.zeros(4, dtype=torch.int32)),
        lambda: plan_experts_device(torch.zeros((3, 2), dtype=torch.int32), 4),
        lambda: combine_experts_device(x, torch.zeros(2, 2), torch.zeros(2, dtype=torch.int32)),
        lambda: combine_experts_device(x, torch.zeros(2, 3), torch.zeros((2, 2), dtype=torch.int32)),
        lambda: combine_experts_device(x, torch.zeros(2, 2), torch.zeros((2, 2), dtype=torch.int32), out=torch.zeros(2, 41)),
        lambda: combine_experts_device(x, torch.zeros(2, 2, requires_grad=True), torch.zeros((2, 2), dtype=torch.int32)),
        lambda: combine_experts_device(x, torch.zeros(2, 2), torch.zeros((2, 2), dtype=torch.int32)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValidationError):
            call()
            pytest.fail(f"case {i} was accepted")


def test_counts_past_32_bits_are_refused():
    many = torch.zeros(1, 1).expand(1 << 31, 1)
    with pytest.raises(ConfigurationError):
        token_logprobs_device(many)
    with pytest.raises(ConfigurationError):
        route_experts_device(torch.zeros(1, 4), top_k=(1 << 32) + 1)
    with pytest.raises(ConfigurationError):
        plan_experts_device(torch.zeros((1, 1), dtype=torch.int32), (1 << 32) + 1)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 97])
def test_pack_allowed(vocab):
    rng = np.random.default_rng(vocab)
    mask = rng.random((5, vocab)) < 0.5
    mask[0] = True
    words = pack_allowed(torch.from_numpy(mask))
    assert words.dtype == torch.int32 and tuple(words.shape) == (5, (vocab + 31) // 32)
    bits = np.unpackbits(words.numpy().view(np.uint8), axis=1, bitorder="little")
    assert np.array_equal(bits[:, :vocab].astype(bool), mask) and not bits[:, vocab:].any()
    assert torch.equal(pack_allowed(torch.from_numpy(mask[1])), words[1])
    with pytest.raises(ValidationError):
        pack_allowed(torch.zeros(4))
    with pytest.raises(ValidationError):
        pack_allowed(torch.zeros(0, dtype=torch.bool))
    assert pack_allowed(torch.zeros((0, vocab), dtype=torch.bool)).shape == (0, (vocab + 31) // 32)


def test_definitions_on_known_answers():
    x = np.log(np.array([[0.5, 0.25, 0.125, 0.125]]))
    lp, ent, top_lp, ids = _heads.logprobs64(x, np.array([[1, -1, 4]]), top=3)
    assert np.allclose(lp[0, :2], [np.log(0.25), 0]) and np.isnan(lp[0, 2])
    assert np.isclose(ent[0], 1.75 * np.log(2)) and ids.tolist() == [[0, 1, 2]]
    w, ids = _heads.route64(np.array([[0.0, 0.0, 5.0, -np.inf]]), 4, renormalise=False)
    assert ids.tolist() == [[2, 0, 1, -1]] and np.isclose(w.sum(), 1.0, atol=1e-6)
    order, slots, offsets = _heads.plan64(np.array([[1, 0], [0, -1], [2, 0]], np.int32), 3)
    assert order.tolist() == [0, 1, 2, 0, 2, -1] and offsets.tolist() == [0, 3, 4, 5]
    assert slots.tolist() == [[3, 0], [1, -1], [4, 2]]
