"""The head operators' results may not lie over their inputs or one another: a plan reads its ids twice
and places what it reads, so ids that its own results replace would send it past the end. The C ABI refuses
by the addresses alone, before it asks for a device: these calls never reach one."""

from __future__ import annotations

import pytest

from shipinfer_b200 import ValidationError, _native
from shipinfer_b200.routing import plan_experts_device

EINVAL = _native.EINVAL
A = 1 << 40  # an address; nothing reads it


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def refused(code, text):
    return code == EINVAL and text in _native.last_error()


def passed_over(code):
    """Not refused for its addresses: what is missing is a device."""
    return code != 0 and "overlaps" not in _native.last_error()


def plan(lib, ids, order, slots, offsets, rows=100, k=2, experts=8):
    return lib.shipk_plan_experts(ids, rows, k, experts, order, slots, offsets, None)


def test_plan(lib):
    far = [A + 4096 * i for i in range(4)]
    assert passed_over(plan(lib, *far))
    assert refused(plan(lib, A, A, far[2], far[3]), "order overlaps ids")
    assert refused(plan(lib, A, far[1], A, far[3]), "slots overlaps ids")
    assert refused(plan(lib, A, far[1], A + 796, far[3]), "slots overlaps ids")  # by its last id
    assert refused(plan(lib, A, far[1], A - 796, far[3]), "slots overlaps ids")  # by its first
    assert passed_over(plan(lib, A, far[1], A + 800, far[3]))
    assert passed_over(plan(lib, A, far[1], A - 800, far[3]))
    assert refused(plan(lib, A, far[1], far[1], far[3]), "slots overlaps order")
    assert refused(plan(lib, A, far[1], far[2], A - 4), "offsets overlaps ids")
    assert refused(plan(lib, A, far[1], far[2], far[2] + 100), "offsets overlaps slots")


def route(lib, logits, weights, ids, *, bias=None, rows=50, experts=64, stride=64, k=4, dtype=0):
    return lib.shipk_route_experts(logits, dtype, rows, experts, stride, bias, k, 0, 1, 1, 0, 1, 1.0, weights, ids, None)


def test_route(lib):
    w, i = A + (1 << 20), A + (2 << 20)
    assert passed_over(route(lib, A, w, i))
    assert refused(route(lib, A, A, i, k=32), "weights overlaps logits")
    assert refused(route(lib, A, w, A + 50 * 64 * 4 - 4), "ids overlaps logits")
    assert passed_over(route(lib, A, w, A + 50 * 64 * 4))
    assert refused(route(lib, A, w, A + 50 * 64 * 2 - 2, dtype=1), "ids overlaps logits")
    assert passed_over(route(lib, A, w, A + 50 * 64 * 2, dtype=1))
    assert refused(route(lib, A, w, w), "ids overlaps weights")
    assert refused(route(lib, A, w, i, bias=w + 796), "weights overlaps bias")


def test_results_between_rows(lib):
    """Rows that lie apart leave room: a result in a gap is apart from them, one that touches a row is not.
    Here 50 rows of 64 float32 (256 bytes), 8192 bytes apart, and results of 800 bytes."""
    w = A - (1 << 20)

    def at(offset, **more):
        return route(lib, A, w, A + offset, stride=2048, **more)

    assert passed_over(at(256)) and passed_over(at(8192 - 800)) and passed_over(at(3 * 8192 + 256))
    assert refused(at(252), "ids overlaps logits") and refused(at(8192 - 796), "ids overlaps logits")
    assert refused(at(49 * 8192 + 252), "ids overlaps logits")
    assert passed_over(at(49 * 8192 + 256)) and passed_over(at(50 * 8192))
    # one row for all of them, and strides that no address space holds
    assert refused(route(lib, A, w, A + 252, stride=0), "ids overlaps logits")
    assert passed_over(route(lib, A, w, A + 256, stride=0))
    assert passed_over(route(lib, A, w, A + 256, stride=(1 << 63) - 1))


def logprobs(lib, logits, lp, ent, top_lp, ids, *, tokens=A + (8 << 20), allowed=None, astride=0, vocab=100, n=2):
    return lib.shipk_token_logprobs(logits, 0, 10, vocab, vocab, tokens, n, allowed, astride, 1.0, 3, lp, ent, top_lp,
                                    ids, None)


def test_logprobs(lib):
    far = [A + (1 << 20) * i for i in range(5)]
    assert passed_over(logprobs(lib, *far))
    for k, name in ((1, "logprobs"), (2, "entropy"), (3, "top_logprobs"), (4, "top_ids")):
        over = list(far)
        over[k] = A + 3996  # the last score
        assert refused(logprobs(lib, *over), f"{name} overlaps logits")
        over[k] = A + (8 << 20) + 152  # the last token
        assert refused(logprobs(lib, *over), f"{name} overlaps tokens")
    assert refused(logprobs(lib, *far, allowed=far[2] + 36), "entropy overlaps allowed")
    assert refused(logprobs(lib, *far, allowed=far[2] - 16 * 4 * 9 - 12, astride=16), "entropy overlaps allowed")
    assert passed_over(logprobs(lib, *far, allowed=far[2] - 16 * 4 * 9 - 16, astride=16))
    assert refused(logprobs(lib, far[0], far[1], far[2], far[1] + 76, far[4]), "top_logprobs overlaps logprobs")
    # counts whose bytes pass 64 bits are no smaller for it
    assert refused(lib.shipk_token_logprobs(A, 0, 2**31 - 1, 100, 100, A + (1 << 45), 2**31 - 1, None, 0, 1.0, 0, A - 4, A - 8,
                                            None, None, None), "logprobs overlaps logits")


def combine(lib, rows, weights, slots, out, *, n=20, stride=32, r=20, k=2, width=32, dtype=2):
    return lib.shipk_combine_experts(rows, dtype, n, stride, weights, slots, r, k, width, out, None)


def test_combine(lib):
    w, s, o = A + (1 << 20), A + (2 << 20), A + (3 << 20)
    assert passed_over(combine(lib, A, w, s, o))
    assert refused(combine(lib, A, w, s, A), "out overlaps in")
    assert refused(combine(lib, A, w, s, w + 156), "out overlaps weights")
    assert refused(combine(lib, A, w, s, s - 1278), "out overlaps slots")
    assert passed_over(combine(lib, A, w, s, s - 1280))
    assert passed_over(combine(lib, None, w, s, o, n=0))


@pytest.mark.gpu
def test_calls_of_one_tensor_are_refused_and_nothing_is_launched(cuda):
    torch = cuda
    ids = torch.randint(0, 8, (5000, 2), device="cuda", dtype=torch.int32)
    before = ids.clone()
    for results in ({"slots": ids}, {"order": ids.view(-1)}):
        with pytest.raises(ValidationError, match="overlaps ids"):
            plan_experts_device(ids, 8, **results)
    torch.cuda.synchronize()
    assert torch.equal(ids, before)
