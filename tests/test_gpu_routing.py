"""Routing to experts on the GPU (shipk_route_experts, _plan_experts, _combine_experts) against
their definitions in 64 bits.

The chosen ids, the plan and the padding are exact. Weights are computed in 64 bits from scores
rounded to 32 and rounded once: half a step, u = 2^-24 relative, plus what the last place of a
64-bit exponential moves a score across a rounding border (another step of its score, 2 u, in the
numerator and in the sum); 6 u. A combined value is a sum of k products in 32 bits, k u times the sum of the
magnitudes, rounded once to the type: half of its step."""

from __future__ import annotations

import numpy as np
import pytest

import _heads
from shipinfer_b200 import ConfigurationError, NormalizeParams, ValidationError
from shipinfer_b200.logprobs import token_logprobs_device
from shipinfer_b200.routing import combine_experts_device, plan_experts_device, route_experts_device

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")


def check(torch, x, k, bias=None, **how):
    """x: a CUDA tensor [rows, experts]; bias: a float32 array or None."""
    w, ids = route_experts_device(x, top_k=k, bias=None if bias is None else torch.from_numpy(bias).cuda(), **how)
    torch.cuda.synchronize()
    want_w, want_ids = _heads.route64(x.double().cpu().numpy(), k, bias=bias, **how)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.double().cpu().numpy()
    tiny = 2.0**-148  # the smallest steps of float32, for weights below its normal range
    assert (np.abs(got - want_w) <= 6 * _heads.EPS32 * np.abs(want_w) + tiny).all()
    return w, ids


def gate(torch, rows, experts, dtype, seed):
    x = np.random.default_rng(seed).normal(0.0, 1.5, (rows, experts))
    return torch.from_numpy(x).to(getattr(torch, dtype)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize(("rows", "experts", "k"), [
    (1, 1, 1), (1, 2, 2), (3, 5, 2), (33, 8, 2), (1, 31, 31), (5, 32, 32), (7, 33, 8), (130, 64, 6), (9, 100, 16),
    (257, 256, 8), (3, 513, 32), (5, 1000, 7), (11, 1024, 32)])
def test_sizes_and_types(cuda, rows, experts, k, dtype, scores):
    x = gate(cuda, rows, experts, dtype, rows + experts)
    bias = np.random.default_rng(experts).normal(0, 0.1, experts).astype(np.float32)
    check(cuda, x, k, scores=scores)
    check(cuda, x, k, bias, scores=scores, renormalise=False, scale=2.5)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize(("experts", "groups", "top_groups", "k"), [
    (4, 2, 1, 2), (256, 8, 4, 8), (160, 8, 3, 6), (63, 7, 2, 8), (64, 32, 5, 8), (32, 32, 4, 6), (1024, 32, 32, 32),
    (96, 3, 1, 32), (1000, 20, 1, 1), (992, 31, 30, 9)])
def test_groups(cuda, experts, groups, top_groups, k, group_score):
    x = gate(cuda, 70, experts, "float32", experts + groups)
    bias = np.random.default_rng(groups).normal(0, 0.1, experts).astype(np.float32)
    for scores in ("softmax", "sigmoid"):
        check(cuda, x, k, bias, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score, scale=2.5)
        check(cuda, x, k, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [1, 4])
def test_masks_ties_and_extremes(cuda, scores, dtype, groups):
    """Equal logits (ties to the lower expert, -0 and +0 alike), masked experts and rows, groups
    with one or no expert left, NaN, infinities, the type's limits, scores that round to 0 or 1."""
    torch = cuda
    t = getattr(torch, dtype)
    experts = 64
    x = torch.zeros((14, experts))
    x[0, ::3] = -0.0
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, [3, 40]] = torch.tensor([1.0, 2.0])
    x[3] = float("nan")
    x[3, 63] = 0.5
    x[4, 7] = float("inf")
    x[4, 9] = float("inf")
    x[5] = torch.finfo(t).min
    x[6] = torch.finfo(t).max
    x[6, 5] = torch.finfo(t).min
    x[7] = torch.linspace(20, 60, experts)
    x[8] = torch.linspace(-200, -90, experts)
    x[9] = -np.inf
    x[9, 16:32] = 1.0
    x[9, 33] = 7.0
    x[10] = torch.arange(experts) // 8
    x[11] = torch.finfo(t).min
    x[11, 50:] = 0.25
    x[12, 1::2] = float("nan")
    x[13] = torch.randn(experts, generator=torch.Generator().manual_seed(3))
    x = x.to(t).cuda()
    bias = np.zeros(experts, np.float32)
    bias[2], bias[20], bias[21], bias[50] = -np.inf, np.nan, np.inf, -3e38
    how = {"scores": scores, "groups": groups, "top_groups": min(groups, 2), "group_score": "top2"}
    for k in (1, 8, 20):
        check(cuda, x, k, **how)
        check(cuda, x, k, bias, renormalise=False, **how)
        check(cuda, x, k, bias, **how)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_close_choices(cuda, scores):
    """Logits a step apart: scores that differ in their last place or only before they are
    rounded, with biases that bring different scores together."""
    rng = np.random.default_rng(17)
    base = np.float32(0.731)
    x = (base.view(np.int32) + rng.integers(-3, 4, (400, 128)).astype(np.int32)).view(np.float32)
    check(cuda, cuda.from_numpy(x).cuda(), 8, scores=scores)
    y = rng.normal(0, 2, (400, 128)).astype(np.float32)
    y[:, 64:] = y[:, :64]
    check(cuda, cuda.from_numpy(y).cuda(), 8, scores=scores)
    s = 1 / (1 + np.exp(-y[0].astype(np.float64)))
    bias = (0.5 - s).astype(np.float32)  # row 0: every choice within a step or two of 0.5
    check(cuda, cuda.from_numpy(np.tile(y[:1], (5, 1))).cuda(), 8, bias, scores="sigmoid")


@pytest.mark.parametrize("dtype", TYPES)
def test_route_strides(cuda, dtype):
    wide = gate(cuda, 20, 150, dtype, 2)
    for lo in (0, 1, 3, 8):
        check(cuda, wide[:, lo : lo + 130], 5)
    check(cuda, wide[::3, 2:66], 5, scores="sigmoid")
    check(cuda, wide[4:5, :70].expand(6, 70), 5)
    check(cuda, wide[:0], 5)


def test_one_wide_row_past_32_bits(cuda):
    stride = (1 << 31) + 32
    flat = cuda.empty(2 * stride, dtype=cuda.float16, device="cuda")
    x = flat.as_strided((2, 100), (stride, 1))
    x.copy_(gate(cuda, 2, 100, "float16", 4))
    check(cuda, x, 5)


# ---- plan -----------------------------------------------------------------------------------

def check_plan(torch, ids, experts, **outs):
    got = plan_experts_device(torch.from_numpy(ids).cuda(), experts, **outs)
    torch.cuda.synchronize()
    for g, w in zip(got, _heads.plan64(ids, experts)):
        assert np.array_equal(g.cpu().numpy(), w)
    return got


@pytest.mark.parametrize(("rows", "k", "experts"), [
    (0, 2, 5), (1, 1, 1), (1, 8, 256), (3, 2, 7), (31, 1, 3), (64, 8, 256), (33, 5, 1024), (513, 2, 8), (1000, 3, 1),
    (4096, 8, 64), (16384, 8, 256), (20011, 7, 1000), (130001, 1, 33), (300000, 4, 1024)])
def test_plans(cuda, rows, k, experts):
    rng = np.random.default_rng(rows + experts)
    ids = rng.integers(0, experts, (rows, k)).astype(np.int32)
    check_plan(cuda, ids, experts)
    skewed = np.minimum(rng.geometric(0.2, (rows, k)) - 1, experts - 1).astype(np.int32)
    skewed[rng.random((rows, k)) < 0.3] = -1
    skewed[rng.random((rows, k)) < 0.05] = experts
    skewed[rng.random((rows, k)) < 0.01] = 2**31 - 1
    check_plan(cuda, skewed, experts)


def test_plan_of_one_expert_and_of_none(cuda):
    check_plan(cuda, np.full((5000, 4), 9, np.int32), 16)
    check_plan(cuda, np.full((700, 2), -1, np.int32), 16)
    check_plan(cuda, np.full((5, 2), -(2**31), np.int32), 16)


def test_plan_writes_nothing_beside_its_results(cuda):
    torch = cuda
    rows, k, experts = 501, 3, 20
    ids = np.random.default_rng(1).integers(-1, experts, (rows, k)).astype(np.int32)
    held = torch.full((3 * rows * k + experts + 1 + 64,), 77, dtype=torch.int32, device="cuda")
    n = rows * k
    order, slots = held[16 : 16 + n], held[32 + n : 32 + 2 * n].view(rows, k)
    offsets = held[48 + 2 * n : 48 + 2 * n + experts + 1]
    check_plan(cuda, ids, experts, order=order, slots=slots, offsets=offsets)
    for lo, hi in ((0, 16), (16 + n, 32 + n), (32 + 2 * n, 48 + 2 * n), (48 + 2 * n + experts + 1, held.numel())):
        assert (held[lo:hi] == 77).all()


# ---- combine --------------------------------------------------------------------------------

def check_combine(torch, y, w, slots, **outs):
    out = combine_experts_device(y, torch.from_numpy(w).cuda(), torch.from_numpy(slots).cuda(), **outs)
    torch.cuda.synchronize()
    want, size = _heads.combine64(y.double().cpu().numpy(), w, slots)
    half = torch.finfo(y.dtype).eps / 2
    tiny = float(torch.finfo(y.dtype).smallest_normal) * torch.finfo(y.dtype).eps
    limit = slots.shape[1] * _heads.EPS32 * size * (1 + half) + half * np.abs(want) + tiny
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= limit).all(), float((err / np.maximum(limit, 1e-300)).max())
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "k", "width"), [
    (1, 1, 1), (3, 2, 7), (64, 2, 512), (33, 8, 130), (5, 32, 1000), (2, 40, 64), (700, 3, 33), (257, 4, 2048), (9, 1, 8),
    (40, 6, 4104)])
def test_combine_sizes_and_types(cuda, rows, k, width, dtype):
    rng = np.random.default_rng(rows + width)
    y = cuda.from_numpy(rng.normal(0, 1, (rows * k, width))).to(getattr(cuda, dtype)).cuda()
    w = rng.random((rows, k)).astype(np.float32)
    slots = rng.permutation(rows * k).reshape(rows, k).astype(np.int32)
    check_combine(cuda, y, w, slots)
    slots[rng.random((rows, k)) < 0.2] = -1
    slots[rng.random((rows, k)) < 0.1] = rows * k  # one past the results
    w[slots < 0] = np.nan  # the weight of nothing
    check_combine(cuda, y, np.where(slots == rows * k, np.inf, w).astype(np.float32), slots)


@pytest.mark.parametrize("dtype", TYPES)
def test_combine_strides_repeats_and_nothing(cuda, dtype):
    torch = cuda
    rng = np.random.default_rng(3)
    wide = torch.from_numpy(rng.normal(0, 1, (50, 300))).to(getattr(torch, dtype)).cuda()
    w = rng.normal(0, 1, (21, 3)).astype(np.float32)
    slots = rng.integers(0, 25, (21, 3)).astype(np.int32)  # the same result for several rows
    for lo, width in ((0, 256), (8, 256), (1, 256), (2, 100), (4, 33)):
        check_combine(torch, wide[::2, lo : lo + width], w, slots)
    check_combine(torch, wide[:25].expand(25, 300), w, np.full((21, 3), -1, np.int32))
    out = combine_experts_device(wide[:0], torch.from_numpy(w).cuda(), torch.from_numpy(slots).cuda())
    assert out.shape == (21, 300) and (out == 0).all()
    held = torch.full((23, 33), 77.0, dtype=wide.dtype, device="cuda")
    check_combine(torch, wide[:25, :33], w, slots, out=held[1:22])
    assert (held[0] == 77).all() and (held[22] == 77).all()


def test_combine_past_32_bits(cuda):
    torch = cuda
    n, width = 70000, 40000
    y = torch.empty((n, width), dtype=torch.float16, device="cuda")  # 5.6 GB, 2.8e9 values
    picked = [0, 1, 53687, 53688, n - 1]
    y[picked] = torch.randn((5, width), device="cuda").half()
    slots = np.array([[0, n - 1], [53688, 53687], [1, -1]], np.int32)
    w = np.array([[0.5, 0.25], [1.0, -1.0], [2.0, 9.0]], np.float32)
    out = combine_experts_device(y, torch.from_numpy(w).cuda(), torch.from_numpy(slots).cuda())
    want = torch.stack([0.5 * y[0].float() + 0.25 * y[n - 1].float(), y[53688].float() - y[53687].float(), 2 * y[1].float()])
    assert torch.equal(out, want.half())  # products by powers of two and one addition: one rounding


# ---- together -------------------------------------------------------------------------------

def test_crops_through_soft_embedders_to_a_reader(cuda, ops, orc):
    """A frame's detections: a gate scores four embedders for each, the plan orders the crops so
    that each embedder's batch is one run of one crop launch, the embeddings come back weighted,
    and a reader's scores over them become log-probabilities."""
    torch = cuda
    rng = np.random.default_rng(12)
    frame = rng.integers(0, 256, (180, 320, 3), dtype=np.uint8)
    n, experts, k, width, vocab = 23, 4, 2, 48, 301
    x0, y0 = rng.uniform(0, 200, n), rng.uniform(0, 100, n)
    boxes = np.stack([x0, y0, x0 + rng.uniform(8, 100, n), y0 + rng.uniform(8, 70, n)], axis=1).astype(np.float32)
    scored = torch.from_numpy(rng.normal(0, 1, (n, experts)).astype(np.float32)).cuda()
    closed = torch.tensor([0.0, 0.0, -np.inf, 0.0], device="cuda")
    weights, ids = route_experts_device(scored, top_k=k, scores="sigmoid", bias=closed)
    order, slots, offsets = plan_experts_device(ids, experts)
    crops = torch.empty((n * k, 3, 16, 8), dtype=torch.float32, device="cuda")
    ops.crop_device([torch.from_numpy(frame).cuda()], torch.from_numpy(boxes).cuda()[order.long()].contiguous(), crops,
                    NormalizeParams())
    embedders = torch.from_numpy(rng.normal(0, 0.1, (experts, 3 * 16 * 8, width)).astype(np.float32)).cuda()
    embedded = torch.zeros((n * k, width), device="cuda")
    bounds = offsets.tolist()
    assert bounds[2] == bounds[3] and bounds[-1] == n * k
    for e in range(experts):
        embedded[bounds[e] : bounds[e + 1]] = (crops[bounds[e] : bounds[e + 1]].flatten(1).double() @ embedders[e].double()).float()
    joined = combine_experts_device(embedded, weights, slots)
    head = torch.from_numpy(rng.normal(0, 0.5, (width, vocab)).astype(np.float32)).cuda()
    logits = (joined.double() @ head.double()).float()
    lp, ent, top_lp, top_ids = token_logprobs_device(logits, torch.arange(n, device="cuda"), top=3)

    want_w, want_ids = _heads.route64(scored.double().cpu().numpy(), k, scores="sigmoid",
                                      bias=np.array([0, 0, -np.inf, 0], np.float32))
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    flat = orc.crop([frame], boxes, (16, 8), None, (0, 0, 0), (255, 255, 255), True).reshape(n, -1).astype(np.float64)
    each = np.einsum("nc,ecw->new", flat, embedders.double().cpu().numpy())
    want = sum(want_w[:, j, None] * each[np.arange(n), want_ids[:, j]] for j in range(k))
    # an embedding is rounded once (u), a weight has 6 u, the sum of two products 2 u
    size = sum(want_w[:, j, None] * np.abs(each[np.arange(n), want_ids[:, j]]) for j in range(k))
    assert (np.abs(joined.double().cpu().numpy() - want) <= 10 * _heads.EPS32 * size).all()
    ref = _heads.logprobs64(logits.double().cpu().numpy(), np.arange(n), top=3)
    assert np.array_equal(top_ids.cpu().numpy(), ref[3])
    # (64 + 64 + 8 |logprob| + 8 ln V) u, as the log-probabilities' own tests derive it
    limit = _heads.EPS32 * (128 + 8 * np.abs(ref[0][:, 0]) + 8 * np.log(vocab + 1))
    assert (np.abs(lp.double().cpu().numpy() - ref[0][:, 0]) <= limit).all()


def test_a_step_replays_from_one_graph(cuda):
    torch = cuda
    rows, experts, k, width, vocab = 300, 32, 4, 64, 1500
    x = gate(cuda, rows, experts, "bfloat16", 1)
    results = torch.randn((rows * k, width), device="cuda", dtype=torch.float16)
    logits, tokens = torch.randn((rows, vocab), device="cuda"), torch.arange(rows, device="cuda")

    def step():
        w, ids = route_experts_device(x, top_k=k)
        order, slots, offsets = plan_experts_device(ids, experts)
        return (w, ids, order, slots, offsets, combine_experts_device(results, w, slots),
                *token_logprobs_device(logits, tokens, top=6))

    step()  # first launches outside capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (2, 3):
        x.copy_(gate(cuda, rows, experts, "bfloat16", seed))
        results.normal_()
        logits.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_explicit_streams(cuda):
    torch = cuda
    side = torch.cuda.Stream()
    x = gate(cuda, 500, 64, "float32", 6)
    y = torch.randn((1000, 96), device="cuda")
    torch.cuda.synchronize()
    s = side.cuda_stream
    w, ids = route_experts_device(x, top_k=2, stream=s)
    order, slots, offsets = plan_experts_device(ids, 64, stream=s)
    out = combine_experts_device(y, w, slots, stream=s)
    side.synchronize()
    want_w, want_ids = route_experts_device(x, top_k=2)
    assert torch.equal(w, want_w) and torch.equal(ids, want_ids)
    assert all(torch.equal(a, b) for a, b in zip((order, slots, offsets), plan_experts_device(ids, 64)))
    assert torch.equal(out, combine_experts_device(y, w, slots))


def test_refusals(cuda):
    torch = cuda
    x = torch.zeros((3, 64), device="cuda")
    with pytest.raises(ConfigurationError):
        route_experts_device(x, top_k=33)
    with pytest.raises(ValidationError):
        route_experts_device(x, top_k=65)
    with pytest.raises(ValidationError):
        route_experts_device(x, top_k=2, groups=5)
    with pytest.raises(ValidationError):
        route_experts_device(x, top_k=2, bias=torch.zeros(64))
    with pytest.raises(ConfigurationError):
        plan_experts_device(torch.zeros((3, 2), dtype=torch.int32, device="cuda"), 1025)
    with pytest.raises(ValidationError):
        plan_experts_device(torch.zeros((3, 0), dtype=torch.int32, device="cuda"), 10)
    with pytest.raises(ValidationError):
        combine_experts_device(x, torch.zeros((3, 2), device="cuda"), torch.zeros((3, 2), dtype=torch.int32))
