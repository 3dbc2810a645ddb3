"""Token log-probabilities on the GPU (shipk_token_logprobs) against their definition in 64 bits.

Tolerances. With d = (x - max) / T <= 0 the kernel has S = sum of e^d and logprob = d - ln S in 32
bits. Half a step is u = 2^-24. d carries three roundings (difference, 1 / T, product): 3 u |d|.
Each e^d is off by its argument's error, times e^d, and by the exponential's own few steps; |d|
e^d < 0.4, so S has the terms' error, under 8 u, and the additions': a thread adds at most
max(64, V / 256) terms one after another and a tree of under 16 joins follows, each with one more
exponential (3 u) and addition. ln S is off by S's relative error and its own two steps. In all
(max(64, V / 256) + 64 + 8 |logprob| + 8 ln V) u bounds it, the last for ln S itself. The entropy
is ln S - (sum of e^d d) / S: the second sum's terms have one sign, so its relative error is S's
and it is at most ln S + ln V in magnitude: the same bound times (1 + 2 ln V). Alternatives' ids are exact.
"""

from __future__ import annotations

import numpy as np
import pytest

import _heads
from shipinfer_b200 import ConfigurationError, ValidationError
from shipinfer_b200.logprobs import pack_allowed, token_logprobs_device

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")


def bound(vocab, values):
    return _heads.EPS32 * (max(64, vocab / 256) + 64 + 8 * np.abs(values) + 8 * np.log(vocab + 1))


def close(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    assert np.isfinite(got[fine]).all()
    err = np.abs(got[fine] - want[fine])
    limit = np.broadcast_to(tol, want.shape)[fine]
    assert (err <= limit).all(), (float(err.max()), float((err / limit).max()))


def check(torch, x, tokens=None, *, allowed=None, top=0, temperature=1.0, **more):
    """x: a CUDA tensor [rows, vocab]; allowed: a bool array or None."""
    words = None if allowed is None else pack_allowed(torch.from_numpy(allowed)).cuda()
    t = None if tokens is None else torch.from_numpy(tokens).cuda()
    got = token_logprobs_device(x, t, top=top, allowed=words, temperature=temperature, **more)
    torch.cuda.synchronize()
    lp, ent, top_lp, ids = (v.cpu().numpy() for v in got)
    want = _heads.logprobs64(x.double().cpu().numpy(), tokens, top=top, allowed=allowed,
                             temperature=float(np.float32(temperature)))
    vocab = x.shape[1]
    assert np.array_equal(ids, want[3])
    with np.errstate(over="ignore"):  # below float32's range is -inf
        w0, w2 = (w.astype(np.float32).astype(np.float64) for w in (want[0].reshape(lp.shape), want[2]))
    close(lp, w0, bound(vocab, np.nan_to_num(w0, posinf=0, neginf=0)))
    close(ent, want[1], bound(vocab, 0.0) * (1 + 2 * np.log(vocab + 1)))
    close(top_lp, w2, bound(vocab, np.nan_to_num(w2, posinf=0, neginf=0)))
    return got


def scores(torch, rows, vocab, dtype, seed, pad=0):
    rng = np.random.default_rng(seed)
    x = rng.normal(-1.0, 2.5, (rows, vocab + pad))
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 9.0
    return torch.from_numpy(x).to(getattr(torch, dtype)).cuda()[:, :vocab]


SIZES = [(1, 1), (3, 2), (2, 31), (5, 32), (7, 33), (300, 97), (4, 255), (3, 1000), (2, 1024), (2, 1025), (9, 2049),
         (3, 4099), (1, 8193), (2, 32000), (150, 5003), (1, 50257), (3, 50257), (20, 20011), (1, 151667), (2, 151667)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "vocab"), SIZES)
def test_sizes_and_types(cuda, rows, vocab, dtype):
    rng = np.random.default_rng(rows * 7919 + vocab)
    x = scores(cuda, rows, vocab, dtype, vocab + rows)
    tokens = rng.integers(-1, vocab, (rows, 3))
    check(cuda, x, tokens, top=min(vocab, 20))
    check(cuda, x, tokens[:, 0].copy(), top=min(vocab, 1), temperature=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [33, 97, 1500, 40001])
@pytest.mark.parametrize("shared", [True, False])
def test_masks(cuda, dtype, vocab, shared):
    """Masks over garbage: what is at a cleared bit may be anything. One row with nothing allowed,
    one with a single token, one with fewer than the alternatives asked for."""
    rows = 6
    rng = np.random.default_rng(vocab)
    x = scores(cuda, rows, vocab, dtype, 5)
    allowed = rng.random((1 if shared else rows, vocab)) < 0.6
    if not shared:
        allowed[1], allowed[2], allowed[3] = False, False, False
        allowed[2, vocab - 1] = True
        allowed[3, rng.integers(0, vocab, 5)] = True
    off = ~np.broadcast_to(allowed, (rows, vocab))
    h = x.float().cpu().numpy()
    junk = rng.choice(np.array([np.nan, np.inf, -np.inf, 6e4, -6e4], np.float32), (rows, vocab))
    x = cuda.from_numpy(np.where(off, junk, h)).to(x.dtype).cuda()
    tokens = rng.integers(0, vocab, (rows, 4))
    check(cuda, x, tokens, allowed=allowed[0] if shared else allowed, top=min(vocab, 8), temperature=1.6)


def extreme_rows(torch, vocab, dtype):
    t = getattr(torch, dtype)
    low = torch.finfo(t).min
    x = torch.zeros((12, vocab), dtype=torch.float32)
    x[0] = -np.inf
    x[1] = low
    x[2] = 3.5
    x[3] = low
    x[3, vocab // 2] = torch.finfo(t).max
    x[4, 5] = float("nan")
    x[5, 6] = float("inf")
    x[6] = torch.linspace(-30, 30, vocab)
    x[7] = torch.linspace(30, -30, vocab)
    x[8, ::2] = -0.0
    x[9, :] = -20.0
    x[9, : vocab // 2 : 16] = torch.arange(len(x[9, : vocab // 2 : 16])).float() % 7
    x[10] = -np.inf
    x[10, vocab - 1] = -3.0
    x[11] = torch.arange(vocab) % 2 * 5.0
    return x.to(t).cuda()


@pytest.mark.parametrize("vocab", [40, 3001, 60000])
@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_rows(cuda, vocab, dtype):
    """Rows of -inf, of the type's lowest value, of one value, of two far ones; NaN and +inf; a
    rising and a falling row; signed zeros; all large values in a few places that one thread reads."""
    x = extreme_rows(cuda, vocab, dtype)
    tokens = np.tile(np.array([0, vocab - 1, -1, vocab // 2, -7], np.int64), (12, 1))
    check(cuda, x, tokens, top=min(vocab, 33))
    check(cuda, x, tokens, top=min(vocab, 64), temperature=0.01)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_middling_length(cuda, dtype):
    """More rows than a row has 16-byte granules, on and off their boundaries: the extreme rows and
    ordinary ones, plain and under masks with cleared and single-token rows."""
    torch = cuda
    for vocab, rows in ((1100, 420), (3001, 800)):
        x = scores(torch, rows, vocab, dtype, vocab, pad=3)
        x[5::7][:12] = extreme_rows(torch, vocab, dtype)[: len(x[5::7][:12])]
        rng = np.random.default_rng(vocab)
        tokens = rng.integers(-1, vocab, (rows, 2))
        check(torch, x, tokens, top=20)
        check(torch, x.contiguous()[:, 1:], np.minimum(tokens, vocab - 2), top=3, temperature=1.6)
        allowed = rng.random((rows, vocab)) < 0.5
        allowed[7], allowed[8] = False, False
        allowed[8, vocab - 2] = True
        allowed[9, 40:] = False
        check(torch, x, tokens, top=8, allowed=allowed)
        check(torch, x, tokens, top=1, allowed=allowed[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "vocab"), [(24, 200), (24, 5003), (900, 5003), (24, 60000)])
def test_entropy_of_sure_rows(cuda, rows, vocab, dtype):
    """One logit far above the rest, early or late in the row: the entropy is small and has to be
    small. A thread's reference is at most 8 (in base 2) below its largest logit, whose y 2^y then has three
    roundings of 8 and as many when the reference moves up, 48 u ln 2 together; log S and the
    quotient add a few u, the other terms (at most 1e-3 of the sum) nothing to speak of: 48 u."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0.0, 0.3, (rows, vocab)).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] = rng.uniform(20, 60, rows)
    x = cuda.from_numpy(x).to(getattr(cuda, dtype)).cuda()
    got = token_logprobs_device(x)[1].double().cpu().numpy()
    want = _heads.logprobs64(x.double().cpu().numpy())[1]
    assert (np.abs(got - want) <= 48 * _heads.EPS32 + bound(vocab, 0.0) * want).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_that_follow_one_another(cuda, dtype):
    """Several long rows for each CTA: a row's copies begin while the one before is ranked."""
    rows, vocab = 1300, 12001
    x = scores(cuda, rows, vocab, dtype, 77, pad=2)
    rng = np.random.default_rng(5)
    tokens = rng.integers(-1, vocab, (rows, 1))
    check(cuda, x, tokens, top=24)
    allowed = rng.random((rows, vocab)) < 0.7
    allowed[600:610] = False
    check(cuda, x, tokens, top=7, allowed=allowed)


@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e3, 1e6])
@pytest.mark.parametrize(("rows", "vocab"), [(5, 97), (2, 5003), (700, 1500)])
def test_far_temperatures(cuda, rows, vocab, temperature):
    for dtype in TYPES:
        x = scores(cuda, rows, vocab, dtype, 6)
        tokens = np.random.default_rng(1).integers(0, vocab, (rows, 2))
        check(cuda, x, tokens, top=5, temperature=temperature)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_large_score_with_one_reader(cuda, dtype):
    """Far more large scores than alternatives, all at places a fixed distance apart: no share of
    the row that a single thread or vector reads may hold them all and lose some."""
    for step in (2, 4, 8, 128, 256, 512, 1024, 2048, 4096, 8192):
        vocab = 90001
        x = np.random.default_rng(step).normal(-8, 1, (2, vocab)).astype(np.float32)
        x[0, 3::step] = np.linspace(1, 9, len(x[0, 3::step]))
        x[1, step - 1 :: step] = 4.0
        check(cuda, cuda.from_numpy(x).to(getattr(cuda, dtype)).cuda(), np.full((2, 1), 3, np.int64), top=20)


def test_tokens_past_the_vocabulary_are_nan(cuda):
    x = scores(cuda, 3, 50, "float32", 1)
    check(cuda, x, np.array([[49, 50], [1 << 40, 0], [-(1 << 40), 60]], np.int64), top=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [97, 1024, 5000, 33333])
def test_strides_and_offsets(cuda, dtype, vocab):
    """Rows apart, rows that start at any element, one row repeated, rows in reverse order."""
    wide = scores(cuda, 6, vocab + 71, dtype, 3)
    tokens = np.random.default_rng(0).integers(0, vocab, (6, 2))
    for lo in (0, 1, 3, 8):
        check(cuda, wide[:, lo : lo + vocab], tokens, top=5)
    check(cuda, wide[::2, :vocab], tokens[:3].copy(), top=5)
    check(cuda, wide[1:2, 2 : 2 + vocab].expand(4, vocab), tokens[:4].copy(), top=5)
    mask = np.random.default_rng(1).random((6, vocab)) < 0.5
    words = pack_allowed(cuda.from_numpy(mask)).cuda()
    spread = cuda.zeros((6, words.shape[1] + 5), dtype=cuda.int32, device="cuda")
    spread[:, 2 : 2 + words.shape[1]] = words
    # against the definition, as everywhere here: a copy that starts at another address is summed
    # in another order, so two calls agree to the sum of their bounds and not to the bit
    x = wide[:, 1 : 1 + vocab]
    _, ent, top_lp, ids = token_logprobs_device(x, top=5, allowed=spread[:, 2 : 2 + words.shape[1]])
    want = _heads.logprobs64(x.double().cpu().numpy(), top=5, allowed=mask)
    assert np.array_equal(ids.cpu().numpy(), want[3])
    close(ent.cpu(), want[1], bound(vocab, 0.0) * (1 + 2 * np.log(vocab + 1)))
    close(top_lp.cpu(), want[2], bound(vocab, want[2]))


def test_offsets_past_32_bits(cuda):
    free = cuda.cuda.mem_get_info()[0]
    assert free > 12 << 30
    stride = (1 << 31) + 96
    flat = cuda.empty(2 * stride, dtype=cuda.bfloat16, device="cuda")
    x = flat.as_strided((2, 40000), (stride, 1))
    x.copy_(scores(cuda, 2, 40000, "bfloat16", 9))
    check(cuda, x, np.array([[1], [39999]], np.int64), top=7)
    small = flat.as_strided((2, 200), (stride, 1))
    check(cuda, small, np.array([[1], [199]], np.int64), top=7)


def test_no_rows_no_tokens_no_alternatives(cuda):
    x = scores(cuda, 4, 300, "float16", 2)
    lp, ent, top_lp, ids = check(cuda, x)
    assert lp.shape == (4, 0) and top_lp.shape == ids.shape == (4, 0)
    lp, ent, top_lp, ids = token_logprobs_device(x[:0], cuda.zeros((0, 2), dtype=cuda.int64, device="cuda"), top=3)
    assert lp.shape == (0, 2) and ent.shape == (0,) and ids.shape == (0, 3)


def test_given_results_are_filled_and_nothing_beside_them(cuda):
    torch = cuda
    x, tokens = scores(cuda, 5, 3500, "bfloat16", 8), torch.arange(5, device="cuda")
    want = token_logprobs_device(x, tokens, top=4)
    held = [torch.full((7, 5), 77.0, device="cuda"), torch.full((7, 5), 77.0, device="cuda"),
            torch.full((7, 4), 77.0, device="cuda"), torch.full((7, 4), 77, dtype=torch.int64, device="cuda")]
    outs = {"logprobs": held[0][1], "entropy": held[1][1], "top_logprobs": held[2][1:6], "top_ids": held[3][1:6]}
    got = token_logprobs_device(x, tokens, top=4, **outs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[3].data_ptr() == outs["top_ids"].data_ptr()
    for h in held:
        assert (h[0] == 77).all() and (h[6] == 77).all()
    assert (held[0][2:] == 77).all()


def test_other_stream_and_repeatability(cuda):
    torch = cuda
    x, tokens = scores(cuda, 64, 50257, "bfloat16", 4), torch.arange(64, device="cuda")
    want = token_logprobs_device(x, tokens, top=8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = token_logprobs_device(x, tokens, top=8, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for _ in range(3):
        again = token_logprobs_device(x, tokens, top=8)
        assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_one_mask_row_and_overlapping_calls(cuda):
    """A mask of one row in two dimensions serves every row; calls that overlap on two streams share
    nothing."""
    torch = cuda
    x = scores(cuda, 700, 9000, "float16", 3)
    mask = torch.rand(9000, device="cuda") < 0.5
    one = token_logprobs_device(x, top=4, allowed=pack_allowed(mask))
    two = token_logprobs_device(x, top=4, allowed=pack_allowed(mask)[None])
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(token_logprobs_device(x, top=4, allowed=pack_allowed(mask)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, one))


def test_two_graphs_and_an_eager_call_share_nothing(cuda):
    torch = cuda
    shapes = [(3, 50257), (300, 97)]
    xs = [scores(cuda, r, v, "float16", r) for r, v in shapes]
    ts = [torch.zeros(r, dtype=torch.int64, device="cuda") for r, _ in shapes]
    for x, t in zip(xs, ts):
        token_logprobs_device(x, t, top=5)  # first launches outside capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, t in zip(xs, ts):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(token_logprobs_device(x, t, top=5))
        graphs.append(g)
    for k in range(2):
        for x, (r, v) in zip(xs, shapes):
            x.copy_(scores(cuda, r, v, "float16", 50 + k))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, t, out in zip(xs, ts, outs):
            want = token_logprobs_device(x, t, top=5)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
    torch = cuda
    x, t = torch.zeros((3, 100), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ConfigurationError):
        token_logprobs_device(x, t, top=65)
    with pytest.raises(ValidationError):
        token_logprobs_device(x[:, :10], t, top=11)
    with pytest.raises(ValidationError):
        token_logprobs_device(x, t, temperature=0.0)
    with pytest.raises(ValidationError):
        token_logprobs_device(x[:, :0], t)
    with pytest.raises(ValidationError):
        token_logprobs_device(x, t.cpu())
    with pytest.raises(ValidationError):
        token_logprobs_device(x.cpu(), t)
    with pytest.raises(ValidationError):
        token_logprobs_device(x, t, entropy=torch.zeros(3))
