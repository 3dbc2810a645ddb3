"""Rows so long that one mark stands for several stages of a thread's granules: alternatives, their
log-probabilities and the entropy against the definition in 64 bits, on a share of the rows.

A thread keeps 16 marks of a row (8 where a warp has a row of its own), and a stage is 4 granules of 16
bytes for each thread. More than 16 stages for each CTA of a row, or 8 for its warp, merge stages into marks:
every shape below does.

Tolerances, u = 2^-24 being half a step. A thread adds its terms to two sums in turn, V / (2 threads) to each,
one rounding each. A term 2^y has y's rounding (|y| u, at most 8 above the reference and with 2^y |y| < 0.54 below it),
the scale's 2 u |y|, and the exponential's 4 u: under 32 u. Moves of a reference, at most one for each 4 that the
logits span in base 2 (under 16 here), cost an exponential, a product and the shift's own rounding, under 8 u each.
The joins over a warp, a CTA and a cluster are under 16 additions and 6 products. With E = V / (2 threads) + 200
the sum is within E u of itself, its logarithm within (E + 2 |ln S|) u. A log-probability d - ln S adds 4 u |d|
and its own rounding. The entropy's second sum has terms of both signs, y up to 8 above 0, each within E u of
its magnitude: with M the mean of |y| its quotient is within 2 E M u, and the entropy within E (1 + 2 M) u."""

from __future__ import annotations

import numpy as np
import pytest

import _heads
from shipinfer_b200.logprobs import pack_allowed, token_logprobs_device

pytestmark = pytest.mark.gpu


def check(torch, x, picked, threads, *, top, tokens, allowed=None):
    """All rows in one call; the rows `picked` against the definition."""
    words = None if allowed is None else pack_allowed(allowed)
    got = token_logprobs_device(x, tokens, top=top, allowed=words)
    torch.cuda.synchronize()
    at = torch.tensor(picked, device="cuda")
    lp, entropy, top_lp, ids = (v[at].cpu().numpy() for v in got)
    sub = x[at].double().cpu().numpy()
    on = None if allowed is None else (allowed[at] if allowed.dim() == 2 else allowed).cpu().numpy()
    want = _heads.logprobs64(sub, tokens[at].cpu().numpy(), top=top, allowed=on)
    assert np.array_equal(ids, want[3])
    vocab = x.shape[1]
    e = vocab / (2 * threads) + 200
    u = _heads.EPS32
    for g, w in ((lp, want[0].reshape(lp.shape)), (top_lp, want[2])):
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine], w[~fine], equal_nan=True)
        # |ln S| is under ln V + 8 and |d| under |logprob| + ln V + 8
        assert (np.abs(g[fine] - w[fine]) <= u * (e + 6 * (np.abs(w[fine]) + np.log(vocab) + 8))).all()
    keep = np.broadcast_to(True if on is None else on, sub.shape)
    y = np.where(keep, sub, -np.inf)
    d = np.maximum(y - y.max(axis=1, keepdims=True), -700.0) * 1.4427
    p = np.where(keep, np.exp2(d), 0.0)
    mean = (p * np.abs(d)).sum(axis=1) / p.sum(axis=1) + 8
    assert (np.abs(entropy - want[1]) <= u * (e * (1 + 2 * mean) + 6 * np.log(vocab))).all()


def rows_by_stage(torch, rows, vocab, dtype, stage, seed):
    """Rows whose 30 best scores are in one stage of the group that reads them, another one from row to
    row; some rows rising, falling, or best at their ends. `stage`: the values of a stage."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((rows, vocab), device="cuda").normal_(-6.0, 1.5, generator=g)
    stages = -(-vocab // stage)
    for r in range(rows):
        lo = r % stages * stage
        hi = min(vocab, lo + stage)
        at = lo + torch.randint(0, hi - lo, (30,), device="cuda", generator=g)
        x[r, at] = 1.0 + torch.rand(30, device="cuda", generator=g) * 8.0
    x[3] = torch.linspace(-20, 0, vocab, device="cuda")
    x[4] = torch.linspace(0, -20, vocab, device="cuda")
    x[5, :20], x[5, -20:] = 9.0, 9.0
    return x.to(getattr(torch, dtype))


def picks(rows, stages):
    """A row for each stage, early and late ones, and those of other kinds."""
    late = [rows - 1 - r for r in range(0, min(stages, rows // 2), 3)]
    return sorted({0, 1, 2, 3, 4, 5, *range(6, min(rows, 6 + stages)), *late, rows // 2})


# (rows, vocab, type, threads that read a row, values of a stage): a CTA a row, once and again; a warp; clusters
SHAPES = [
    (310, 151667, "float32", 256, 4096),
    (700, 70001, "float32", 256, 4096),
    (700, 151667, "bfloat16", 256, 8192),
    (1300, 5003, "float32", 32, 512),
    (2600, 20011, "bfloat16", 32, 1024),
    (2600, 20011, "float16", 32, 1024),
    (3, 1200001, "bfloat16", 2048, 8192),
    (2, 700001, "float32", 2048, 4096),
]


@pytest.mark.parametrize(("rows", "vocab", "dtype", "threads", "stage"), SHAPES)
@pytest.mark.parametrize("top", [3, 20])
def test_best_scores_in_any_stage(cuda, rows, vocab, dtype, threads, stage, top):
    torch = cuda
    if rows < 6:
        rows_ = [rows_by_stage(torch, 8, vocab, dtype, stage, 7)[i * 3 : i * 3 + rows] for i in range(2)]
    else:
        rows_ = [rows_by_stage(torch, rows, vocab, dtype, stage, 7)]
    for x in rows_:
        tokens = torch.randint(0, vocab, (rows, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        picked = list(range(rows)) if rows < 6 else picks(rows, -(-vocab // stage))
        check(torch, x, picked, threads, top=top, tokens=tokens)


@pytest.mark.parametrize(("rows", "vocab", "dtype", "threads", "stage"), SHAPES)
def test_best_scores_in_any_stage_under_masks(cuda, rows, vocab, dtype, threads, stage):
    torch = cuda
    x = rows_by_stage(torch, max(rows, 6), vocab, dtype, stage, 8)[:rows]
    g = torch.Generator(device="cuda").manual_seed(3)
    allowed = torch.rand((rows, vocab), device="cuda", generator=g) < 0.7
    tokens = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)
    picked = list(range(rows)) if rows < 6 else picks(rows, -(-vocab // stage))
    check(torch, x, picked, threads, top=12, tokens=tokens, allowed=allowed)


@pytest.mark.parametrize(("rows", "vocab"), [(310, 151667), (700, 70001)])
def test_many_alternatives_of_merged_marks(cuda, rows, vocab):
    torch = cuda
    x = rows_by_stage(torch, rows, vocab, "float32", 4096, 9)
    tokens = torch.zeros((rows, 1), dtype=torch.int64, device="cuda")
    check(torch, x, picks(rows, -(-vocab // 4096)), 256, top=64, tokens=tokens)
