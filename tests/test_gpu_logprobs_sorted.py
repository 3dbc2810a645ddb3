"""Rows whose large scores lie together: a vocabulary sorted by frequency, rising and falling rows, plateaus. A
few threads read all of them, so that the bound from the threads' maxima lets more pass than a group holds.
Alternatives are exact; their log-probabilities are held to the definition in 64 bits.

Tolerance, u = 2^-24: a thread adds its V / (2 threads) terms of a sum one after another, each term is within
32 u (its argument's rounding, the scale's and the exponential's), the references' moves and the joins are under
168 u: ln S is within E = V / (2 threads) + 200 of u. A log-probability d - ln S adds 4 u |d|, 2 u |ln S| and its own u, with
|d| and |ln S| under |logprob| + ln V + 8."""

from __future__ import annotations

import numpy as np
import pytest

import _heads
from shipinfer_b200.logprobs import pack_allowed, token_logprobs_device

pytestmark = pytest.mark.gpu


def rows_of(rng, rows, vocab):
    """float32 [rows, vocab], a kind for each row in turn."""
    ids = np.arange(1, vocab + 1, dtype=np.float32)
    x = np.empty((rows, vocab), np.float32)
    for r in range(rows):
        kind = r % 9
        noise = rng.normal(0, 0.3, vocab).astype(np.float32)
        if kind < 2:
            x[r] = -np.log(ids) + noise
        elif kind == 2:
            x[r] = -np.log(ids[::-1]) + noise
        elif kind == 3:
            x[r] = -20 * ids / vocab
        elif kind == 4:
            x[r] = 20 * ids / vocab
        elif kind == 5:  # a block of good scores in the row's midst, all above the rest
            x[r] = -10 + noise
            lo = int(rng.integers(0, vocab - 700))
            x[r, lo : lo + 700] = 5 + rng.random(700)
        elif kind == 6:  # a plateau below a rising block
            x[r] = -4
            lo = int(rng.integers(0, vocab - 600))
            x[r, lo : lo + 600] = np.arange(600) // 7
        elif kind == 7:  # alternating rise: later ones a little better than earlier ones
            x[r] = np.where(ids % 3 == 0, ids * np.float32(8 / vocab), np.float32(-5))
        else:  # one value, and a few better
            x[r] = 1.5
            x[r, rng.integers(0, vocab, 6)] = 3
    return x


# a warp, a CTA that ends, a CTA that walks on, a cluster (and its threads)
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize(("rows", "vocab", "threads"), [
    (2600, 2003, 32), (1300, 5003, 32), (180, 20011, 256), (700, 20011, 256), (700, 9001, 256), (27, 70001, 512)])
def test_large_scores_that_lie_together(cuda, rows, vocab, threads, dtype):
    torch = cuda
    rng = np.random.default_rng(rows + vocab)
    few = rows_of(rng, 45, vocab)
    x = torch.from_numpy(few).to(getattr(torch, dtype)).cuda()
    # copies of the 45 kinds in a matrix whose rows start off the 16-byte boundaries
    wide = torch.zeros((rows, vocab + 4), dtype=x.dtype, device="cuda")
    wide[:, 1 : 1 + vocab] = x[torch.arange(rows, device="cuda") % len(few)]
    allowed = torch.rand((len(few), vocab), generator=torch.Generator().manual_seed(vocab)) < 0.8
    for mask in (None, allowed):
        words = None if mask is None else pack_allowed(mask).cuda()[torch.arange(rows, device="cuda") % len(few)].contiguous()
        for top in (1, 5, 20, 64):
            _, _, top_lp, ids = token_logprobs_device(wide[:, 1 : 1 + vocab], top=top, allowed=words)
            on = None if mask is None else mask.numpy()
            want = _heads.logprobs64(x.double().cpu().numpy(), top=top, allowed=on)
            picked = torch.arange(rows, device="cuda") % len(few)
            assert torch.equal(ids, torch.from_numpy(want[3]).cuda()[picked])
            w = torch.from_numpy(want[2]).cuda()[picked]
            e = vocab / (2 * threads) + 200
            limit = _heads.EPS32 * (e + 7 * (w.abs() + np.log(vocab) + 8))
            assert ((top_lp.double() - w).abs() <= limit).all()


def test_more_large_scores_with_one_thread_than_bounds_can_tame(cuda):
    """15,600 rising scores at the places that the first thread of the first of eight CTAs reads: each bound
    from what is held passes some 500 of them, so the alternatives are found one by one."""
    torch = cuda
    vocab, top = 32_000_001, 20
    x = torch.empty((1, vocab), device="cuda").normal_(-9.0, 1.0, generator=torch.Generator(device="cuda").manual_seed(1))
    granule = torch.arange(0, vocab // 8 // 4, 256, device="cuda")
    at = (granule[:, None] * 4 + torch.arange(4, device="cuda")).flatten()
    x[0, at] = torch.linspace(1, 9, len(at), device="cuda")
    assert len(at) > 15_000
    _, entropy, top_lp, ids = token_logprobs_device(x, top=top)
    assert torch.equal(ids[0], at.flip(0)[:top])
    lp = torch.log_softmax(x.double(), dim=1)
    want = lp[0, ids[0]]
    e = vocab / (2 * 2048) + 200
    assert ((top_lp[0].double() - want).abs() <= _heads.EPS32 * (e + 7 * (want.abs() + np.log(vocab) + 8))).all()
    # y is within 8 + (ln V + 18) / ln 2 of the reference where it has weight; E (1 + 2 M) u as for merged marks
    assert abs(float(entropy[0]) + float((lp.exp() * lp).sum())) <= _heads.EPS32 * e * (1 + 2 * 60)
