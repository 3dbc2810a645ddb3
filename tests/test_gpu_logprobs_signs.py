"""A log-probability is at most 0 and an entropy at least 0, whatever a row's sums round to.

A row that is all but certain has both within a few roundings of 0, and a caller may take a root
or a logarithm of the entropy: the signs are part of the definition, so there is no tolerance here.
"""

from __future__ import annotations

import numpy as np
import pytest

from shipinfer_b200.logprobs import token_logprobs_device

pytestmark = pytest.mark.gpu

# a warp's registers, a warp, a CTA and a cluster per row
SHAPES = [(200, 700), (900, 5003), (300, 5003), (24, 60000)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize(("rows", "vocab"), SHAPES)
def test_signs_of_sure_rows(cuda, rows, vocab, temperature, dtype):
    """One logit far above the rest, or a few above them and the others far below: certain rows, and
    rows whose largest logit is anywhere above the one that the sums are relative to."""
    torch = cuda
    rng = np.random.default_rng(rows + vocab)
    x = rng.normal(-60.0, 1.0, (rows, vocab)).astype(np.float32)
    at = rng.integers(0, vocab, rows)
    x[np.arange(rows), at] = rng.uniform(-20, 40, rows)
    # an earlier logit just below the largest, which later ones need not move the reference from
    near = rng.integers(0, vocab, rows)
    half = np.arange(rows) % 2 == 0
    x[half, near[half]] = np.maximum(x[half, near[half]], x[half, at[half]] - rng.uniform(16, 30, half.sum()).astype(np.float32))
    scores = torch.from_numpy(x).to(getattr(torch, dtype)).cuda()
    tokens = torch.from_numpy(at).cuda()
    lp, entropy, top_lp, _ = token_logprobs_device(scores, tokens, top=5, temperature=temperature)
    assert (entropy >= 0).all(), (int((entropy < 0).sum()), float(entropy.min()))
    assert (lp <= 0).all(), (int((lp > 0).sum()), float(lp.max()))
    assert (top_lp <= 0).all(), float(top_lp.max())


@pytest.mark.parametrize(("rows", "vocab"), SHAPES)
def test_signs_of_single_tokens_and_nothing(cuda, rows, vocab):
    """A row with one token left has log-probability and entropy 0; NaN stays NaN."""
    torch = cuda
    x = torch.full((rows, vocab), -float("inf"), device="cuda")
    at = torch.arange(rows, device="cuda") * 37 % vocab
    x[torch.arange(rows), at] = torch.linspace(-30, 30, rows, device="cuda")
    x[3, 5] = float("nan")
    x[4] = -float("inf")
    lp, entropy, _, _ = token_logprobs_device(x, at, top=2)
    assert torch.isnan(lp[3]) and torch.isnan(entropy[3])
    assert lp[4] == -float("inf") and entropy[4] == 0
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[3:5] = False
    assert (entropy[rest] >= 0).all() and (lp[rest] <= 0).all()
    # one rounding of log S and one of the product with the slip, each of 1
    assert (entropy[rest] <= 2.0**-22).all() and (lp[rest] >= -(2.0**-22)).all()
