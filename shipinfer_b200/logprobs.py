"""Token log-probabilities on the device: what a reader or captioner answered, and how surely.

A recogniser behind a crop (a hull number, a name) or a captioner answers with a row of scores
over a vocabulary for each token. :func:`token_logprobs_device` takes these rows where the engine
left them and leaves the log-probabilities of given tokens, the entropy of each row and its top
alternatives on the device (``shipk_token_logprobs``), in one pass over the scores. The reference
has no counterpart: its heads end in host code.
"""

from __future__ import annotations

from typing import Any

import torch

from shipinfer_b200 import _native
from shipinfer_b200._heads import check_dense, check_device, check_matrix, element_code, empty, guard, handle_of, ptr, small
from shipinfer_b200.errors import ValidationError

__all__ = ["pack_allowed", "token_logprobs_device"]


def pack_allowed(mask: Any) -> Any:
    """A bool mask ``[vocab]`` or ``[rows, vocab]`` as the bits :func:`token_logprobs_device`
    reads: int32 ``[words]`` or ``[rows, words]``, token ``v`` in bit ``v % 32`` of word ``v // 32``."""
    if mask.dtype != torch.bool or mask.dim() not in (1, 2) or mask.shape[-1] == 0:
        raise ValidationError(f"mask must be a bool [vocab] or [rows, vocab] tensor; got {mask.dtype} {list(mask.shape)}")
    vocab = int(mask.shape[-1])
    bits = torch.nn.functional.pad(mask, (0, -vocab % 32)).unflatten(-1, (-1, 32)).to(torch.int64)
    words = (bits << torch.arange(32, device=mask.device)).sum(dim=-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def token_logprobs_device(
    logits: Any,
    tokens: Any = None,
    *,
    top: int = 0,
    allowed: Any = None,
    temperature: float = 1.0,
    logprobs: Any = None,
    entropy: Any = None,
    top_logprobs: Any = None,
    top_ids: Any = None,
    stream: int | None = None,
) -> tuple[Any, Any, Any, Any]:
    """Log-probabilities of given tokens, entropy and top alternatives of rows of scores.

    Args:
        logits: CUDA float32, float16 or bfloat16 ``[rows, vocab]``; rows may lie apart (a head
            that pads its vocabulary: ``scores[:, :vocab]``).
        tokens: CUDA int64 ``[rows]`` or ``[rows, n]``, the tokens to score, or ``None``. A
            negative one is padding and scores 0; one past the vocabulary gives NaN.
        top: alternatives per row, up to 64.
        allowed: CUDA int32 bits ``[words]`` (one mask for every row) or ``[rows, words]`` from
            :func:`pack_allowed`, or ``None``: every token. What is not allowed, and a score of
            -inf, has probability 0; the values at cleared bits do not matter.
        temperature: divides the scores, 1e-6 to 1e6.
        logprobs, entropy, top_logprobs, top_ids: optional results to fill: float32 of the tokens'
            shape, ``[rows]``, ``[rows, top]`` and int64 ``[rows, top]``, apart from the inputs and
            from one another.
        stream: CUDA stream handle; torch's current stream when ``None``.

    Returns:
        ``(logprobs, entropy, top_logprobs, top_ids)`` on the device: natural logarithms, entropy
        in nats, alternatives best first with equal scores by the lower id; past the last
        alternative id -1 and -inf. A row with nothing allowed has -inf, entropy 0 and no
        alternatives; a NaN or +inf among the allowed scores makes its numbers NaN.
    """
    rows, vocab = check_matrix(logits, "logits")
    code = element_code(logits, "logits")
    top = small(top, "top")
    if tokens is None:
        n, shape = 0, (rows, 0)
    else:
        shape = tokens.shape
        if len(shape) not in (1, 2) or shape[0] != rows:
            raise ValidationError(f"tokens must be [{rows}] or [{rows}, n]; got {list(shape)}")
        n = 1 if len(shape) == 1 else small(shape[1], "tokens per row")
        check_dense(tokens, "tokens", torch.int64, shape)
    allowed_stride = 0
    if allowed is not None:
        words = (vocab + 31) // 32
        if (allowed.dtype != torch.int32 or allowed.dim() not in (1, 2) or int(allowed.shape[-1]) < words
                or (allowed.dim() == 2 and int(allowed.shape[0]) not in (1, rows))
                or (words > 1 and int(allowed.stride(-1)) != 1)):
            raise ValidationError(
                f"allowed must be int32 bits [{words}] or [{rows}, {words}], the words of a row adjacent "
                f"(see pack_allowed); got {allowed.dtype} {list(allowed.shape)}"
            )
        if allowed.dim() == 2 and int(allowed.shape[0]) > 1:
            allowed_stride = int(allowed.stride(0))
    if logprobs is not None:
        check_dense(logprobs, "logprobs", torch.float32, shape)
    if entropy is not None:
        check_dense(entropy, "entropy", torch.float32, (rows,))
    if top_logprobs is not None:
        check_dense(top_logprobs, "top_logprobs", torch.float32, (rows, top))
    if top_ids is not None:
        check_dense(top_ids, "top_ids", torch.int64, (rows, top))
    dev = check_device(logits, tokens, allowed, logprobs, entropy, top_logprobs, top_ids)
    if logprobs is None:
        logprobs = empty(shape, torch.float32, dev, stream)
    if entropy is None:
        entropy = empty((rows,), torch.float32, dev, stream)
    if top_logprobs is None:
        top_logprobs = empty((rows, max(top, 0)), torch.float32, dev, stream)
    if top_ids is None:
        top_ids = empty((rows, max(top, 0)), torch.int64, dev, stream)
    with guard(dev):
        _native.check(
            _native.lib().shipk_token_logprobs(
                ptr(logits), code, rows, vocab, logits.stride(0) if rows > 1 else vocab, ptr(tokens), n, ptr(allowed),
                allowed_stride, float(temperature), top, ptr(logprobs), ptr(entropy), ptr(top_logprobs), ptr(top_ids),
                handle_of(dev, stream),
            )
        )
    return logprobs, entropy, top_logprobs, top_ids
