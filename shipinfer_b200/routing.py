"""Routing rows to experts on the device: a gate's scores -> who works on which row, and back.

The reference's ``CropStage`` (``csrc/shipinfer/pipeline/graph/stages.cpp:195-245``) sends each
detection's crop to the embedder of its class. Where a gate scores several embedders per
detection instead:

* :func:`route_experts_device` chooses each row's experts and their weights
  (``shipk_route_experts``);
* :func:`plan_experts_device` groups the rows by expert (``shipk_plan_experts``): with its order,
  ``boxes[order]`` into ``NativeImageOps.crop_device`` makes every expert's batch in one launch;
* :func:`combine_experts_device` joins the experts' results per row (``shipk_combine_experts``).

All of it stays on the device; nothing synchronises, so a step captures in a CUDA graph.
"""

from __future__ import annotations

from typing import Any

import torch

from shipinfer_b200 import _native
from shipinfer_b200._heads import check_dense, check_device, check_matrix, element_code, empty, guard, handle_of, ptr, small
from shipinfer_b200.errors import ValidationError

__all__ = ["combine_experts_device", "plan_experts_device", "route_experts_device"]

_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


def route_experts_device(
    logits: Any,
    *,
    top_k: int,
    scores: str = "softmax",
    bias: Any = None,
    groups: int = 1,
    top_groups: int = 1,
    group_score: str = "max",
    renormalise: bool = True,
    scale: float = 1.0,
    weights: Any = None,
    ids: Any = None,
    stream: int | None = None,
) -> tuple[Any, Any]:
    """The experts of each row and their weights.

    Args:
        logits: CUDA float32, float16 or bfloat16 ``[rows, experts]`` (up to 1024 experts); rows
            may lie apart. -inf or NaN: this expert cannot be chosen.
        top_k: experts per row, up to 32.
        scores: "softmax" or "sigmoid" of the logits.
        bias: CUDA float32 ``[experts]`` added to the scores for the choice only (a balance), or
            ``None``; -inf there closes an expert to every row.
        groups, top_groups, group_score: with more than one group, the experts form ``groups``
            runs (up to 32) and only the ``top_groups`` best can be chosen from, by their best
            expert ("max") or the sum of their two best ("top2").
        renormalise: divide the chosen scores by their sum.
        scale: multiplies the weights; finite in float32.
        weights, ids: optional results to fill: float32 and int32 ``[rows, top_k]``, apart from the
            inputs and from each other.
        stream: CUDA stream handle; torch's current stream when ``None``.

    Returns:
        ``(weights, ids)`` on the device, best first, ties to the lower expert; past the last
        expert that can be chosen, id -1 and weight 0. The scores are computed in 64 bits and
        rounded once, so the choice does not depend on how a sum was ordered.
    """
    rows, experts = check_matrix(logits, "logits")
    code = element_code(logits, "logits")
    top_k, groups, top_groups = small(top_k, "top_k"), small(groups, "groups"), small(top_groups, "top_groups")
    if scores not in _SCORES:
        raise ValidationError(f"scores must be 'softmax' or 'sigmoid', got {scores!r}")
    if group_score not in _GROUP_SCORES:
        raise ValidationError(f"group_score must be 'max' or 'top2', got {group_score!r}")
    if bias is not None:
        check_dense(bias, "bias", torch.float32, (experts,))
    if weights is not None:
        check_dense(weights, "weights", torch.float32, (rows, top_k))
    if ids is not None:
        check_dense(ids, "ids", torch.int32, (rows, top_k))
    dev = check_device(logits, bias, weights, ids)
    if weights is None:
        weights = empty((rows, max(top_k, 0)), torch.float32, dev, stream)
    if ids is None:
        ids = empty((rows, max(top_k, 0)), torch.int32, dev, stream)
    with guard(dev):
        _native.check(
            _native.lib().shipk_route_experts(
                ptr(logits), code, rows, experts, logits.stride(0) if rows > 1 else experts, ptr(bias), top_k,
                _SCORES[scores], groups, top_groups, _GROUP_SCORES[group_score], int(bool(renormalise)),
                float(scale), ptr(weights), ptr(ids), handle_of(dev, stream),
            )
        )
    return weights, ids


def plan_experts_device(
    ids: Any,
    experts: int,
    *,
    order: Any = None,
    slots: Any = None,
    offsets: Any = None,
    stream: int | None = None,
) -> tuple[Any, Any, Any]:
    """Group the rows by expert.

    Args:
        ids: CUDA int32 ``[rows, k]`` from :func:`route_experts_device`; an id outside
            ``[0, experts)`` is nobody's.
        experts: how many there are, up to 1024.
        order, slots, offsets: optional results to fill: int32 ``[rows * k]``, ``[rows, k]`` and
            ``[experts + 1]``, apart from the ids (which are read twice) and from one another.
        stream: CUDA stream handle; torch's current stream when ``None``.

    Returns:
        ``(order, slots, offsets)`` on the device. Expert ``e`` works on the rows
        ``order[offsets[e]:offsets[e + 1]]``, ascending; places past ``offsets[experts]`` hold -1.
        ``slots[r, j]`` is the place of row r's j-th expert, -1 where there is none.
    """
    if ids.dim() != 2:
        raise ValidationError(f"ids must be int32 [rows, k]; got {list(ids.shape)}")
    rows, k = small(ids.shape[0], "rows"), small(ids.shape[1], "k")
    experts = small(experts, "experts")
    check_dense(ids, "ids", torch.int32, (rows, k))
    if order is not None:
        check_dense(order, "order", torch.int32, (rows * k,))
    if slots is not None:
        check_dense(slots, "slots", torch.int32, (rows, k))
    if offsets is not None:
        check_dense(offsets, "offsets", torch.int32, (experts + 1,))
    dev = check_device(ids, order, slots, offsets)
    if order is None:
        order = empty((rows * k,), torch.int32, dev, stream)
    if slots is None:
        slots = empty((rows, k), torch.int32, dev, stream)
    if offsets is None:
        offsets = empty((max(experts, 0) + 1,), torch.int32, dev, stream)
    with guard(dev):
        _native.check(
            _native.lib().shipk_plan_experts(ptr(ids), rows, k, experts, ptr(order), ptr(slots), ptr(offsets),
                                             handle_of(dev, stream))
        )
    return order, slots, offsets


def combine_experts_device(
    rows: Any,
    weights: Any,
    slots: Any,
    *,
    out: Any = None,
    stream: int | None = None,
) -> Any:
    """Join the experts' results: ``out[r] = sum over j of weights[r, j] * rows[slots[r, j]]``.

    Args:
        rows: CUDA float32, float16 or bfloat16 ``[n, width]``, the experts' results at the
            places of the plan; rows may lie apart.
        weights: CUDA float32 ``[r, k]``; slots: CUDA int32 ``[r, k]``. A slot outside ``[0, n)``
            adds nothing, whatever its weight.
        out: optional result to fill, ``[r, width]`` of the rows' type, apart from the inputs.
        stream: CUDA stream handle; torch's current stream when ``None``.

    Returns:
        ``[r, width]`` on the device, summed in 32 bits in the order of j and rounded once.
    """
    n, width = check_matrix(rows, "rows")
    code = element_code(rows, "rows")
    if slots.dim() != 2:
        raise ValidationError(f"slots must be int32 [rows, k]; got {list(slots.shape)}")
    r, k = small(slots.shape[0], "rows"), small(slots.shape[1], "k")
    check_dense(slots, "slots", torch.int32, (r, k))
    check_dense(weights, "weights", torch.float32, (r, k))
    if out is not None:
        check_dense(out, "out", rows.dtype, (r, width))
    dev = check_device(slots, weights, rows, out)
    if out is None:
        out = empty((r, width), rows.dtype, dev, stream)
    with guard(dev):
        _native.check(
            _native.lib().shipk_combine_experts(
                ptr(rows), code, n, rows.stride(0) if n > 1 else width, ptr(weights), ptr(slots), r, k, width, ptr(out),
                handle_of(dev, stream),
            )
        )
    return out
