"""The head operators' measured cases: what the framework computes from a model's scores.

Each operator is here twice: in its plain form, elementary torch operations in 32 bits (64 for
the routing scores, whose order decides), and as the calls a user makes of ``shipinfer_b200``.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------

def _logprobs(rows, vocab, dtype, top, **more):
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "stride": more.get("stride", vocab), "dtype": dtype,
            "top": top, "tokens": more.get("tokens", 1), "allowed": more.get("allowed", "none"),
            "temperature": more.get("temperature", 1.0)}


def _route(rows, experts, k, dtype, scores, **more):
    return {"op": "route", "rows": rows, "experts": experts, "k": k, "dtype": dtype, "scores": scores,
            "bias": more.get("bias", False), "groups": more.get("groups", 1), "top_groups": more.get("top_groups", 1),
            "group_score": more.get("group_score", "max"), "renormalise": more.get("renormalise", True),
            "scale": more.get("scale", 1.0)}


def listed():
    return [
        # one step of one reader: the smallest call, where launch latency counts
        {"name": "logprobs, one step", **_logprobs(1, 32000, "f16", 5)},
        # a character reader over a frame batch's crops: 512 crops x 8 positions, a small alphabet, part of it allowed
        {"name": "logprobs, characters", **_logprobs(4096, 97, "f32", 3, allowed="shared")},
        # a decoding batch, an odd vocabulary in rows that an engine pads, a temperature
        {"name": "logprobs, batch", **_logprobs(64, 50257, "bf16", 8, stride=50304, temperature=0.7)},
        # ragged candidate scoring in float32 with a grammar of its own for each row, rows not 16-byte aligned
        {"name": "logprobs, grammar", **_logprobs(333, 151667, "f32", 20, tokens=4, allowed="rows")},
        # whole prompts scored at once: the largest
        {"name": "logprobs, prompts", **_logprobs(4096, 128256, "bf16", 20)},
        # one row through a small gate
        {"name": "route, one row", **_route(1, 64, 6, "f32", "softmax")},
        # a frame batch's crops over a handful of embedders
        {"name": "route, crops", **_route(512, 8, 2, "f16", "softmax")},
        # a long batch: sigmoid scores, a balancing bias, groups
        {"name": "route, long", **_route(16384, 256, 8, "f32", "sigmoid", bias=True, groups=8, top_groups=4,
                                         group_score="top2", scale=2.5)},
        # a decoding batch's assignments by expert
        {"name": "plan, batch", "op": "plan", "rows": 64, "experts": 256, "k": 8, "dropped": 0.0},
        # a long batch's, some of them dropped
        {"name": "plan, long", "op": "plan", "rows": 16384, "experts": 256, "k": 8, "dropped": 0.05},
        # the embeddings of a frame batch's crops, two embedders each
        {"name": "combine, crops", "op": "combine", "rows": 512, "k": 2, "width": 512, "dtype": "f16", "dropped": 0.0},
        # a long batch of wide rows
        {"name": "combine, long", "op": "combine", "rows": 16384, "k": 8, "width": 2048, "dtype": "bf16",
         "dropped": 0.02},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "logprobs", "route", "route", "plan", "combine"))
    if op == "logprobs":
        vocab = _log_int(rng, 2, 160000)
        rows = _log_int(rng, 1, max(1, min(16384, 250_000_000 // vocab)))
        return _logprobs(rows, vocab, rng.choice(("f32", "f16", "bf16")), min(vocab, rng.choice((0, 1, 5, 20, 64))),
                         stride=vocab + rng.choice((0, 0, 1, 64 - vocab % 64)), tokens=rng.choice((0, 1, 1, 5)),
                         allowed=rng.choice(("none", "none", "shared", "rows")),
                         temperature=rng.choice((1.0, 1.0, 0.7, 1.6)))
    if op == "route":
        scores = rng.choice(("softmax", "sigmoid"))
        dtype = rng.choice(("f32", "f16", "bf16"))
        if rng.random() < 0.5:
            groups = rng.choice((2, 4, 8, 16))
            experts = groups * _log_int(rng, 2, 1024 // groups)
            rows = _log_int(rng, 1, min(16384, 4_194_304 // experts))
            top_groups = rng.randint(1, groups)
            k = min(rng.choice((1, 2, 6, 8)), top_groups * (experts // groups))
            return _route(rows, experts, k, dtype, scores, bias=rng.random() < 0.6, groups=groups,
                          top_groups=top_groups, group_score=rng.choice(("max", "top2")),
                          renormalise=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)))
        experts = _log_int(rng, 2, 1024)
        rows = _log_int(rng, 1, min(16384, 4_194_304 // experts))
        return _route(rows, experts, min(experts, rng.choice((1, 2, 4, 8, 16))), dtype, scores,
                      bias=rng.random() < 0.5, renormalise=rng.random() < 0.7)
    if op == "plan":
        return {"op": "plan", "rows": _log_int(rng, 1, 16384), "experts": _log_int(rng, 1, 1024),
                "k": rng.randint(1, 8), "dropped": rng.choice((0.0, 0.0, 0.1))}
    k, width = rng.randint(1, 8), _log_int(rng, 1, 2048)
    return {"op": "combine", "rows": _log_int(rng, 1, min(16384, 150_000_000 // ((k + 1) * width))), "k": k,
            "width": width, "dtype": rng.choice(("f32", "f16", "bf16")), "dropped": rng.choice((0.0, 0.1))}


def work(case):
    rows = case["rows"]
    if case["op"] == "logprobs":
        words = (case["vocab"] + 31) // 32 * 4
        masks = {"none": 0, "shared": words, "rows": rows * words}[case["allowed"]]
        values = rows * case["vocab"]
        return {"bytes": values * SIZE[case["dtype"]] + masks + rows * (12 * case["tokens"] + 4 + 12 * case["top"]),
                "flops": 6 * values}
    if case["op"] == "route":
        values = rows * case["experts"]
        return {"bytes": values * SIZE[case["dtype"]] + 4 * case["experts"] * case["bias"] + 8 * rows * case["k"],
                "flops": 6 * values}
    pairs = rows * case["k"]
    if case["op"] == "plan":
        return {"bytes": 12 * pairs + 4 * (case["experts"] + 1), "flops": 0}
    return {"bytes": (pairs + rows) * case["width"] * SIZE[case["dtype"]] + 8 * pairs, "flops": 2 * pairs * case["width"]}


# ---- inputs ---------------------------------------------------------------------------------

def _assignments(rows, experts, k, dropped, g):
    """Distinct experts per row, unevenly loaded; some assignments dropped."""
    load = torch.linspace(1.5, 0.0, experts, device="cuda")
    noise = torch.empty((rows, experts), device="cuda").exponential_(1.0, generator=g)
    ids = (load - noise.log()).topk(min(k, experts), dim=1).indices
    if k > experts:
        ids = torch.cat([ids, torch.full((rows, k - experts), -1, device="cuda")], dim=1)
    lost = torch.rand(ids.shape, device="cuda", generator=g) < dropped
    return torch.where(lost, -1, ids).to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, state = case["rows"], {"case": case}
    if case["op"] == "logprobs":
        vocab, dtype = case["vocab"], TYPES[case["dtype"]]
        # a head's logits: a wide bulk, a few likely tokens in each row
        logits = torch.empty((rows, case["stride"]), device="cuda", dtype=dtype)
        logits.normal_(-1.0, 2.5, generator=g)
        likely = torch.randint(0, vocab, (rows, 4), device="cuda", generator=g)
        lift = torch.rand((rows, 4), device="cuda", generator=g) * 12.0
        logits.scatter_(1, likely, lift.to(dtype))
        state["logits"] = logits[:, :vocab]
        n = case["tokens"]
        tokens = torch.randint(0, vocab, (rows, n), device="cuda", generator=g)
        tokens[:, : min(n, 4)] = likely[:, : min(n, 4)]
        if n:
            tokens[torch.rand((rows, n), device="cuda", generator=g) < 0.03] = -1  # padding
        state["tokens"] = tokens
        state["allowed"] = None
        if case["allowed"] != "none":
            count = 1 if case["allowed"] == "shared" else rows
            words = (vocab + 31) // 32
            bits = torch.randint(-(2**31), 2**31, (2, count, words), device="cuda", generator=g, dtype=torch.int64)
            state["allowed"] = (bits[0] | bits[1]).to(torch.int32)  # three tokens in four
        state["logprobs"] = torch.empty((rows, n), device="cuda")
        state["entropy"] = torch.empty((rows,), device="cuda")
        state["top_logprobs"] = torch.empty((rows, case["top"]), device="cuda")
        state["top_ids"] = torch.empty((rows, case["top"]), device="cuda", dtype=torch.int64)
    elif case["op"] == "route":
        logits = torch.empty((rows, case["experts"]), device="cuda").normal_(0.0, 1.5, generator=g)
        state["logits"] = logits.to(TYPES[case["dtype"]])
        state["bias"] = torch.empty(case["experts"], device="cuda").normal_(0.0, 0.05, generator=g) if case["bias"] else None
        state["weights"] = torch.empty((rows, case["k"]), device="cuda")
        state["ids"] = torch.empty((rows, case["k"]), device="cuda", dtype=torch.int32)
    elif case["op"] == "plan":
        pairs = rows * case["k"]
        state["ids"] = _assignments(rows, case["experts"], case["k"], case["dropped"], g)
        state["order"] = torch.empty((pairs,), device="cuda", dtype=torch.int32)
        state["slots"] = torch.empty((rows, case["k"]), device="cuda", dtype=torch.int32)
        state["offsets"] = torch.empty((case["experts"] + 1,), device="cuda", dtype=torch.int32)
    else:
        pairs = rows * case["k"]
        y = torch.empty((pairs, case["width"]), device="cuda").normal_(0.0, 1.0, generator=g)
        state["rows"] = y.to(TYPES[case["dtype"]])
        state["weights"] = torch.rand((rows, case["k"]), device="cuda", generator=g)
        slots = torch.randperm(pairs, device="cuda", generator=g).reshape(rows, case["k"])
        lost = torch.rand(slots.shape, device="cuda", generator=g) < case["dropped"]
        state["slots"] = torch.where(lost, -1, slots).to(torch.int32)
        state["out"] = torch.empty((rows, case["width"]), device="cuda", dtype=state["rows"].dtype)
    return state


# ---- the plain forms ------------------------------------------------------------------------

def _descending_keys(x):
    """int64 keys whose order is the values' and, among equal values, the lower index first."""
    bits = (x + 0.0).view(torch.int32)
    rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    n = x.shape[-1]
    return (rank << 32) + (n - 1 - torch.arange(n, device=x.device))


def _highest(x, k):
    """Indices of the k highest values in a row, ties to the lower index."""
    if k == 0:
        return torch.empty((*x.shape[:-1], 0), device=x.device, dtype=torch.int64)
    return x.shape[-1] - 1 - (_descending_keys(x).topk(k, dim=-1).values & 0xFFFFFFFF)


def _plain_logprobs(s):
    case, x = s["case"], s["logits"].float()
    if s["allowed"] is not None:
        v = torch.arange(case["vocab"], device=x.device)
        x = torch.where(((s["allowed"][:, v >> 5] >> (v & 31)) & 1) == 1, x, -math.inf)
    y = x / case["temperature"] if case["temperature"] != 1.0 else x
    high = y.amax(dim=1, keepdim=True)
    some = high > -math.inf
    d = torch.where(y > -math.inf, y - high, -math.inf)
    e = d.exp()
    total = e.sum(dim=1, keepdim=True)
    log_total = torch.where(some, total.log(), 0.0)
    mean = torch.where(y > -math.inf, e * d, 0.0).sum(dim=1, keepdim=True) / torch.where(some, total, 1.0)
    entropy = (log_total - mean).squeeze(1)
    t = s["tokens"]
    logprobs = torch.where(t < 0, 0.0, d.gather(1, t.clamp(min=0)) - log_total)
    ids = _highest(x, case["top"])
    top = d.gather(1, ids) - log_total
    return logprobs, entropy, top, torch.where(x.gather(1, ids) > -math.inf, ids, -1)


def _plain_route(s):
    case, x = s["case"], s["logits"].double()
    if case["scores"] == "sigmoid":
        score = (1.0 / (1.0 + (-x).exp())).float()
    else:
        e = (x - x.amax(dim=1, keepdim=True)).exp()
        score = (e / e.sum(dim=1, keepdim=True)).float()
    choice = score if s["bias"] is None else score + s["bias"]
    if case["groups"] > 1:
        grouped = choice.reshape(case["rows"], case["groups"], -1)
        best = grouped.gather(2, _highest(grouped, min(2, grouped.shape[2])))
        value = best.sum(dim=2) if case["group_score"] == "top2" else best[:, :, 0]
        kept = torch.zeros_like(value, dtype=torch.bool).scatter_(1, _highest(value, case["top_groups"]), True)
        choice = torch.where(kept[:, :, None], grouped, -math.inf).reshape(case["rows"], -1)
    ids = _highest(choice, case["k"])
    weights = score.gather(1, ids).double()
    if case["renormalise"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    return (weights * case["scale"]).float(), ids.to(torch.int32)


def _plain_plan(s):
    case, ids = s["case"], s["ids"].reshape(-1).long()
    experts, k = case["experts"], case["k"]
    ids = torch.where((ids >= 0) & (ids < experts), ids, experts)
    pairs = ids.numel()
    by_expert = ids.argsort(stable=True)
    offsets = torch.zeros(experts + 2, device=ids.device, dtype=torch.int64).scatter_add_(
        0, ids + 1, torch.ones_like(ids)).cumsum(0)[: experts + 1]
    place = torch.arange(pairs, device=ids.device)
    here = place < offsets[experts]
    order = torch.where(here, by_expert // k, -1)
    slots = torch.empty_like(ids).scatter_(0, by_expert, torch.where(here, place, -1))
    return order.to(torch.int32), slots.reshape(case["rows"], k).to(torch.int32), offsets.to(torch.int32)


def _plain_combine(s):
    slots = s["slots"].long()
    kept = slots >= 0
    weights = torch.where(kept, s["weights"], 0.0)
    taken = s["rows"].float()[slots.clamp(min=0)]
    return (taken * weights[:, :, None]).sum(dim=1).to(s["rows"].dtype)


# ---- the framework's calls ------------------------------------------------------------------

def _own(s):
    from shipinfer_b200 import logprobs, routing

    case = s["case"]
    if case["op"] == "logprobs":
        return logprobs.token_logprobs_device(
            s["logits"], s["tokens"], top=case["top"], allowed=s["allowed"], temperature=case["temperature"],
            logprobs=s["logprobs"], entropy=s["entropy"], top_logprobs=s["top_logprobs"], top_ids=s["top_ids"])
    if case["op"] == "route":
        return routing.route_experts_device(
            s["logits"], top_k=case["k"], scores=case["scores"], bias=s["bias"], groups=case["groups"],
            top_groups=case["top_groups"], group_score=case["group_score"], renormalise=case["renormalise"],
            scale=case["scale"], weights=s["weights"], ids=s["ids"])
    if case["op"] == "plan":
        return routing.plan_experts_device(s["ids"], case["experts"], order=s["order"], slots=s["slots"],
                                           offsets=s["offsets"])
    return routing.combine_experts_device(s["rows"], s["weights"], s["slots"], out=s["out"])


def run(state):
    if own:
        return _own(state)
    return {"logprobs": _plain_logprobs, "route": _plain_route, "plan": _plain_plan,
            "combine": _plain_combine}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        logprobs, entropy, top = [], [], []
        for lo in range(0, case["rows"], 512):
            x = s["logits"][lo : lo + 512].double()
            if s["allowed"] is not None:
                words = s["allowed"] if case["allowed"] == "shared" else s["allowed"][lo : lo + 512]
                bit = torch.arange(32, device=x.device)
                on = ((words[:, :, None] >> bit) & 1).bool().flatten(1)[:, : case["vocab"]]
                x = x.masked_fill(~on, -math.inf)
            y = x / case["temperature"]
            lp = y - torch.logsumexp(y, dim=1, keepdim=True)
            lp = torch.where(y > -math.inf, lp, -math.inf)  # an empty row too
            entropy.append(-torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(dim=1))
            t = s["tokens"][lo : lo + 512]
            logprobs.append(torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0))))
            top.append(lp.topk(case["top"], dim=1).values)
        return torch.cat(logprobs), torch.cat(entropy), torch.cat(top), None
    if case["op"] == "route":
        x = s["logits"].double()
        score = torch.sigmoid(x) if case["scores"] == "sigmoid" else torch.softmax(x, dim=1)
        choice = score.float() + (0.0 if s["bias"] is None else s["bias"])
        if case["groups"] > 1:
            grouped = choice.view(case["rows"], case["groups"], -1).sort(dim=2, descending=True).values
            value = grouped[..., 0]
            if case["group_score"] == "top2" and grouped.shape[2] > 1:
                value = value + grouped[..., 1]
            order = value.sort(dim=1, descending=True, stable=True).indices[:, case["top_groups"] :]
            group = torch.arange(case["experts"], device=x.device) // (case["experts"] // case["groups"])
            closed = (order[:, :, None] == group).any(dim=1)
            choice = choice.masked_fill(closed, -math.inf)
        ids = choice.sort(dim=1, descending=True, stable=True).indices[:, : case["k"]]
        weights = score.gather(1, ids)
        if case["renormalise"]:
            weights = weights / weights.sum(dim=1, keepdim=True)
        return weights * case["scale"], None
    if case["op"] == "plan":
        return None
    out = torch.zeros((case["rows"], case["width"]), device="cuda", dtype=torch.float64)
    for j in range(case["k"]):
        kept = s["slots"][:, j] >= 0
        out[kept] += s["weights"][kept, j, None].double() * s["rows"][s["slots"][kept, j].long()].double()
    return out
