"""Performance cases of the routed and 8-bit integer products: what a serving program calls, over the range it calls it in.

A case is a dict of plain values.  Five kinds, one per call that a model makes:

  route     ``ops.moe_route``: router logits -> expert ids and weights of every token
  quantize  ``ops.int8_quantize``: rows of floats -> 8-bit integers and one scale a row
  linear    ``ops.int8_mul_mat``: a linear layer with 8-bit integer weights, one scale a row, on float activations, which
            it quantizes by the token
  moe       ``ops.int8_fused_moe``: the routed expert step on 8-bit integer weights, from ids and weights to the sum
  layer     the expert layer as a model runs it: route, then moe

With ``own`` false, ``run`` computes the same in elementary torch operations.

What the operators are, in exact arithmetic:

  quantize  a = max |x| of the row, scale = a / 127, code = x * 127 / a rounded to the nearest integer, halves to the even
            one.  A row of zeros has scale 0 and codes 0.
  linear    y[t, n] = (sum over k of code[t, k] * W[n, k]) * scale[t] * w_scale[n] + bias[n]
  route     scores s = softmax or sigmoid of the row's logits; an expert whose logit is -inf or NaN is masked.  The choice
            goes by s + bias with a bias, by s without one.  With groups, an expert's group has to be among the `topk_group`
            best, by the sum of the group's two best choices with a bias, by its best one without.  The top_k best are
            taken, the best first, equals by the lower index; weights are their s (without bias), divided by their sum if
            `renormalize`, times `scale`.  A place for which no unmasked expert is left has id -1 and weight 0.
  moe       h = act(gate) * up for every routed (token, expert), gate and up as `linear` has them; h quantized by the row as
            `quantize` has it; y[t] = sum over j of weight[t, j] * down(h[t, j]).  Ids of -1 contribute nothing.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
MOST_LINEAR = 4096 * 14336 * 4096      # multiply-adds of one linear pass
MOST_MOE = 2048 * 8 * 3 * 2048 * 1024  # ... of one expert step
MOST_DENSE = 2048 * 64 * 2048 * 1024   # tokens * experts * hidden * intermediate
INF = float("inf")


def listed():
    return [
        # one token of a decode step: nothing but latency
        {"name": "route 1", "kind": "route", "tokens": 1, "experts": 64, "top_k": 8, "scoring": "softmax", "groups": 1, "topk_group": 1,
         "bias": False, "renormalize": True, "scale": 1.0, "masked": 0, "padding": 0, "dtype": "bfloat16"},
        # a batch of requests, padded to the size of its captured graph, odd number of experts, three of them switched off
        {"name": "route 333 masked", "kind": "route", "tokens": 333, "experts": 60, "top_k": 4, "scoring": "softmax", "groups": 1,
         "topk_group": 1, "bias": False, "renormalize": False, "scale": 1.0, "masked": 3, "padding": 13, "dtype": "float32"},
        # a large prefill chunk of a model with many experts in groups, balanced by a bias
        {"name": "route 8192 grouped", "kind": "route", "tokens": 8192, "experts": 256, "top_k": 8, "scoring": "sigmoid", "groups": 8,
         "topk_group": 4, "bias": True, "renormalize": True, "scale": 2.5, "masked": 0, "padding": 0, "dtype": "float32"},
        # one token's activations ahead of several products that share them
        {"name": "quantize 1", "kind": "quantize", "rows": 1, "k": 4096, "dtype": "bfloat16"},
        # a large weight matrix at loading
        {"name": "quantize 28672", "kind": "quantize", "rows": 28672, "k": 8192, "dtype": "float16"},
        # decode: one token through a square projection, a batch through an MLP one
        {"name": "linear 1", "kind": "linear", "tokens": 1, "n": 4096, "k": 4096, "bias": False, "dtype": "bfloat16"},
        {"name": "linear 27", "kind": "linear", "tokens": 27, "n": 14336, "k": 4096, "bias": False, "dtype": "float16"},
        # prefill: an ordinary chunk through the down projection with a bias, the largest chunk
        {"name": "linear 500 bias", "kind": "linear", "tokens": 500, "n": 4096, "k": 14336, "bias": True, "dtype": "bfloat16"},
        {"name": "linear 4096", "kind": "linear", "tokens": 4096, "n": 14336, "k": 4096, "bias": False, "dtype": "bfloat16"},
        # mixture of experts: a decode batch, a prefill chunk
        {"name": "moe 8", "kind": "moe", "tokens": 8, "experts": 64, "top_k": 8, "hidden": 2048, "inter": 1024, "act": "silu",
         "dtype": "float16"},
        {"name": "moe 2048", "kind": "moe", "tokens": 2048, "experts": 64, "top_k": 8, "hidden": 2048, "inter": 1024, "act": "silu",
         "dtype": "bfloat16"},
        # router and experts together, an ordinary batch with a padded end
        {"name": "layer 200", "kind": "layer", "tokens": 200, "experts": 32, "top_k": 4, "hidden": 1536, "inter": 768, "act": "gelu",
         "scoring": "sigmoid", "groups": 4, "topk_group": 2, "bias": True, "renormalize": True, "scale": 1.5, "masked": 0, "padding": 7,
         "dtype": "bfloat16"},
    ]


# ---- drawn cases -------------------------------------------------------------------------------------------


def _log(rng, lo, hi, step=1):
    """Log-uniform between lo and hi, a multiple of `step`."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _draw_route(rng, experts, tokens):
    groups = rng.choice([g for g in (1, 1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
    topk_group = rng.randint(1, groups)
    return {"top_k": rng.randint(1, min(16, topk_group * (experts // groups))), "scoring": rng.choice(["softmax", "sigmoid"]), "groups": groups,
            "topk_group": topk_group, "bias": rng.random() < 0.5, "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 1.0, 1.5, 2.5]),
            "masked": rng.choice([0, 0, rng.randint(1, experts // 2)]), "padding": rng.choice([0, 0, rng.randint(0, tokens // 4)])}


def draw(rng):
    kind = rng.choice(["route", "route", "quantize", "linear", "linear", "linear", "moe", "moe", "layer"])
    if kind == "route":
        tokens, experts = _log(rng, 1, 8192), rng.choice([8, 16, 32, 60, 64, 72, 96, 128, 160, 256])
        return {"kind": kind, "tokens": tokens, "experts": experts, **_draw_route(rng, experts, tokens), "dtype": rng.choice(sorted(DTYPES))}
    if kind == "quantize":
        k = _log(rng, 64, 28672, rng.choice([1, 2, 8, 256]))
        return {"kind": kind, "rows": _log(rng, 1, min(28672, 28672 * 8192 // k)), "k": k, "dtype": rng.choice(["float16", "bfloat16", "float32"])
                if k < 4096 else rng.choice(["float16", "bfloat16"])}
    if kind == "linear":
        n, k = _log(rng, 256, 28672, rng.choice([1, 8, 128])), _log(rng, 256, 14336, rng.choice([1, 16, 256]))
        return {"kind": kind, "tokens": _log(rng, 1, max(1, min(4096, MOST_LINEAR // (n * k)))), "n": n, "k": k, "bias": rng.random() < 0.3,
                "dtype": rng.choice(["float16", "bfloat16", "bfloat16"])}
    experts = rng.choice([8, 16, 32, 64])
    hidden = _log(rng, 512, 4096, rng.choice([16, 128]))
    inter = min(_log(rng, 256, 4096, rng.choice([8, 128])), MOST_DENSE // (64 * hidden * experts) // 8 * 8)
    if kind == "moe":
        top_k = rng.choice([1, 2, 4, 6, 8])
        most = min(MOST_DENSE // (experts * hidden * inter), MOST_MOE // (3 * hidden * inter * top_k), 4096)
        return {"kind": kind, "tokens": _log(rng, 1, max(1, most)), "experts": experts, "top_k": top_k, "hidden": hidden, "inter": inter,
                "act": rng.choice(["silu", "silu", "gelu"]), "dtype": rng.choice(["float16", "bfloat16"])}
    tokens = _log(rng, 1, max(1, min(MOST_DENSE // (experts * hidden * inter), MOST_MOE // (3 * hidden * inter * 16), 1024)))
    return {"kind": kind, "tokens": tokens, "experts": experts, **_draw_route(rng, experts, tokens), "hidden": hidden, "inter": inter,
            "act": rng.choice(["silu", "gelu"]), "dtype": rng.choice(["float16", "bfloat16"])}


# ---- inputs ------------------------------------------------------------------------------------------------


def _ops():
    path = os.path.join(os.getcwd(), "vllm-gguf-plugin-prism_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vllm_gguf_plugin import ops

    return ops


def _activations(gen, rows, k, dtype):
    """N(0, 1) with a few channels eight times as large, as the residual stream of a trained model has them."""
    x = torch.randn(rows, k, device="cuda", generator=gen)
    loud = torch.randint(0, k, (max(1, k // 512),), device="cuda", generator=gen)
    x[:, loud] *= 8
    return x.to(dtype)


def _codes(gen, rows, k):
    """int8 [rows, k] of normally distributed codes, rows a multiple of 16 bytes apart, and a scale for every row."""
    buf = torch.empty(rows, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    for r in range(0, rows, 8192):
        part = buf[r:r + 8192]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen).mul_(36).round_().clamp_(-127, 127))
    return buf[:, :k], (0.5 + torch.rand(rows, device="cuda", generator=gen)) * (0.8 / 36 / math.sqrt(k))


def _router(gen, case):
    t, e = case["tokens"], case["experts"]
    logits = torch.randn(t, e, device="cuda", generator=gen) * 1.5
    if case["masked"]:
        off = torch.randperm(e, device="cuda", generator=gen)[:case["masked"]]
        logits[:, off] = -INF
    if case["padding"]:
        logits[t - case["padding"]:] = -INF
    bias = torch.randn(e, device="cuda", generator=gen) * 0.1 if case["bias"] else None
    return logits.to(DTYPES[case["dtype"]]), bias


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind in ("route", "layer"):
        state["logits"], state["bias"] = _router(gen, case)
    if kind == "quantize":
        state["x"] = _activations(gen, case["rows"], case["k"], dtype)
    if kind == "linear":
        state["w"], state["w_scale"] = _codes(gen, case["n"], case["k"])
        state["x"] = _activations(gen, case["tokens"], case["k"], dtype)
        state["b"] = torch.randn(case["n"], device="cuda", generator=gen).to(dtype) if case["bias"] else None
    if kind in ("moe", "layer"):
        e, h, i = case["experts"], case["hidden"], case["inter"]
        w13, s13 = _codes(gen, e * 2 * i, h)
        w2, s2 = _codes(gen, e * h, i)
        state["w13"], state["s13"] = w13.unflatten(0, (e, 2 * i)), s13.view(e, 2 * i)
        state["w2"], state["s2"] = w2.unflatten(0, (e, h)), s2.view(e, h)
        state["x"] = _activations(gen, case["tokens"], h, dtype)
    if kind == "moe":
        p = (torch.randn(case["tokens"], case["experts"], device="cuda", generator=gen) * 1.5).softmax(-1)
        weights, ids = p.topk(case["top_k"], dim=-1)
        state["weights"], state["ids"] = weights.contiguous(), ids.to(torch.int32)
    if own:
        state["ops"] = _ops()
    return state


# ---- one pass ----------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return _plain(state)
    ops = state["ops"]
    if kind == "quantize":
        return ops.int8_quantize(state["x"])
    if kind == "linear":
        return ops.int8_mul_mat(state["w"], state["w_scale"], state["x"], bias=state["b"])
    if kind == "moe":
        weights, ids = state["weights"], state["ids"]
    else:
        weights, ids = ops.moe_route(state["logits"], case["top_k"], scoring=case["scoring"], bias=state["bias"], n_group=case["groups"],
                                     topk_group=case["topk_group"], renormalize=case["renormalize"], scale=case["scale"])
        if kind == "route":
            return weights, ids
    y = ops.int8_fused_moe(state["x"], state["w13"], state["s13"], state["w2"], state["s2"], weights, ids, case["act"])
    return y if kind == "moe" else (y, weights, ids)


def _plain_quantize(x):
    x = x.double()   # a code next to a half is lost in 32 bits
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * 127 / torch.where(top > 0, top, 1.0))
    return codes, (top / torch.full_like(top, 127)).squeeze(-1).float()


def _plain_act(name, gate):
    return gate / (1 + torch.exp(-gate)) if name == "silu" else 0.5 * gate * (1 + torch.erf(gate * math.sqrt(0.5)))


def _plain_route(state):
    case, bias = state["case"], state["bias"]
    x = state["logits"].double()   # two choices next to one another are lost in 32 bits
    x = torch.where(torch.isnan(x), -INF, x).clamp_(max=torch.finfo(torch.float32).max)
    if case["scoring"] == "softmax":
        top = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(top == -INF, 0.0, top))
        s = e / e.sum(-1, keepdim=True).clamp_(min=1e-300)
    else:
        s = 1 / (1 + torch.exp(-x))
    choice = torch.where(x == -INF, -INF, x if bias is None else s + bias.double())
    if case["groups"] > 1:
        g = choice.unflatten(-1, (case["groups"], -1))
        best = g.sort(dim=-1, descending=True).values
        score = best[..., 0]
        if bias is not None and g.shape[-1] > 1:
            score = score + torch.where(best[..., 1] == -INF, 0.0, best[..., 1])
        picked = score.sort(dim=-1, descending=True, stable=True).indices[:, :case["topk_group"]]
        keep = torch.zeros_like(score).scatter_(1, picked, 1.0) > 0
        choice = torch.where(keep[..., None], g, -INF).flatten(1)
    values, ids = choice.sort(dim=-1, descending=True, stable=True)
    values, ids = values[:, :case["top_k"]], ids[:, :case["top_k"]]
    weights = torch.where(values == -INF, 0.0, s.gather(1, ids))
    if case["renormalize"]:
        total = weights.sum(-1, keepdim=True)
        weights = weights / torch.where(total > 0, total, 1.0)
    return (weights * case["scale"]).float(), torch.where(values == -INF, -1, ids).to(torch.int32)


def _plain_moe(state, weights, ids):
    case, x = state["case"], state["x"]
    codes, scales = _plain_quantize(x)
    out = torch.zeros(x.shape, device=x.device)
    half = case["inter"]
    for e in range(case["experts"]):
        share = torch.where(ids == e, weights, 0.0).sum(-1)[:, None]
        gate_up = (codes @ state["w13"][e].double().T).float() * scales[:, None] * state["s13"][e]   # (in 64 bits: its codes come next)
        h, h_scale = _plain_quantize(_plain_act(case["act"], gate_up[:, :half]) * gate_up[:, half:])
        out += share * ((h.float() @ state["w2"][e].float().T) * h_scale[:, None] * state["s2"][e])
    return out.to(x.dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        codes, scales = _plain_quantize(state["x"])
        return codes.to(torch.int8), scales
    if kind == "linear":
        codes, scales = _plain_quantize(state["x"])
        y = (codes.float() @ state["w"].float().T) * scales[:, None] * state["w_scale"]
        return (y if state["b"] is None else y + state["b"].float()).to(state["x"].dtype)
    if kind == "moe":
        return _plain_moe(state, state["weights"], state["ids"])
    weights, ids = _plain_route(state)
    return (weights, ids) if kind == "route" else (_plain_moe(state, weights, ids), weights, ids)


# ---- what has to move and to be computed -------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (size + 1) + 4 * case["rows"], "flops": 3 * n}
    t = case["tokens"]
    if kind == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": n * k + 4 * n + size * (t * (n + k) + (n if case["bias"] else 0)), "flops": 2 * t * n * k}
    bytes_ = flops = 0
    if kind in ("route", "layer"):
        e = case["experts"]
        bytes_ += t * e * size + 8 * t * case["top_k"] + (4 * e if case["bias"] else 0)
        flops += t * e * (5 + case["top_k"])
    if kind in ("moe", "layer"):
        e, k, h, i = case["experts"], case["top_k"], case["hidden"], case["inter"]
        used = e * (1 - (1 - k / e) ** t)     # experts that some token asks for
        bytes_ += int(used * (3 * h * i + 4 * (2 * i + h))) + 2 * size * t * h + 8 * t * k
        flops += 6 * t * k * h * i
    return {"bytes": bytes_, "flops": flops}


# ---- the operators from their definitions, in 64 bits ------------------------------------------------------


def _exact_codes(x):
    """(codes, scales): 127 fractions of the row's largest value."""
    x = x.double()
    a = torch.linalg.vector_norm(x, INF, dim=1)
    return torch.round(x.mul(127).div_(a.masked_fill(a == 0, 1.0).unsqueeze(1))), a / 127


def _exact_route(state):
    import numpy as np

    case = state["case"]
    x = np.minimum(state["logits"].double().cpu().numpy(), float(torch.finfo(torch.float32).max))
    x[np.isnan(x)] = -INF
    live = x > -INF
    if case["scoring"] == "softmax":
        top = np.where(live.any(1), np.where(live, x, -1e308).max(1), 0.0)
        with np.errstate(over="ignore", under="ignore"):
            s = np.where(live, np.exp(np.where(live, x, 0.0) - top[:, None]), 0.0)
        total = s.sum(1)
        s = s / np.where(total > 0, total, 1.0)[:, None]
    else:
        z = np.exp(-np.abs(np.where(live, x, 0.0)))
        s = np.where(live, np.where(x >= 0, 1 / (1 + z), z / (1 + z)), 0.0)
    choice = np.where(live, x if state["bias"] is None else s + state["bias"].double().cpu().numpy(), -INF)
    rows = np.arange(len(x))
    if case["groups"] > 1:
        per = case["experts"] // case["groups"]
        score = np.full((len(x), case["groups"]), -INF)
        for g in range(case["groups"]):
            part = choice[:, g * per:(g + 1) * per].copy()
            first = part.argmax(1)
            score[:, g] = part[rows, first]
            if state["bias"] is not None:
                part[rows, first] = -INF
                score[:, g] += np.where(part.max(1) > -INF, part.max(1), 0.0)
        allowed = np.zeros_like(live)
        taken = np.zeros_like(score, dtype=bool)
        for _ in range(case["topk_group"]):
            free = np.where(taken, np.nan, score)
            g = np.array([int(np.nanargmax(r)) for r in free]) if len(x) else rows
            taken[rows, g] = True
            for c in range(per):
                allowed[rows, g * per + c] = True
        choice = np.where(allowed, choice, -INF)
    weights, ids = np.zeros((len(x), case["top_k"])), np.full((len(x), case["top_k"]), -1, dtype=np.int32)
    for j in range(case["top_k"]):
        at = choice.argmax(1)
        ok = choice[rows, at] > -INF
        ids[ok, j] = at[ok]
        weights[ok, j] = s[rows, at][ok]
        choice[rows, at] = -INF
    if case["renormalize"]:
        total = weights.sum(1, keepdims=True)
        weights = np.divide(weights, total, out=np.zeros_like(weights), where=total > 0)
    return torch.from_numpy(weights * case["scale"]), torch.from_numpy(ids)


def _exact_moe(state, weights, ids):
    case, x = state["case"], state["x"]
    codes, scales = _exact_codes(x)
    out = torch.zeros(x.shape, device=x.device, dtype=torch.float64)
    half, weights, ids = case["inter"], weights.to(x.device).double(), ids.to(x.device)
    for e in ids.unique().tolist():
        if e < 0:
            continue
        token, place = (ids == e).nonzero(as_tuple=True)
        both = torch.einsum("tk,nk->tn", codes[token], state["w13"][e].double())
        both = both * torch.outer(scales[token], state["s13"][e].double())
        gate, up = both.split(half, dim=1)
        h, h_scale = _exact_codes(up * (gate * torch.sigmoid(gate) if case["act"] == "silu" else gate * torch.special.ndtr(gate)))
        down = torch.einsum("tk,nk->tn", h, state["w2"][e].double()) * torch.outer(h_scale, state["s2"][e].double())
        out.index_add_(0, token, down * weights[token, place][:, None])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        codes, scales = _exact_codes(state["x"])
        return codes.to(torch.int8), scales
    if kind == "linear":
        codes, scales = _exact_codes(state["x"])
        y = torch.einsum("tk,nk->tn", codes, state["w"].double()) * torch.outer(scales, state["w_scale"].double())
        return y if state["b"] is None else y + state["b"].double()
    if kind == "moe":
        return _exact_moe(state, state["weights"], state["ids"])
    weights, ids = _exact_route(state)
    return (weights, ids) if kind == "route" else (_exact_moe(state, weights, ids), weights, ids)
