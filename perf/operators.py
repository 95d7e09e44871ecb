"""The routed feed-forward and the fused projection of this framework, measured call by call.

Three operators (``op`` of a case):

* ``route``    ``route_experts``: every token's experts and their weights from the router's logits.
* ``experts``  ``expert_mlp``: the gated feed-forward of the chosen experts, weighted, summed and added to a residual.
* ``linear``   ``fused_linear``: a projection with bias, activation or gate, and residual in its epilogue.

``run`` computes the plain form (elementary torch operations in 32 bits, choices in 64) or, where ``own`` is set, calls
the framework.  Widths and feed-forward sizes are those of the decoders this framework serves, or generic.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


def _route(name, tokens, experts, top_k, scores="softmax", bias=False, groups=1, top_groups=1, group_best=1,
           renormalize=True, scale=1.0, dtype="float32"):
    case = {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "scores": scores, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_best": group_best, "renormalize": renormalize,
            "scale": scale, "dtype": dtype}
    return {"name": name, **case} if name else case


def _experts(name, tokens, width, experts, ff, top_k, skew=0.5, activation="silu", residual=True):
    case = {"op": "experts", "tokens": tokens, "width": width, "experts": experts, "ff": ff, "top_k": top_k,
            "skew": skew, "activation": activation, "residual": residual}
    return {"name": name, **case} if name else case


def _linear(name, tokens, k, n, bias=False, activation="none", gated=False, residual=False):
    """``n``: columns of the result; a gated weight has twice as many rows."""

    case = {"op": "linear", "tokens": tokens, "k": k, "n": n, "bias": bias, "activation": activation, "gated": gated,
            "residual": residual}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One user's next token: the router of one layer.
        _route("route-1", 1, 128, 8),
        # A prompt batch under a balance bias and groups of experts, as large expert pools are routed.
        _route("route-grouped-4096", 4096, 256, 8, scores="sigmoid", bias=True, groups=8, top_groups=4, group_best=2,
               scale=2.5),
        # Many packed prompts; 16-bit logits, weights of the full softmax.
        _route("route-30011", 30011, 64, 6, renormalize=False, dtype="bfloat16"),
        # One user's next token through a pool of small experts: their weights once.
        _experts("experts-decode-1", 1, 2048, 128, 768, 8),
        # A decode batch that reaches nearly every expert with a few tokens each.
        _experts("experts-decode-40", 40, 2048, 128, 768, 8),
        # A prompt chunk over fewer, wider experts; ragged loads, no residual.
        _experts("experts-chunk-777", 777, 2560, 64, 1408, 6, skew=1.0, residual=False),
        # Prompts prefilled whole.
        _experts("experts-prefill-8192", 8192, 2048, 128, 768, 8),
        # One user's next token: gate and up of a dense feed-forward, gated in the epilogue.
        _linear("linear-gated-1", 1, 2048, 6144, activation="silu", gated=True),
        # A decode batch's down projection onto the residual stream.
        _linear("linear-residual-24", 24, 9728, 2560, residual=True),
        # A prompt chunk with bias and gelu; no size a whole number of tiles.
        _linear("linear-gelu-1021", 1021, 2056, 5003, bias=True, activation="gelu"),
        # Prompts: gate and up in one product.
        _linear("linear-gated-4096", 4096, 2560, 9728, activation="silu", gated=True),
        # Prompts: the down projection of the widest feed-forward.
        _linear("linear-residual-8192", 8192, 12288, 4096, bias=True, residual=True),
    ]


MOST_FLOPS = 0.8e12  # of a drawn case: below the largest listed one
MOST_WEIGHTS = 1.2e9  # bytes


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "linear", "linear"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_uniform(rng, max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(10, top_groups * (experts // groups)))
        return _route(None, _log_uniform(rng, 1, 32768), experts, top_k, scores=rng.choice(["softmax", "sigmoid"]),
                      bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                      group_best=rng.randint(1, min(2, experts // groups)), renormalize=rng.random() < 0.7,
                      scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]))
    if op == "experts":
        width = 8 * _log_uniform(rng, 48, 512)
        ff = 8 * _log_uniform(rng, 16, 256)
        experts = min(_log_uniform(rng, 4, 160), int(MOST_WEIGHTS / (6 * width * ff)))
        top_k = rng.randint(1, min(10, experts))
        tokens = min(_log_uniform(rng, 1, 8192), int(MOST_FLOPS / (6 * top_k * width * ff)))
        return _experts(None, tokens, width, experts, ff, top_k, skew=rng.choice([0.0, 0.5, 1.0, 2.0]),
                        activation=rng.choice(["silu", "silu", "gelu"]), residual=rng.random() < 0.6)
    gated = rng.random() < 0.5
    k = 8 * _log_uniform(rng, 32, 1536)
    n = _log_uniform(rng, 200, 16384)
    n = n if rng.random() < 0.25 else 8 * (n // 8)
    tokens = min(_log_uniform(rng, 1, 8192), int(MOST_FLOPS / (2 * k * n * (2 if gated else 1))))
    return _linear(None, tokens, k, n, bias=rng.random() < 0.4,
                   activation=rng.choice(["silu", "gelu"] if gated else ["none", "none", "gelu", "relu", "silu"]),
                   gated=gated, residual=rng.random() < 0.5)


# -- inputs -----------------------------------------------------------------------------------------------

def _router_logits(generator, tokens, experts, skew):
    """Logits of spread one, with experts that are more popular than others by ``skew``."""

    z = torch.randn(tokens, experts, generator=generator, device=DEVICE)
    return z + skew * torch.randn(experts, generator=generator, device=DEVICE)


def _bf16(generator, *shape, scale=1.0):
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEVICE)
    return out.normal_(0.0, scale, generator=generator)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    tokens = case["tokens"]
    if case["op"] == "route":
        logits = _router_logits(g, tokens, case["experts"], 0.5)
        bias = 0.05 * torch.randn(case["experts"], generator=g, device=DEVICE) if case["bias"] else None
        return {**state, "logits": logits.to(getattr(torch, case["dtype"])), "bias": bias}
    if case["op"] == "experts":
        width, experts, ff = case["width"], case["experts"], case["ff"]
        z = _router_logits(g, tokens, experts, case["skew"])
        top, ids = torch.sort(z, dim=1, descending=True, stable=True)
        weights = torch.softmax(top[:, :case["top_k"]], dim=1)
        return {**state, "x": _bf16(g, tokens, width), "ids": ids[:, :case["top_k"]].to(torch.int32).contiguous(),
                "weights": weights.contiguous(),
                "gate_up": _bf16(g, experts, 2 * ff, width, scale=width ** -0.5),
                "down": _bf16(g, experts, width, ff, scale=ff ** -0.5),
                "residual": _bf16(g, tokens, width) if case["residual"] else None}
    k, n = case["k"], case["n"]
    rows = 2 * n if case["gated"] else n
    return {**state, "x": _bf16(g, tokens, k), "weight": _bf16(g, rows, k, scale=k ** -0.5),
            "bias": _bf16(g, rows, scale=0.5) if case["bias"] else None,
            "residual": _bf16(g, tokens, n) if case["residual"] else None}


# -- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return {"route": _run_route, "experts": _run_experts, "linear": _run_linear}[state["case"]["op"]](state)


def _run_route(state):
    c, logits, bias = state["case"], state["logits"], state["bias"]
    if own:
        from mini_inference_engine_b200.engine.kernels.experts import route_experts

        ids, weights = route_experts(logits, c["top_k"], scores=c["scores"], bias=bias, groups=c["groups"],
                                     top_groups=c["top_groups"], group_best=c["group_best"],
                                     renormalize=c["renormalize"], scale=c["scale"], status=state["status"])
        return {"ids": ids, "weights": weights}
    z = logits.double()  # scores next to each other decide which experts are taken
    if c["scores"] == "softmax":
        e = torch.exp(z - z.max(dim=1, keepdim=True).values)
        s = e / e.sum(dim=1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    choice = s if bias is None else s + bias.double()
    if c["groups"] > 1:
        grouped = choice.view(c["tokens"], c["groups"], -1)
        best = torch.sort(grouped, dim=2, descending=True).values[:, :, :c["group_best"]].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        mask = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        choice = grouped.masked_fill(mask.unsqueeze(2), -math.inf).view(c["tokens"], -1)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    weights = torch.gather(s, 1, ids)
    if c["renormalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": (weights * c["scale"]).float()}


def _activate(z, kind):
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    return z


def _run_experts(state):
    c, x, ids, weights = state["case"], state["x"], state["ids"], state["weights"]
    gate_up, down, residual = state["gate_up"], state["down"], state["residual"]
    if own:
        from mini_inference_engine_b200.engine.kernels.experts import expert_mlp

        return expert_mlp(x, ids, weights, gate_up, down, activation=c["activation"], residual=residual,
                          status=state["status"])
    tokens, top_k, ff, experts = c["tokens"], c["top_k"], c["ff"], c["experts"]
    flat = ids.reshape(-1).long()
    pairs = tokens * top_k
    if pairs <= experts:  # a few tokens: every pair with its own expert's weights
        rows = x.float().repeat_interleave(top_k, dim=0).unsqueeze(2)
        z = torch.bmm(gate_up[flat].float(), rows).squeeze(2)
        hidden = _activate(z[:, :ff], c["activation"]) * z[:, ff:]
        out = torch.bmm(down[flat].float(), hidden.unsqueeze(2)).squeeze(2)
    else:  # rows sorted by expert, every expert's padded to the longest
        order = torch.sort(flat, stable=True).indices
        count = torch.zeros(experts, dtype=torch.int64, device=x.device).index_add_(0, flat, torch.ones_like(flat))
        first = torch.cumsum(count, 0) - count
        place = torch.arange(pairs, device=x.device) - first[flat[order]]
        most = int(count.max())
        rows = torch.zeros(experts, most, c["width"], dtype=torch.float32, device=x.device)
        rows[flat[order], place] = x[order // top_k].float()
        z = torch.bmm(rows, gate_up.float().transpose(1, 2))
        hidden = _activate(z[:, :, :ff], c["activation"]) * z[:, :, ff:]
        out = torch.empty(pairs, c["width"], dtype=torch.float32, device=x.device)
        out[order] = torch.bmm(hidden, down.float().transpose(1, 2))[flat[order], place]
    y = (out.view(tokens, top_k, -1) * weights.unsqueeze(2)).sum(dim=1)
    if residual is not None:
        y = y + residual.float()
    return y.to(torch.bfloat16)


def _run_linear(state):
    c, x, weight, bias, residual = state["case"], state["x"], state["weight"], state["bias"], state["residual"]
    if own:
        from mini_inference_engine_b200.engine.kernels.linear import fused_linear

        return fused_linear(x, weight, bias, activation=c["activation"], gated=c["gated"], residual=residual,
                            status=state["status"])
    y = torch.matmul(x.float(), weight.float().t())
    if bias is not None:
        y = y + bias.float()
    if c["gated"]:
        y = _activate(y[:, :c["n"]], c["activation"]) * y[:, c["n"]:]
    else:
        y = _activate(y, c["activation"])
    if residual is not None:
        y = y + residual.float()
    return y.to(torch.bfloat16)


# -- what a pass cannot do without ------------------------------------------------------------------------

def work(case):
    t = case["tokens"]
    if case["op"] == "route":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": t * case["experts"] * size + t * case["top_k"] * 8 + (4 * case["experts"] if case["bias"] else 0),
                "flops": 4.0 * t * case["experts"]}
    if case["op"] == "experts":
        h, f, e, k = case["width"], case["ff"], case["experts"], case["top_k"]
        # Experts that a batch reaches: all that t k draws without skew would; one token reaches top_k.
        used = e * (1.0 - (1.0 - k / e) ** t)
        return {"bytes": used * 6 * h * f + t * h * (6 if case["residual"] else 4) + t * k * 8, "flops": 6.0 * t * k * h * f}
    rows = case["n"] * (2 if case["gated"] else 1)
    return {"bytes": 2.0 * (t * case["k"] + rows * case["k"] + t * case["n"] * (2 if case["residual"] else 1)
                            + (rows if case["bias"] else 0)),
            "flops": 2.0 * t * rows * case["k"]}


# -- the definition, in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "experts": _exact_experts, "linear": _exact_linear}[case["op"]](case, state)


def _exact_route(case, state):
    z = state["logits"].double().cpu().numpy()
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    if case["scores"] == "softmax":
        score = np.exp(z - np.logaddexp.reduce(z, axis=1, keepdims=True))
    else:
        score = np.where(z >= 0, 1.0, np.exp(np.minimum(z, 0))) / (1.0 + np.exp(-np.abs(z)))
    key = score.copy() if state["bias"] is None else score + state["bias"].double().cpu().numpy()[None, :]
    if case["groups"] > 1:
        size = experts // case["groups"]
        best = np.partition(key.reshape(tokens, case["groups"], size), size - case["group_best"], axis=2)
        best = best[:, :, size - case["group_best"]:].sum(axis=2)
        rank = np.lexsort((np.broadcast_to(np.arange(case["groups"]), best.shape), -best), axis=1)
        for row in range(tokens):
            for group in rank[row, case["top_groups"]:]:
                key[row, group * size:(group + 1) * size] = -np.inf
    ids = np.lexsort((np.broadcast_to(np.arange(experts), key.shape), -key), axis=1)[:, :k]
    w = np.take_along_axis(score, ids, axis=1)
    if case["renormalize"]:
        w = w / w.sum(axis=1, keepdims=True)
    return {"ids": ids.astype(np.int32), "weights": w * case["scale"]}


def _exact_activation(z, kind):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return torch.clamp(z, min=0) if kind == "relu" else z


def _exact_experts(case, state):
    x, ids, weights = state["x"].double(), state["ids"].long(), state["weights"].double()
    y = torch.zeros_like(x) if state["residual"] is None else state["residual"].double()
    for e in range(case["experts"]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            gate, up = (x[token] @ state["gate_up"][e].double().t()).chunk(2, dim=1)
            hidden = _exact_activation(gate, case["activation"]) * up
            y.index_add_(0, token, weights[token, slot, None] * (hidden @ state["down"][e].double().t()))
    return y


def _exact_linear(case, state):
    y = state["x"].double() @ state["weight"].double().t()
    if state["bias"] is not None:
        y += state["bias"].double()
    if case["gated"]:
        gate, up = y.chunk(2, dim=1)
        y = _exact_activation(gate, case["activation"]) * up
    else:
        y = _exact_activation(y, case["activation"])
    return y if state["residual"] is None else y + state["residual"].double()
