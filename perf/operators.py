"""The float operators of a language model that this package has, as cases that can be timed one by one.

  linear    one product with its epilogue, y = act(x . w^T * w_scale + b) + r: float16 or float32, or float16 rows against
            int8 weights; from one row (a token being generated) to a prompt's
  experts   the same product with a weight matrix for each expert, over rows that a routing has sent to them
  routing   scores of the experts, the choice of k of them, their weights, and the rows in the experts' order
  combine   the weighted sum of a row's k expert results, with the residual
  logprobs  log probabilities of given tokens, the entropy of each row and the best alternatives

With `own` false, run() computes them in elementary torch operations; with `own` true it makes the package's calls.
"""
import importlib
import math

import torch

own = False

PACKAGE = "chainer-compiler_amd"  # (not an identifier: imported by name)
_TYPES = {"float16": torch.float16, "float32": torch.float32, "int8": torch.int8}


def _ops():
    pkg = importlib.import_module(PACKAGE)
    pkg.capi.init(0)
    return pkg.ops


# ---- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # one token through a square projection: the latency of a single small read of weights
        {"name": "linear_token_f16", "op": "linear", "type": "float16", "weights": "float16", "m": 1, "k": 4096, "n": 4096, "act": "silu",
         "bias": False, "residual": False, "gap": 0},
        # a batch of tokens being generated, quantized weights: the bytes of the weights are the time
        {"name": "linear_batch_i8", "op": "linear", "type": "float16", "weights": "int8", "m": 24, "k": 4096, "n": 16384, "act": "gelu",
         "bias": True, "residual": False, "gap": 0},
        # a prompt through a feed-forward layer's first product: the matrix cores are the time
        {"name": "linear_prompt_f16", "op": "linear", "type": "float16", "weights": "float16", "m": 4096, "k": 4096, "n": 16384, "act": "gelu",
         "bias": True, "residual": False, "gap": 0},
        # odd extents everywhere, in float32: an encoder's layer whose rows are not whole vectors
        {"name": "linear_ragged_f32", "op": "linear", "type": "float32", "weights": "float32", "m": 197, "k": 770, "n": 1001, "act": "relu",
         "bias": True, "residual": True, "gap": 0},
        # a few tokens being generated, most experts with a row or two
        {"name": "experts_tokens", "op": "experts", "type": "float16", "weights": "float16", "tokens": 16, "experts": 64, "top": 8, "k": 2048, "n": 1536,
         "act": "silu", "bias": False, "fanned": True},
        # a prompt, the experts unevenly loaded, the layer's second product
        {"name": "experts_prompt", "op": "experts", "type": "float16", "weights": "float16", "tokens": 4096, "experts": 32, "top": 4, "k": 4096, "n": 2048,
         "act": "", "bias": True, "fanned": False},
        # the routing of a few tokens: latency
        {"name": "routing_tokens", "op": "routing", "type": "float32", "tokens": 16, "experts": 256, "top": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_best": 2, "normalize": True},
        # a prompt's
        {"name": "routing_prompt", "op": "routing", "type": "float16", "tokens": 8192, "experts": 128, "top": 6, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_best": 1, "normalize": True},
        # the sums behind the experts' second product, of a few tokens and of a prompt
        {"name": "combine_tokens", "op": "combine", "type": "float16", "tokens": 16, "top": 8, "n": 2048, "residual": True},
        {"name": "combine_prompt", "op": "combine", "type": "float16", "tokens": 8192, "top": 4, "n": 4096, "residual": True},
        # what a server reports for each generated token: few rows, a large vocabulary, so that each row is split
        {"name": "logprobs_tokens", "op": "logprobs", "type": "float32", "rows": 6, "vocabulary": 100003, "top": 20},
        # the scores of a whole text under a model
        {"name": "logprobs_text", "op": "logprobs", "type": "float16", "rows": 4096, "vocabulary": 65536, "top": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng, lo, hi, whole):
    """A size between lo and hi: any, or (two times of three) a multiple of `whole`."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 1 / 3 else max(whole, v // whole * whole)


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "experts", "routing", "combine", "logprobs", "logprobs"])
    if op == "linear":
        kind, weights = rng.choice([("float16", "float16"), ("float16", "float16"), ("float16", "int8"), ("float32", "float32")])
        m, k, n = _log(rng, 1, 8192), _shape(rng, 48, 12288, 64), _shape(rng, 48, 20480, 32)
        most = 2 ** 38 if kind == "float16" else 2 ** 35  # multiply-adds
        m = max(1, min(m, most // (k * n)))
        return {"op": op, "type": kind, "weights": weights, "m": m, "k": k, "n": n, "act": rng.choice(["", "relu", "gelu", "gelu_tanh", "silu"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "gap": rng.choice([0, 0, 8, 5])}
    if op == "experts":
        kind, weights = rng.choice([("float16", "float16"), ("float16", "float16"), ("float16", "int8"), ("float32", "float32")])
        e = rng.choice([4, 8, 16, 32, 60, 64, 128])
        top = rng.choice([1, 2, 4, 6, 8] if e > 8 else [1, 2])
        k, n = _shape(rng, 64, 4096, 64), _shape(rng, 64, 4096, 32)
        while e * k * n > 2 ** 29:
            e //= 2
        top = min(top, e)
        most = 2 ** 37 if kind == "float16" else 2 ** 34
        t = max(1, min(_log(rng, 1, 4096), most // (top * k * n)))
        return {"op": op, "type": kind, "weights": weights, "tokens": t, "experts": e, "top": top, "k": k, "n": n,
                "act": rng.choice(["", "relu", "gelu", "silu"]), "bias": rng.random() < 0.5, "fanned": rng.random() < 0.5}
    if op == "routing":
        e = rng.choice([8, 16, 60, 64, 128, 160, 256, 384, 512])
        groups = rng.choice([1, 1, 4, 8] if e > 8 else [1, 4])
        groups = 1 if e % groups else groups
        top_groups = rng.randint(max(1, groups // 2), groups)
        top = rng.randint(1, min(12, top_groups * (e // groups)))
        return {"op": op, "type": rng.choice(["float16", "float32"]), "tokens": _log(rng, 1, 8192), "experts": e, "top": top,
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_best": rng.choice([1, 2]) if e // groups > 1 else 1, "normalize": rng.random() < 0.7}
    if op == "combine":
        top = rng.choice([1, 2, 4, 6, 8])
        n = _shape(rng, 64, 8192, 64)
        return {"op": op, "type": rng.choice(["float16", "float32"]), "tokens": max(1, min(_log(rng, 1, 16384), 2 ** 26 // (top * n))), "top": top, "n": n,
                "residual": rng.random() < 0.5}
    v = _log(rng, 1, 200000)
    return {"op": op, "type": rng.choice(["float16", "float32"]), "rows": max(1, min(_log(rng, 1, 8192), 2 ** 27 // v)), "vocabulary": v,
            "top": min(v, rng.choice([0, 1, 5, 20, 40]))}


# ---- inputs -------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _weights(g, c, lead=()):
    """(w [.., n, k], w_scale [.., n] or None, b [.., n] or None): outputs of about 1."""
    n, k = c["n"], c["k"]
    scale = None
    if c["weights"] == "int8":
        w = torch.randint(-127, 128, lead + (n, k), generator=g, device="cuda", dtype=torch.int8)
        scale = (torch.rand(lead + (n,), generator=g, device="cuda") + 0.5) / (73.0 * math.sqrt(k))
    else:
        w = _normal(g, lead + (n, k), _TYPES[c["weights"]], 1.0 / math.sqrt(k))
    return w, scale, _normal(g, lead + (n,), _TYPES[c["type"]], 0.5) if c["bias"] else None


def _routed(g, tokens, experts, top):
    """(order [tokens * top], offsets [experts + 1]) of a routing in which some experts are asked for far more often than others."""
    liked = torch.randn(experts, generator=g, device="cuda")
    chosen = (torch.randn((tokens, experts), generator=g, device="cuda") + 0.7 * liked).topk(top, dim=1).indices.reshape(-1)
    order = torch.sort(chosen, stable=True).indices
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.bincount(chosen, minlength=experts).cumsum(0)
    return order.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g, c = _generator(seed), case
    kind = _TYPES[c["type"]]
    if c["op"] == "linear":
        s = {"x": _normal(g, (c["m"], c["k"] + c["gap"]), kind)[:, : c["k"]]}
        s["w"], s["scale"], s["b"] = _weights(g, c)
        s["r"] = _normal(g, (c["m"], c["n"]), kind) if c["residual"] else None
    elif c["op"] == "experts":
        s = {"x": _normal(g, (c["tokens"] * (1 if c["fanned"] else c["top"]), c["k"]), kind)}
        s["w"], s["scale"], s["b"] = _weights(g, c, (c["experts"],))
        s["order"], s["offsets"] = _routed(g, c["tokens"], c["experts"], c["top"])
        s["most"] = int(s["offsets"].diff().max())  # rows of the expert with the most: what the plain form's batch is as high as
    elif c["op"] == "routing":
        s = {"logits": _normal(g, (c["tokens"], c["experts"]), kind, 1.5)}
        s["bias"] = torch.randn(c["experts"], generator=g, device="cuda") * 0.05 if c["bias"] else None
    elif c["op"] == "combine":
        s = {"x": _normal(g, (c["tokens"] * c["top"], c["n"]), kind)}
        s["weights"] = torch.softmax(torch.randn((c["tokens"], c["top"]), generator=g, device="cuda"), dim=1)
        s["r"] = _normal(g, (c["tokens"], c["n"]), kind) if c["residual"] else None
    else:
        rows, v = c["rows"], c["vocabulary"]
        s = {"logits": _normal(g, (rows, v), kind, 2.5)}
        s["tokens"] = torch.randint(0, v, (rows,), generator=g, device="cuda")
        if rows > 2 and v > 8:
            s["logits"][1, torch.rand(v, generator=g, device="cuda") < 0.9] = -math.inf  # a row that a grammar leaves few tokens
            s["logits"][1, s["tokens"][1]] = 1.0
            s["tokens"][2] = -1  # a place without a token
    s["case"] = dict(case)
    if own and "w" in s:  # the layer's weights, laid out once when a program loads them
        s["plan"] = _ops().LinearPlan(s["w"], b=s["b"], w_scale=s["scale"])
    return s


# ---- one pass -----------------------------------------------------------------------------------

def _act(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _linear(s):
    c, x = s["case"], s["x"]
    if own:
        return s["plan"].run(x, activation=c["act"], r=s["r"])
    v = x.float() @ s["w"].float().t()
    if s["scale"] is not None:
        v = v * s["scale"]
    if s["b"] is not None:
        v = v + s["b"].float()
    v = _act(v, c["act"])
    return (v if s["r"] is None else v + s["r"].float()).to(x.dtype)


def _experts(s):
    c, x = s["case"], s["x"]
    if own:
        return s["plan"].run_experts(x, s["order"], s["offsets"], activation=c["act"])
    # every expert's rows, as many as the fullest has; places behind an expert's last one go to a row that is dropped
    total = c["tokens"] * c["top"]
    begin, end = s["offsets"][:-1, None].long(), s["offsets"][1:, None].long()
    at = begin + torch.arange(s["most"], device=x.device)
    row = torch.where(at < end, s["order"].long()[at.clamp(max=total - 1)], total)
    source = row.clamp(max=total - 1) // (total // x.shape[0])
    v = torch.bmm(x[source.reshape(-1)].float().reshape(c["experts"], -1, c["k"]), s["w"].float().transpose(1, 2).contiguous())
    if s["scale"] is not None:
        v = v * s["scale"][:, None]
    if s["b"] is not None:
        v = v + s["b"].float()[:, None]
    y = torch.empty((total + 1, c["n"]), dtype=x.dtype, device=x.device)
    y[row.reshape(-1)] = _act(v, c["act"]).to(x.dtype).reshape(-1, c["n"])
    return y[:total]


def _routing(s):
    c, logits = s["case"], s["logits"]
    if own:
        return _ops().ExpertRouting(logits, c["top"], bias=s["bias"], score=c["score"], groups=c["groups"], top_groups=c["top_groups"],
                                    group_best=c["group_best"], normalize=c["normalize"], scale=1.5)
    # (64 bits: the choice is between values that may differ in the last of 32)
    t, e, x = c["tokens"], c["experts"], logits.double()
    score = torch.softmax(x, dim=1) if c["score"] == "softmax" else 1 / (1 + torch.exp(-x))
    key = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        of_group = torch.sort(key.reshape(t, c["groups"], -1), dim=2, descending=True).values[:, :, : c["group_best"]].sum(2)
        best = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        taken = torch.zeros((t, c["groups"]), dtype=torch.bool, device=x.device).scatter_(1, best, True)
        key = torch.where(taken.repeat_interleave(e // c["groups"], dim=1), key, -math.inf)
    experts = torch.sort(key, dim=1, descending=True, stable=True).indices[:, : c["top"]]
    weights = score.gather(1, experts)
    if c["normalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    flat = experts.reshape(-1)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=x.device)
    offsets[1:] = (flat[:, None] == torch.arange(e, device=x.device)).sum(0).cumsum(0)
    return experts.to(torch.int32), (1.5 * weights).float(), torch.sort(flat, stable=True).indices.to(torch.int32), offsets


def _combine(s):
    c, x = s["case"], s["x"]
    if own:
        return _ops().ExpertCombine(x, s["weights"], r=s["r"])
    v = (x.reshape(c["tokens"], c["top"], -1).float() * s["weights"][:, :, None]).sum(1)
    return (v if s["r"] is None else v + s["r"].float()).to(x.dtype)


def _logprobs(s):
    c, logits, tokens = s["case"], s["logits"], s["tokens"]
    if own:
        return _ops().TokenLogProbs(logits, tokens, top=c["top"])
    x = logits.float()
    d = x - x.max(dim=1, keepdim=True).values
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logp = d - torch.log(total)
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, d * e, 0.0).sum(1) / total[:, 0]
    given = torch.where(tokens < 0, 0.0, logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0])
    best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : c["top"]]
    return given, entropy, logp.gather(1, best), best


def run(state):
    return {"linear": _linear, "experts": _experts, "routing": _routing, "combine": _combine, "logprobs": _logprobs}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] in ("linear", "experts"):
        root = math.sqrt(2.0)
        acts = {"": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.erfc(-v / root) / 2,
                "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}
        scale = 1.0 if s["scale"] is None else s["scale"].double()[..., None, :]
        bias = 0.0 if s["b"] is None else s["b"].double()[..., None, :]
    if c["op"] == "linear":
        y = acts[c["act"]](torch.mm(s["x"].double(), s["w"].double().T) * scale + bias)
        return y if s["r"] is None else y + s["r"].double()
    if c["op"] == "experts":
        total = c["tokens"] * c["top"]
        y = torch.zeros((total, c["n"]), dtype=torch.float64, device="cuda")
        bounds, per = s["offsets"].tolist(), total // s["x"].shape[0]
        for e in range(c["experts"]):
            rows = s["order"][bounds[e] : bounds[e + 1]].long()
            v = torch.mm(s["x"][rows // per].double(), s["w"][e].double().T)
            y[rows] = acts[c["act"]](v * (1.0 if s["scale"] is None else scale[e]) + (0.0 if s["b"] is None else bias[e]))
        return y
    if c["op"] == "routing":
        x = s["logits"].double().cpu()
        p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)) if c["score"] == "softmax" else torch.sigmoid(x)
        key = p + (0.0 if s["bias"] is None else s["bias"].double().cpu())
        if c["groups"] > 1:
            each = key.view(c["tokens"], c["groups"], -1)
            rank = each.topk(c["group_best"], dim=2).values.sum(2).argsort(dim=1, descending=True, stable=True).argsort(dim=1)
            key = each.masked_fill((rank >= c["top_groups"])[:, :, None], -math.inf).flatten(1)
        experts = key.argsort(dim=1, descending=True, stable=True)[:, : c["top"]]
        w = p.gather(1, experts)
        w = 1.5 * w / w.sum(1, keepdim=True) if c["normalize"] else 1.5 * w
        return None, w, None, None
    if c["op"] == "combine":
        y = torch.bmm(s["weights"].double()[:, None], s["x"].double().view(c["tokens"], c["top"], -1))[:, 0]
        return y if s["r"] is None else y + s["r"].double()
    given, entropy, top = [], [], []
    for rows, tokens in zip(s["logits"].split(256), s["tokens"].split(256)):
        logp = torch.log_softmax(rows.double(), dim=1)
        given.append(torch.where(tokens < 0, torch.zeros((), dtype=torch.float64, device="cuda"), logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]))
        entropy.append(torch.special.entr(torch.exp(logp)).sum(1))
        top.append(logp.topk(c["top"], dim=1).values)
    return torch.cat(given), torch.cat(entropy), torch.cat(top), None


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    c = case
    size = 2 if c["type"] == "float16" else 4
    if c["op"] in ("linear", "experts"):
        m = c["m"] if c["op"] == "linear" else c["tokens"] * c["top"]
        rows = m if c["op"] == "linear" or not c["fanned"] else c["tokens"]
        # an expert that no row is sent to is not read: rows * (1 - (1 - 1 / experts) ^ rows) of them are, where all are asked for alike
        e = 1 if c["op"] == "linear" else c["experts"] * (1 - (1 - 1 / c["experts"]) ** m)
        per = c["k"] * (1 if c["weights"] == "int8" else size) + (4 if c["weights"] == "int8" else 0) + (size if c["bias"] else 0)
        more = (m * c["n"] * size if c.get("residual") else 0) + (4 * m + 4 * c["experts"] if c["op"] == "experts" else 0)
        return {"bytes": rows * c["k"] * size + e * c["n"] * per + m * c["n"] * size + more, "flops": 2 * m * c["n"] * c["k"]}
    if c["op"] == "routing":
        t, e, k = c["tokens"], c["experts"], c["top"]
        return {"bytes": t * e * size + 12 * t * k + 4 * (e + 1) + (4 * e if c["bias"] else 0), "flops": 8 * t * e}
    if c["op"] == "combine":
        t, k, n = c["tokens"], c["top"], c["n"]
        return {"bytes": t * n * size * (k + 1 + (1 if c["residual"] else 0)) + 4 * t * k, "flops": 2 * t * k * n}
    r, v = c["rows"], c["vocabulary"]
    return {"bytes": r * v * size + r * (16 + 12 * c["top"]), "flops": 6 * r * v}
