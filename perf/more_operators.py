"""Operators of a training step with a mixture of experts, as cases that can be timed and checked.

``route``     ``route``: from a router's logits the experts of each token and their weights.
``exchange``  ``expert_plan``, ``dispatch`` and ``combine``: tokens copied to rows in the order of the experts, and the experts' results
              added up where the tokens came from.
``linear``    ``expert_linear``: a product of every expert's rows with that expert's weights, and its activation.
``clip``      ``clip_grad_norm``: the norm of all gradients of a model, and the gradients cut back to a limit.

A case with ``"backward": True`` is a training step of the operator: its outputs and the gradients of all its inputs from given
gradients of the outputs. The others are calls for inference, or have no gradient.
"""
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
HIDDEN, FFN, LAYERS, KV, VOCAB = 2048, 5632, 22, 256, 32000     # the decoder of the training benchmark
TOKENS = 8 * 2048                                               # its micro-batch


def listed():
    return [
        # eight sequences take one decoding step: latency is everything
        {"name": "route_step", "kind": "route", "tokens": 8, "experts": 64, "k": 6, "scores": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max",
         "renormalize": True, "scale": 1.0, "dtype": "float32", "padded": 0.0, "backward": False},
        # the training benchmark's micro-batch over many small experts: balanced by a bias, in groups that stand for ranks
        {"name": "route_train", "kind": "route", "tokens": TOKENS, "experts": 256, "k": 8, "scores": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2",
         "renormalize": True, "scale": 2.5, "dtype": "float32", "padded": 0.0, "backward": True},
        # a batch of odd size in fp16, a tenth of whose tokens are padding, no power of two of experts, weights as the softmax gives them
        {"name": "route_padded", "kind": "route", "tokens": 1021, "experts": 60, "k": 4, "scores": "softmax", "bias": True, "groups": 5, "top_groups": 3, "group_score": "max",
         "renormalize": False, "scale": 1.0, "dtype": "float16", "padded": 0.1, "backward": True},
        # the same decoding step between router and experts
        {"name": "exchange_step", "kind": "exchange", "tokens": 8, "k": 6, "experts": 64, "width": HIDDEN, "dtype": "bfloat16", "dropped": 0.0, "backward": False},
        # a short batch of odd sizes in fp16, a fifth of whose places no expert had room for
        {"name": "exchange_dropped", "kind": "exchange", "tokens": 1021, "k": 3, "experts": 11, "width": 1451, "dtype": "float16", "dropped": 0.2, "backward": True},
        # the micro-batch of the training benchmark
        {"name": "exchange_train", "kind": "exchange", "tokens": TOKENS, "k": 4, "experts": 64, "width": HIDDEN, "dtype": "bfloat16", "dropped": 0.0, "backward": True},
        # eight tokens with two experts each: the weights of the experts that anyone goes to are read once and that is the time
        {"name": "linear_step", "kind": "linear", "rows": 16, "experts": 8, "width": HIDDEN, "out": FFN, "act": "gelu", "dtype": "bfloat16", "dropped": 0.0, "backward": False},
        # a small fp16 model of odd sizes, no row of its weights on a 16-byte boundary, some rows of nobody
        {"name": "linear_odd", "kind": "linear", "rows": 777, "experts": 5, "width": 1001, "out": 2731, "act": "silu", "dtype": "float16", "dropped": 0.1, "backward": True},
        # the training benchmark's micro-batch through the first product of eight experts
        {"name": "linear_train", "kind": "linear", "rows": TOKENS, "experts": 8, "width": HIDDEN, "out": FFN, "act": "gelu", "dtype": "bfloat16", "dropped": 0.0, "backward": True},
        # gradients of the tests' decoder, cut back into the buffers that the optimizer reads: a few launches' latency
        {"name": "clip_tiny", "kind": "clip", "layers": 2, "hidden": 128, "kv": 64, "ffn": 256, "vocab": 512, "dtype": "bfloat16", "odd": False, "limited": True},
        # gradients in two types, places and sizes that no vector access likes, and a norm below the limit: nothing is written
        {"name": "clip_below", "kind": "clip", "layers": 3, "hidden": 517, "kv": 131, "ffn": 1451, "vocab": 8009, "dtype": "float16", "odd": True, "limited": False},
        # all gradients of the training benchmark's decoder
        {"name": "clip_train", "kind": "clip", "layers": LAYERS, "hidden": HIDDEN, "kv": KV, "ffn": FFN, "vocab": VOCAB, "dtype": "bfloat16", "odd": False, "limited": True},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "exchange", "linear", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "route":
        groups = rng.choice([1, 1, 1, 2, 4, 5, 8])
        experts = groups * _spread(rng, 4, 512 // groups)
        top = rng.randint(1, groups)
        k = rng.randint(1, min(12, top * (experts // groups)))
        return {"kind": kind, "tokens": _spread(rng, 1, min(TOKENS, (1 << 22) // experts)), "experts": experts, "k": k,
                "scores": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.6, "groups": groups, "top_groups": top, "group_score": rng.choice(["max", "top2"]),
                "renormalize": k > 1 and rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]),
                "padded": rng.choice([0.0, 0.0, 0.3]), "backward": rng.random() < 0.6}
    if kind == "exchange":
        experts, width = _spread(rng, 2, 256), rng.choice([_spread(rng, 33, 8192), 8 * _spread(rng, 8, 1024)])
        k = rng.randint(1, min(8, experts))
        return {"kind": kind, "tokens": _spread(rng, 1, max(1, min(TOKENS, (TOKENS * HIDDEN * 4) // (k * width)))), "k": k, "experts": experts, "width": width,
                "dtype": rng.choice([dtype, dtype, "float32"]), "dropped": rng.choice([0.0, 0.0, 0.2]), "backward": rng.random() < 0.6}
    if kind == "linear":
        experts = _spread(rng, 1, 64)
        width, out = rng.choice([_spread(rng, 40, 4096), 8 * _spread(rng, 8, 512)]), rng.choice([_spread(rng, 40, 6144), 8 * _spread(rng, 8, 768)])
        experts = max(1, min(experts, 8 * HIDDEN * FFN // (width * out)))
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(TOKENS, TOKENS * HIDDEN * FFN // (width * out)))), "experts": experts, "width": width, "out": out,
                "act": rng.choice(["none", "gelu", "silu", "gelu_tanh"]), "dtype": dtype, "dropped": rng.choice([0.0, 0.0, 0.1]), "backward": rng.random() < 0.5}
    hidden = rng.choice([_spread(rng, 64, HIDDEN), 64 * rng.randint(1, HIDDEN // 64)])
    return {"kind": kind, "layers": _spread(rng, 1, LAYERS), "hidden": hidden, "kv": max(1, hidden // rng.choice([1, 4, 8])), "ffn": _spread(rng, hidden, FFN), "vocab": _spread(rng, 256, VOCAB),
            "dtype": rng.choice([dtype, dtype, "float32"]) if hidden <= 1024 else dtype, "odd": rng.random() < 0.4, "limited": rng.random() < 0.7}


def _shapes(case):
    """The parameters of a decoder, in the order of its modules."""
    h, kv, f, v = case["hidden"], case["kv"], case["ffn"], case["vocab"]
    block = [(h,), (h,), (h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f)]
    return [(v, h)] + case["layers"] * block + [(h,), (v, h)]


def _places(case):
    """(shape, type, first element in the buffer of that type) of every gradient, and the sizes of the buffers."""
    places, ends, dtype = [], {}, TYPES[case["dtype"]]
    for i, shape in enumerate(_shapes(case)):
        t = torch.float32 if case["odd"] and len(shape) == 1 else dtype
        at = -(-ends.get(t, 0) // 8) * 8 + (i % 8 if case["odd"] else 0)
        places.append((shape, t, at))
        ends[t] = at + math.prod(shape)
    return places, ends


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def randn(*shape, std=1.0, dtype=dtype):
        return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    s = {"case": case}
    if case["kind"] == "route":
        t, e = case["tokens"], case["experts"]
        # some experts are liked better than others, by every token
        s["logits"] = (randn(t, e, std=1.5, dtype=torch.float32) + randn(e, std=0.5, dtype=torch.float32)).to(dtype)
        if case["padded"]:
            s["logits"][rand(t) < case["padded"]] = -math.inf
        s["bias"] = randn(e, std=0.05, dtype=torch.float32) if case["bias"] else None
        if case["backward"]:
            s["dweights"] = randn(t, case["k"], std=0.02, dtype=torch.float32)
            s["logits"].requires_grad_(True)
    elif case["kind"] in ("exchange", "linear"):
        tokens, k = (case["tokens"], case["k"]) if case["kind"] == "exchange" else (case["rows"], 1)
        liked = randn(case["experts"], std=0.7, dtype=torch.float32)
        chance = liked - torch.log(-torch.log(rand(tokens, case["experts"]) * (1 - 2e-7) + 1e-7))
        experts = chance.topk(k, -1).indices.int()
        if case["dropped"]:
            experts = torch.where(rand(tokens, k) < case["dropped"], torch.full_like(experts, -1), experts)
        if case["kind"] == "exchange":
            w = case["width"]
            s["experts"] = experts
            s["x"], s["done"] = randn(tokens, w), randn(tokens * k, w)
            s["weights"] = torch.softmax(randn(tokens, k, dtype=torch.float32), -1)
            leaves = ["x", "done", "weights"]
            if case["backward"]:
                s["drows"], s["dy"] = randn(tokens * k, w, std=0.02), randn(tokens, w, std=0.02)
        else:
            counts = (experts.reshape(-1, 1) == torch.arange(case["experts"], device="cuda")).sum(0).tolist()
            s["bounds"] = [sum(counts[:e]) for e in range(case["experts"] + 1)]
            s["starts"] = torch.tensor(s["bounds"], dtype=torch.int32, device="cuda")
            s["x"] = randn(tokens, case["width"])
            s["weight"] = randn(case["experts"], case["out"], case["width"], std=1 / math.sqrt(case["width"]))
            leaves = ["x", "weight"]
            if case["backward"]:
                s["dh"] = randn(tokens, case["out"], std=0.02)
        if case["backward"]:
            for name in leaves:
                s[name].requires_grad_(True)
    else:
        # gradients are views of flat buffers, one for each type, and differ a thousandfold in size from tensor to tensor; odd ones begin anywhere
        places, ends = _places(case)
        s["flat"] = {t: torch.zeros(n, device="cuda", dtype=t) for t, n in ends.items()}
        s["grads"] = [s["flat"][t][at:at + math.prod(shape)].view(shape) for shape, t, at in places]
        for i, g in enumerate(s["grads"]):
            g.copy_(randn(*g.shape, std=10.0 ** (-3 - 3 * (i % 5) / 4), dtype=torch.float32))
        if case["limited"]:
            s["flat_out"] = {t: torch.zeros_like(f) for t, f in s["flat"].items()}
            s["out"] = [s["flat_out"][t][at:at + math.prod(shape)].view(shape) for shape, t, at in places]
        else:
            s["flat_out"], s["out"] = s["flat"], None
        # a quarter of the norm, about: a fifth of the elements have most of it
        s["limit"] = 1e-4 * math.sqrt(sum(g.numel() for g in s["grads"])) if case["limited"] else 1e4
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls

def _route_own(s):
    from dccl_b200 import ops
    c = s["case"]
    weights, experts = ops.route(s["logits"], c["k"], scores=c["scores"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"], group_score=c["group_score"],
                                 renormalize=c["renormalize"], scale=c["scale"])
    if not c["backward"]:
        return {"weights": weights, "experts": experts}
    dlogits, = torch.autograd.grad(weights, s["logits"], s["dweights"])
    return {"weights": weights, "experts": experts, "dlogits": dlogits}


def _exchange_own(s):
    from dccl_b200 import ops
    c = s["case"]
    plan = ops.expert_plan(s["experts"], c["experts"])
    rows = ops.dispatch(s["x"], plan)
    y = ops.combine(s["done"], plan, s["weights"])
    out = {"counts": plan.counts, "places": plan.rows, "rows": rows, "y": y}
    if c["backward"]:
        out["dx"], out["ddone"], out["dweights"] = torch.autograd.grad((rows, y), (s["x"], s["done"], s["weights"]), (s["drows"], s["dy"]))
    return out


def _linear_own(s):
    from dccl_b200 import ops
    c = s["case"]
    h = ops.expert_linear(s["x"], s["weight"], s["starts"], activation=None if c["act"] == "none" else c["act"])
    if not c["backward"]:
        return {"h": h}
    dx, dw = torch.autograd.grad(h, (s["x"], s["weight"]), s["dh"])
    return {"h": h, "dx": dx, "dweight": dw}


def _clip_own(s):
    from dccl_b200 import ops
    norm = ops.clip_grad_norm(s["grads"], s["limit"], out=s["out"])
    return {"norm": norm, "grads": list(s["flat_out"].values())}


# ---------------------------------------------------------------------------------------------- the plain forms

def _route_plain(s):
    c, k = s["case"], s["case"]["k"]
    with torch.no_grad():
        z = s["logits"].float()
        t, e = z.shape
        # what is compared is held in 64 bits: of two scores that 32 cannot tell apart, one may be the better all the same
        z64 = s["logits"].double()
        open_ = z64 > -math.inf
        if s["bias"] is None and c["group_score"] == "max":
            score = z64                                             # both scores grow with the logit
        elif c["scores"] == "softmax":
            grown = torch.exp(z64 - torch.where(open_, z64, -math.inf).max(-1, keepdim=True).values.clamp(min=-1e300))
            score = grown / grown.sum(-1, keepdim=True)
        else:
            score = 1 / (1 + torch.exp(-z64))
        if s["bias"] is not None:
            score = score + s["bias"].double()
        score = torch.where(open_, score, -math.inf)
        if c["groups"] > 1:
            by_group = score.view(t, c["groups"], -1)
            best, at = by_group.max(-1)
            if c["group_score"] == "top2" and by_group.shape[-1] > 1:
                second = by_group.scatter(-1, at.unsqueeze(-1), -math.inf).max(-1).values
                best = best + torch.where(second > -math.inf, second, 0.0)
            kept = torch.zeros(t, c["groups"], dtype=torch.bool, device=z.device)
            for _ in range(c["top_groups"]):
                at = torch.where(kept, -math.inf, best).max(-1, keepdim=True).indices
                kept = kept.scatter(-1, at, True)
            score = torch.where(kept.unsqueeze(-1), by_group, -math.inf).view(t, e)
        experts = []
        for _ in range(k):
            value, at = score.max(-1, keepdim=True)
            experts.append(torch.where(value > -math.inf, at, -1))
            score = score.scatter(-1, at, -math.inf)
        experts = torch.cat(experts, -1)
        chosen = experts >= 0
        if c["scores"] == "softmax":
            grown = torch.exp(z - z.max(-1, keepdim=True).values.clamp(min=-1e30))
            p = grown / grown.sum(-1, keepdim=True).clamp(min=1e-30)
        else:
            p = 1 / (1 + torch.exp(-z))
        pc = torch.where(chosen, p.gather(-1, experts.clamp(min=0)), 0.0)
        share = pc / pc.sum(-1, keepdim=True).clamp(min=1e-30) if c["renormalize"] else pc
        out = {"weights": c["scale"] * share, "experts": experts.int()}
        if c["backward"]:
            g = torch.where(chosen, c["scale"] * s["dweights"], 0.0)
            if c["renormalize"]:
                d = share * (g - (g * share).sum(-1, keepdim=True))
                if c["scores"] == "sigmoid":
                    d = d * (1 - pc)
                dz = torch.zeros_like(z).scatter_add(-1, experts.clamp(min=0).long(), d)
            elif c["scores"] == "sigmoid":
                dz = torch.zeros_like(z).scatter_add(-1, experts.clamp(min=0).long(), g * pc * (1 - pc))
            else:
                full = torch.zeros_like(z).scatter_add(-1, experts.clamp(min=0).long(), g)
                dz = p * (full - (g * pc).sum(-1, keepdim=True))
            out["dlogits"] = dz.to(s["logits"].dtype)
        return out


def _exchange_plain(s):
    c = s["case"]
    tokens, k, e, w = c["tokens"], c["k"], c["experts"], c["width"]
    with torch.no_grad():
        dtype, flat = s["x"].dtype, s["experts"].reshape(-1)
        hit = flat.unsqueeze(-1) == torch.arange(e, device=flat.device)
        counts = hit.sum(0)
        starts = counts.cumsum(0) - counts
        before = torch.where(hit, hit.int().cumsum(0) - 1 + starts, 0).sum(-1)
        routed = flat >= 0
        places = torch.where(routed, before, -1)
        to, token = places[routed], torch.arange(tokens * k, device=flat.device)[routed] // k
        rows = torch.zeros(tokens * k, w, dtype=dtype, device=flat.device)
        rows[to] = s["x"][token]

        def at_tokens(r):       # [tokens, k, width] of the rows, zeros where there are none
            return torch.where(routed.unsqueeze(-1), r[before].float(), 0.0).view(tokens, k, w)

        done = at_tokens(s["done"])
        out = {"counts": counts.int(), "places": places.int().view(tokens, k), "rows": rows, "y": (done * s["weights"].unsqueeze(-1)).sum(1).to(dtype)}
        if c["backward"]:
            out["dx"] = at_tokens(s["drows"]).sum(1).to(dtype)
            dy = s["dy"].float()
            ddone = torch.zeros(tokens * k, w, dtype=dtype, device=flat.device)
            ddone[to] = (dy.unsqueeze(1) * s["weights"].unsqueeze(-1)).to(dtype).view(tokens * k, w)[routed]
            out["ddone"] = ddone
            out["dweights"] = (done * dy.unsqueeze(1)).sum(-1)
        return out


def _act(z, name):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def _linear_plain(s):
    c, dtype = s["case"], s["x"].dtype
    with torch.no_grad():
        h = torch.zeros(c["rows"], c["out"], dtype=dtype, device="cuda")
        out = {"h": h}
        if c["backward"]:
            out["dx"], out["dweight"] = torch.zeros_like(s["x"]), torch.zeros_like(s["weight"])
        for e in range(c["experts"]):
            mine = slice(s["bounds"][e], s["bounds"][e + 1])
            if mine.start == mine.stop:
                continue
            x, w = s["x"][mine].float(), s["weight"][e].float()
            a, da = _act(x @ w.t(), c["act"])
            h[mine] = a.to(dtype)
            if c["backward"]:
                dz = s["dh"][mine].float() * da
                out["dx"][mine], out["dweight"][e] = (dz @ w).to(dtype), (dz.t() @ x).to(dtype)
        return out


def _clip_plain(s):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        total = total + (g.double() * g.double()).sum()     # a billion squares: 64 bits
    norm = total.sqrt()
    factor = (s["limit"] / (norm + 1e-6)).clamp(max=1.0).float()
    for g, o in zip(s["grads"], s["out"] or s["grads"]):
        o.copy_(g.float() * factor)
    return {"norm": norm.float(), "grads": list(s["flat_out"].values())}


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"route": _route_own, "exchange": _exchange_own, "linear": _linear_own, "clip": _clip_own}[kind](s)
    return {"route": _route_plain, "exchange": _exchange_plain, "linear": _linear_plain, "clip": _clip_plain}[kind](s)


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits

def _best(score, n):
    """Indices of the n largest of each row, the largest first and of equal ones the first; -1 for those of minus infinity."""
    value, at = torch.sort(score, dim=-1, descending=True, stable=True)
    return torch.where(value[:, :n] > -math.inf, at[:, :n], -1)


def _route_exact(case, s):
    z = s["logits"].detach().double().requires_grad_(case["backward"])
    closed = torch.isneginf(z)
    empty = closed.all(-1, keepdim=True)
    p = torch.sigmoid(z) if case["scores"] == "sigmoid" else torch.softmax(z.masked_fill(empty, 0.0), -1)
    score = (p if s["bias"] is None else p + s["bias"].double()).detach()
    if s["bias"] is None and (case["groups"] == 1 or case["group_score"] == "max"):
        score = z.detach()
    score = score.masked_fill(closed, -math.inf)
    if case["groups"] > 1:
        g = score.unflatten(-1, (case["groups"], -1))
        top = torch.sort(g, dim=-1, descending=True).values[..., :1 if case["group_score"] == "max" else 2]
        of_group = torch.where(torch.isneginf(top), 0.0, top).sum(-1).masked_fill(torch.isneginf(top).all(-1), -math.inf)
        open_ = (_best(of_group, case["top_groups"]).unsqueeze(-1) == torch.arange(case["groups"], device=z.device)).any(1)
        score = g.masked_fill(~open_.unsqueeze(-1), -math.inf).flatten(1)
    experts = _best(score, case["k"])
    there = experts >= 0
    w = torch.where(there, torch.take_along_dim(p, experts.clamp(min=0), -1), 0.0)
    if case["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    w = w * case["scale"]
    out = {"weights": w.detach(), "experts": experts.int()}
    if case["backward"]:
        dz, = torch.autograd.grad(w, z, s["dweights"].double())
        out["dlogits"] = dz.masked_fill(closed, 0.0)
    return out


def _exchange_exact(case, s):
    flat = s["experts"].flatten().long()
    k, last = case["k"], case["experts"]
    order = torch.sort(torch.where(flat < 0, last, flat), stable=True).indices
    routed = order[:int((flat >= 0).sum())]
    places = torch.full_like(flat, -1)
    places[routed] = torch.arange(routed.numel(), device=flat.device)
    token, n = routed // k, routed.numel()
    out = {"counts": torch.bincount(flat[flat >= 0], minlength=last).int(), "places": places.int().view(-1, k)}
    x, done, weights = s["x"].detach().double(), s["done"].detach().double(), s["weights"].detach().double().flatten()
    rows = torch.zeros_like(done)
    rows[:n] = x[token]
    out["rows"] = rows
    out["y"] = torch.zeros_like(x).index_add_(0, token, done[:n] * weights[routed].unsqueeze(-1))
    if case["backward"]:
        dy = s["dy"].double()
        out["dx"] = torch.zeros_like(x).index_add_(0, token, s["drows"][:n].double())
        out["ddone"] = torch.zeros_like(done)
        out["ddone"][:n] = dy[token] * weights[routed].unsqueeze(-1)
        dw = torch.zeros_like(weights)
        dw[routed] = torch.einsum("nw,nw->n", done[:n], dy[token])
        out["dweights"] = dw.view(-1, k)
    return out


def _linear_exact(case, s):
    x, weight = s["x"].detach().double().requires_grad_(case["backward"]), s["weight"].detach().double().requires_grad_(case["backward"])
    sizes = [b - a for a, b in zip(s["bounds"], s["bounds"][1:])]
    parts = []
    for part, w in zip(x[:s["bounds"][-1]].split(sizes), weight):
        z = torch.nn.functional.linear(part, w)
        parts.append({"none": lambda v: v, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.ndtr(v),
                      "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}[case["act"]](z))
    h = torch.cat(parts + [x.new_zeros(case["rows"] - s["bounds"][-1], case["out"])])
    out = {"h": h.detach()}
    if case["backward"]:
        out["dx"], out["dweight"] = torch.autograd.grad(h, (x, weight), s["dh"].double())
    return out


def _clip_exact(case, s):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
    factor = min(1.0, s["limit"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"), "grads": [f.double() * factor for f in s["flat"].values()]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _route_exact, "exchange": _exchange_exact, "linear": _linear_exact, "clip": _clip_exact}[case["kind"]](case, s)


def work(case):
    """Each input read once, each output written once. A forward and a backward pass, called one after the other, need the inputs of the
    second too; what the first could leave to it does not count."""
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    if case["kind"] == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        moved = size * t * e * (2 if case["backward"] else 1) + 8 * t * k + (4 * t * k if case["backward"] else 0) + (4 * e if case["bias"] else 0)
        return {"bytes": moved, "flops": t * e * (12 if case["backward"] else 6)}
    if case["kind"] == "exchange":
        # forward: x, rows, done, y; backward: drows, dx, dy, ddone; places and weights beside them
        rows, tokens, w = case["tokens"] * case["k"], case["tokens"], case["width"]
        moved = size * w * 2 * (rows + tokens) + rows * 12 + 4 * case["experts"]
        if case["backward"]:
            moved += size * w * 2 * (rows + tokens) + rows * 4
        return {"bytes": moved, "flops": rows * w * (6 if case["backward"] else 2)}
    if case["kind"] == "linear":
        n, e, w, f = case["rows"], case["experts"], case["width"], case["out"]
        seen = e * (1 - (1 - 1 / e) ** n) if e > 1 else 1        # experts that any row goes to
        if case["backward"]:
            return {"bytes": int(size * (2 * n * w + (seen + e) * f * w + 2 * n * f)), "flops": 6 * n * w * f}
        return {"bytes": int(size * (n * w + seen * f * w + n * f)), "flops": 2 * n * w * f}
    elements = [(math.prod(shape), t.itemsize) for shape, t, _ in _places(case)[0]]
    return {"bytes": sum(n * b for n, b in elements) * (2 if case["limited"] else 1), "flops": sum(n for n, _ in elements) * (3 if case["limited"] else 2)}
