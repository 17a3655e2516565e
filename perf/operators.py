"""Operators of a decoder block, as cases that can be timed and checked.

Three operators, each in the forms in which a block of ``dccl_b200.models`` meets it:

``norm``    ``residual_norm``: the residual add at the end of one sub-block (the sub-block's own norm, a gate and a scale with it
            where the case has them) together with the norm at the entry of the next.
``rotary``  ``rotary``: queries and keys turned by angles that grow with the position, halves or neighbours paired, the whole head
            or part of it.
``gated``   ``gated_linear``: act(x Wg^T) * (x Wu^T), the two projections of a gated feed-forward layer.

A case with ``"backward": True`` is a training step of the operator: its outputs and the gradients of all its inputs from
given gradients of the outputs. The others are calls for inference.
"""
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
EPS = 1e-5
HIDDEN, FFN, HEADS, KV_HEADS, HEAD = 2048, 5632, 32, 4, 64      # the decoder of the training benchmark
TOKENS = 8 * 2048                                               # its micro-batch


def listed():
    return [
        # eight sequences take one decoding step through the end of a sub-block: latency is everything
        {"name": "norm_step", "kind": "norm", "batch": 8, "seq": 1, "width": HIDDEN, "dtype": "bfloat16", "post": False, "gate": "none", "scale": 1.0, "backward": False},
        # the micro-batch of the training benchmark
        {"name": "norm_train", "kind": "norm", "batch": 8, "seq": 2048, "width": HIDDEN, "dtype": "bfloat16", "post": False, "gate": "none", "scale": 1.0, "backward": True},
        # a short ragged batch in fp16, norms on both sides of the sub-block, a gate per sequence, a residual scale, an odd width
        {"name": "norm_ragged", "kind": "norm", "batch": 3, "seq": 517, "width": 1451, "dtype": "float16", "post": True, "gate": "sequence", "scale": 0.7071, "backward": True},
        # a wide model: norms on both sides and a gate per channel
        {"name": "norm_wide", "kind": "norm", "batch": 2, "seq": 4096, "width": 8192, "dtype": "bfloat16", "post": True, "gate": "channel", "scale": 0.5, "backward": True},
        # sixteen sequences of different lengths take one decoding step, far into a context that was stretched eightfold
        {"name": "rotary_step", "kind": "rotary", "batch": 16, "seq": 1, "heads": HEADS, "kv_heads": KV_HEADS, "head": HEAD, "rotary": HEAD, "interleaved": False,
         "dtype": "bfloat16", "furthest": 131072, "stretch": 8.0, "backward": False},
        # queries and keys of the training benchmark's micro-batch
        {"name": "rotary_train", "kind": "rotary", "batch": 8, "seq": 2048, "heads": HEADS, "kv_heads": KV_HEADS, "head": HEAD, "rotary": HEAD, "interleaved": False,
         "dtype": "bfloat16", "furthest": 2048, "stretch": 1.0, "backward": True},
        # documents packed into one odd-length row, fp32, neighbours paired over less than half of the head
        {"name": "rotary_packed", "kind": "rotary", "batch": 1, "seq": 5003, "heads": 12, "kv_heads": 12, "head": 80, "rotary": 34, "interleaved": True,
         "dtype": "float32", "furthest": 1000000, "stretch": 4.0, "backward": True},
        # one token of one sequence: the weights are read once and that is the time
        {"name": "gated_token", "kind": "gated", "tokens": 1, "width": HIDDEN, "ffn": FFN, "act": "silu", "dtype": "bfloat16", "backward": False},
        # a decoding step of a batch of forty sequences
        {"name": "gated_batch", "kind": "gated", "tokens": 40, "width": HIDDEN, "ffn": FFN, "act": "silu", "dtype": "bfloat16", "backward": False},
        # a prompt of 2000 tokens
        {"name": "gated_prompt", "kind": "gated", "tokens": 2000, "width": HIDDEN, "ffn": FFN, "act": "silu", "dtype": "bfloat16", "backward": False},
        # a small fp16 model of odd sizes, no row of its weights on a 16-byte boundary, gelu
        {"name": "gated_odd", "kind": "gated", "tokens": 777, "width": 1001, "ffn": 2731, "act": "gelu", "dtype": "float16", "backward": True},
        # the micro-batch of the training benchmark
        {"name": "gated_train", "kind": "gated", "tokens": TOKENS, "width": HIDDEN, "ffn": FFN, "act": "silu", "dtype": "bfloat16", "backward": True},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "gated"])
    if kind == "norm":
        batch, width = rng.choice([1, 2, 3, 8, 31]), rng.choice([_spread(rng, 33, 8192), 8 * _spread(rng, 8, 1024)])
        seq = _spread(rng, 1, max(1, min(4096, (1 << 26) // (width * batch))))
        return {"kind": kind, "batch": batch, "seq": seq, "width": width, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "channel", "sequence"]), "scale": rng.choice([1.0, 0.5, 0.125]), "backward": rng.random() < 0.6}
    if kind == "rotary":
        head = rng.choice([32, 64, 80, 128, 256, 2 * rng.randrange(5, 65)])
        rotary = rng.choice([head, head, 2 * rng.randrange(1, head // 2 + 1)])
        kv = rng.choice([1, 2, 4, 8])
        heads, batch = kv * rng.choice([1, 2, 8]), rng.choice([1, 2, 5, 16])
        seq = _spread(rng, 1, max(1, min(8192, (1 << 25) // (batch * (heads + kv) * head))))
        return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv, "head": head, "rotary": rotary, "interleaved": rng.random() < 0.5,
                "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "furthest": max(seq, _spread(rng, 1000, 1000000)),
                "stretch": rng.choice([1.0, 4.0, 32.0]), "backward": rng.random() < 0.5}
    width, ffn = rng.choice([_spread(rng, 40, 4096), 8 * _spread(rng, 8, 512)]), rng.choice([_spread(rng, 40, 12288), 8 * _spread(rng, 8, 1536)])
    most = max(1, min(TOKENS, TOKENS * HIDDEN * FFN // (width * ffn)))
    return {"kind": kind, "tokens": _spread(rng, 1, most), "width": width, "ffn": ffn, "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh"]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16"]), "backward": rng.random() < 0.5}


def _frequencies(case, device):
    """Radians per position of each pair: geometric, and where the context was stretched the slow ones (fewer than one turn in
    the original length) are slowed by that much, the fast ones kept, those between mixed."""
    pairs = case["rotary"] // 2
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    turns = f * (case["furthest"] / case["stretch"]) / (2 * math.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    return f * (keep + (1 - keep) / case["stretch"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32) * std).to(dtype)

    s = {"case": case}
    if case["kind"] == "norm":
        b, n, w = case["batch"], case["seq"], case["width"]
        # a residual stream has a few channels that are much larger than the others
        loud = 1 + 15 * (torch.rand(w, device="cuda", generator=gen) < 0.01).float()
        s["x"] = (torch.randn((b, n, w), device="cuda", generator=gen) * loud).to(dtype)
        s["branch"] = randn(b, n, w, std=0.5)
        s["weight"] = (1 + 0.1 * torch.randn(w, device="cuda", generator=gen)).to(dtype)
        s["post"] = (1 + 0.1 * torch.randn(w, device="cuda", generator=gen)).to(dtype) if case["post"] else None
        s["gate"] = {"none": lambda: None, "channel": lambda: randn(w, std=0.5), "sequence": lambda: randn(b, 1, w, std=0.5)}[case["gate"]]()
        leaves = ["x", "branch", "weight", "post", "gate"]
        if case["backward"]:
            s["dy"], s["dn"] = randn(b, n, w, std=0.02), randn(b, n, w, std=0.02)
    elif case["kind"] == "rotary":
        b, n = case["batch"], case["seq"]
        s["q"], s["k"] = randn(b, n, case["heads"], case["head"]), randn(b, n, case["kv_heads"], case["head"])
        s["freqs"] = _frequencies(case, "cuda")
        # every sequence (for a step) or every document (packed into a row) has its own place
        start = torch.randint(0, case["furthest"] - n + 1, (b, 1), device="cuda", generator=gen)
        s["positions"] = start + torch.arange(n, device="cuda")
        leaves = ["q", "k"]
        if case["backward"]:
            s["dq"], s["dk"] = randn(b, n, case["heads"], case["head"], std=0.02), randn(b, n, case["kv_heads"], case["head"], std=0.02)
    else:
        t, w, f = case["tokens"], case["width"], case["ffn"]
        s["x"] = randn(t, w)
        s["w_gate"], s["w_up"] = randn(f, w, std=1 / math.sqrt(w)), randn(f, w, std=1 / math.sqrt(w))
        leaves = ["x", "w_gate", "w_up"]
        if case["backward"]:
            s["dh"] = randn(t, f, std=0.02)
    if case["backward"]:
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _norm_own(s):
    from dccl_b200 import ops
    c = s["case"]
    y, n = ops.residual_norm(s["x"], s["branch"], s["weight"], eps=EPS, post_weight=s["post"], gate=s["gate"], scale=c["scale"])
    if not c["backward"]:
        return {"y": y, "n": n}
    names = [k for k in ("x", "branch", "weight", "post", "gate") if s[k] is not None]
    grads = torch.autograd.grad((y, n), [s[k] for k in names], (s["dy"], s["dn"]))
    return {"y": y, "n": n, **{"d" + k: g for k, g in zip(names, grads)}}


def _norm_plain(s):
    c = s["case"]
    with torch.no_grad():
        x, b, w = s["x"].float(), s["branch"].float(), s["weight"].float()
        gate = s["gate"].float() if s["gate"] is not None else None
        p = b
        if s["post"] is not None:
            w2 = s["post"].float()
            rb = torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS)
            p = b * rb * w2
        y = x + c["scale"] * (p if gate is None else gate * p)
        ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        yh = y * ry
        out = {"y": y.to(s["x"].dtype), "n": (yh * w).to(s["x"].dtype)}
        if c["backward"]:
            dn = s["dn"].float()
            out["dweight"] = (dn * yh).sum((0, 1)).to(s["weight"].dtype)
            t = dn * w
            dy = s["dy"].float() + ry * (t - yh * (t * yh).mean(-1, keepdim=True))
            out["dx"] = dy.to(s["x"].dtype)
            dp = c["scale"] * dy
            if gate is not None:
                out["dgate"] = (dp * p).sum((0, 1) if c["gate"] == "channel" else 1).reshape(s["gate"].shape).to(s["gate"].dtype)
                dp = dp * gate
            if s["post"] is not None:
                bh = b * rb
                out["dpost"] = (dp * bh).sum((0, 1)).to(s["post"].dtype)
                u = dp * w2
                dp = rb * (u - bh * (u * bh).mean(-1, keepdim=True))
            out["dbranch"] = dp.to(s["x"].dtype)
        return out


def _rotary_own(s):
    from dccl_b200 import ops
    c = s["case"]
    q, k = ops.rotary(s["q"], s["k"], s["freqs"], positions=s["positions"], interleaved=c["interleaved"])
    if not c["backward"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _turn(x, cos, sin, interleaved):
    r, v = 2 * cos.shape[-1], x.float()
    if interleaved:
        a, b = v[..., 0:r:2], v[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = v[..., :r // 2], v[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, v[..., r:]), -1).to(x.dtype)


def _rotary_plain(s):
    c = s["case"]
    with torch.no_grad():
        # 64 bits: an angle of a million radians has no digit behind the point to spare in 32
        angle = (s["positions"].double().unsqueeze(-1) * s["freqs"]).unsqueeze(2)
        cos, sin = angle.cos().float(), angle.sin().float()
        out = {"q": _turn(s["q"], cos, sin, c["interleaved"]), "k": _turn(s["k"], cos, sin, c["interleaved"])}
        if c["backward"]:
            out["dq"], out["dk"] = _turn(s["dq"], cos, -sin, c["interleaved"]), _turn(s["dk"], cos, -sin, c["interleaved"])
        return out


def _gated_own(s):
    from dccl_b200 import ops
    c = s["case"]
    h = ops.gated_linear(s["x"], s["w_gate"], s["w_up"], activation=c["act"])
    if not c["backward"]:
        return {"h": h}
    dx, dg, du = torch.autograd.grad(h, (s["x"], s["w_gate"], s["w_up"]), s["dh"])
    return {"h": h, "dx": dx, "dw_gate": dg, "dw_up": du}


def _act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        e = 1 / (1 + torch.exp(-g))
        return g * e, e * (1 + g * (1 - e))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _gated_plain(s):
    c, dtype = s["case"], s["x"].dtype
    with torch.no_grad():
        x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
        g, u = x @ wg.t(), x @ wu.t()
        a, da = _act(g, c["act"])
        out = {"h": (a * u).to(dtype)}
        if c["backward"]:
            dh = s["dh"].float()
            dg, du = dh * u * da, dh * a
            out["dx"] = (dg @ wg + du @ wu).to(dtype)
            out["dw_gate"], out["dw_up"] = (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)
        return out


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"norm": _norm_own, "rotary": _rotary_own, "gated": _gated_own}[kind](s)
    return {"norm": _norm_plain, "rotary": _rotary_plain, "gated": _gated_plain}[kind](s)


def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor)}
    if case["backward"]:
        for k, t in s.items():
            if isinstance(t, torch.Tensor) and t.requires_grad:
                v[k].requires_grad_(True)
    if case["kind"] == "norm":
        rms = lambda t: t / ((t ** 2).sum(-1, keepdim=True) / case["width"] + EPS).sqrt()  # noqa: E731
        inner = rms(v["branch"]) * v["post"] if "post" in v else v["branch"]
        y = v["x"] + inner * v.get("gate", 1.0) * case["scale"]
        outs, given = {"y": y, "n": rms(y) * v["weight"]}, ("dy", "dn")
    elif case["kind"] == "rotary":
        spin = torch.polar(torch.ones_like(v["freqs"]), v["freqs"] * v["positions"].unsqueeze(-1)).unsqueeze(2)
        r = case["rotary"]

        def turn(t):
            pair = t[..., :r].unflatten(-1, (r // 2, 2) if case["interleaved"] else (2, r // 2))
            pair = pair if case["interleaved"] else pair.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * spin)
            return torch.cat(((z if case["interleaved"] else z.transpose(-1, -2)).reshape(*t.shape[:-1], r), t[..., r:]), -1)

        outs, given = {"q": turn(v["q"]), "k": turn(v["k"])}, ("dq", "dk")
    else:
        g, u = torch.nn.functional.linear(v["x"], v["w_gate"]), torch.nn.functional.linear(v["x"], v["w_up"])
        if case["act"] == "silu":
            a = g * torch.sigmoid(g)
        elif case["act"] == "gelu":
            a = g * torch.special.ndtr(g)
        else:
            a = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        outs, given = {"h": a * u}, ("dh",)
    if case["backward"]:
        names = [k for k, t in v.items() if t.requires_grad]
        grads = torch.autograd.grad(list(outs.values()), [v[k] for k in names], [v[k] for k in given])
        outs.update({"d" + k: g for k, g in zip(names, grads)})
    return {k: t.detach() for k, t in outs.items()}


def work(case):
    """Each input read once, each output written once. A forward and a backward pass, called one after the other, need the inputs of the
    second too; what the first could leave to it does not count."""
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    if case["kind"] == "norm":
        elements = case["batch"] * case["seq"] * case["width"]
        vectors = case["width"] * (1 + case["post"] + {"none": 0, "channel": 1, "sequence": case["batch"]}[case["gate"]])
        arrays, flops = (8, 30) if case["backward"] else (4, 8)
        return {"bytes": size * (arrays * elements + vectors * (2 if case["backward"] else 1)), "flops": flops * elements}
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["seq"]
        elements = tokens * (case["heads"] + case["kv_heads"]) * case["head"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * 2 * size * elements + 8 * tokens + 4 * case["rotary"], "flops": passes * 3 * elements}
    t, w, f = case["tokens"], case["width"], case["ffn"]
    if case["backward"]:
        return {"bytes": size * (2 * t * w + 4 * f * w + 2 * t * f), "flops": 12 * t * w * f}
    return {"bytes": size * (t * w + 2 * f * w + t * f), "flops": 4 * t * w * f}
