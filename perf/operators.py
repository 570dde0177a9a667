"""Operators around the matrix products of a decoder, as cases that can be timed and compared.

Four operators, each through the entry point that a user's program calls:

* ``rope``     ``ops.rope`` / ``ops.rope_`` with an ``ops.Rotary``: rotary positions in both pairings, of a part of the head,
  scaled for long contexts, at positions of the user's own;
* ``qk_norm``  ``ops.qk_norm_rope`` / ``ops.qk_norm_rope_``: the norm of every query and key head and the rotation in one pass;
* ``route``    ``ops.moe.route``: softmax or sigmoid scores, a bias for balance, groups of experts, weights of the chosen ones;
* ``clip``     ``ops.clip_grad_norm_``: the norm of all gradients and their clipping.

``listed()`` names twelve cases, ``draw(rng)`` gives more of the same ranges.  ``run`` takes the plain form in elementary
operations where ``own`` is false and the framework's calls where it is true; ``exact`` states the definition in 64 bits.
"""
import functools
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# The gradients of a decoder: GPT-2-XL and Llama-3-8B widths are the package's own configurations.
_GPT2_XL = dict(family="gpt2", d_model=1600, heads=25, kv_heads=25, ffn=6400, vocab=50257)
_LLAMA_8B = dict(family="llama", d_model=4096, heads=32, kv_heads=8, ffn=14336, vocab=128256)


def listed():
    return [
        # one new token of each of eight sequences, at positions of its own: a decoding step, where only latency counts
        dict(name="rope_decode", kind="rope", batch=8, seq=1, heads=32, kv_heads=8, head_dim=128, dim=128, dtype="bf16",
             interleaved=False, scaling="bands", factor=8.0, positions=True, inplace=True, train=False),
        # prompts of an odd length whose heads rotate in part, neighbours paired, read in fp16 (evaluation)
        dict(name="rope_prompts", kind="rope", batch=2, seq=1531, heads=16, kv_heads=16, head_dim=80, dim=32,
             dtype="fp16", interleaved=True, scaling="none", factor=1.0, positions=False, inplace=True, train=False),
        # long-context training, one sequence of four times the length that the frequencies were made for
        dict(name="rope_train_long", kind="rope", batch=1, seq=16384, heads=32, kv_heads=8, head_dim=128, dim=128,
             dtype="bf16", interleaved=False, scaling="yarn", factor=4.0, positions=False, inplace=False, train=True),
        # a decoding step of one sequence, far into a long context
        dict(name="qk_norm_decode", kind="qk_norm", batch=1, seq=1, heads=16, kv_heads=4, head_dim=128, dim=128,
             dtype="bf16", wide_weights=False, interleaved=False, scaling="linear", factor=4.0, positions=True,
             inplace=True, train=False),
        # training on documents of a ragged length; part of the head rotates, weights kept in fp32
        dict(name="qk_norm_ragged", kind="qk_norm", batch=3, seq=1000, heads=16, kv_heads=4, head_dim=128, dim=64,
             dtype="bf16", wide_weights=True, interleaved=True, scaling="none", factor=1.0, positions=False,
             inplace=False, train=True),
        # a training step's attention input at Llama-3-8B widths, two sequences of 8192
        dict(name="qk_norm_train", kind="qk_norm", batch=2, seq=8192, heads=32, kv_heads=8, head_dim=128, dim=128,
             dtype="bf16", wide_weights=False, interleaved=False, scaling="none", factor=1.0, positions=False,
             inplace=False, train=True),
        # the router of a serving step: few tokens, many experts in groups, a bias that only chooses
        dict(name="route_decode", kind="route", tokens=64, experts=256, width=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", renormalize=True, scale=2.5, capacity=1.25, dtype="bf16",
             train=False),
        # an expert layer in training whose experts are no power of two (the projection is padded), plain softmax weights
        dict(name="route_odd", kind="route", tokens=4095, experts=60, width=64, top_k=4, score="softmax", bias=False,
             groups=1, top_groups=1, group_score="max", renormalize=False, scale=1.0, capacity=1.25, dtype="bf16",
             train=True),
        # a large expert layer in training, logits in fp32
        dict(name="route_train", kind="route", tokens=16384, experts=256, width=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", renormalize=True, scale=2.5, capacity=1.25, dtype="fp32",
             train=True),
        # the gradients of the smallest decoder that the package trains (its smoke run): launches count
        dict(name="clip_tiny", kind="clip", family="llama", d_model=512, heads=4, kv_heads=2, ffn=1024, vocab=4096,
             layers=2, dtype="bf16", wide_norms=False),
        # GPT-2-XL widths, four layers: matrices, biases and norm weights, 53 tensors of very different sizes
        dict(name="clip_gpt2", kind="clip", layers=4, dtype="bf16", wide_norms=True, **_GPT2_XL),
        # two layers at Llama-3-8B widths with the whole vocabulary, accumulated in fp32: the largest case
        dict(name="clip_llama", kind="clip", layers=2, dtype="fp32", wide_norms=False, **_LLAMA_8B),
    ]


# ------------------------------------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    """An integer between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng, c):
    c["head_dim"] = rng.choice((40, 64, 80, 96, 128, 128, 192, 256))
    c["kv_heads"] = rng.choice((1, 2, 3, 4, 8))
    c["heads"] = c["kv_heads"] * rng.choice((1, 2, 4, 5, 8))
    whole = rng.random() < 0.6
    c["dim"] = c["head_dim"] if whole else 2 * rng.randint(1, c["head_dim"] // 2)
    c["interleaved"] = rng.random() < 0.5
    c["scaling"] = rng.choice(("none", "linear", "ntk", "yarn", "bands"))
    c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice((2.0, 4.0, 8.0, 32.0))
    if c["scaling"] in ("ntk", "yarn") and c["dim"] < 4:
        c["dim"] = 4
    most = 16384 * 48 * 128 // ((c["heads"] + 2 * c["kv_heads"]) * c["head_dim"])
    tokens = _log(rng, 1, min(32768, most))
    c["seq"] = 1 if rng.random() < 0.3 else _log(rng, 1, tokens)
    c["batch"] = max(1, min(512, tokens // c["seq"]))
    c["positions"] = rng.random() < 0.5
    c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if c["dtype"] == "fp32":
        c["batch"], c["seq"] = max(1, c["batch"] // 2), (c["seq"] + 1) // 2
    c["train"] = rng.random() < 0.6
    c["inplace"] = not c["train"]


def draw(rng):
    kind = rng.choice(("rope", "qk_norm", "route", "clip"))
    c = dict(kind=kind)
    if kind in ("rope", "qk_norm"):
        _draw_heads(rng, c)
        if kind == "qk_norm":
            c["wide_weights"] = rng.random() < 0.5
    elif kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        each = _log(rng, 3, 512 // groups)
        c["experts"] = groups * each
        c["width"] = (c["experts"] + 7) // 8 * 8 if rng.random() < 0.7 else c["experts"]
        c["groups"], c["top_groups"] = groups, rng.randint(1, groups)
        c["top_k"] = rng.randint(1, min(10, c["top_groups"] * each))
        c["tokens"] = _log(rng, 1, 16384)
        if c["tokens"] * c["experts"] > 16384 * 256:
            c["tokens"] = 16384 * 256 // c["experts"]
        c["score"] = rng.choice(("softmax", "sigmoid"))
        c["bias"] = rng.random() < 0.5
        c["group_score"] = rng.choice(("max", "top2"))
        c["renormalize"] = rng.random() < 0.6
        c["scale"] = rng.choice((1.0, 2.5, 16.0))
        c["capacity"] = rng.choice((1.0, 1.25, 2.0))
        c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        c["train"] = rng.random() < 0.6
    else:
        c["family"] = rng.choice(("llama", "gpt2"))
        hd = rng.choice((64, 128))
        c["heads"] = _log(rng, 2, 4096 // hd)
        c["kv_heads"] = c["heads"] if c["family"] == "gpt2" else rng.choice([k for k in range(1, c["heads"] + 1)
                                                                           if c["heads"] % k == 0])
        c["d_model"] = hd * c["heads"]
        c["ffn"] = int(c["d_model"] * rng.uniform(2, 3.5))
        c["vocab"] = _log(rng, 500, 128256)
        c["layers"] = rng.randint(1, 4 if c["family"] == "gpt2" else 2 if c["d_model"] > 2048 else 6)
        c["dtype"] = rng.choice(("bf16", "fp16", "fp32"))
        c["wide_norms"] = rng.random() < 0.5
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _grad_shapes(c):
    """The trainable tensors of a decoder: (shape, whether it is a norm's or a bias)."""
    d, f, hd = c["d_model"], c["ffn"], c["d_model"] // c["heads"]
    qkv = (c["heads"] + 2 * c["kv_heads"]) * hd
    gpt = c["family"] == "gpt2"
    shapes = [((c["vocab"], d), False)] + ([((1024, d), False)] if gpt else [])
    for _ in range(c["layers"]):
        for rows, cols in ((qkv, d), (d, d), (f if gpt else 2 * f, d), (d, f)):
            shapes.append(((rows, cols), False))
            if gpt:
                shapes.append(((rows,), True))
        shapes += [((d,), True)] * (4 if gpt else 2)
    return shapes + [((d,), True)] * (2 if gpt else 1) + [((c["vocab"], d), False)]


def _rotary_args(c):
    """The settings of the rotation, as an ``ops.Rotary`` takes them."""
    how = dict(theta=500000.0, dim=c["dim"], interleaved=c["interleaved"])
    if c["scaling"] != "none":
        how.update(scaling=c["scaling"], factor=c["factor"])
        if c["scaling"] in ("yarn", "bands"):
            how["original"] = 4096
    return how


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[c["dtype"]]
    s = dict(case=c)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale)

    if c["kind"] in ("rope", "qk_norm"):
        tokens, total = c["batch"] * c["seq"], c["heads"] + 2 * c["kv_heads"]
        s["qkv"] = normal(tokens, total, c["head_dim"]).to(dt)
        s["positions"] = None
        if c["positions"]:
            # every sequence at a place of its own in a long context, its tokens one after the other
            start = torch.randint(0, 100000, (c["batch"], 1), generator=gen, device="cuda")
            s["positions"] = (start + torch.arange(c["seq"], device="cuda")).reshape(-1)
        if c["kind"] == "qk_norm":
            wdt = torch.float32 if c["wide_weights"] else dt
            s["wq"] = (1 + normal(c["head_dim"], scale=0.1)).to(wdt)
            s["wk"] = (1 + normal(c["head_dim"], scale=0.1)).to(wdt)
        if c["train"]:
            s["dout"] = normal(tokens, total, c["head_dim"]).to(dt)
            for name in ("qkv", "wq", "wk"):
                if name in s:
                    s[name].requires_grad_(True)
    elif c["kind"] == "route":
        T, E = c["tokens"], c["experts"]
        # some experts are liked more than others, as in training
        s["logits"] = (normal(T, c["width"]) + normal(1, c["width"], scale=0.5)).to(dt)
        s["bias"] = normal(E, scale=0.05) if c["bias"] else None
        s["capacity"] = int(math.ceil(c["capacity"] * T * c["top_k"] / E / 8.0) * 8)
        if c["train"]:
            s["logits"].requires_grad_(True)
            s["dw"] = normal(T, c["top_k"])
            s["dprob"] = normal(E, scale=0.01)
    else:
        s["grads"] = [normal(*shape, scale=1e-3).to(torch.float32 if vector and c["wide_norms"] else dt)
                      for shape, vector in _grad_shapes(c)]
        # Some way below the norm at first; each pass asks for a little less than the one before, so that every one of them clips
        # (gradients that the last pass has clipped are what this one finds).
        s["max_norm"] = 0.37e-3 * math.sqrt(sum(g.numel() for g in s["grads"]))
    return s


# ---------------------------------------------------------------------------------------------------- run
def _frequencies(c, device):
    """Angle per position of every pair, fp64."""
    n, theta, factor = c["dim"], 500000.0, c["factor"]
    if c["scaling"] == "ntk":
        theta = theta * factor ** (n / (n - 2))
    f = theta ** (-torch.arange(0, n, 2, device=device, dtype=torch.float64) / n)
    if c["scaling"] == "linear":
        f = f / factor
    elif c["scaling"] == "yarn":
        # pairs that turn more than 32 times over the original length stay, those that turn less than once are slowed down
        lo, hi = (n * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(theta)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
        ramp = ((torch.arange(n // 2, device=device, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
    elif c["scaling"] == "bands":
        g = ((4096 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        f = f * ((1 - g) / factor + g)
    return f


def _magnitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "yarn" else 1.0


def _angles(s):
    """(cos, sin) [tokens, 1, dim / 2] in fp32, times the magnitude."""
    c, dev = s["case"], s["qkv"].device
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(c["batch"] * c["seq"], device=dev) % c["seq"]
    angle = (pos.double().unsqueeze(1) * _frequencies(c, dev)).unsqueeze(1)
    return (_magnitude(c) * angle.cos()).float(), (_magnitude(c) * angle.sin()).float()


def _turn(x, cos, sin, c):
    """The pairs of the leading ``dim`` components of fp32 heads ``x`` turned by (cos, sin)."""
    n = c["dim"]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if c["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    y, z = a * cos - b * sin, b * cos + a * sin
    both = torch.stack([y, z], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([y, z], dim=-1)
    return torch.cat([both, x[..., n:]], dim=-1)


def _plain_rope(s):
    c, x = s["case"], s["qkv"].detach()
    nh = c["heads"] + c["kv_heads"]
    cos, sin = _angles(s)
    turned = _turn(x[:, :nh].float(), cos, sin, c).to(x.dtype)
    if c["inplace"]:
        x[:, :nh] = turned
        return [x]
    out = [torch.cat([turned, x[:, nh:]], dim=1)]
    if c["train"]:
        d = s["dout"]
        out.append(torch.cat([_turn(d[:, :nh].float(), cos, -sin, c).to(d.dtype), d[:, nh:]], dim=1))
    return out


def _plain_qk_norm(s):
    c, x = s["case"], s["qkv"].detach()
    hq, nh = c["heads"], c["heads"] + c["kv_heads"]
    cos, sin = _angles(s)
    h = x[:, :nh].float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    w = torch.cat([s["wq"].detach().float().expand(hq, -1), s["wk"].detach().float().expand(nh - hq, -1)])
    unit = h * r
    turned = _turn(unit * w, cos, sin, c).to(x.dtype)
    if c["inplace"]:
        x[:, :nh] = turned
        return [x]
    out = [torch.cat([turned, x[:, nh:]], dim=1)]
    if c["train"]:
        d = s["dout"]
        g = _turn(d[:, :nh].float(), cos, -sin, c)
        dw = (g * unit).sum(0)
        gw = g * w
        dh = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
        out += [torch.cat([dh.to(x.dtype), d[:, nh:]], dim=1), dw[:hq].sum(0).to(s["wq"].dtype),
                dw[hq:].sum(0).to(s["wk"].dtype)]
    return out


def _plain_route(s):
    # in 64 bits: two experts whose scores are nearly alike must not change places
    c, E, k = s["case"], s["case"]["experts"], s["case"]["top_k"]
    logits = s["logits"].detach()
    T = logits.shape[0]
    l64 = logits[:, :E].double()
    if c["score"] == "softmax":
        e = torch.exp(l64 - l64.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
        prob, slope = score, torch.ones_like(score)
    else:
        score = 1 / (1 + torch.exp(-l64))
        prob, slope = score / score.sum(-1, keepdim=True), 1 - score
    choice = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by_group = choice.reshape(T, c["groups"], E // c["groups"])
        ranked = by_group.sort(dim=-1, descending=True).values
        value = ranked[..., 0] if c["group_score"] == "max" or ranked.shape[-1] == 1 else ranked[..., 0] + ranked[..., 1]
        best = value.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        live = torch.zeros_like(value).scatter(1, best, 1.0) > 0
        choice = torch.where(live.unsqueeze(-1), by_group, -math.inf).reshape(T, E)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]         # ties: the lowest expert
    chosen = score.gather(1, ids)
    w = chosen / chosen.sum(-1, keepdim=True) if c["renormalize"] else chosen
    # a pair's slot: its rank, in the order of the pairs, among those of its expert
    flat = ids.reshape(-1)
    counts = torch.zeros(E, dtype=torch.int64, device=flat.device).scatter_add(0, flat, torch.ones_like(flat))
    order = flat.sort(stable=True).indices
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device=flat.device) - (counts.cumsum(0) - counts)[flat[order]]
    slot = torch.where(rank < s["capacity"], rank, -1)
    out = [(c["scale"] * w).float(), prob.sum(0).float(), flat.int(), slot.int(), counts.int()]
    if c["train"]:
        dw = c["scale"] * s["dw"].double()
        if c["renormalize"]:
            part = w * (dw - (w * dw).sum(-1, keepdim=True))
            dl = torch.zeros_like(score).scatter(1, ids, part)
        else:
            dl = torch.zeros_like(score).scatter(1, ids, w * dw)
            if c["score"] == "softmax":
                dl = dl - score * (w * dw).sum(-1, keepdim=True)
        coef = s["dprob"].double()
        dl = slope * (dl + prob * (coef - (prob * coef).sum(-1, keepdim=True)))
        grad = torch.zeros(T, c["width"], dtype=logits.dtype, device=logits.device)
        grad[:, :E] = dl.to(logits.dtype)
        out.append(grad)
    return out


def _plain_clip(s):
    # (the sums in 64 bits: up to 1.5e9 squares)
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt().float()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return [norm] + [g.copy_(g.float() * scale) for g in s["grads"]]


def run(state):
    s, c = state, state["case"]
    if not own:
        out = {"rope": _plain_rope, "qk_norm": _plain_qk_norm, "route": _plain_route, "clip": _plain_clip}[c["kind"]](s)
    else:
        out = _own(s, c)
    if c["kind"] == "clip":
        s["max_norm"] *= 0.9999
    return out


@functools.lru_cache(maxsize=None)
def _rotary(settings):
    """The ``ops.Rotary`` that a program makes once, next to its model."""
    from distdl_b200 import ops
    return ops.Rotary(**dict(settings))


def _own(s, c):
    from distdl_b200 import ops
    if c["kind"] == "clip":
        return [ops.clip_grad_norm_(s["grads"], s["max_norm"]), *s["grads"]]
    if c["kind"] == "route":
        w, prob, ids, slot, counts = ops.moe.route(
            s["logits"], c["experts"], c["top_k"], s["capacity"], score=c["score"], bias=s["bias"], groups=c["groups"],
            top_groups=c["top_groups"], group_score=c["group_score"], renormalize=c["renormalize"], scale=c["scale"])
        if not c["train"]:
            return [w, prob, ids, slot, counts]
        (dl,) = torch.autograd.grad((w, prob), s["logits"], (s["dw"], s["dprob"]))
        return [w.detach(), prob.detach(), ids, slot, counts, dl]
    where = dict(rotary=_rotary(tuple(_rotary_args(c).items())), positions=s["positions"])
    if c["kind"] == "rope":
        nh = c["heads"] + c["kv_heads"]
        if c["inplace"]:
            return [ops.rope_(s["qkv"], c["seq"], nh, **where)]
        y = ops.rope(s["qkv"], c["seq"], nh, **where)
        leaves = (s["qkv"],)
    else:
        args = (s["qkv"], c["seq"], c["heads"], c["kv_heads"], s["wq"], s["wk"])
        if c["inplace"]:
            return [ops.qk_norm_rope_(*args, eps=1e-6, **where)]
        y = ops.qk_norm_rope(*args, eps=1e-6, **where)
        leaves = (s["qkv"], s["wq"], s["wk"])
    if not c["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dout"])]


# ------------------------------------------------------------------------------------------------ the work
def work(case):
    c = dict(case)
    size = 2 if c["dtype"] != "fp32" else 4
    if c["kind"] in ("rope", "qk_norm"):
        tokens, nh, hd = c["batch"] * c["seq"], c["heads"] + c["kv_heads"], c["head_dim"]
        every = tokens * (nh + c["kv_heads"]) * hd * size
        touched = tokens * nh * (c["dim"] if c["kind"] == "rope" else hd) * size
        # in place: what changes, read and written; in training x and its output, the gradient and its own
        moved = 2 * touched if c["inplace"] else (4 if c["train"] else 2) * every
        per = (3 if c["kind"] == "rope" else 7) if not c["train"] else (6 if c["kind"] == "rope" else 20)
        return {"bytes": moved + (8 * tokens if c["positions"] else 0), "flops": per * touched // size}
    if c["kind"] == "route":
        T, E, k = c["tokens"], c["experts"], c["top_k"]
        moved = T * E * size + 12 * T * k + 8 * E + (4 * E if c["bias"] else 0)
        if c["train"]:
            moved += T * c["width"] * size + 4 * T * k + 4 * E
        return {"bytes": moved, "flops": T * E * (12 if c["train"] else 6)}
    wide = sum(math.prod(shape) for shape, vector in _grad_shapes(c) if vector and c["wide_norms"])
    n = sum(math.prod(shape) for shape, _ in _grad_shapes(c))
    return {"bytes": 2 * ((n - wide) * size + wide * 4), "flops": 3 * n}


# ------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_rotation(c, s):
    """e^(i angle) times the magnitude [tokens, dim / 2], complex128: position by position, pair by pair."""
    n, base = c["dim"], 500000.0
    if c["scaling"] == "ntk":
        base *= c["factor"] ** (n / (n - 2.0))
    f = []
    for i in range(n // 2):
        w = math.exp(-2.0 * i / n * math.log(base))
        turns = 4096 * w / (2 * math.pi)                       # over the original length
        if c["scaling"] == "linear":
            w /= c["factor"]
        elif c["scaling"] == "bands":
            keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            w = keep * w + (1.0 - keep) * w / c["factor"]
        elif c["scaling"] == "yarn":
            first = max(0, math.floor(n / 2 * math.log(4096 / (32.0 * 2 * math.pi)) / math.log(base)))
            last = min(n - 1, math.ceil(n / 2 * math.log(4096 / (2 * math.pi)) / math.log(base)))
            slow = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            w = (1.0 - slow) * w + slow * w / c["factor"]
        f.append(w)
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    if s["positions"] is None:
        pos = torch.arange(c["seq"], dtype=torch.float64, device="cuda").repeat(c["batch"])
    else:
        pos = s["positions"].to(torch.float64)
    return torch.polar(torch.full((1, 1), _magnitude(c), dtype=torch.float64, device="cuda"), torch.outer(pos, f))


def _exact_turn(x, z, c):
    """Complex multiplication of the pairs of fp64 heads ``x [tokens, heads, head_dim]`` by ``z``."""
    n = c["dim"]
    lead = x[..., :n]
    pairs = lead.unflatten(-1, (n // 2, 2)) if c["interleaved"] else lead.unflatten(-1, (2, n // 2)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z.unsqueeze(1))
    turned = turned if c["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), x[..., n:]], dim=-1)


def _exact_heads(c, s):
    hq, nh = c["heads"], c["heads"] + c["kv_heads"]
    z = _exact_rotation(c, s)
    x = s["qkv"].detach().double()
    leaves = [x]
    if c["train"]:
        x.requires_grad_(True)
    h = x[:, :nh]
    if c["kind"] == "qk_norm":
        wq, wk = (s[n].detach().double().requires_grad_(c["train"]) for n in ("wq", "wk"))
        leaves += [wq, wk]
        h = h / (h.pow(2).sum(-1, keepdim=True) / c["head_dim"] + 1e-6).sqrt()
        h = torch.cat([h[:, :hq] * wq, h[:, hq:] * wk], dim=1)
    y = torch.cat([_exact_turn(h, z, c), x[:, nh:]], dim=1)
    if not c["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dout"].double())]


def _exact_route(c, s):
    E, G = c["experts"], c["groups"]
    l64 = s["logits"].detach().double().requires_grad_(c["train"])
    kept = l64[:, :E]
    score = torch.softmax(kept, -1) if c["score"] == "softmax" else torch.sigmoid(kept)
    prob = score / score.sum(-1, keepdim=True)
    want = score.detach() + (0.0 if s["bias"] is None else s["bias"].double())
    T = want.shape[0]
    if G > 1:
        best = want.reshape(T, G, -1).topk(min(2 if c["group_score"] == "top2" else 1, E // G), -1).values.sum(-1)
        # groups by value, then by number
        place = (best.unsqueeze(1) > best.unsqueeze(2)).sum(-1)
        number = torch.arange(G, device=best.device)
        place = place + ((best.unsqueeze(1) == best.unsqueeze(2)) & (number.unsqueeze(0) < number.unsqueeze(1))).sum(-1)
        want = want.masked_fill((place >= c["top_groups"]).repeat_interleave(E // G, dim=1), -math.inf)
    ids, left = [], want.clone()
    index = torch.arange(E, device=left.device).expand_as(left)
    for _ in range(c["top_k"]):
        top = left.amax(-1, keepdim=True)
        pick = torch.where(left == top, index, E).amin(-1, keepdim=True)
        ids.append(pick)
        left.scatter_(1, pick, -math.inf)
    ids = torch.cat(ids, 1)
    w = score.gather(1, ids)
    w = c["scale"] * (w / w.sum(-1, keepdim=True) if c["renormalize"] else w)
    total = prob.sum(0)
    out = [w.detach(), total.detach(), None, None, None]
    if c["train"]:
        out += torch.autograd.grad((w, total), l64, (s["dw"].double(), s["dprob"].double()))
    return out


def _exact_clip(s):
    total = 0.0
    for g in s["grads"]:
        for part in g.reshape(-1).split(1 << 26):
            p = part.double()
            total += float(torch.dot(p, p))
    norm = math.sqrt(total)
    scale = min(1.0, s["max_norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64)] + [g.double() * scale for g in s["grads"]]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "clip":
        return _exact_clip(s)
    return _exact_route(c, s) if c["kind"] == "route" else _exact_heads(c, s)
