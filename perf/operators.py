"""The operators of a transformer block around the FP4 expert layer, as measured cases.

* ``dense``  ``dense_matmul``: a product with bias, activation and residual in its epilogue
  (the router's logits, the shared expert's two projections, any dense projection);
* ``route``  ``route_grouped_topk``: top-k routing limited to the best groups of experts;
* ``norm``   ``pre_norm`` / ``post_norm``: the norms before and after a block, with the
  block's gate, its scale and the residual's scale.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run``
makes one pass (the plain form in elementary torch operations, or with ``own`` the
framework's call), ``exact`` computes the same in 64 bits, ``work`` says what a pass has to move.
"""

import math

import torch

own = False

ACTS = ("none", "silu", "gelu", "gelu_tanh", "swiglu", "swiglu_clamp")
LIMIT = 7.0  # swiglu_clamp: gate <= LIMIT, |up| <= LIMIT
EPS = 1e-6

# The largest listed cases, which bound the drawn ones.
MOST_MACS = 8192 * 4096 * 4096
MOST_SCORES = 32771 * 256
MOST_ROWS = 8192 * 4096


def listed():
    return [
        # The router's logits of one decoded token: 2 MB of weights, so latency.
        dict(name="router, one token", op="dense", m=1, k=4096, n=256, act="none", bias=False,
             residual="", out="f32"),
        # The shared expert's gated up projection for a decode batch of 64: 33 MB of weights.
        dict(name="shared up, decode", op="dense", m=64, k=4096, n=4096, act="swiglu", bias=False,
             residual="", out="bf16"),
        # A projection with nothing even about it: rows, columns and k off every tile.
        dict(name="projection, odd sizes", op="dense", m=333, k=1000, n=777, act="gelu", bias=True,
             residual="bf16", out="bf16"),
        # The shared expert's down projection added to the routed sum, a prompt of 1024.
        dict(name="shared down, prompt", op="dense", m=1024, k=2048, n=4096, act="none", bias=True,
             residual="f32", out="bf16"),
        # The shared expert's up projection for 8192 tokens of prompts: tensor-core bound.
        dict(name="shared up, prompts", op="dense", m=8192, k=4096, n=4096, act="swiglu_clamp",
             bias=False, residual="", out="bf16"),
        # One decoded token's routing: latency.
        dict(name="routing, one token", op="route", t=1, e=256, groups=8, keep=4, k=8,
             scoring="sigmoid", group_score="top2", bias=True, renorm=True, logits="f32"),
        # A prompt of 1024 with bf16 logits (many exact ties).
        dict(name="routing, prompt, bf16", op="route", t=1024, e=256, groups=8, keep=4, k=8,
             scoring="sigmoid", group_score="top2", bias=True, renorm=True, logits="bf16"),
        # A large batch of prompts, softmax scores, groups of 20 experts by their best one.
        dict(name="routing, prompts, softmax", op="route", t=32771, e=160, groups=8, keep=3, k=6,
             scoring="softmax", group_score="max", bias=False, renorm=False, logits="f32"),
        # The norm before the block for one decoded token: latency.
        dict(name="norm before, one token", op="norm", t=1, h=4096, form="pre", kind="rms",
             stream="bf16", gate="", inner=False, next=True),
        # After the block for a decode batch: norm, gate of each token, residual, next norm.
        dict(name="norm after, decode", op="norm", t=64, h=4096, form="post", kind="rms",
             stream="bf16", gate="token", inner=True, next=True),
        # The same for 8192 tokens of prompts, gate of each channel: bandwidth.
        dict(name="norm after, prompts", op="norm", t=8192, h=4096, form="post", kind="rms",
             stream="bf16", gate="channel", inner=True, next=True),
        # An f32 residual stream of odd width, layer norm, a gate value for each element.
        dict(name="layer norm after, odd, f32", op="norm", t=1023, h=5003, form="post",
             kind="layer", stream="f32", gate="full", inner=True, next=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dense", "dense", "route", "norm"))
    if op == "dense":
        k = 8 * _log(rng, 8, 1024)  # rows of x and w start on 16 bytes
        m = _log(rng, 1, 8192)
        n = min(_log(rng, 16, 8192), max(16, MOST_MACS // (m * k)))
        act = rng.choice(ACTS)
        if act.startswith("swiglu"):
            n -= n % 2
        return dict(op="dense", m=m, k=k, n=n, act=act, bias=rng.random() < 0.5,
                    residual=rng.choice(("", "", "bf16", "f32")),
                    out=rng.choice(("bf16", "bf16", "f32")))
    if op == "route":
        groups = rng.choice((1, 2, 4, 8, 16))
        per = rng.randint(2, 32)
        e = groups * per
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, keep * per))
        t = min(_log(rng, 1, 32768), MOST_SCORES // e)
        return dict(op="route", t=t, e=e, groups=groups, keep=keep, k=k,
                    scoring=rng.choice(("softmax", "sigmoid", "sqrtsoftplus")),
                    group_score=rng.choice(("max", "top2")), bias=rng.random() < 0.6,
                    renorm=rng.random() < 0.7, logits=rng.choice(("bf16", "f32")))
    h = _log(rng, 64, 16384)
    if rng.random() < 0.5:
        h = max(64, h - h % 64)
    t = min(_log(rng, 1, 16384), MOST_ROWS // h)
    form = rng.choice(("pre", "post", "post"))
    post = form == "post"
    return dict(op="norm", t=t, h=h, form=form, kind=rng.choice(("rms", "layer")),
                stream=rng.choice(("bf16", "f32")),
                gate=rng.choice(("", "token", "channel", "full")) if post else "",
                inner=post and rng.random() < 0.6, next=not post or rng.random() < 0.8)


_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0, dtype=torch.bfloat16):
        v = torch.randn(shape, generator=g, device="cuda")
        return (v * scale + mean).to(dtype)

    c = dict(case)
    if c["op"] == "dense":
        n_out = c["n"] // 2 if c["act"].startswith("swiglu") else c["n"]
        c["x"] = normal(c["m"], c["k"])
        c["w"] = normal(c["n"], c["k"], scale=c["k"] ** -0.5)
        c["b"] = normal(c["n"], scale=0.1, dtype=torch.float32) if c["bias"] else None
        c["r"] = normal(c["m"], n_out, dtype=_DT[c["residual"]]) if c["residual"] else None
        c["rs"] = 0.5 if c["residual"] else 1.0
    elif c["op"] == "route":
        c["x"] = normal(c["t"], c["e"], scale=1.5, dtype=_DT[c["logits"]])
        c["b"] = normal(c["e"], scale=0.05, dtype=torch.float32) if c["bias"] else None
        c["ws"] = 2.5
    else:
        t, h, dt = c["t"], c["h"], _DT[c["stream"]]
        c["y"] = normal(t, h, scale=0.7, mean=0.05)  # the block's output: bf16 activations
        c["r"] = normal(t, h, scale=2.0, mean=0.1, dtype=dt)
        c["w1"], c["b1"] = normal(h, scale=0.2, mean=1.0), None
        c["w2"], c["b2"] = (normal(h, scale=0.2, mean=1.0), None) if c["inner"] else (None, None)
        if c["kind"] == "layer":
            c["b1"] = normal(h, scale=0.1)
            c["b2"] = normal(h, scale=0.1) if c["inner"] else None
        c["g"] = {"": None, "token": (t, 1), "channel": (h,), "full": (t, h)}[c["gate"]]
        if c["g"] is not None:
            c["g"] = normal(*c["g"], scale=0.3, mean=0.5)
        c["ys"], c["rs"] = 1.25, 0.75
    return c


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _own(c):
    import dw_tpu_b200 as dw

    if c["op"] == "dense":
        return dw.dense_matmul(c["x"], c["w"], bias=c["b"],
                               act=None if c["act"] == "none" else c["act"], act_limit=LIMIT,
                               residual=c["r"], residual_scale=c["rs"], out_dtype=_DT[c["out"]])
    if c["op"] == "route":
        w, ids = dw.route_grouped_topk(c["x"], c["k"], c["groups"], c["keep"],
                                       renormalize=c["renorm"], scoring_fn=c["scoring"],
                                       group_score=c["group_score"], routed_scale=c["ws"],
                                       bias=c["b"], dtype=torch.float32)
        return {"weights": w, "ids": ids}
    if c["form"] == "pre":
        return dw.pre_norm(c["r"], c["w1"], c["b1"], eps=EPS, kind=c["kind"])
    r, h = dw.post_norm(c["y"], c["r"], norm_weight=c["w2"], norm_bias=c["b2"], gate=c["g"],
                        scale=c["ys"], residual_scale=c["rs"],
                        next_weight=c["w1"] if c["next"] else None,
                        next_bias=c["b1"] if c["next"] else None, eps=EPS, kind=c["kind"])
    return {"residual": r, "next": h} if c["next"] else r


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _act_plain(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act.startswith("swiglu"):
        half = z.shape[1] // 2
        gate, up = z[:, :half], z[:, half:]
        if act == "swiglu_clamp":
            gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
        return gate / (1.0 + torch.exp(-gate)) * up
    return z


def _dense_plain(c):
    z = torch.matmul(c["x"].float(), c["w"].float().t())
    if c["b"] is not None:
        z = z + c["b"]
    z = _act_plain(z, c["act"])
    if c["r"] is not None:
        z = c["rs"] * c["r"].float() + z
    return z.to(_DT[c["out"]])


def _route_plain(c):
    # In 64 bits: experts whose scores differ in the last place of 32 are ordered rightly, and
    # equal ones go to the lower index (a stable sort).
    x = c["x"].double()
    t, e = x.shape
    if c["scoring"] == "softmax":
        ex = torch.exp(x - x.amax(dim=1, keepdim=True))
        s = ex / ex.sum(dim=1, keepdim=True)
    elif c["scoring"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        s = torch.sqrt(torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs())))
    choice = s if c["b"] is None else s + c["b"].double()
    per = e // c["groups"]
    by_group = choice.reshape(t, c["groups"], per)
    if c["group_score"] == "max":
        value = by_group.amax(dim=2)
    else:
        value = torch.sort(by_group, dim=2, descending=True)[0][:, :, :2].sum(dim=2)
    best = torch.sort(value, dim=1, descending=True, stable=True)[1][:, :c["keep"]]
    kept = torch.zeros((t, c["groups"]), dtype=torch.bool, device=x.device)
    kept.scatter_(1, best, True)
    masked = torch.where(kept[:, :, None], by_group, -math.inf).reshape(t, e)
    ids = torch.sort(masked, dim=1, descending=True, stable=True)[1][:, :c["k"]]
    w = torch.gather(s, 1, ids)
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return {"weights": (w * c["ws"]).float(), "ids": ids.int()}


def _norm_one(v, w, b, kind):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * w.float()
    return v if b is None else v + b.float()


def _norm_plain(c):
    dt = _DT[c["stream"]]
    if c["form"] == "pre":
        return _norm_one(c["r"].float(), c["w1"], c["b1"], c["kind"]).to(torch.bfloat16)
    y = c["y"].float()
    if c["inner"]:
        y = _norm_one(y, c["w2"], c["b2"], c["kind"])
    if c["g"] is not None:
        y = y * c["g"].float()
    r = c["rs"] * c["r"].float() + c["ys"] * y
    if not c["next"]:
        return r.to(dt)
    return {"residual": r.to(dt),
            "next": _norm_one(r, c["w1"], c["b1"], c["kind"]).to(torch.bfloat16)}


def run(state):
    if own:
        return _own(state)
    return {"dense": _dense_plain, "route": _route_plain, "norm": _norm_plain}[state["op"]](state)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    c = prepare(case, seed)
    up = {k: v.to(torch.float64) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    if c["op"] == "dense":
        z = torch.einsum("mk,nk->mn", up["x"], up["w"])
        if up["b"] is not None:
            z += up["b"][None, :]
        n = c["n"]
        if c["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif c["act"] == "gelu":
            z = z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
        elif c["act"] == "gelu_tanh":
            # 1 + tanh(a) = 2 sigmoid(2 a)
            z = z * torch.sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z.pow(3)))
        elif c["act"] in ("swiglu", "swiglu_clamp"):
            lim = LIMIT if c["act"] == "swiglu_clamp" else math.inf
            a = torch.minimum(z[:, :n // 2], torch.full_like(z[:, :n // 2], lim))
            z = a * torch.sigmoid(a) * z[:, n // 2:].clamp(min=-lim, max=lim)
        return z if up["r"] is None else torch.add(z, up["r"], alpha=c["rs"])
    if c["op"] == "route":
        x = up["x"]
        if c["scoring"] == "softmax":
            s = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
        elif c["scoring"] == "sigmoid":
            s = torch.sigmoid(x)
        else:
            s = torch.logaddexp(x, torch.zeros_like(x)).sqrt()
        choice = s.clone() if up["b"] is None else s + up["b"]
        t, e = x.shape
        per = e // c["groups"]
        rows = torch.arange(t, device=x.device)
        # Groups, then experts, one at a time: the largest value's first index.
        left = choice.reshape(t, c["groups"], per).clone()
        first, at = left.max(dim=2)
        if c["group_score"] == "max":
            value = first
        else:
            left.scatter_(2, at[:, :, None], -math.inf)
            value = first + left.max(dim=2)[0]

        def first_largest(v):
            top = v.amax(dim=1, keepdim=True)
            index = torch.arange(v.shape[1], device=v.device).expand_as(v)
            return torch.where(v == top, index, v.shape[1]).amin(dim=1)

        open_ = torch.zeros((t, c["groups"]), dtype=torch.bool, device=x.device)
        for _ in range(c["keep"]):
            best = first_largest(value)
            open_[rows, best] = True
            value[rows, best] = -math.inf
        choice[~open_.repeat_interleave(per, dim=1)] = -math.inf
        weights = torch.empty((t, c["k"]), dtype=torch.float64, device=x.device)
        for j in range(c["k"]):
            best = first_largest(choice)
            weights[:, j] = s[rows, best]
            choice[rows, best] = -math.inf
        if c["renorm"]:
            weights /= weights.sum(dim=1, keepdim=True)
        return {"weights": weights * c["ws"], "ids": None}

    def norm(v, w, b):
        mean = v.mean(dim=1, keepdim=True) if c["kind"] == "layer" else 0.0
        out = (v - mean) * torch.rsqrt((v - mean).pow(2).mean(dim=1, keepdim=True) + EPS) * w
        return out if b is None else out + b

    if c["form"] == "pre":
        return norm(up["r"], up["w1"], up["b1"])
    y = norm(up["y"], up["w2"], up["b2"]) if c["inner"] else up["y"]
    r = c["rs"] * up["r"] + c["ys"] * (y if up["g"] is None else up["g"] * y)
    return {"residual": r, "next": norm(r, up["w1"], up["b1"])} if c["next"] else r


def work(case):
    c = case
    size = {"": 0, "bf16": 2, "f32": 4}
    if c["op"] == "dense":
        m, k, n = c["m"], c["k"], c["n"]
        n_out = n // 2 if c["act"].startswith("swiglu") else n
        return {"bytes": 2 * (m * k + n * k) + (4 * n if c["bias"] else 0)
                + m * n_out * (size[c["residual"]] + size[c["out"]]),
                "flops": 2 * m * n * k}
    if c["op"] == "route":
        t, e, k = c["t"], c["e"], c["k"]
        # A score is some 20 operations, its comparisons for the groups and the top k as many.
        return {"bytes": t * e * size[c["logits"]] + (4 * e if c["bias"] else 0) + t * k * 8,
                "flops": 40 * t * e}
    t, h, es = c["t"], c["h"], size[c["stream"]]
    vectors = 2 * h * ((1 + (c["kind"] == "layer")) * (c["inner"] + c["next"]))
    if c["form"] == "pre":
        return {"bytes": t * h * (es + 2) + vectors, "flops": 6 * t * h}
    gate = {"": 0, "token": t, "channel": h, "full": t * h}[c["gate"]] * 2
    return {"bytes": t * h * (2 + 2 * es + (2 if c["next"] else 0)) + gate + vectors,
            "flops": t * h * (4 + 6 * (c["inner"] + c["next"]))}
