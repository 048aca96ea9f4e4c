"""The operators around the experts' products of a mixture-of-experts layer, and the products with 4-bit weights.

* ``route``: router logits -> chosen experts and their weights (scores, balancing bias, expert groups), with the gradient.
* ``gated``: the gated activation between the experts' two products, with the gradient.
* ``int4``: a linear layer with 4-bit weights and group scales, from one token to a long prompt.
* ``int4_moe``: the same for all experts of a layer over expert-sorted rows.

``listed()`` names the cases, ``draw(rng)`` gives one more of their ranges, ``prepare`` builds what a program holds before
the call, ``run`` makes one pass - in elementary torch operations, or through the library where ``own`` is true -,
``work`` counts what a pass cannot do without, and ``exact`` states the same result in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda"
MAX_FLOPS = 2.7e11     # bounds of a drawn case: the largest listed ones
MAX_BYTES = 8.1e8


def listed():
    return [
        # Router of a generation batch: 64 tokens over the 64 experts of the layer's example script.
        dict(name="route_decode", kind="route", tokens=64, experts=64, topk=8, score="softmax", bias=False, groups=1,
             topk_groups=1, group_top=1, renorm=True, scale=1.0, dtype="fp32", train=False),
        # Router of a prompt of 8192 tokens over many small experts: sigmoid scores, a balancing bias, half of the groups.
        dict(name="route_groups", kind="route", tokens=8192, experts=256, topk=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, group_top=2, renorm=True, scale=2.5, dtype="fp32", train=False),
        # Router in training: the tokens of one rank's batch, an expert count that is no power of two, gradient included.
        dict(name="route_train", kind="route", tokens=16384, experts=120, topk=6, score="softmax", bias=False, groups=1,
             topk_groups=1, group_top=1, renorm=False, scale=1.0, dtype="bf16", train=True),
        # Activation between the two products while generating: 64 tokens times eight experts.
        dict(name="gated_decode", kind="gated", rows=512, ffn=1536, act="silu", packed=True, weighted=False, counted=False,
             dtype="bf16", train=False),
        # The same in training, weighted with the router's output, gradients of the halves and of the weights.
        dict(name="gated_train", kind="gated", rows=32768, ffn=2048, act="silu", packed=True, weighted=True, counted=False,
             dtype="bf16", train=True),
        # Two weight groups (gate | up), a width that fits no vector, a buffer longer than the rows that arrived.
        dict(name="gated_ragged", kind="gated", rows=5000, ffn=1001, act="gelu", packed=False, weighted=True, counted=True,
             dtype="fp16", train=False),
        # One token through the up projection of the MLP block of the example script.
        dict(name="int4_token", kind="int4", m=1, n=16384, k=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # A generation batch through the down projection: zero points, smaller groups, a bias.
        dict(name="int4_batch", kind="int4", m=16, n=4096, k=16384, group=64, zeros=True, bias=True, dtype="fp16"),
        # A few speculative tokens of several sequences; sizes that fit no tile (odd vocabulary cut).
        dict(name="int4_odd", kind="int4", m=45, n=5003, k=4128, group=32, zeros=True, bias=False, dtype="bf16"),
        # A chunk of a prompt: bound by the operations, not by the weights.
        dict(name="int4_prefill", kind="int4", m=2048, n=12288, k=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # First product (gate and up) of a generation batch: about eight rows for each of 64 experts.
        dict(name="int4_moe_decode", kind="int4_moe", tokens=64, topk=8, experts=64, n=4096, k=4096, group=128, zeros=False,
             dtype="bf16"),
        # Second product over a prompt: a few hundred rows for each expert.
        dict(name="int4_moe_prefill", kind="int4_moe", tokens=1536, topk=6, experts=32, n=4096, k=2048, group=64,
             zeros=True, dtype="fp16"),
    ]


# ------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi, step=1):
    """Log-uniform between lo and hi, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, min(int(round(v / step)) * step, hi // step * step))


def draw(rng):
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


def _draw_one(rng):
    kind = rng.choice(["route", "gated", "int4", "int4", "int4_moe"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = _log(rng, 8, 512) if groups == 1 else groups * _log(rng, 4, 512 // groups)
        topk_groups = 1 if groups == 1 else rng.randint(1, groups)
        topk = min(rng.choice([1, 2, 4, 6, 8]), experts // groups * topk_groups)
        return dict(kind=kind, tokens=_log(rng, 1, 16384), experts=experts, topk=topk,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    topk_groups=topk_groups, group_top=rng.choice([1, 2]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    train=rng.random() < 0.5)
    if kind == "gated":
        return dict(kind=kind, rows=_log(rng, 1, 32768), ffn=_log(rng, 64, 8192, rng.choice([1, 8, 64])),
                    act=rng.choice(["silu", "silu", "gelu", "relu"]), packed=rng.random() < 0.6,
                    weighted=rng.random() < 0.5, counted=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    train=rng.random() < 0.5)
    group = rng.choice([32, 64, 128, 128])
    n, k = _log(rng, 128, 16384, rng.choice([1, 8, 128])), _log(rng, 512, 16384, max(group, rng.choice([32, 128])))
    if kind == "int4":
        return dict(kind=kind, m=_log(rng, 1, 2048), n=n, k=k, group=group, zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    experts = rng.choice([8, 16, 32, 64, 128])
    return dict(kind=kind, tokens=_log(rng, 1, 2048), topk=rng.choice([1, 2, 4, 6, 8]), experts=experts,
                n=_log(rng, 128, 8192, rng.choice([1, 8, 128])), k=_log(rng, 512, 8192, max(group, rng.choice([32, 128]))),
                group=group, zeros=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16"]))


# ------------------------------------------------------------------------------------------ inputs
class _Inputs:
    """Values from one seed, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, std=1.0, mean=0.0):
        return torch.empty(shape, device=DEVICE, dtype=dtype).normal_(mean, std, generator=self.g)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device=DEVICE, dtype=torch.float32).uniform_(lo, hi, generator=self.g)

    def bytes(self, *shape, below=256):
        return torch.randint(0, below, shape, device=DEVICE, dtype=torch.uint8, generator=self.g)


def _weights4(made, case, lead):
    """Packed 4-bit weights, group scales and zero points, as a quantiser leaves them: scales near the spread of a row of
    normal weights over 15 steps, zero points in the middle of the range."""
    n, k, gs, dt = case["n"], case["k"], case["group"], DTYPES[case["dtype"]]
    q = made.bytes(*lead, n, k // 2)
    scales = made.uniform(*lead, n, k // gs, lo=0.4, hi=1.6).mul_(0.3 / math.sqrt(k)).to(dt)
    zeros = made.bytes(*lead, n, k // gs, below=8).add_(4) if case["zeros"] else None
    return q, scales, zeros


def _inputs(case, seed):
    made, dt, kind = _Inputs(seed), DTYPES[case["dtype"]], case["kind"]
    s = {}
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = made.normal(t, e, std=1.5).to(dt)
        s["bias"] = made.normal(e, std=0.05) if case["bias"] else None
        s["grad"] = made.normal(t, case["topk"]) if case["train"] else None
    elif kind == "gated":
        r, f = case["rows"], case["ffn"]
        if case["packed"]:
            s["gate"], s["up"] = made.normal(r, 2 * f, dtype=dt), None
        else:
            s["gate"], s["up"] = made.normal(r, f, dtype=dt), made.normal(r, f, dtype=dt)
        s["row_weight"] = made.uniform(r) if case["weighted"] else None
        # (what a device-side sum of the splits gives: about nine tenths of the buffer are in use)
        s["num_rows"] = torch.full((1,), r - r // 10, dtype=torch.int32, device=DEVICE) if case["counted"] else None
        s["grad"] = made.normal(r, f, dtype=dt) if case["train"] else None
    elif kind == "int4":
        s["x"] = made.normal(case["m"], case["k"], dtype=dt)
        s["q"], s["scales"], s["zeros"] = _weights4(made, case, ())
        s["bias"] = made.normal(case["n"], std=0.1).to(dt) if case["bias"] else None
    else:
        e, t = case["experts"], case["tokens"]
        topk = min(case["topk"], e)
        # (some experts are more popular than others)
        scores = made.normal(t, e) + 0.5 * made.normal(e)
        chosen = scores.argsort(dim=1, descending=True)[:, :topk]
        s["splits"] = torch.bincount(chosen.reshape(-1), minlength=e).to(torch.int32)
        s["x"] = made.normal(t * topk, case["k"], dtype=dt)
        s["q"], s["scales"], s["zeros"] = _weights4(made, case, (e,))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if own:
        import tempname_new_b200 as flux
        if case.get("train"):
            for name in ("logits", "gate", "up", "row_weight"):
                if s.get(name) is not None:
                    s[name].requires_grad_(True)
        if kind == "int4":
            s["op"] = flux.Int4Gemm(s["q"], s["scales"], s["zeros"])
        elif kind == "int4_moe":
            s["op"] = flux.Int4GemmGrouped(s["q"], s["scales"], s["zeros"])
    elif kind == "int4_moe":
        s["host_splits"] = s["splits"].tolist()
    return s


# ------------------------------------------------------------------------------------------ the library's calls
def _own_route(s, c):
    import tempname_new_b200 as flux
    experts, weights = flux.moe_route(s["logits"], c["topk"], score_func=c["score"], bias=s["bias"], num_groups=c["groups"],
                                      topk_groups=c["topk_groups"], group_top=c["group_top"], renormalize=c["renorm"],
                                      scale=c["scale"])
    if not c["train"]:
        return experts, weights
    grad, = torch.autograd.grad(weights, s["logits"], s["grad"])
    return experts, weights.detach(), grad


def _own_gated(s, c):
    import tempname_new_b200 as flux
    y = flux.gated_act(s["gate"], s["up"], act=c["act"], row_weight=s["row_weight"], num_rows=s["num_rows"])
    if not c["train"]:
        return y
    leaves = [t for t in (s["gate"], s["up"], s["row_weight"]) if t is not None]
    return (y.detach(),) + torch.autograd.grad(y, leaves, s["grad"])


def _own(s):
    c = s["case"]
    if c["kind"] == "route":
        return _own_route(s, c)
    if c["kind"] == "gated":
        return _own_gated(s, c)
    if c["kind"] == "int4":
        return s["op"].forward(s["x"], bias=s["bias"])
    return s["op"].forward(s["x"], s["splits"])


# ------------------------------------------------------------------------------------------ plain form
def _best(values, count):
    """Places of the ``count`` largest values of every row, largest first, ties to the lowest place."""
    return values.sort(dim=-1, descending=True, stable=True).indices[..., :count]


def _plain_route(s, c):
    # (which scores are the largest is decided in 64 bits: neighbours may be closer than 32 bits tell apart)
    x = s["logits"].double()
    t, e = x.shape
    if c["score"] == "softmax":
        p = (x - x.amax(dim=1, keepdim=True)).exp()
        score = p / p.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + (-x).exp())
    choice = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by_group = choice.view(t, c["groups"], e // c["groups"])
        ranks = by_group.sort(dim=2, descending=True).values[:, :, :c["group_top"]].sum(dim=2)
        kept = torch.zeros(t, c["groups"], dtype=torch.bool, device=x.device)
        kept.scatter_(1, _best(ranks, c["topk_groups"]), True)
        choice = by_group.masked_fill(~kept.unsqueeze(2), -math.inf).view(t, e)
    experts = _best(choice, c["topk"])
    score = score.float()
    picked = score.gather(1, experts)
    total = picked.sum(dim=1, keepdim=True)
    weights = picked / total * c["scale"] if c["renorm"] else picked * c["scale"]
    if not c["train"]:
        return experts.int(), weights
    g = s["grad"] * c["scale"]
    ds = (g - (g * picked).sum(dim=1, keepdim=True) / total) / total if c["renorm"] else g
    if c["score"] == "softmax":
        dense = torch.zeros_like(score).scatter_(1, experts, ds)
        grad = score * (dense - (ds * picked).sum(dim=1, keepdim=True))
    else:
        grad = torch.zeros_like(score).scatter_(1, experts, ds * picked * (1.0 - picked))
    return experts.int(), weights, grad.to(s["logits"].dtype)


_GELU_A, _GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def _act_and_slope(g, act):
    if act == "silu":
        sig = 1.0 / (1.0 + (-g).exp())
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if act == "relu":
        return g.clamp(min=0.0), (g > 0).to(g.dtype)
    th = (_GELU_A * (g + _GELU_B * g * g * g)).tanh()
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * _GELU_A * (1.0 + 3.0 * _GELU_B * g * g)


def _plain_gated(s, c):
    f, dt = c["ffn"], s["gate"].dtype
    g = (s["gate"][:, :f] if c["packed"] else s["gate"]).float()
    u = (s["gate"][:, f:] if c["packed"] else s["up"]).float()
    live = None
    if c["counted"]:
        live = torch.arange(c["rows"], device=g.device).unsqueeze(1) < s["num_rows"]
    a, slope = _act_and_slope(g, c["act"])
    r = s["row_weight"].unsqueeze(1) if c["weighted"] else 1.0
    mask = (lambda t: t) if live is None else (lambda t: torch.where(live, t, torch.zeros_like(t)))
    y = mask(r * a * u).to(dt)
    if not c["train"]:
        return y
    dy = s["grad"].float()
    dg, du = mask(r * dy * u * slope).to(dt), mask(r * dy * a).to(dt)
    grads = (torch.cat([dg, du], dim=1),) if c["packed"] else (dg, du)
    if c["weighted"]:
        grads += (mask((dy * a * u).sum(dim=1, keepdim=True)).squeeze(1),)
    return (y,) + grads


def _plain_weight(q, scales, zeros, group):
    low, high = q & 15, q >> 4
    w = torch.stack([low, high], dim=-1).view(q.shape[0], -1, group).float()
    z = 8.0 if zeros is None else zeros.float().unsqueeze(2)
    return ((w - z) * scales.float().unsqueeze(2)).view(q.shape[0], -1)


def _plain_int4(s, c):
    y = s["x"].float() @ _plain_weight(s["q"], s["scales"], s["zeros"], c["group"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_int4_moe(s, c):
    y = torch.empty(s["x"].shape[0], c["n"], dtype=s["x"].dtype, device=DEVICE)
    row = 0
    for e, count in enumerate(s["host_splits"]):
        if count:
            w = _plain_weight(s["q"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e], c["group"])
            y[row:row + count] = s["x"][row:row + count].float() @ w.t()
        row += count
    return y


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    plain = {"route": _plain_route, "gated": _plain_gated, "int4": _plain_int4, "int4_moe": _plain_int4_moe}[c["kind"]]
    return plain(state, c)


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_route(s, c):
    x = s["logits"].double()
    t, e = x.shape
    score = torch.softmax(x, dim=1) if c["score"] == "softmax" else torch.sigmoid(x)
    choice = score.clone()
    if s["bias"] is not None:
        choice += s["bias"].double()
    size = e // c["groups"]
    lowest = torch.full_like(choice, -math.inf)
    if c["groups"] > 1:
        left = choice.view(t, c["groups"], size).clone()
        total = torch.zeros(t, c["groups"], dtype=torch.float64, device=x.device)
        for _ in range(min(c["group_top"], size)):
            top, place = left.max(dim=2, keepdim=True)
            total += top.squeeze(2)
            left.scatter_(2, place, -math.inf)
        allowed = torch.zeros(t, c["groups"], dtype=torch.bool, device=x.device)
        for _ in range(c["topk_groups"]):
            allowed.scatter_(1, _first_max(total), True)
            total.masked_fill_(allowed, -math.inf)
        choice = torch.where(allowed.repeat_interleave(size, dim=1), choice, lowest)
    experts = []
    for _ in range(c["topk"]):
        place = _first_max(choice)
        experts.append(place)
        choice = choice.scatter(1, place, -math.inf)
    experts = torch.cat(experts, dim=1)
    p = score.gather(1, experts)
    norm = p.sum(dim=1, keepdim=True) if c["renorm"] else torch.ones_like(p[:, :1])
    w = c["scale"] * p / norm
    if not c["train"]:
        return experts.int(), w
    # L = sum_i grad_i w_i; with w = scale p / norm and norm = sum p (or 1)
    grad = s["grad"].double()
    dp = c["scale"] * grad / norm
    if c["renorm"]:
        dp = dp - (grad * w).sum(dim=1, keepdim=True) / norm
    ds = torch.zeros_like(score)
    ds.scatter_(1, experts, dp)
    if c["score"] == "softmax":
        dx = score * (ds - (ds * score).sum(dim=1, keepdim=True))
    else:
        dx = ds * score * (1.0 - score)
    return experts.int(), w, dx


def _first_max(values):
    """[rows, 1]: the lowest place of each row's largest value."""
    top = values.max(dim=1, keepdim=True).values
    places = torch.arange(values.shape[1], device=values.device).expand_as(values)
    return torch.where(values == top, places, values.shape[1]).min(dim=1, keepdim=True).values


def _exact_gated_part(g, u, r, dy, act):
    g, u = g.double(), u.double()
    if act == "silu":
        a, da = g * torch.sigmoid(g), torch.sigmoid(g) + g * torch.sigmoid(g) * torch.sigmoid(-g)
    elif act == "relu":
        a, da = torch.relu(g), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    else:
        inner = math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
        a = 0.5 * g * (1.0 + torch.tanh(inner))
        da = 0.5 * (1.0 + torch.tanh(inner)) + (0.5 * g / torch.cosh(inner) ** 2
                                                * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * g ** 2))
    r = torch.ones_like(g[:, :1]) if r is None else r.double().unsqueeze(1)
    if dy is None:
        return r * a * u, None, None, None
    dy = dy.double()
    return r * a * u, dy * r * u * da, dy * r * a, (dy * a * u).sum(dim=1)


def _exact_gated(s, c):
    f, rows = c["ffn"], c["rows"]
    live = int(s["num_rows"]) if c["counted"] else rows
    kinds = 4 if c["train"] else 1
    parts = [[] for _ in range(kinds)]
    for lo in range(0, live, 4096):
        hi = min(lo + 4096, live)
        both = s["gate"][lo:hi]
        g, u = (both[:, :f], both[:, f:]) if c["packed"] else (both, s["up"][lo:hi])
        r = s["row_weight"][lo:hi] if c["weighted"] else None
        got = _exact_gated_part(g, u, r, s["grad"][lo:hi] if c["train"] else None, c["act"])
        for kept, t in zip(parts, got):
            kept.append(t)
    out = []
    for kept in parts:
        t = torch.cat(kept)
        out.append(torch.cat([t, t.new_zeros((rows - live,) + t.shape[1:])]))
    if not c["train"]:
        return out[0]
    y, dg, du, dr = out
    return (y,) + ((torch.cat([dg, du], dim=1),) if c["packed"] else (dg, du)) + ((dr,) if c["weighted"] else ())


def _exact_linear(x, q, scales, zeros, group):
    """x [m, k] times the weights (q - z) * s, a few thousand output columns at a time."""
    n, k = q.shape[0], 2 * q.shape[1]
    cols = max(1, 2 ** 26 // k)
    out = []
    for lo in range(0, n, cols):
        part = q[lo:lo + cols]
        w = torch.empty(part.shape[0], k, dtype=torch.float64, device=q.device)
        w[:, 0::2] = part.remainder(16).double()
        w[:, 1::2] = part.div(16, rounding_mode="floor").double()
        which = torch.arange(k, device=q.device) // group
        w -= 8.0 if zeros is None else zeros[lo:lo + cols].double()[:, which]
        w *= scales[lo:lo + cols].double()[:, which]
        out.append(torch.matmul(x.double(), w.t()))
    return torch.cat(out, dim=1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "route":
        return _exact_route(s, case)
    if case["kind"] == "gated":
        return _exact_gated(s, case)
    if case["kind"] == "int4":
        y = _exact_linear(s["x"], s["q"], s["scales"], s["zeros"], case["group"])
        return y if s["bias"] is None else y + s["bias"].double()
    out, row = [], 0
    for e, count in enumerate(s["splits"].tolist()):
        if count:
            out.append(_exact_linear(s["x"][row:row + count], s["q"][e], s["scales"][e],
                                     None if s["zeros"] is None else s["zeros"][e], case["group"]))
        row += count
    return torch.cat(out)


# ------------------------------------------------------------------------------------------ work
def work(case):
    kind, elt = case["kind"], SIZE[case["dtype"]]
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        passes = 2 if case["train"] else 1
        bytes_ = t * e * elt + t * k * 8 + (4 * e if case["bias"] else 0)
        if case["train"]:
            bytes_ += t * k * 4 + t * e * elt
        return {"bytes": bytes_, "flops": passes * 4 * t * e}
    if kind == "gated":
        r, f = case["rows"], case["ffn"]
        live = r - r // 10 if case["counted"] else r
        bytes_ = live * 2 * f * elt + r * f * elt + (4 * live if case["weighted"] else 0)
        if case["train"]:
            bytes_ += live * f * elt + r * 2 * f * elt + (4 * r if case["weighted"] else 0)
        return {"bytes": bytes_, "flops": live * f * (16 if case["train"] else 6)}
    n, k = case["n"], case["k"]
    weights = n * k // 2 + n * (k // case["group"]) * (elt + (1 if case["zeros"] else 0))
    if kind == "int4":
        m = case["m"]
        return {"bytes": weights + elt * (m * k + m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    e, topk = case["experts"], min(case["topk"], case["experts"])
    rows = case["tokens"] * topk
    # (experts that a token out of ``tokens`` chooses, were all equally popular)
    used = e * (1.0 - (1.0 - topk / e) ** case["tokens"])
    return {"bytes": int(used * weights) + elt * rows * (k + n) + 4 * e, "flops": 2 * rows * n * k}
