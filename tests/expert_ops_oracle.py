"""Plain statements in 64 bits of routing, gated activation and 4-bit products, row by row, and the error bounds of the
kernels. Written from the definitions, apart from the library's own PyTorch statements."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}    # half a step, relative
# smallest step of the type (results below the normal range are rounded to it)
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def _rank(value, index):
    """Sort key: largest first, NaN behind everything, then the lower index."""
    return (1, 0.0, index) if math.isnan(value) else (0, -value, index)


def _sigmoid(v):
    return 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0


def route_choice(logits, topk, score, bias=None, groups=1, topk_groups=1, group_top=1):
    """[tokens][topk] expert indices of logits [tokens, E] (a CPU tensor)."""
    out = []
    for row in logits.double().tolist():
        if score == "sigmoid":
            s = [_sigmoid(v) if not math.isnan(v) else v for v in row]
        else:
            top = max(row)
            if any(map(math.isnan, row)):
                s = [math.nan] * len(row)                      # (a NaN reaches the whole sum)
            elif top == -math.inf:
                s = [0.0] * len(row)
            else:
                p = [math.exp(v - top) for v in row]
                s = [v / math.fsum(p) for v in p]
        # (without a bias the order of the scores is that of the logits)
        choice = row if bias is None else [a + b for a, b in zip(s, bias.double().tolist())]
        ranked_by = choice if bias is not None or group_top == 1 else s
        size = len(row) // groups
        best = []
        for g in range(groups):
            inside = sorted(ranked_by[g * size:(g + 1) * size], key=lambda v: _rank(v, 0))
            best.append(sum(inside[:group_top]))
        kept = sorted(range(groups), key=lambda g: _rank(best[g], g))[:topk_groups]
        inside = [e for e in range(len(row)) if groups == 1 or e // size in kept]
        out.append(sorted(inside, key=lambda e: _rank(choice[e], e))[:topk])
    return torch.tensor(out, dtype=torch.int64)


def route_weights(logits, experts, score, renorm, scale):
    """Weights and, as a function of the gradient, the logits' gradient with its bound; 64 bits."""
    x = logits.double()
    chosen = x.gather(1, experts)
    if score == "softmax":
        p_all = torch.softmax(x, dim=1)
        p = p_all.gather(1, experts)
        own = torch.softmax(chosen, dim=1)                     # over the chosen ones
        share = own
    else:
        p_all, p = torch.sigmoid(x), torch.sigmoid(chosen)
        log = torch.nn.functional.logsigmoid(chosen)
        share = torch.softmax(log, dim=1)
    w = scale * (share if renorm else p)

    def grad(g):
        g = g.double()
        dot, size = (w * g).sum(1, keepdim=True), (w * g).abs().sum(1, keepdim=True)
        d, b = torch.zeros_like(x), torch.zeros_like(x)
        if renorm:
            part, bound = w * (g - dot / scale), w.abs() * (g.abs() + size / abs(scale))
        else:
            part, bound = w * g, (w * g).abs()
        if score == "sigmoid":
            part, bound = part * torch.sigmoid(-chosen), bound * torch.sigmoid(-chosen)
        if score == "softmax" and not renorm:
            d, b = -p_all * dot, p_all * size
        return d.scatter_add(1, experts, part), b.scatter_add(1, experts, bound)

    return w, grad


# relative error of a weight in units of 2^-24: the difference of two logits (|l| up to 32 here) and its exponential
# (32 + 4), sums of up to 512 positive terms, 16 in a lane and five steps across lanes (21), quotient and scale (2)
ROUTE_RTOL = 64 * 2.0 ** -24


def gated(gate, up, act, weight=None, dy=None):
    """(y, dgate, dup, dweight) and their bounds for the fp32 arithmetic, all in 64 bits. Units of 2^-24: exp 4, the inner
    argument 6 |z| for gelu and 0 otherwise, quotient and products 8."""
    g, u = gate.double(), up.double()
    if act == "relu":
        z = torch.zeros_like(g)
        a, da, da_size = torch.clamp(g, min=0.0), (g > 0).double(), (g > 0).double()
    else:
        z = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        dz = torch.ones_like(g) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
        s = torch.sigmoid(z)
        a, da = g * s, s + g * dz * s * torch.sigmoid(-z)
        # (1 - s is taken in 32 bits: its error is one unit of 1)
        da_size = s + (g * dz * s).abs() * (torch.sigmoid(-z) + 2.0 ** -2)
    unit = 2.0 ** -24 * (16 + 8 * z.abs())
    # Below 2^-126 fp32 has steps of 2^-149 whatever the value, so the relative bounds end there. exp(-|z|) and the products
    # that follow (at most four, each factor after the first at most `scale` in all) are each off by half such a step, and
    # what is off by then is multiplied by the factors that are still to come: 5 * 2^-150 * max(1, scale) together.
    low = 5 * 2.0 ** -150
    r = torch.ones_like(g[:, :1]) if weight is None else weight.double().unsqueeze(1)
    y = r * a * u
    if dy is None:
        return y, y.abs() * unit + low * (1 + g.abs()) * (1 + u.abs()) * (1 + r.abs())
    d = dy.double()
    terms = d * a * u
    n = g.shape[1]
    slope = 1 + (g.abs() if act != "relu" else 0) * (dz if act != "relu" else 1)
    scale = low * (1 + g.abs()) * (1 + d.abs()) * (1 + r.abs())
    return ((y, r * d * u * da, r * d * a, terms.sum(1)),
            (y.abs() * unit + low * (1 + g.abs()) * (1 + u.abs()) * (1 + r.abs()),
             (r * d * u).abs() * da_size * unit + scale * (1 + u.abs()) * slope, (r * d * a).abs() * unit + scale,
             (terms.abs() * (unit + 2.0 ** -24 * (n / 32 + 16)) + scale * (1 + u.abs())).sum(1)))


def weights4(q, scales, zeros, group):
    """[N, K] in 64 bits, column by column of the bytes."""
    n, half = q.shape
    w = torch.empty(n, 2 * half, dtype=torch.float64, device=q.device)
    w[:, 0::2] = (q % 16).double()
    w[:, 1::2] = (q // 16).double()
    at = torch.arange(2 * half, device=q.device) // group
    return (w - (8.0 if zeros is None else zeros.double()[:, at])) * scales.double()[:, at]


def product4(x, w, group, bias=None):
    """x @ w^T (+ bias) and its bound: the tensor cores add 16 products to a sum at a time (one unit of 2^-23 of the
    magnitudes each, for sums that are cut off instead of rounded), then groups, warps and blocks are added in fp32."""
    y, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    k = x.shape[1]
    unit = 2.0 ** -23 * (min(group, 128) / 16 + k / min(group, 128) + 16)
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size * unit


def assert_within(got, ref, bound, what=""):
    """|got - ref| <= bound + half a step of got's type."""
    limit = bound + EPS[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    error = (got.double() - ref).abs()
    bad = ~(error <= limit)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(error / limit).max():.3g} of the limit"
