"""Routing, gated activation and 4-bit products on the GPU against plain statements in 64 bits."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda", 0)


@pytest.fixture(scope="module")
def flux():
    import tempname_new_b200
    return tempname_new_b200


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


# ------------------------------------------------------------------------------------------ routing
ROUTES = [
    # tokens, experts, topk, score, bias, groups, topk_groups, group_top, renorm, scale
    (1, 1, 1, "softmax", False, 1, 1, 1, True, 1.0),
    (5, 8, 2, "softmax", False, 1, 1, 1, False, 1.0),
    (64, 64, 8, "softmax", False, 1, 1, 1, True, 1.0),
    (33, 65, 6, "sigmoid", True, 1, 1, 1, True, 2.5),
    (130, 120, 6, "softmax", True, 1, 1, 1, False, 1.0),
    (67, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (31, 160, 6, "softmax", False, 8, 3, 1, False, 16.0),
    (40, 96, 8, "softmax", True, 4, 2, 2, True, 1.0),
    (29, 60, 4, "sigmoid", False, 5, 2, 2, False, 1.0),
    (17, 512, 32, "sigmoid", True, 32, 31, 2, True, 1.0),
    (9, 511, 32, "softmax", False, 1, 1, 1, True, -0.5),
    (12, 264, 8, "sigmoid", False, 1, 1, 1, True, 1.0),
]


def _route_inputs(dev, tokens, experts, bias, dtype):
    g = _gen(dev, tokens * 1000 + experts)
    x = (torch.randn(tokens, experts, device=dev, generator=g) * 2).clamp(-8, 8).to(dtype)
    return x, torch.randn(experts, device=dev, generator=g) * 0.1 if bias else None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ROUTES, ids=lambda c: "-".join(map(str, c[:6])))
def test_route(dev, flux, case, dtype):
    tokens, experts, topk, score, has_bias, groups, topk_groups, group_top, renorm, scale = case
    x, bias = _route_inputs(dev, tokens, experts, has_bias, dtype)
    x.requires_grad_(True)
    idx, w = flux.moe_route(x, topk, score, bias, groups, topk_groups, group_top, renorm, scale)
    ref = oracle.route_choice(x.detach().cpu(), topk, score, None if bias is None else bias.cpu(), groups, topk_groups,
                              group_top)
    assert idx.dtype == torch.int32 and torch.equal(idx.cpu().long(), ref)
    w_ref, grad_of = oracle.route_weights(x.detach(), idx.long(), score, renorm, scale)
    oracle.assert_within(w, w_ref, w_ref.abs() * oracle.ROUTE_RTOL, "weights")
    gw = torch.randn(tokens, topk, device=dev, generator=_gen(dev, 5))
    dx, = torch.autograd.grad(w, x, gw)
    d_ref, d_size = grad_of(gw)
    assert dx.dtype == dtype
    oracle.assert_within(dx, d_ref, d_size * 2 * oracle.ROUTE_RTOL, "gradient")
    # without gradients: the same numbers
    with torch.no_grad():
        idx2, w2 = flux.moe_route(x, topk, score, bias, groups, topk_groups, group_top, renorm, scale)
    assert torch.equal(idx, idx2) and torch.equal(w.detach(), w2)


def test_route_ties_and_neighbours(dev, flux):
    """Equal logits go to the lower index; scores that 32 bits cannot tell apart are ordered all the same."""
    x = torch.zeros(4, 96, device=dev)
    x[1, 40:] = 1.0
    x[2] = -0.0
    x[2, 5] = 0.0
    x[3] = torch.arange(96, device=dev) % 3
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(96, device=dev)):
            idx, _ = flux.moe_route(x, 8, score, bias)
            ref = oracle.route_choice(x.cpu(), 8, score, None if bias is None else bias.cpu())
            assert torch.equal(idx.cpu().long(), ref), (score, bias is not None)
    # sigmoid(l) + b with values one rounding of 32 bits apart
    g = _gen(dev, 3)
    n = 2000
    base = torch.randn(n, 1, device=dev, generator=g)
    x = base + torch.randint(-3, 4, (n, 64), device=dev, generator=g) * 2.0 ** -23
    bias = torch.randint(-1, 2, (64,), device=dev, generator=g) * 2.0 ** -25
    for groups, keep, top in ((1, 1, 1), (8, 4, 2), (8, 2, 1)):
        for score in ("sigmoid", "softmax"):
            idx, _ = flux.moe_route(x, 6, score, bias, groups, keep, top)
            ref = oracle.route_choice(x.cpu(), 6, score, bias.cpu(), groups, keep, top)
            assert torch.equal(idx.cpu().long(), ref), (groups, score)
    # saturated scores keep the order of their logits
    x = torch.linspace(20, 80, 64, device=dev).flip(0).repeat(3, 1)
    idx, _ = flux.moe_route(x, 5, "sigmoid")
    assert idx.cpu().tolist() == [[0, 1, 2, 3, 4]] * 3


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_masked_and_nan(dev, flux, score, renorm):
    inf, nan = math.inf, math.nan
    lowest = torch.finfo(torch.float32).min
    rows = [[-inf] * 8, [-inf] * 6 + [1.0, -inf], [lowest] * 8, [lowest] * 7 + [0.0], [nan] + [0.0] * 7,
            [-inf, nan] + [-inf] * 6, [-90.0, -95.0, -100.0, -91.0] + [-inf] * 4, [nan] * 8]
    x = torch.tensor(rows, device=dev, requires_grad=True)
    for bias in (None, torch.linspace(0.5, -0.5, 8, device=dev)):
        idx, w = flux.moe_route(x, 3, score, bias, renormalize=renorm)
        ref = oracle.route_choice(x.detach().cpu(), 3, score, None if bias is None else bias.cpu())
        assert torch.equal(idx.cpu().long(), ref), bias is None
        cpu_idx, cpu_w = flux.moe_route(x.detach().cpu(), 3, score, None if bias is None else bias.cpu(), renormalize=renorm)
        assert torch.equal(cpu_idx.long(), ref)
        torch.testing.assert_close(w.detach().cpu(), cpu_w, rtol=2.0 ** -17, atol=2.0 ** -140, equal_nan=True)
        assert w[0].tolist() == [0.0, 0.0, 0.0]                     # nothing left: weights of zero
        dx, = torch.autograd.grad(w.sum(), x, retain_graph=True)
        assert bool((dx[0] == 0).all()) and bool(torch.isfinite(dx[1:4]).all())


def test_route_strides_streams_and_graphs(dev, flux):
    g = _gen(dev, 11)
    wide = torch.randn(50, 200, device=dev, generator=g)
    for x in (wide[:, 3:131], wide[:, :128], wide.t()[:64].t(), wide[::2, 8:136]):
        idx, w = flux.moe_route(x, 4, "sigmoid")
        idx2, w2 = flux.moe_route(x.contiguous(), 4, "sigmoid")
        assert torch.equal(idx, idx2) and torch.equal(w, w2)
    assert flux.moe_route(wide[:0], 4)[0].shape == (0, 4)
    x = torch.randn(300, 128, device=dev, generator=g)
    want = flux.moe_route(x, 6, num_groups=4, topk_groups=2, group_top=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = flux.moe_route(x, 6, num_groups=4, topk_groups=2, group_top=2)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf, gw = torch.zeros_like(x).requires_grad_(True), torch.randn(300, 6, device=dev, generator=g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gi, gwt = flux.moe_route(buf, 6, num_groups=4, topk_groups=2, group_top=2)
        gdx, = torch.autograd.grad(gwt, buf, gw)
    with torch.no_grad():
        buf.copy_(x)
    graph.replay()
    x.requires_grad_(True)
    dx, = torch.autograd.grad(flux.moe_route(x, 6, num_groups=4, topk_groups=2, group_top=2)[1], x, gw)
    assert torch.equal(gi, want[0]) and torch.equal(gwt.detach(), want[1]) and torch.equal(gdx, dx)


def test_route_gradient_by_differences(dev, flux):
    """Central differences of the kernel's own weights in directions that do not change the choice."""
    g = _gen(dev, 21)
    x = torch.randn(6, 16, device=dev, generator=g) + torch.arange(16, device=dev) * 0.5
    h = 2.0 ** -7
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            xr = x.clone().requires_grad_(True)
            idx, w = flux.moe_route(xr, 4, score, renormalize=renorm)
            gw = torch.randn(6, 4, device=dev, generator=g)
            dx, = torch.autograd.grad(w, xr, gw)
            for e in range(16):
                step = torch.zeros_like(x)
                step[:, e] = h
                (ia, wa), (ib, wb) = flux.moe_route(x + step, 4, score, renormalize=renorm), \
                    flux.moe_route(x - step, 4, score, renormalize=renorm)
                same = ((ia == idx) & (ib == idx)).all(1)
                slope = ((wa - wb).double() * gw).sum(1) / (2 * h)
                # third derivatives of the weights stay below 1: h^2 / 6 each; two roundings of 32 bits over 2 h
                limit = gw.abs().sum(1) * (h * h / 6 + 2 * oracle.ROUTE_RTOL / (2 * h)) + 1e-6
                assert bool((((slope - dx[:, e]).abs() <= limit) | ~same).all()), (score, renorm, e)


# ------------------------------------------------------------------------------------------ gated activation
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,cols,packed", [(1, 1, False), (3, 1, True), (7, 33, False), (5, 36, True), (64, 1536, True),
                                              (130, 1001, True), (130, 1001, False), (9, 8200, True), (300, 64, False)])
def test_gated(dev, flux, rows, cols, packed, act, dtype):
    g = _gen(dev, rows * 10000 + cols)
    gate = (torch.randn(rows, cols, device=dev, generator=g) * 4).to(dtype)
    up = torch.randn(rows, cols, device=dev, generator=g).to(dtype)
    dy = torch.randn(rows, cols, device=dev, generator=g).to(dtype)
    for weighted in (False, True):
        weight = torch.randn(rows, device=dev, generator=g) if weighted else None
        leaves = [torch.cat([gate, up], 1)] if packed else [gate.clone(), up.clone()]
        leaves = [t.requires_grad_(True) for t in leaves + ([weight] if weighted else [])]
        y = flux.gated_act(leaves[0], None if packed else leaves[1], act, leaves[-1] if weighted else None)
        grads = torch.autograd.grad(y, leaves, dy)
        dg, du = (grads[0][:, :cols], grads[0][:, cols:]) if packed else grads[:2]
        refs, bounds = oracle.gated(gate, up, act, weight, dy)
        got = (y.detach(), dg, du) + ((grads[-1],) if weighted else ())
        for name, t, ref, bound in zip(("y", "dgate", "dup", "dweight"), got, refs, bounds):
            oracle.assert_within(t, ref, bound, name)
        with torch.no_grad():
            assert torch.equal(y, flux.gated_act(leaves[0], None if packed else leaves[1], act, weight))


@pytest.mark.parametrize("count_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("count", [0, 1, 37, 50, 99, -3])
def test_gated_rows_in_use(dev, flux, count, count_type):
    """Rows behind the count: zeros in a fresh result and in the gradients, untouched in a given buffer, never read into
    the others."""
    g = _gen(dev, 8)
    both = torch.randn(50, 2 * 70, device=dev, generator=g).bfloat16()
    n = max(0, min(50, count))
    both[n:] = math.nan
    weight = torch.rand(50, device=dev, generator=g)
    num = torch.tensor([count], device=dev, dtype=count_type)
    ref, bound = oracle.gated(both[:n, :70], both[:n, 70:], "silu", weight[:n])
    y = flux.gated_act(both, row_weight=weight, num_rows=num)
    oracle.assert_within(y[:n], ref, bound)
    assert bool((y[n:] == 0).all())
    out = torch.full((52, 80), 7.0, device=dev, dtype=torch.bfloat16)
    assert flux.gated_act(both, row_weight=weight, num_rows=num, out=out[:50, :70]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:n, :70], y[:n]) and bool((out[n:] == 7).all()) and bool((out[:, 70:] == 7).all())
    both.requires_grad_(True), weight.requires_grad_(True)
    y = flux.gated_act(both, row_weight=weight, num_rows=num)
    db, dw = torch.autograd.grad(y, (both, weight), torch.ones_like(y))
    assert bool((db[n:] == 0).all()) and bool((dw[n:] == 0).all()) and bool(torch.isfinite(db).all())


def test_gated_values_at_the_edges(dev, flux):
    """Large magnitudes, both infinities, NaN: as the formula has them, gradients finite wherever the inputs are."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 80.0, -80.0, 3e4, -3e4, 1e30, -1e30, math.inf, math.nan], device=dev)
    one = torch.ones_like(v).unsqueeze(0)
    for act in ("silu", "gelu", "relu"):
        gate = v.unsqueeze(0).clone().requires_grad_(True)
        y = flux.gated_act(gate, one, act)
        d, = torch.autograd.grad(y, gate, one)
        assert bool(torch.isfinite(y[0, :10]).all()) and bool(torch.isfinite(d[0, :10]).all()), act
        assert math.isnan(y[0, 11]) and y[0, 10] == math.inf
        assert d[0, 8] == 1.0 and d[0, 9] == 0.0


def test_gated_strides_streams_and_graphs(dev, flux):
    g = _gen(dev, 9)
    wide = torch.randn(40, 400, device=dev, generator=g).half()
    for gate, up in ((wide[:, :96], wide[:, 96:192]), (wide[:, 1:97], wide[:, 200:296]), (wide[::2, :64], wide[1::2, 4:68]),
                     (wide.t()[:40].t(), wide.t()[40:80].t()), (wide[:1].expand(40, 400), wide)):
        assert torch.equal(flux.gated_act(gate, up), flux.gated_act(gate.contiguous(), up.contiguous()))
    # a broadcast input gets the sum of its rows' gradients; a gradient that is itself broadcast is fine
    leaf = wide[:1].clone().requires_grad_(True)
    y = flux.gated_act(leaf.expand(40, 400), wide)
    d, = torch.autograd.grad(y.sum(), leaf)
    full = wide[:1].repeat(40, 1).requires_grad_(True)
    d2, = torch.autograd.grad(flux.gated_act(full, wide).sum(), full)
    torch.testing.assert_close(d[0].float(), d2.float().sum(0), rtol=2.0 ** -10, atol=2.0 ** -6)
    assert flux.gated_act(wide[:0]).shape == (0, 200) and flux.gated_act(wide[:, :0]).shape == (40, 0)
    want = flux.gated_act(wide)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = flux.gated_act(wide)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    buf = torch.zeros_like(wide).requires_grad_(True)
    weight = torch.rand(40, device=dev, generator=g).requires_grad_(True)
    num = torch.tensor([40], device=dev, dtype=torch.int32)
    dy = torch.randn(40, 200, device=dev, generator=g).half()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy = flux.gated_act(buf, row_weight=weight, num_rows=num)
        gd = torch.autograd.grad(gy, (buf, weight), dy)
    for n in (40, 13):
        with torch.no_grad():
            buf.copy_(wide)
        num.fill_(n)
        graph.replay()
        x = wide.clone().requires_grad_(True)
        y = flux.gated_act(x, row_weight=weight, num_rows=num)
        d = torch.autograd.grad(y, (x, weight), dy)
        assert torch.equal(gy, y) and all(torch.equal(a, b) for a, b in zip(gd, d))


def test_gated_in_place(dev, flux):
    """The result may go where the gate, the up values or the gate's half of both were."""
    x = torch.randn(33, 2 * 1000, device=dev, generator=_gen(dev, 10)).bfloat16()
    for cols in (1000, 999, 64, 3):
        both = x[:, :2 * cols]
        want = flux.gated_act(both)
        for place in range(3):
            work = both.clone()
            gate, up = work[:, :cols], work[:, cols:]
            if place == 0:
                got = flux.gated_act(work, out=gate)
            else:
                got = flux.gated_act(gate, up, out=gate if place == 1 else up)
            assert torch.equal(got, want)
            assert torch.equal(*((up, both[:, cols:]) if place < 2 else (gate, both[:, :cols])))


def test_tangents_are_refused(dev, flux):
    """Forward-mode derivatives have no rule on the device: an error, not a result without its tangent."""
    x = torch.randn(4, 16, device=dev, generator=_gen(dev, 11))
    q, s, _ = _made4(dev, (), 8, 128, 128, False, 1)
    wide = torch.ones(4, 128, device=dev, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: flux.moe_route(dual, 2), lambda: flux.gated_act(dual), lambda: flux.gated_act(x, dual),
                  lambda: flux.Int4Gemm(q, s).forward(forward_ad.make_dual(wide, torch.ones_like(wide)))):
            with pytest.raises(RuntimeError):
                f()
        assert flux.gated_act(x).shape == (4, 8) and flux.moe_route(x, 2)[0].shape == (4, 2)


# ------------------------------------------------------------------------------------------ 4-bit products
def _made4(dev, lead, n, k, group, zeros, seed, scale_dtype=torch.bfloat16):
    g = _gen(dev, seed)
    q = torch.randint(0, 256, (*lead, n, k // 2), device=dev, dtype=torch.uint8, generator=g)
    s = (torch.rand((*lead, n, k // group), device=dev, generator=g) + 0.25).mul_(0.1).to(scale_dtype)
    z = torch.randint(0, 16, (*lead, n, k // group), device=dev, dtype=torch.uint8, generator=g) if zeros else None
    return q, s, z


SHAPES4 = [
    # M, N, K, group
    (1, 64, 128, 128), (1, 1, 32, 32), (2, 5, 96, 32), (3, 100, 64, 64), (7, 129, 192, 64), (8, 64, 1024, 128),
    (9, 200, 2176, 128), (16, 333, 512, 32), (17, 64, 256, 256), (24, 192, 4096, 128), (31, 130, 640, 64), (32, 128, 384, 128),
    (33, 128, 128, 32), (47, 257, 4128, 32), (64, 512, 256, 128), (65, 72, 1152, 128), (100, 1000, 320, 64),
    (128, 256, 4096, 64), (129, 384, 512, 512), (200, 640, 96, 32), (257, 130, 1024, 128), (513, 300, 2048, 64),
    (1, 4096, 8192, 128), (5, 9000, 2048, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", SHAPES4)
def test_int4_exact_integers(dev, flux, m, n, k, group, zeros, dtype):
    """Small integers and scales of powers of two: every sum is exact in 32 bits, so the result is the exactly rounded one
    and any misplaced weight, scale, zero point or activation shows."""
    g = _gen(dev, m * 7 + n * 3 + k)
    q, s, z = _made4(dev, (), n, k, group, zeros, k + n)
    s = (2.0 ** torch.randint(-3, 1, s.shape, device=dev, generator=g)).to(dtype)
    x = torch.randint(-4, 5, (m, k), device=dev, generator=g).to(dtype) / (64 if dtype == torch.float16 else 1)
    y = flux.Int4Gemm(q, s, z).forward(x)
    ref = x.double() @ oracle.weights4(q, s, z, group).t()
    assert torch.equal(y, ref.to(dtype))


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                               (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("m,n,k,group", SHAPES4)
def test_int4(dev, flux, m, n, k, group, dtype, scale_dtype):
    g = _gen(dev, m + n + k)
    for zeros, biased in ((False, False), (True, True)):
        q, s, z = _made4(dev, (), n, k, group, zeros, m + k, scale_dtype)
        x = torch.randn(m, k, device=dev, generator=g).to(dtype)
        bias = torch.randn(n, device=dev, generator=g).to(dtype) if biased else None
        y = flux.Int4Gemm(q, s, z).forward(x, bias=bias)
        ref, bound = oracle.product4(x, oracle.weights4(q, s, z, group), group, bias)
        assert y.dtype == dtype
        oracle.assert_within(y, ref, bound)


# (m, n, k) -> the kernel, rows of x per tile and CTAs per tile that the rules choose on 148 SMs
VARIANTS4 = [
    (1, 16400, 256, "int4_rows", 8, 1), (7, 9400, 8448, "int4_rows", 8, 2), (8, 1000, 4096, "int4_rows", 8, 4),
    (3, 600, 8192, "int4_rows", 8, 4), (9, 16300, 384, "int4_rows", 16, 1), (16, 520, 16384, "int4_rows", 16, 4),
    (17, 300, 128, "int4_tiles", 32, 1), (40, 1000, 1024, "int4_tiles", 32, None), (100, 1000, 8192, "int4_tiles", 32, None),
    (33, 5003, 4224, "int4_tiles", None, 3), (200, 700, 4096, "int4_tiles", 64, None),
    (60, 16384, 1024, "int4_tiles", 64, 1), (57, 16001, 640, "int4_tiles", 64, 1), (64, 5000, 6144, "int4_tiles", None, None),
    (120, 16384, 1024, "int4_tiles", 128, 1), (101, 15999, 1152, "int4_tiles", 128, 1),
    (512, 8192, 1024, "int4_tiles", 256, 1), (433, 8100, 1152, "int4_tiles", 256, 1), (385, 8192, 1024, "int4_tiles", 256, 1),
    (900, 2000, 4096, "int4_tiles", 256, None),
]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k,kernel,rows,splits", VARIANTS4)
def test_int4_variants(dev, flux, m, n, k, kernel, rows, splits, group):
    """Every kernel, tile and split with every group size, on integers whose sums are exact (as above)."""
    g = _gen(dev, m + n)
    q, s, z = _made4(dev, (), n, k, group, True, k)
    s = (2.0 ** torch.randint(-3, 1, s.shape, device=dev, generator=g)).bfloat16()
    x = torch.randint(-3, 4, (m, k), device=dev, generator=g).bfloat16()
    bias = torch.randint(-8, 9, (n,), device=dev, generator=g).bfloat16()
    op = flux.Int4Gemm(q, s, z)
    y = op.forward(x, bias=bias)
    took = flux._native.last_gemm()
    assert took["kernel"] == kernel
    if group == 128:
        assert rows in (None, took["tile_m"]) and splits in (None, took["splits"]), took
    ref = x.double() @ oracle.weights4(q, s, z, group).t() + bias.double()
    assert torch.equal(y, ref.bfloat16())
    op.check_status()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("splits,n,k", [([600, 0, 257, 300], 8192, 1024), ([128, 129, 127, 1, 0, 383], 4000, 1152),
                                        ([3, 0, 40, 8], 16000, 640), ([0, 5, 0, 0], 300, 4096), ([70, 60, 64, 1], 8200, 1024)])
def test_int4_grouped_variants(dev, flux, splits, n, k, group):
    g = _gen(dev, n + k)
    rows, E = sum(splits), len(splits)
    q, s, z = _made4(dev, (E,), n, k, group, True, k)
    s = (2.0 ** torch.randint(-3, 1, s.shape, device=dev, generator=g)).half()
    x = torch.randint(-3, 4, (rows, k), device=dev, generator=g).half() / 32
    op = flux.Int4GemmGrouped(q, s, z)
    y = op.forward(x, torch.tensor(splits, device=dev, dtype=torch.int32))
    row = 0
    for e, count in enumerate(splits):
        ref = x[row:row + count].double() @ oracle.weights4(q[e], s[e], z[e], group).t()
        assert torch.equal(y[row:row + count], ref.half()), (e, flux._native.last_gemm())
        row += count
    op.check_status()


def test_int4_outliers(dev, flux):
    """One huge activation next to small ones, a large mean: nothing cancels on the way."""
    q, s, z = _made4(dev, (), 200, 1024, 128, True, 4)
    g = _gen(dev, 4)
    for m in (1, 12, 40, 150):
        x = torch.randn(m, 1024, device=dev, generator=g)
        x[:, 17] = 3000.0
        x[:, 512:] += 50.0
        x = x.bfloat16()
        ref, bound = oracle.product4(x, oracle.weights4(q, s, z, 128), 128)
        oracle.assert_within(flux.Int4Gemm(q, s, z).forward(x), ref, bound)
        # infinities and NaN reach the rows that hold them and no other
        x[0, 5], x[0, 900] = math.inf, math.nan
        y = flux.Int4Gemm(q, s, z).forward(x)
        assert bool(torch.isnan(y[0]).all())
        if m > 1:
            oracle.assert_within(y[1:], ref[1:], bound[1:])


@pytest.mark.parametrize("m", [1, 5, 20, 70, 140])
def test_int4_views(dev, flux, m):
    """Inputs with any strides and alignment; buffers that are part of something larger."""
    q, s, z = _made4(dev, (), 190, 256, 64, True, 6)
    op = flux.Int4Gemm(q, s, z)
    wide = torch.randn(2 * m, 600, device=dev, generator=_gen(dev, 6)).half()
    for x in (wide[:m, :256], wide[:m, 8:264], wide[:m, 1:257], wide[::2, 300:556], wide[:1, :256].expand(m, 256),
              wide[:256].t()[:m, :256] if m >= 128 else torch.randn(256, m, device=dev).half().t()):
        assert x.shape == (m, 256)
        want = op.forward(x.contiguous())
        assert torch.equal(op.forward(x), want)
        out = torch.full((m + 2, 220), 3.0, device=dev, dtype=torch.float16)
        got = op.forward(x, output_buf=out[1:m + 1, 7:197])
        assert torch.equal(got, want) and got.data_ptr() == out[1:, 7:].data_ptr()
        out[1:m + 1, 7:197] = 3.0
        assert bool((out == 3).all())
    assert op.forward(wide[:0, :256]).shape == (0, 190)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("splits", [[3, 0, 9, 1, 0, 17, 2, 8], [0] * 8, [40, 0, 0, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 0, 0, 300],
                                    [1] * 8, [33, 65, 7, 128, 0, 129, 16, 1], [260, 5, 130, 0, 64, 31, 257, 90]])
def test_int4_grouped(dev, flux, splits, zeros):
    g = _gen(dev, sum(splits))
    rows = sum(splits)
    for n, k, group, dtype in ((130, 384, 128, torch.bfloat16), (64, 96, 32, torch.float16), (200, 2048, 64, torch.bfloat16)):
        q, s, z = _made4(dev, (8,), n, k, group, zeros, n)
        op = flux.Int4GemmGrouped(q, s, z)
        x = torch.randn(rows + 5, k, device=dev, generator=g).to(dtype)
        x[rows:] = math.nan                                       # (rows that belong to nobody)
        sp = torch.tensor(splits, device=dev, dtype=torch.int32)
        out = torch.full((rows + 5, n), 5.0, device=dev, dtype=dtype)
        assert op.forward(x, sp, output_buf=out) is out
        assert bool((out[rows:] == 5).all())
        row = 0
        for e, count in enumerate(splits):
            w = oracle.weights4(q[e], s[e], None if z is None else z[e], group)
            ref, bound = oracle.product4(x[row:row + count], w, group)
            oracle.assert_within(out[row:row + count], ref, bound, f"expert {e}")
            row += count
        if rows:
            assert torch.equal(op.forward(x, sp)[:rows], out[:rows])
            assert torch.equal(op.forward(x, sp.cpu())[:rows], out[:rows])
        # counts that claim more rows than there are end at the last row
        more = sp.clone()
        more[7] += 1000
        short = torch.full((rows + 5, n), 5.0, device=dev, dtype=dtype)
        x[rows:] = 0.0
        op.forward(x, more, output_buf=short)
        assert torch.equal(short[:rows - splits[7]], out[:rows - splits[7]]) and bool((short[rows:] == 0).all())


def test_offsets_beyond_32_bits(dev, flux):
    """Rows and experts whose elements lie more than 2^31 behind the first: as in a call of their own. Activations -1, 0, 1
    and scales of a power of two make every sum exact, so that tiles of any shape agree to the bit."""
    g = _gen(dev, 5)
    x = torch.randint(-1, 2, (300_000, 8192), device=dev, generator=g, dtype=torch.int8).bfloat16()
    q, s, _ = _made4(dev, (), 130, 8192, 128, False, 1)
    op = flux.Int4Gemm(q, torch.full_like(s, 0.0625))
    y = op.forward(x)
    assert torch.equal(y[-70:], op.forward(x[-70:])) and torch.equal(y[262_100:262_200], op.forward(x[262_100:262_200]))
    both = x.view(150_000, 16384)[-140_000:]
    act = flux.gated_act(both)
    for part in (slice(-9, None), slice(131_060, 131_080)):
        assert torch.equal(act[part], flux.gated_act(both[part]))
    del both, act, y
    idx, w = flux.moe_route(x.view(-1, 512)[:, 100:356], 4, "sigmoid")
    few = flux.moe_route(x.view(-1, 512)[-40:, 100:356], 4, "sigmoid")
    assert torch.equal(idx[-40:], few[0]) and torch.equal(w[-40:], few[1])
    x = x[:40]
    q = torch.randint(0, 256, (70, 8192, 4096), device=dev, dtype=torch.uint8, generator=g)
    s = torch.full((70, 8192, 64), 0.0625, device=dev, dtype=torch.bfloat16)
    splits = torch.zeros(70, device=dev, dtype=torch.int32)
    splits[0], splits[-2], splits[-1] = 3, 20, 17
    y = flux.Int4GemmGrouped(q, s).forward(x, splits)
    for e, rows in ((0, slice(0, 3)), (68, slice(3, 23)), (69, slice(23, 40))):
        assert torch.equal(y[rows], flux.Int4Gemm(q[e], s[e]).forward(x[rows]))


def test_int4_streams_and_graphs(dev, flux):
    q, s, z = _made4(dev, (4,), 256, 512, 128, False, 2)
    dense, grouped = flux.Int4Gemm(q[0], s[0]), flux.Int4GemmGrouped(q, s)
    g = _gen(dev, 2)
    for m in (4, 30, 100, 300):
        x = torch.randn(m, 512, device=dev, generator=g).bfloat16()
        sp = torch.tensor([m // 2, 0, m - m // 2 - 1, 1], device=dev, dtype=torch.int32)
        want = dense.forward(x), grouped.forward(x, sp)
        side = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for st in side:                                            # two calls of one op at once
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append((dense.forward(x), grouped.forward(x, sp)))
        for st in side:
            torch.cuda.current_stream().wait_stream(st)
        for pair in got:
            assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])
        buf, bsp = torch.zeros_like(x), torch.zeros_like(sp)
        graphs = []
        for _ in range(2):                                         # two graphs of one op
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = dense.forward(buf), grouped.forward(buf, bsp)
            graphs.append((graph, outs))
        buf.copy_(x), bsp.copy_(sp)
        for graph, _ in graphs:
            graph.replay()
        for _, outs in graphs:
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_calls_from_several_threads(dev, flux):
    """One op used by four threads at once, each with its own stream, sizes and outputs."""
    import threading
    q, s, z = _made4(dev, (6,), 200, 384, 64, True, 4)
    dense, grouped = flux.Int4Gemm(q[0], s[0], z[0]), flux.Int4GemmGrouped(q, s, z)
    g = _gen(dev, 4)
    work = []
    for m in (3, 20, 75, 310):
        x = torch.randn(m, 384, device=dev, generator=g).bfloat16()
        splits = torch.tensor([m // 3, 0, m // 4, 0, 1, m - m // 3 - m // 4 - 1], device=dev, dtype=torch.int32)

        def calls(x=x, splits=splits):
            leaf = x.clone().requires_grad_(True)
            idx, w = flux.moe_route(leaf[:, :64], 8, "sigmoid")
            d, = torch.autograd.grad(w.sum() + flux.gated_act(leaf).sum(), leaf)
            return idx, w.detach(), d, dense.forward(x), grouped.forward(x, splits)
        work.append((calls, calls()))
    torch.cuda.synchronize()
    wrong = []

    def run(calls, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = calls()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        wrong.append("result")
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_expert_layer_together(dev, flux):
    """Router, index build, both products with 4-bit weights, activation with the routing weights, sum over the chosen
    experts - as a layer runs them - against the same steps in 64 bits on the rounded values in between."""
    T, E, topk, H, F, group = 37, 16, 4, 256, 192, 64
    g = _gen(dev, 77)
    x = torch.randn(T, H, device=dev, generator=g).bfloat16()
    logits = torch.randn(T, E, device=dev, generator=g)
    bias = torch.randn(E, device=dev, generator=g) * 0.05
    up, down = _made4(dev, (E,), 2 * F, H, group, True, 1), _made4(dev, (E,), H, F, group, False, 2)
    experts, weights = flux.moe_route(logits, topk, "sigmoid", bias, 4, 2, 2, True, 2.0)
    splits, offsets, scatter, gather, place = flux.moe_index_build(experts, E)
    row_weight = weights.reshape(-1)[gather.long() * topk + place.long()]
    rows = x[gather.long()]
    h = flux.Int4GemmGrouped(*up).forward(rows, splits)
    act = flux.gated_act(h, row_weight=row_weight, num_rows=offsets[-1:])
    y = flux.Int4GemmGrouped(*down).forward(act, splits)
    out = flux.topk_scatter_reduce(y, scatter.reshape(-1), topk)

    assert torch.equal(experts.cpu().long(), oracle.route_choice(logits.cpu(), topk, "sigmoid", bias.cpu(), 4, 2, 2))
    w_ref, _ = oracle.route_weights(logits, experts.long(), "sigmoid", True, 2.0)
    oracle.assert_within(weights, w_ref, w_ref.abs() * oracle.ROUTE_RTOL)
    flat = experts.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    assert torch.equal(rows, x[order // topk]) and torch.equal(row_weight, weights.reshape(-1)[order])
    row = 0
    for e, count in enumerate(torch.bincount(flat, minlength=E).tolist()):
        part = slice(row, row + count)
        for got, src, (q, s, z) in ((h, rows, up), (y, act, down)):
            ref, bound = oracle.product4(src[part], oracle.weights4(q[e], s[e], None if z is None else z[e], group), group)
            oracle.assert_within(got[part], ref, bound, f"expert {e}")
        row += count
    ref, bound = oracle.gated(h[:, :F], h[:, F:], "silu", row_weight)
    oracle.assert_within(act, ref, bound)
    ref = y[scatter.long()].double()
    oracle.assert_within(out, ref.sum(1), ref.abs().sum(1) * 4 * 2.0 ** -24)


@pytest.mark.parametrize("args,op", [
    (["route", "--tokens", "500", "--experts", "64", "--groups", "4", "--topk-groups", "2", "--bias", "--train"], "moe_route"),
    (["gated", "--rows", "300", "--cols", "128", "--train"], "gated_act"),
    (["int4", "--m", "5", "--n", "256", "--k", "512", "--zeros"], "int4"),
    (["int4", "--m", "64", "--n", "256", "--k", "512", "--group", "32", "--experts", "8"], "int4")])
def test_microbench_commands(dev, args, op, capsys):
    import json
    from tempname_new_b200.utils import microbench
    microbench.main(args + ["--iters", "2", "--warmup", "1", "--no-flush"])
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["op"] == op and line["ms"] > 0
