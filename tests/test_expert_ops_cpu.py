"""Routing, gated activation and 4-bit products without a GPU: the PyTorch statements against the 64-bit oracle, and what
the entry points refuse."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import expert_ops_oracle as oracle
import tempname_new_b200 as flux


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (4, 2, 1), (4, 2, 2), (8, 8, 2)])
@pytest.mark.parametrize("renorm,scale", [(True, 1.0), (False, 2.5)])
def test_route(score, groups, keep, top, renorm, scale):
    torch.manual_seed(groups * 10 + keep)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(40, 48).mul_(2).to(dtype).requires_grad_(True)
        for bias in (None, torch.randn(48) * 0.1):
            idx, w = flux.moe_route(x, 6, score, bias, groups, keep, top, renorm, scale)
            assert torch.equal(idx.long(), oracle.route_choice(x.detach(), 6, score, bias, groups, keep, top))
            w_ref, grad_of = oracle.route_weights(x.detach(), idx.long(), score, renorm, scale)
            oracle.assert_within(w, w_ref, w_ref * 2.0 ** -24)
            gw = torch.randn(40, 6)
            dx, = torch.autograd.grad(w, x, gw)
            d_ref, size = grad_of(gw)
            oracle.assert_within(dx, d_ref, size * oracle.ROUTE_RTOL)


def test_route_masked():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 6, [-inf] * 5 + [1.0], [nan] + [0.0] * 5], requires_grad=True)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            idx, w = flux.moe_route(x, 2, score, renormalize=renorm)
            assert idx.tolist() == [[0, 1], [5, 0], [1, 2]]
            assert w[0].tolist() == [0.0, 0.0] and w[1, 1] == 0.0
            assert bool(torch.isnan(w[2]).all()) == (score == "softmax")
            dx, = torch.autograd.grad(w[:2].sum(), x)
            assert bool((dx[0] == 0).all())


def test_route_refusals():
    x = torch.randn(4, 16)
    for bad in (dict(topk=0), dict(topk=17), dict(topk=2, score_func="relu"), dict(topk=2, num_groups=3),
                dict(topk=2, num_groups=4, topk_groups=5), dict(topk=2, num_groups=4, topk_groups=0),
                dict(topk=5, num_groups=4, topk_groups=1), dict(topk=2, num_groups=4, topk_groups=2, group_top=3),
                dict(topk=1, num_groups=16, topk_groups=2, group_top=2), dict(topk=2, scale=0.0),
                dict(topk=2, scale=math.inf), dict(topk=2, scale=math.nan), dict(topk=2, bias=torch.zeros(15)),
                dict(topk=2, bias=torch.zeros(16, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            flux.moe_route(x, **bad)
    with pytest.raises(ValueError):
        flux.moe_route(x[0], 2)
    with pytest.raises(ValueError):
        flux.moe_route(torch.randn(2, 513), 2)
    with pytest.raises(ValueError):
        flux.moe_route(torch.randn(2, 64), 33)
    with pytest.raises(TypeError):
        flux.moe_route(x.double(), 2)
    assert flux.moe_route(x[:0], 2)[0].shape == (0, 2)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated(act):
    torch.manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        both = torch.randn(9, 34).mul_(3).to(dtype).requires_grad_(True)
        weight = torch.randn(9, requires_grad=True)
        y = flux.gated_act(both, act=act, row_weight=weight)
        dy = torch.randn(9, 17).to(dtype)
        db, dw = torch.autograd.grad(y, (both, weight), dy)
        refs, bounds = oracle.gated(both.detach()[:, :17], both.detach()[:, 17:], act, weight.detach(), dy)
        for got, ref, bound in zip((y.detach(), db[:, :17], db[:, 17:], dw), refs, bounds):
            oracle.assert_within(got, ref, 4 * bound)
        two = flux.gated_act(both.detach()[:, :17], both.detach()[:, 17:], act, weight.detach())
        assert torch.equal(two, y.detach())
    num = torch.tensor(4)
    out = torch.full((9, 17), 2.0)
    x = torch.randn(9, 34)
    flux.gated_act(x, act=act, num_rows=num, out=out)
    y = flux.gated_act(x, act=act, num_rows=num)
    assert bool((out[4:] == 2).all()) and bool((y[4:] == 0).all()) and torch.equal(out[:4], y[:4])


def test_gated_refusals():
    x = torch.randn(4, 16)
    with pytest.raises(ValueError):
        flux.gated_act(torch.randn(4, 15))
    with pytest.raises(ValueError):
        flux.gated_act(x, x[:, :8])
    with pytest.raises(ValueError):
        flux.gated_act(x[0])
    with pytest.raises(TypeError):
        flux.gated_act(x.double())
    with pytest.raises(TypeError):
        flux.gated_act(x, x.bfloat16())
    for bad in (dict(act="tanh"), dict(act=None), dict(row_weight=torch.ones(5)), dict(row_weight=torch.ones(4).bfloat16()),
                dict(row_weight=torch.ones(4, 1)), dict(num_rows=torch.tensor([1, 2])), dict(num_rows=torch.tensor(1.0)),
                dict(out=torch.empty(4, 16)), dict(out=torch.empty(4, 8).bfloat16()), dict(out=torch.empty(8, 4).t()),
                dict(out=torch.empty(1, 8).expand(4, 8))):
        with pytest.raises(ValueError):
            flux.gated_act(x, **bad)
    with pytest.raises(ValueError):
        flux.gated_act(x.clone().requires_grad_(True), out=torch.empty(4, 8))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 256])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float16])
def test_quantize_int4(symmetric, group, scale_dtype):
    torch.manual_seed(group)
    w = torch.randn(2, 10, 256)
    w[0, 3, :group] = 0.0                                       # a group of zeros
    w[1, 4] = w[1, 4].abs()
    q, s, z = flux.quantize_int4(w, group, symmetric, scale_dtype)
    assert q.shape == (2, 10, 128) and s.shape == (2, 10, 256 // group) and s.dtype == scale_dtype
    assert (z is None) == symmetric
    back = flux.dequantize_int4(q, s, z)
    for e in range(2):
        ref = oracle.weights4(q[e], s[e], None if z is None else z[e], group)
        assert torch.equal(back[e].double(), ref)
    # half a step, and what the rounded scale leaves at the end of the range: 7 (or 15) steps of half a step of its type;
    # with zero points their rounding moves the range by another half step
    step = s.float().repeat_interleave(group, dim=2)
    assert bool(((back - w).abs() <= step * (0.5 + 15 * oracle.EPS[scale_dtype] + (0.0 if symmetric else 0.5)) + 1e-6).all())
    assert bool((back[0, 3, :group] == 0).all())
    one = flux.quantize_int4(w[0], group, symmetric, scale_dtype)
    assert torch.equal(one[0], q[0]) and torch.equal(one[1], s[0])


def test_int4_statement():
    torch.manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16):
        w = torch.randn(3, 20, 128)
        q, s, z = flux.quantize_int4(w, 64, False)
        x = torch.randn(7, 128).to(dtype)
        bias = torch.randn(20).to(dtype)
        ref, bound = oracle.product4(x, oracle.weights4(q[0], s[0], z[0], 64), 64, bias)
        oracle.assert_within(flux.Int4Gemm(q[0], s[0], z[0]).forward(x, bias=bias), ref, bound)
        splits = torch.tensor([4, 0, 2], dtype=torch.int32)
        out = torch.full((7, 20), 9.0, dtype=dtype)
        flux.Int4GemmGrouped(q, s, z).forward(x, splits, output_buf=out)
        for e, part in ((0, slice(0, 4)), (2, slice(4, 6))):
            ref, bound = oracle.product4(x[part], oracle.weights4(q[e], s[e], z[e], 64), 64)
            oracle.assert_within(out[part], ref, bound)
        assert bool((out[6:] == 9).all())


def test_int4_refusals():
    w = torch.randn(8, 128)
    for bad in (dict(group_size=48), dict(group_size=16), dict(group_size=96), dict(group_size=256)):
        with pytest.raises(ValueError):
            flux.quantize_int4(w, **bad)
    with pytest.raises(ValueError):
        flux.quantize_int4(torch.full((8, 128), math.nan))
    with pytest.raises(ValueError):
        flux.quantize_int4(torch.full((8, 128), 1e9), scale_dtype=torch.float16)
    with pytest.raises(TypeError):
        flux.quantize_int4(w, scale_dtype=torch.float32)
    with pytest.raises(ValueError):
        flux.quantize_int4(w[0])
    q, s, z = flux.quantize_int4(w, 32, False)
    for args in ((q.int(), s, z), (q[0], s, z), (q, s[:4], z), (q, s[:, :3], None), (q, s, z[:, :2]), (q, s, z.int())):
        with pytest.raises(ValueError):
            flux.Int4Gemm(*args)
    with pytest.raises(TypeError):
        flux.Int4Gemm(q, s.float(), z)
    with pytest.raises(ValueError):
        flux.Int4GemmGrouped(q, s, z)
    op = flux.Int4Gemm(q, s, z)
    x = torch.randn(3, 128)
    for bad in (x[:, :64], x[0], torch.randn(2, 3, 128)):
        with pytest.raises(ValueError):
            op.forward(bad)
    with pytest.raises(TypeError):
        op.forward(x.double())
    with pytest.raises(RuntimeError):
        op.forward(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError):
        op.forward(x, bias=torch.zeros(8, requires_grad=True))
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        op.forward(forward_ad.make_dual(x, torch.ones_like(x)))
    with torch.no_grad():
        op.forward(x.clone().requires_grad_(True), bias=torch.zeros(8, requires_grad=True))
    for bad in (dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8).bfloat16()), dict(output_buf=torch.empty(3, 7)),
                dict(output_buf=torch.empty(8, 3).t()), dict(output_buf=torch.empty(3, 8).half()),
                dict(output_buf=torch.empty(1, 8).expand(3, 8))):
        with pytest.raises(ValueError):
            op.forward(x, **bad)
    many = flux.Int4GemmGrouped(q.unsqueeze(0), s.unsqueeze(0), z.unsqueeze(0))
    for bad in (torch.tensor([1, 2]), torch.tensor([1.0]), torch.tensor([True])):
        with pytest.raises(ValueError):
            many.forward(x, bad)


def test_native_argument_checks(lib_built):
    """The C entry points answer bad sizes with an error code before anything reaches the device."""
    import ctypes

    from tempname_new_b200.ops import gated as G
    from tempname_new_b200.ops import int4 as I
    from tempname_new_b200.ops import route as R
    lib = lib_built.lib()
    a = R.RouteArgs(tokens=1, num_experts=600, topk=1, num_groups=1, topk_groups=1, group_top=1, scale=1.0)
    assert lib.fluxb_moe_route(ctypes.byref(a)) == 1 and lib.fluxb_moe_route_bwd(ctypes.byref(a)) == 1
    a = R.RouteArgs(tokens=1, num_experts=64, topk=9, num_groups=8, topk_groups=1, group_top=1, scale=1.0)
    assert lib.fluxb_moe_route(ctypes.byref(a)) == 1
    a = R.RouteArgs(tokens=0, num_experts=64, topk=8, num_groups=8, topk_groups=1, group_top=1, scale=1.0)
    assert lib.fluxb_moe_route(ctypes.byref(a)) == 0
    a = R.RouteArgs(tokens=1, num_experts=64, topk=8, num_groups=1, topk_groups=1, group_top=1, scale=1.0, logits=16, experts=16,
                    weights=16, grad=16, dlogits=24)
    assert lib.fluxb_moe_route_bwd(ctypes.byref(a)) == 1 and b"dlogits" in lib.fluxb_last_error()
    b = G.GatedArgs(rows=3, cols=4, act=3)
    assert lib.fluxb_gated_act(ctypes.byref(b)) == 1 and lib.fluxb_gated_act_bwd(ctypes.byref(b)) == 1
    c = I.Int4Layout(experts=1, N=8, K=48, group=32)
    assert lib.fluxb_int4_layout(ctypes.byref(c)) == 1
    for bad in (dict(K=40, group=40), dict(K=64, group=128), dict(experts=2), dict(experts=0), dict(N=0), dict(M=-1),
                dict(dtype=3), dict(scale_dtype=3), dict(ldx=60), dict(x=8)):
        f = dict(x=16, packed=16, scales=16, out=16, M=1, ldx=64, ldo=8, experts=1, N=8, K=64, group=32, dtype=0, scale_dtype=0)
        f.update(bad)
        d = I.Int4GemmArgs(**f)
        assert lib.fluxb_int4_gemm(ctypes.byref(d)) == 1, bad
    for f in (lib.fluxb_moe_route, lib.fluxb_gated_act, lib.fluxb_int4_layout, lib.fluxb_int4_gemm):
        assert f(None) == 1


def test_sizes_beyond_the_arguments():
    """Sizes that 32-bit arguments would wrap are refused."""
    from tempname_new_b200.ops import gated as G
    side = 1 << 25
    with pytest.raises(ValueError):
        flux.Int4Gemm(torch.empty(side, 16, dtype=torch.uint8, device="meta"),
                      torch.empty(side, 1, dtype=torch.bfloat16, device="meta"))
    with pytest.raises(ValueError):
        G._args(torch.empty(1, 1 << 33, device="meta"), None, "silu", None, None, torch.device("cpu"))


def test_forward_mode_on_the_cpu():
    """Tangents pass through the statements in PyTorch: here they match the gradient's product with the direction."""
    g = torch.Generator().manual_seed(3)
    x, v = torch.randn(5, 16, generator=g, dtype=torch.float32), torch.randn(5, 16, generator=g)
    for f in (lambda t: flux.moe_route(t, 3)[1], lambda t: flux.gated_act(t, act="gelu")):
        with forward_ad.dual_level():
            tangent = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v))).tangent
        leaf = x.clone().requires_grad_(True)
        y = f(leaf)
        d = torch.randn(y.shape, generator=g)
        grad, = torch.autograd.grad(y, leaf, d)
        torch.testing.assert_close((tangent * d).sum(), (grad * v).sum(), rtol=1e-4, atol=1e-4)


def test_example_with_int4_weights():
    import os
    import subprocess
    import sys
    from conftest import ROOT, free_port
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "1", "--master-addr", "127.0.0.1",
           "--master-port", str(free_port()), os.path.join(ROOT, "examples", "moe_layer.py"), "--tokens-per-rank", "16",
           "--hidden", "64", "--ffn", "32", "--experts", "4", "--topk", "2", "--int4"]
    r = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "MoE layer E=4 top2" in r.stdout, r.stdout[-1500:] + r.stderr[-3000:]
