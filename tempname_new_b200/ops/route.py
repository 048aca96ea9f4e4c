"""``moe_route``: the choice of a token's experts and their weights from the router's logits, with the gradient of the
weights. It stands in front of ``moe_index_build``, which sorts the choices; the reference's tests use a softmax and a
top-k of the framework there (``python/flux/testing/moe_utils.py``). The kernel and the definition are in
``csrc/aux/route.cu``; ``moe_route_torch`` states the same in PyTorch (CPU path and test oracle)."""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from ._dense import current_stream_ptr, device_guard, dtype_code, has_tangent

_VP = ctypes.c_void_p
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_TOPK, MAX_GROUPS = 512, 32, 32


class RouteArgs(ctypes.Structure):
    _fields_ = [
        ("logits", _VP), ("bias", _VP), ("experts", _VP), ("weights", _VP), ("grad", _VP), ("dlogits", _VP),
        ("tokens", ctypes.c_int64), ("row_stride", ctypes.c_int64),
        ("num_experts", ctypes.c_int32), ("topk", ctypes.c_int32),
        ("num_groups", ctypes.c_int32), ("topk_groups", ctypes.c_int32), ("group_top", ctypes.c_int32),
        ("score", ctypes.c_int32), ("renormalize", ctypes.c_int32), ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float), ("reserved", ctypes.c_int32),
        ("stream", _VP),
    ]


def _order(values: torch.Tensor) -> torch.Tensor:
    """Places of a row's values, largest first, ties to the lowest place, NaN last of all."""
    lowest = torch.where(torch.isnan(values), torch.full_like(values, -math.inf), values)
    # (two stable sorts: NaN behind -inf)
    first = lowest.sort(dim=-1, descending=True, stable=True).indices
    return first.gather(-1, torch.isnan(values).gather(-1, first).sort(dim=-1, stable=True).indices)


def _choose_torch(logits, topk, score_func, bias, num_groups, topk_groups, group_top):
    x = logits.double()
    t, e = x.shape
    masked = (x.amax(dim=1, keepdim=True) == -math.inf) if e else None
    if score_func == "softmax":
        score = torch.where(masked, torch.zeros_like(x), torch.softmax(x, dim=1))
    else:
        score = torch.sigmoid(x)
    if bias is not None:
        choice = by_group = score + bias.double()
    else:
        choice, by_group = x, (score if group_top == 2 else x)
    if num_groups > 1:
        size = e // num_groups
        split = by_group.view(t, num_groups, size)
        best = split.gather(2, _order(split)[:, :, :group_top]).sum(dim=2)
        kept = torch.zeros(t, num_groups, dtype=torch.bool, device=x.device)
        kept.scatter_(1, _order(best)[:, :topk_groups], True)
        # (candidates in front of the others, whatever their values)
        out = ~kept.repeat_interleave(size, dim=1)
        first = _order(choice)
        order = first.gather(1, out.gather(1, first).sort(dim=1, stable=True).indices)
    else:
        order = _order(choice)
    return order[:, :topk]


def moe_route_torch(logits: torch.Tensor, topk: int, score_func: str = "softmax", bias: Optional[torch.Tensor] = None,
                    num_groups: int = 1, topk_groups: int = 1, group_top: int = 1, renormalize: bool = True,
                    scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The operator in PyTorch, differentiable by autograd; scores and sums in 64 bits."""
    with torch.no_grad():
        experts = _choose_torch(logits.detach(), topk, score_func, bias, num_groups, topk_groups, group_top)
    x = logits.double()
    picked = x.gather(1, experts)
    none = x.detach().amax(dim=1, keepdim=True) == -math.inf
    if score_func == "softmax":
        # (rows without an expert: any finite numbers, replaced by zeros below)
        x = torch.where(none, torch.zeros_like(x), x)
        w = torch.softmax(x, dim=1).gather(1, experts)
        if renormalize:
            nan = torch.isnan(x.detach()).any(dim=1, keepdim=True)
            safe = torch.where(none, torch.zeros_like(picked), picked)
            w = torch.where(nan, torch.full_like(w, math.nan), torch.softmax(safe, dim=1))
    else:
        none = picked.detach().amax(dim=1, keepdim=True) == -math.inf
        picked = torch.where(none, torch.zeros_like(picked), picked)
        log = torch.nn.functional.logsigmoid(picked)
        w = torch.softmax(log, dim=1) if renormalize else log.exp()
    w = torch.where(none, torch.zeros_like(w), w)
    return experts.to(torch.int32), (w * scale).float()


@functools.lru_cache(maxsize=256)
def _plan(E: int, dtype: torch.dtype, topk: int, score_func: str, num_groups: int, topk_groups: int, group_top: int,
          renormalize: bool, scale: float) -> RouteArgs:
    """The checked arguments that do not depend on the tensors; to be copied by each call."""
    if dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {dtype}")
    if score_func not in _SCORES:
        raise ValueError(f"score_func must be one of {tuple(_SCORES)}, got {score_func!r}")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"between 1 and {MAX_EXPERTS} experts, got {E}")
    if not 1 <= num_groups <= MAX_GROUPS or E % num_groups:
        raise ValueError(f"{E} experts do not divide over {num_groups} groups (at most {MAX_GROUPS})")
    if not 1 <= topk_groups <= num_groups:
        raise ValueError("topk_groups must be between 1 and num_groups")
    if group_top not in (1, 2) or (num_groups > 1 and group_top > E // num_groups):
        raise ValueError("group_top must be 1 or 2, and no more than the experts of a group")
    if not 1 <= topk <= min(MAX_TOPK, E // num_groups * topk_groups):
        raise ValueError(f"topk must be between 1 and {min(MAX_TOPK, E // num_groups * topk_groups)}, got {topk}")
    if not 2.0 ** -126 <= abs(scale) < 2.0 ** 127:
        raise ValueError("scale must be finite and not zero (in 32 bits)")
    a = RouteArgs()
    a.num_experts, a.topk, a.num_groups = E, topk, num_groups
    a.topk_groups, a.group_top = (topk_groups, group_top) if num_groups > 1 else (1, 1)
    a.score, a.renormalize, a.scale, a.dtype = _SCORES[score_func], renormalize, scale, dtype_code(dtype)
    return a


def _args(plan, x, experts, weights, device) -> RouteArgs:
    a = RouteArgs.from_buffer_copy(plan)
    a.logits, a.row_stride, a.tokens = x.data_ptr(), x.stride(0), x.shape[0]
    a.experts, a.weights = experts.data_ptr(), weights.data_ptr()
    a.stream = current_stream_ptr(device)
    return a


def _forward(logits, bias, plan):
    x = logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()
    device, shape = x.device, (x.shape[0], plan.topk)
    experts, weights = x.new_empty(shape, dtype=torch.int32), x.new_empty(shape, dtype=torch.float32)
    with device_guard(device):
        a = _args(plan, x, experts, weights, device)
        if bias is not None:
            a.bias = bias.data_ptr()
        _native.check(_native.lib().fluxb_moe_route(ctypes.byref(a)), "fluxb_moe_route")
    return x, experts, weights


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, plan):
        x, experts, weights = _forward(logits, bias, plan)
        ctx.save_for_backward(x, experts, weights)
        ctx.plan = plan
        ctx.mark_non_differentiable(experts)
        return experts, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _, grad):
        x, experts, weights = ctx.saved_tensors
        grad = grad.to(torch.float32).contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        with device_guard(x.device):
            a = _args(ctx.plan, x, experts, weights, x.device)
            a.grad, a.dlogits = grad.data_ptr(), dx.data_ptr()
            _native.check(_native.lib().fluxb_moe_route_bwd(ctypes.byref(a)), "fluxb_moe_route_bwd")
        return dx, None, None


def moe_route(logits: torch.Tensor, topk: int, score_func: str = "softmax", bias: Optional[torch.Tensor] = None,
              num_groups: int = 1, topk_groups: int = 1, group_top: int = 1, renormalize: bool = True,
              scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(choosed_experts [tokens, topk] int32, weights [tokens, topk] float32)`` from ``logits [tokens, experts]``.

    The scores are the softmax of a row or the sigmoid of each logit (``score_func``). ``bias [experts]`` (float32, no
    gradient) is added to them for the choice only. With ``num_groups`` groups of consecutive experts, the
    ``topk_groups`` groups whose ``group_top`` (1 or 2) best experts have the largest sum stay. Experts come best first,
    equal ones by their index. The weights are the chosen experts' scores, divided by their sum (``renormalize``), times
    ``scale``; they carry the gradient to the logits. An expert whose logit is -inf is chosen only when no other is left,
    with weight 0; NaN ranks lowest and shows in the weights."""
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError(f"logits must be [tokens, experts], got {tuple(shape)}")
    E = shape[1]
    plan = _plan(E, logits.dtype, int(topk), score_func, int(num_groups), int(topk_groups), int(group_top), bool(renormalize),
                 float(scale))
    if bias is not None:
        if bias.shape != (E,) or bias.dtype != torch.float32 or bias.device != logits.device:
            raise ValueError("bias must be float32 [experts] on the device of the logits")
        bias = bias.detach().contiguous()
    if not logits.is_cuda:
        return moe_route_torch(logits, plan.topk, score_func, bias, plan.num_groups, plan.topk_groups, plan.group_top,
                               renormalize, plan.scale)
    if (logits.requires_grad and torch.is_grad_enabled()) or has_tangent(logits):   # (a tangent is refused there)
        return _Route.apply(logits, bias, plan)
    return _forward(logits, bias, plan)[1:]
