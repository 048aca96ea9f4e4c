"""``gated_act``: the gated activation ``row_weight * act(gate) * up`` between the two products of an MLP or of a layer's
experts, with its gradient. The reference leaves it to its callers (``examples/moe_flux_only.py``). Kernel and formulas are
in ``csrc/aux/gated.cu``; ``gated_act_torch`` states the same in PyTorch (CPU path and test oracle)."""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from ._dense import ACT, current_stream_ptr, device_guard, dtype_code, has_tangent

_VP = ctypes.c_void_p
_GELU_A, _GELU_B = 2.0 * math.sqrt(2.0 / math.pi), 0.044715
_ACTS = ("silu", "gelu", "gelu_tanh", "relu")


class GatedArgs(ctypes.Structure):
    _fields_ = [
        ("gate", _VP), ("up", _VP), ("row_weight", _VP), ("num_rows", _VP), ("out", _VP), ("grad", _VP), ("dgate", _VP),
        ("dup", _VP), ("drow", _VP),
        ("rows", ctypes.c_int64), ("gate_stride", ctypes.c_int64), ("up_stride", ctypes.c_int64),
        ("out_stride", ctypes.c_int64), ("grad_stride", ctypes.c_int64), ("dgate_stride", ctypes.c_int64),
        ("dup_stride", ctypes.c_int64),
        ("cols", ctypes.c_int32), ("dtype", ctypes.c_int32), ("act", ctypes.c_int32), ("num_rows_64", ctypes.c_int32),
        ("zero_rest", ctypes.c_int32), ("reserved", ctypes.c_int32),
        ("stream", _VP),
    ]


def gated_act_torch(gate: torch.Tensor, up: torch.Tensor, act: str = "silu", row_weight: Optional[torch.Tensor] = None,
                    num_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The operator in PyTorch, differentiable by autograd; rows that are not in use are zeros."""
    wide = torch.promote_types(gate.dtype, torch.float32)
    g = gate.to(wide)
    if act == "relu":
        y = torch.relu(g) * up.to(wide)
    else:                                   # (the sigmoid form loses no digits where the result is close to zero)
        z = g if act == "silu" else _GELU_A * (g + _GELU_B * g * g * g)
        y = g * torch.sigmoid(z) * up.to(wide)
    if row_weight is not None:
        y = y * row_weight.to(wide).unsqueeze(1)
    if num_rows is not None:
        live = torch.arange(gate.shape[0], device=gate.device).unsqueeze(1) < num_rows.reshape(1, 1)
        y = torch.where(live, y, torch.zeros_like(y))
    return y.to(gate.dtype)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _args(gate, up, act, row_weight, num_rows, device) -> GatedArgs:
    """``up`` None: both halves are in ``gate``."""
    a = GatedArgs()
    rows, cols = gate.shape
    a.gate, a.gate_stride = gate.data_ptr(), gate.stride(0)
    if up is None:
        cols //= 2
        a.up, a.up_stride = gate.data_ptr() + cols * gate.element_size(), gate.stride(0)
    else:
        a.up, a.up_stride = up.data_ptr(), up.stride(0)
    if cols >= 1 << 31:
        raise ValueError(f"rows of {cols} columns are not supported")
    a.rows, a.cols = rows, cols
    a.dtype, a.act = dtype_code(gate.dtype), ACT[act]
    if row_weight is not None:
        a.row_weight = row_weight.data_ptr()
    if num_rows is not None:
        a.num_rows, a.num_rows_64 = num_rows.data_ptr(), int(num_rows.dtype == torch.int64)
    a.stream = current_stream_ptr(device)
    return a


def _forward(gate, up, act, row_weight, num_rows, out):
    gate, up = _rows(gate), None if up is None else _rows(up)
    fresh, device = out is None, gate.device
    if fresh:
        out = gate.new_empty((gate.shape[0], gate.shape[1] // 2 if up is None else gate.shape[1]))
    with device_guard(device):
        a = _args(gate, up, act, row_weight, num_rows, device)
        a.out, a.out_stride, a.zero_rest = out.data_ptr(), out.stride(0), fresh
        _native.check(_native.lib().fluxb_gated_act(ctypes.byref(a)), "fluxb_gated_act")
    return out


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, row_weight, act, num_rows):
        ctx.save_for_backward(gate, up, row_weight, num_rows)
        ctx.act = act
        return _forward(gate, up, act, row_weight, num_rows, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        gate, up, row_weight, num_rows = ctx.saved_tensors
        grad, gate, up = _rows(grad), _rows(gate), None if up is None else _rows(up)
        device = gate.device
        dgate = torch.empty(gate.shape, dtype=gate.dtype, device=device)
        dup = torch.empty(up.shape, dtype=gate.dtype, device=device) if up is not None else None
        drow = torch.empty_like(row_weight) if row_weight is not None and ctx.needs_input_grad[2] else None
        with device_guard(device):
            a = _args(gate, up, ctx.act, row_weight, num_rows, device)
            a.grad, a.grad_stride = grad.data_ptr(), grad.stride(0)
            a.dgate, a.dgate_stride = dgate.data_ptr(), dgate.stride(0)
            if up is None:
                a.dup, a.dup_stride = dgate.data_ptr() + a.cols * gate.element_size(), dgate.stride(0)
            else:
                a.dup, a.dup_stride = dup.data_ptr(), dup.stride(0)
            a.drow = drow.data_ptr() if drow is not None else None
            _native.check(_native.lib().fluxb_gated_act_bwd(ctypes.byref(a)), "fluxb_gated_act_bwd")
        return dgate, dup, drow, None, None


def gated_act(gate: torch.Tensor, up: Optional[torch.Tensor] = None, act: str = "silu",
              row_weight: Optional[torch.Tensor] = None, num_rows: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``row_weight * act(gate) * up``, [rows, cols]; ``act`` is "silu", "gelu" (tanh form) or "relu".

    Without ``up``, ``gate`` is [rows, 2 * cols] and holds the gate in its first half, as the product with stacked gate and
    up weights leaves it. ``row_weight [rows]`` (float32) scales whole rows: the routing weight of each expert-sorted row.
    ``num_rows`` (one int32 or int64 on the device) is the number of rows in use, for buffers that are sized without asking
    the device; the rows behind it become zeros, in ``out`` they stay as they are. Gradients reach ``gate``, ``up`` and
    ``row_weight``; ``out`` is for calls without them, and may be ``gate`` or ``up`` (or the gate's half of ``gate``)."""
    if gate.dim() != 2 or (up is not None and up.shape != gate.shape):
        raise ValueError("gate and up must be [rows, cols] of one shape, or gate [rows, 2 * cols] alone")
    if up is None and gate.shape[1] % 2:
        raise ValueError(f"gate without up holds two halves, got {gate.shape[1]} columns")
    if gate.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"gate must be bfloat16, float16 or float32, got {gate.dtype}")
    if up is not None and (up.dtype != gate.dtype or up.device != gate.device):
        raise TypeError("gate and up must share type and device")
    if act not in _ACTS:
        raise ValueError(f"act must be one of {_ACTS}, got {act!r}")
    rows, cols = gate.shape if up is not None else (gate.shape[0], gate.shape[1] // 2)
    if row_weight is not None and (row_weight.shape != (rows,) or row_weight.dtype != torch.float32
                                   or row_weight.device != gate.device):
        raise ValueError("row_weight must be float32 [rows] on the device of gate")
    if num_rows is not None and (num_rows.numel() != 1 or num_rows.dtype not in (torch.int32, torch.int64)
                                 or num_rows.device != gate.device):
        raise ValueError("num_rows must be one int32 or int64 on the device of gate")
    grads = torch.is_grad_enabled() and (gate.requires_grad or (up is not None and up.requires_grad)
                                         or (row_weight is not None and row_weight.requires_grad))
    grads = grads or has_tangent(gate, up, row_weight)             # (a tangent is refused by the function below)
    if out is not None:
        if grads:
            raise ValueError("out cannot be used where gradients are recorded")
        if out.shape != (rows, cols) or out.dtype != gate.dtype or out.device != gate.device or (
                cols > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < cols):
            raise ValueError("out must be [rows, cols] of the type of gate, on its device, with contiguous rows that do not "
                             "overlap")
    if not gate.is_cuda:
        g, u = (gate, up) if up is not None else (gate[:, :cols], gate[:, cols:])
        y = gated_act_torch(g, u, act, row_weight, num_rows)
        if out is None:
            return y
        n = rows if num_rows is None else max(0, min(rows, int(num_rows)))
        out[:n].copy_(y[:n])
        return out
    if row_weight is not None and not row_weight.is_contiguous():
        row_weight = row_weight.contiguous()
    if grads:
        return _Gated.apply(gate, up, row_weight, act, num_rows)
    return _forward(gate, up, act, row_weight, num_rows, out)
