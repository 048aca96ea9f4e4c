"""Linear layers with 4-bit weights and group scales: ``Int4Gemm`` (dense, beside ``GemmOnly`` and ``BlockScaleGemm``) and
``Int4GemmGrouped`` (one weight matrix per expert over expert-sorted rows, beside ``GemmGroupedV3``), for inference, from one
token to a long prompt. The reference has no 4-bit weights. Kernels and layouts: ``csrc/sm100/gemm_int4.cuh``.

Interchange format, as ``quantize_int4`` writes it: ``qweight [N, K / 2]`` uint8 (column 2j in the low half of byte j),
``scales [N, K / group]`` bf16 or fp16, ``zeros [N, K / group]`` uint8 in 0 .. 15 or None for 8; experts as a leading
dimension. ``w[n, k] = (q[n, k] - z[n, k // group]) * s[n, k // group]``."""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _native
from ..parallel.symm import FluxTimeoutError
from ._dense import current_stream_ptr, device_guard, dtype_code, has_tangent

_VP = ctypes.c_void_p
_HALF = (torch.bfloat16, torch.float16)
MAX_EXPERTS, MAX_SIDE = 512, 1 << 24


class Int4Layout(ctypes.Structure):
    _fields_ = [
        ("q", _VP), ("scales", _VP), ("zeros", _VP), ("packed", _VP), ("scales_out", _VP), ("zeros_out", _VP),
        ("experts", ctypes.c_int32), ("N", ctypes.c_int32), ("K", ctypes.c_int32), ("group", ctypes.c_int32),
        ("stream", _VP),
    ]


class Int4GemmArgs(ctypes.Structure):
    _fields_ = [
        ("x", _VP), ("packed", _VP), ("scales", _VP), ("zeros", _VP), ("bias", _VP), ("splits", _VP), ("out", _VP),
        ("M", ctypes.c_int64), ("ldx", ctypes.c_int64), ("ldo", ctypes.c_int64),
        ("experts", ctypes.c_int32), ("N", ctypes.c_int32), ("K", ctypes.c_int32), ("group", ctypes.c_int32),
        ("dtype", ctypes.c_int32), ("scale_dtype", ctypes.c_int32),
        ("status", _VP), ("stream", _VP),
    ]


def _check_group(K: int, group: int) -> None:
    if K < 32 or group < 32 or K % group or (group not in (32, 64) and group % 128):
        raise ValueError(f"groups of {group} along K = {K}: 32, 64 or a multiple of 128 that divides K")


def quantize_int4(weight: torch.Tensor, group_size: int = 128, symmetric: bool = True,
                  scale_dtype: Optional[torch.dtype] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``(qweight, scales, zeros)`` of ``weight [..., N, K]``, rounded to the nearest step of each group: -7 .. 7 times the
    largest magnitude / 7 (``symmetric``; zeros None), or 15 steps from the smallest to the largest value, zero among them.
    ``scale_dtype`` is bf16 or fp16 (default: the weight's own, bf16 for fp32)."""
    if weight.dim() not in (2, 3) or not weight.is_floating_point():
        raise ValueError("weight must be a floating-point [N, K] or [experts, N, K]")
    K = weight.shape[-1]
    _check_group(K, group_size)
    if scale_dtype is None:
        scale_dtype = weight.dtype if weight.dtype in _HALF else torch.bfloat16
    if scale_dtype not in _HALF:
        raise TypeError("scale_dtype must be bfloat16 or float16")
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("weight holds values that are not finite")
    parts = []
    for w in (weight if weight.dim() == 3 else weight.unsqueeze(0)):
        x = w.detach().float().view(w.shape[0], K // group_size, group_size)
        if symmetric:
            zero = torch.full(x.shape[:2], 8.0, device=x.device)
            scale = x.abs().amax(dim=2) / 7.0
        else:
            low, high = x.amin(dim=2).clamp(max=0.0), x.amax(dim=2).clamp(min=0.0)
            scale = (high - low) / 15.0
        scale = scale.to(scale_dtype)
        used = scale.float()
        if not bool(torch.isfinite(used).all()):
            raise ValueError(f"a group's scale does not fit {scale_dtype}")
        used = torch.where(used == 0, torch.ones_like(used), used)
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        if not symmetric:
            zero = (-low / used).round().clamp(0.0, 15.0)
        q = ((x / used.unsqueeze(2)).round() + zero.unsqueeze(2)).clamp(0.0, 15.0).to(torch.uint8).view(w.shape)
        parts.append((q[:, 0::2] | (q[:, 1::2] << 4), scale, None if symmetric else zero.to(torch.uint8)))
    if weight.dim() == 2:
        return parts[0]
    return (torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]),
            None if symmetric else torch.stack([p[2] for p in parts]))


def dequantize_int4(qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights that the format stands for, fp32 [..., N, K]."""
    q = torch.stack([qweight & 15, qweight >> 4], dim=-1).flatten(-2)
    group = q.shape[-1] // scales.shape[-1]
    w = q.unflatten(-1, (scales.shape[-1], group)).float()
    w = w - (8.0 if zeros is None else (zeros & 15).float().unsqueeze(-1))
    return (w * scales.float().unsqueeze(-1)).flatten(-2)


class _Int4Weights:
    """4-bit weights in the kernels' layout; on the CPU as they were given."""

    def __init__(self, qweight, scales, zeros, dims: int):
        if qweight.dim() != dims or qweight.dtype != torch.uint8:
            raise ValueError("qweight must be uint8 " + ("[N, K / 2]" if dims == 2 else "[experts, N, K / 2]"))
        if scales.dim() != dims or scales.shape[:-1] != qweight.shape[:-1] or scales.shape[-1] < 1:
            raise ValueError("scales must be [..., N, K / group] beside qweight [..., N, K / 2]")
        if scales.dtype not in _HALF:
            raise TypeError("scales must be bfloat16 or float16")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8):
            raise ValueError("zeros must be uint8 in the shape of scales")
        if any(t is not None and t.device != qweight.device for t in (scales, zeros)):
            raise ValueError("qweight, scales and zeros must share a device")
        self.N, self.K = qweight.shape[-2], 2 * qweight.shape[-1]
        if self.N > MAX_SIDE or self.K > MAX_SIDE:
            raise ValueError(f"weights of at most {MAX_SIDE} rows and columns, got {self.N} and {self.K}")
        if self.N < 1 or self.K % scales.shape[-1]:
            raise ValueError(f"{scales.shape[-1]} scales per row do not divide K = {self.K}")
        self.group = self.K // scales.shape[-1]
        _check_group(self.K, self.group)
        self.E = qweight.shape[0] if dims == 3 else 1
        if not 1 <= self.E <= MAX_EXPERTS:
            raise ValueError(f"between 1 and {MAX_EXPERTS} experts, got {self.E}")
        self.device, self.scale_dtype = qweight.device, scales.dtype
        self.qweight = self.scales = self.zeros = None
        qweight, scales = qweight.detach().contiguous(), scales.detach().contiguous()
        zeros = zeros.contiguous() if zeros is not None else None
        if not qweight.is_cuda:
            self.qweight, self.scales, self.zeros = qweight, scales, zeros
            return
        if qweight.data_ptr() % 2:
            qweight = qweight.clone()
        Np, Kp = -(-self.N // 128) * 128, -(-self.K // 128) * 128
        groups = Kp // min(self.group, 128)
        self.packed = torch.empty(self.E * Np * Kp // 2, dtype=torch.uint8, device=self.device)
        self.packed_scales = torch.empty(self.E * groups * Np, dtype=self.scale_dtype, device=self.device)
        self.packed_zeros = torch.empty(self.E * groups * Np, dtype=torch.uint8, device=self.device) \
            if zeros is not None else None
        a = Int4Layout()
        a.q, a.scales, a.zeros = qweight.data_ptr(), scales.data_ptr(), zeros.data_ptr() if zeros is not None else None
        a.packed, a.scales_out = self.packed.data_ptr(), self.packed_scales.data_ptr()
        a.zeros_out = self.packed_zeros.data_ptr() if zeros is not None else None
        a.experts, a.N, a.K, a.group = self.E, self.N, self.K, self.group
        self._status = torch.zeros(4, dtype=torch.int32, device=self.device)
        with device_guard(self.device):
            a.stream = current_stream_ptr(self.device)
            _native.check(_native.lib().fluxb_int4_layout(ctypes.byref(a)), "fluxb_int4_layout")
        a = self._args = Int4GemmArgs()                # what every call has in common
        a.packed, a.scales = self.packed.data_ptr(), self.packed_scales.data_ptr()
        if self.packed_zeros is not None:
            a.zeros = self.packed_zeros.data_ptr()
        a.experts, a.N, a.K, a.group = self.E, self.N, self.K, self.group
        a.scale_dtype, a.status = dtype_code(self.scale_dtype), self._status.data_ptr()

    def check_status(self) -> None:
        """Raises if a wait inside a launch so far ran out of time (its results are then not to be used)."""
        if self.device.type == "cuda" and self._status.tolist()[0] != 0:
            self._status.zero_()
            raise FluxTimeoutError("product with 4-bit weights: a wait inside the kernel timed out")

    # ------------------------------------------------------------------------------
    def _check_input(self, x, output_buf, bias=None):
        shape, dtype = x.shape, x.dtype
        if len(shape) != 2 or shape[1] != self.K:
            raise ValueError(f"input must be [rows, {self.K}], got {tuple(shape)}")
        if dtype not in _HALF and (x.is_cuda or dtype != torch.float32):
            raise TypeError(f"input must be bfloat16 or float16, got {dtype}")
        if x.device != self.device:
            raise ValueError(f"input is on {x.device}, the weights on {self.device}")
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)) \
                or has_tangent(x, bias):
            raise RuntimeError("products with 4-bit weights have no backward; call them under torch.no_grad()")
        if output_buf is not None and (output_buf.shape != (shape[0], self.N) or output_buf.dtype != dtype
                                       or output_buf.device != self.device or (self.N > 1 and output_buf.stride(1) != 1)
                                       or (shape[0] > 1 and output_buf.stride(0) < self.N)):
            raise ValueError("output_buf must be [rows, N] of the input's type, on its device, with contiguous rows that do "
                             "not overlap")

    def _launch(self, x, bias, splits, output_buf):
        rows = x.shape[0]
        out = output_buf if output_buf is not None else x.new_empty((rows, self.N))
        ldx, inner = x.stride()
        if rows == 1:
            ldx = self.K
        ptr = x.data_ptr()
        if inner != 1 or ldx % 8 or ptr % 16:          # (the kernels read rows in 16-byte pieces)
            x = x.clone(memory_format=torch.contiguous_format)
            ldx, ptr = self.K, x.data_ptr()
        a = Int4GemmArgs.from_buffer_copy(self._args)  # (a copy: calls may come from several threads)
        a.x, a.out, a.M, a.ldx, a.ldo = ptr, out.data_ptr(), rows, ldx, out.stride(0)
        if bias is not None:
            a.bias = bias.data_ptr()
        if splits is not None:
            a.splits = splits.data_ptr()
        a.dtype = dtype_code(x.dtype)
        with device_guard(self.device):
            a.stream = current_stream_ptr(self.device)
            _native.check(_native.lib().fluxb_int4_gemm(ctypes.byref(a)), "fluxb_int4_gemm")
        return out


class Int4Gemm(_Int4Weights):
    """``forward(input [M, K]) -> [M, N]`` = input @ w^T (+ bias [N]) with the 4-bit weights laid out at construction."""

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None):
        super().__init__(qweight, scales, zeros, 2)

    def forward(self, input: torch.Tensor, bias: Optional[torch.Tensor] = None,
                output_buf: Optional[torch.Tensor] = None) -> torch.Tensor:
        self._check_input(input, output_buf, bias)
        if bias is not None:
            if bias.numel() != self.N or bias.shape[-1] != self.N or bias.dtype != input.dtype \
                    or bias.device != input.device:
                raise ValueError("bias must be [N] or [1, N] in the input's type, on its device")
            bias = bias.detach().reshape(-1).contiguous()
        if input.is_cuda:
            return self._launch(input, bias, None, output_buf)
        y = input.float() @ dequantize_int4(self.qweight, self.scales, self.zeros).t()
        if bias is not None:
            y = y + bias.float()
        y = y.to(input.dtype)
        return y if output_buf is None else output_buf.copy_(y)

    __call__ = forward


class Int4GemmGrouped(_Int4Weights):
    """``forward(input [rows, K], splits [experts]) -> [rows, N]``: rows sorted by expert, ``splits[e]`` of them (int32, on
    the device; nothing is read back) times the weights of expert e. Rows behind the last expert's stay as they are in
    ``output_buf`` and are undefined in a fresh result."""

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None):
        super().__init__(qweight, scales, zeros, 3)

    def forward(self, input: torch.Tensor, splits: torch.Tensor, output_buf: Optional[torch.Tensor] = None) -> torch.Tensor:
        self._check_input(input, output_buf)
        if splits.numel() != self.E or splits.is_floating_point() or splits.dtype == torch.bool:
            raise ValueError(f"splits must hold one row count for each of {self.E} experts")
        if input.is_cuda:
            if splits.dtype != torch.int32 or splits.device != self.device or not splits.is_contiguous():
                splits = splits.to(device=self.device, dtype=torch.int32, non_blocking=True).contiguous()
            return self._launch(input, None, splits, output_buf)
        y = output_buf if output_buf is not None else torch.zeros((input.shape[0], self.N), dtype=input.dtype)
        row = 0
        for e, count in enumerate(splits.reshape(-1).tolist()):
            count = max(0, min(count, input.shape[0] - row))
            w = dequantize_int4(self.qweight[e], self.scales[e], None if self.zeros is None else self.zeros[e])
            y[row:row + count] = (input[row:row + count].float() @ w.t()).to(input.dtype)
            row += count
        return y

    __call__ = forward
