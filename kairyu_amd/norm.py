"""The norms around a decoder block, fused with its gate and residual scale.

``block_norm`` runs what lies between a block's output projection and the next
block's first one: the norm after the block, its gate and residual scale, the
residual sum, and the norm before the next block, whose rows come out in 16 bits
or quantized as this package's activation quantizers lay them out.  The library's
W8A8 and block-FP8 GEMM entries (``include/kairyu_quant.h``) take quantized rows and
their scales; the module classes and packs take 16-bit rows and quantize them
themselves.  Counterpart of the reference's RMS norm kernels
(kairyu/kernels/rms_norm_gpu.py).
"""

from __future__ import annotations

import torch

from kairyu_amd import _native
from kairyu_amd.kernels import kv_cache_hip as hip

__all__ = ["block_norm"]

MODES = {None: 0, "fp8": 1, "int8": 2, "fp8_block": 3}
Y_DTYPES = (None, torch.float8_e4m3fn, torch.int8, torch.float8_e4m3fn)
MAX_HIDDEN = 32768


def block_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, *,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               residual_scale: float = 1.0, eps: float = 1e-6, unit_offset: bool = False,
               quantize: str | None = None) -> tuple[torch.Tensor, ...]:
    """``r = residual + residual_scale * gate * (x / rms(x) * post_weight)`` and
    ``y = r / rms(r) * weight`` for rows ``x [..., H]``, ``rms(z) =
    sqrt(mean(z^2) + eps)``.

    ``x``, the weights ``[H]`` and ``gate`` (``[H]``, or a row for each of ``x``'s)
    are fp16 or bf16 alike; ``residual`` is of that dtype or fp32 and shaped like
    ``x`` (None: zero, and ``r`` of ``x``'s dtype).  Without ``post_weight`` the
    block's output is not normed, without ``gate`` not gated; ``unit_offset`` keeps
    the norms' weights as their difference from one.  All is computed in fp32; ``r``
    and ``y`` are each rounded once.

    Returns ``(r, y)``, or with ``quantize`` ``(r, yq, scales)`` as the activation
    quantizers lay them out: ``"fp8"`` / ``"int8"`` per row (scales ``[..., 1]``),
    ``"fp8_block"`` per 128 elements (scales ``[..., ceil(H / 128)]``)."""

    mode = MODES.get(quantize)
    if mode is None:
        raise ValueError(f"quantize must be one of {tuple(MODES)}, got {quantize!r}")
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_HIDDEN:
        raise ValueError(f"rows must have 1 to {MAX_HIDDEN} elements, got {tuple(shape)}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"block_norm supports float16/bfloat16 rows, got {dtype}")
    hidden = shape[-1]
    for name, t in (("weight", weight), ("post_weight", post_weight), ("gate", gate)):
        if t is None:
            continue
        if t.dtype is not dtype or t.device != device:
            raise ValueError(f"{name} must have the rows' dtype and device, got {t.dtype} on {t.device}")
        if t.shape != (hidden,) and not (name == "gate" and t.shape == shape):
            raise ValueError(f"{name} {tuple(t.shape)} does not match rows {tuple(shape)}")
    r_dtype = dtype
    if residual is not None:
        r_dtype = residual.dtype
        if residual.shape != shape or residual.device != device:
            raise ValueError(f"residual {tuple(residual.shape)} on {residual.device} does not match rows "
                             f"{tuple(shape)} on {device}")
        if r_dtype is not dtype and r_dtype is not torch.float32:
            raise ValueError(f"residual must be {dtype} or float32, got {r_dtype}")
    if torch.is_grad_enabled():
        for t in (x, residual, weight, post_weight, gate):
            if t is not None and t.requires_grad:
                raise RuntimeError("block_norm is for inference: an input requires a gradient")
    if not x.is_cuda:
        return _plain(x, residual, weight, post_weight, gate, residual_scale, eps, unit_offset, quantize)
    hip.require_device(device, "block_norm")
    flat, pitch, rows = _rows(x, hidden)
    res, res_pitch, _ = (None, 0, 0) if residual is None else _rows(residual, hidden)
    gates, gate_pitch = gate, 0
    if gate is not None:
        if len(shape) == 1 or gate.dim() > 1:
            gates, gate_pitch, _ = _rows(gate, hidden)
        else:
            gates = gate.contiguous()
    r = torch.empty_like(x, dtype=r_dtype, memory_format=torch.contiguous_format)
    y = torch.empty_like(x, dtype=Y_DTYPES[mode], memory_format=torch.contiguous_format) if mode else torch.empty_like(
        x, memory_format=torch.contiguous_format)
    scales = None
    if mode:
        scales = torch.empty((*shape[:-1], -(-hidden // 128) if mode == 3 else 1), device=device, dtype=torch.float32)
    weight = weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    hip.call_on(
        device, "kq_block_norm", flat.data_ptr(), _native.dtype_code(dtype), rows, hidden, pitch, _native.ptr(res),
        _native.dtype_code(r_dtype), res_pitch, _native.ptr(post_weight), _native.ptr(gates), gate_pitch, residual_scale,
        weight.data_ptr(), 1.0 if unit_offset else 0.0, eps, mode, r.data_ptr(), y.data_ptr(), _native.ptr(scales),
    )
    return (r, y) if scales is None else (r, y, scales)


def _rows(x: torch.Tensor, hidden: int) -> tuple[torch.Tensor, int, int]:
    """``x`` as rows of unit stride (a view where it has them, else a copy), the pitch
    from one to the next, at least their width, and their number."""

    if x.is_contiguous():
        return x, hidden, x.numel() // hidden
    if x.dim() != 2:
        x = x.reshape(-1, hidden)
    rows, (pitch, unit) = x.shape[0], x.stride()
    if unit == 1 and pitch >= hidden:
        return x, pitch, rows
    return x.contiguous(), hidden, rows


def _rms(x, weight, offset, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * (weight.to(torch.float32) + offset)


def _plain(x, residual, weight, post_weight, gate, residual_scale, eps, unit_offset, quantize):
    """The definition in fp32 torch operations (CPU tensors)."""

    offset = 1.0 if unit_offset else 0.0
    b = x.to(torch.float32)
    if post_weight is not None:
        b = _rms(b, post_weight, offset, eps)
    if gate is not None:
        b = b * gate.to(torch.float32)
    r = residual_scale * b if residual is None else residual.to(torch.float32) + residual_scale * b
    y = _rms(r, weight, offset, eps)
    r = r.to(x.dtype if residual is None else residual.dtype)
    if quantize is None:
        return r, y.to(x.dtype)
    if quantize == "fp8_block":
        hidden = y.shape[-1]
        y = torch.nn.functional.pad(y, (0, -hidden % 128)).unflatten(-1, (-1, 128))
    most = 127.0 if quantize == "int8" else 448.0
    scales = y.abs().amax(-1, keepdim=True).clamp(min=1e-12) / most
    z = (y / scales).clamp(-most, most)
    if quantize == "int8":
        return r, z.round().to(torch.int8), scales
    z = z.to(torch.float8_e4m3fn)
    return (r, z.flatten(-2)[..., :hidden].contiguous(), scales[..., 0]) if quantize == "fp8_block" else (r, z, scales)
