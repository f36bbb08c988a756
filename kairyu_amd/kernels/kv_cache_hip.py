"""Launches of the paged e4m3 key/value cache's kernels: the rotation and append,
and attention.  Shapes and types are checked by the public functions
(``kairyu_amd/attention.py``); both launch on torch's current stream of the
tensors' device and read lengths and tables on the device only."""

from __future__ import annotations

from functools import lru_cache

import torch

from kairyu_amd import _native
from kairyu_amd.kernels.quant_gemm_hip import REQUIRED_ARCH, _arch_of


@lru_cache(maxsize=None)
def _supported(index: int) -> str:
    """The device's architecture; raises without the library."""

    _native.library()
    return _arch_of(index)


def require_device(device: torch.device, what: str) -> None:
    try:
        arch = _supported(device.index)
    except RuntimeError as error:
        raise RuntimeError(f"{what} on a device requires the kairyu_amd HIP library: {error}") from error
    if arch != REQUIRED_ARCH:
        raise RuntimeError(f"{what} requires {REQUIRED_ARCH}, got {arch}")


def call_on(device: torch.device, entry: str, *args) -> None:
    """``entry`` on torch's current stream of ``device``, with that device current
    for the launch."""

    if device.index == torch.cuda.current_device():
        _native.call(entry, *args, _native.stream_handle(device))
        return
    with torch.cuda.device(device):
        _native.call(entry, *args, _native.stream_handle(device))


def aligned(x: torch.Tensor) -> torch.Tensor:
    """fp16 / bf16 ``x`` with unit stride in its last dimension and every row 16-byte
    aligned: itself where it is so, else a contiguous copy."""

    *outer, unit = x.stride()
    if unit == 1 and x.data_ptr() % 16 == 0 and not any(s % 8 for s in outer):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def rotate_append(q, k, v, shape, cache, cache_shape, table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps):
    device = q.device
    require_device(device, "the key/value append")
    q, k, v = aligned(q), aligned(k), aligned(v)
    rows, heads, dim = shape
    pages, kv_heads, page, _ = cache_shape
    out = torch.empty(shape, device=device, dtype=q.dtype)
    (q_row, q_head, _), (k_row, k_head, _), (v_row, v_head, _) = q.stride(), k.stride(), v.stride()
    angles = (0, 0) if cos_sin is None else cos_sin.shape
    seqs, width = table.shape
    call_on(
        device, "kq_kv_rotate_append", q.data_ptr(), q_row, q_head, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
        _native.dtype_code(q.dtype), rows, heads, kv_heads, dim, cache[0].data_ptr(), cache[1].data_ptr(),
        cache[2].data_ptr(), cache[3].data_ptr(), pages, page, table.data_ptr(), _pitch(table, seqs, width), width,
        cu_rows.data_ptr(), lengths.data_ptr(), seqs, _native.ptr(cos_sin), angles[0], angles[1], interleaved,
        _native.ptr(q_norm), _native.ptr(k_norm), eps, out.data_ptr(),
    )
    return out


def _pitch(table: torch.Tensor, seqs: int, width: int) -> int:
    return table.stride(0) if seqs > 1 else width


@lru_cache(maxsize=4096)
def _attention_bytes(*shape: int) -> int:
    return int(_native.library().kq_kv_attention_workspace_size(*shape))


def attention(q, shape, cache, cache_shape, table, cu_rows, lengths, scale, causal, window):
    device = q.device
    require_device(device, "attention over a key/value cache")
    q = aligned(q)
    rows, heads, dim = shape
    pages, kv_heads, page, _ = cache_shape
    seqs, width = table.shape
    out = torch.empty(shape, device=device, dtype=q.dtype)
    # partial results of split sequences, of the call's own: torch's allocator keeps
    # them to the calling stream and, under capture, to the graph
    need = _attention_bytes(rows, heads, kv_heads, dim, page, width, seqs)
    scratch = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    q_row, q_head, _ = q.stride()
    call_on(
        device, "kq_kv_attention", q.data_ptr(), q_row, q_head, _native.dtype_code(q.dtype), rows, heads, kv_heads, dim,
        cache[0].data_ptr(), cache[1].data_ptr(), cache[2].data_ptr(), cache[3].data_ptr(), pages, page, table.data_ptr(),
        _pitch(table, seqs, width), width, cu_rows.data_ptr(), lengths.data_ptr(), seqs, scale, causal, window,
        out.data_ptr(), _native.ptr(scratch), need,
    )
    return out
