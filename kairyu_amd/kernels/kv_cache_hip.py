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


def _heads(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """fp16 / bf16 ``x [rows, heads, dim]`` with unit stride in its last dimension and
    every head 16-byte aligned (itself where it is so, else a contiguous copy), its
    address and its pitches from row to row and head to head."""

    row, head, unit = x.stride()
    at = x.data_ptr()
    if unit != 1 or at & 15 or (row | head) & 7:
        x = x.clone(memory_format=torch.contiguous_format)
        row, head, unit = x.stride()
        at = x.data_ptr()
    return x, at, row, head


def _weight(w: torch.Tensor | None) -> torch.Tensor | None:
    """Norm weights, contiguous and 16-byte aligned."""

    if w is None or (w.is_contiguous() and not w.data_ptr() & 15):
        return w
    return w.clone(memory_format=torch.contiguous_format)


def rotate_append(q, k, v, shape, cache, cache_shape, table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps):
    device = q.device
    require_device(device, "the key/value append")
    q, q_at, q_row, q_head = _heads(q)
    k, k_at, k_row, k_head = _heads(k)
    v, v_at, v_row, v_head = _heads(v)
    q_norm, k_norm = _weight(q_norm), _weight(k_norm)
    rows, heads, dim = shape
    pages, kv_heads, page, _ = cache_shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    angles = (0, 0) if cos_sin is None else cos_sin.shape
    seqs, width = table.shape
    call_on(
        device, "kq_kv_rotate_append", q_at, q_row, q_head, k_at, k_row, k_head, v_at, v_row, v_head,
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
    q, q_at, q_row, q_head = _heads(q)
    rows, heads, dim = shape
    pages, kv_heads, page, _ = cache_shape
    seqs, width = table.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    # partial results of split sequences, of the call's own: torch's allocator keeps
    # them to the calling stream and, under capture, to the graph
    need = _attention_bytes(rows, heads, kv_heads, dim, page, width, seqs)
    scratch = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    call_on(
        device, "kq_kv_attention", q_at, q_row, q_head, _native.dtype_code(q.dtype), rows, heads, kv_heads, dim,
        cache[0].data_ptr(), cache[1].data_ptr(), cache[2].data_ptr(), cache[3].data_ptr(), pages, page, table.data_ptr(),
        _pitch(table, seqs, width), width, cu_rows.data_ptr(), lengths.data_ptr(), seqs, scale, causal, window,
        out.data_ptr(), _native.ptr(scratch), need,
    )
    return out
