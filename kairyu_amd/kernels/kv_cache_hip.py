"""Launches of the paged e4m3 key/value cache's kernels: the rotation and append,
and attention.  Shapes and types are checked by the public functions
(``kairyu_amd/attention.py``); both launch on torch's current stream of the
tensors' device and read lengths and tables on the device only."""

from __future__ import annotations

from functools import lru_cache

import torch

from kairyu_amd import _native
from kairyu_amd.kernels.quant_gemm_hip import REQUIRED_ARCH, _device_arch


def require_device(device: torch.device, what: str) -> None:
    try:
        _native.library()
    except RuntimeError as error:
        raise RuntimeError(f"{what} on a device requires the kairyu_amd HIP library: {error}") from error
    if _device_arch(device) != REQUIRED_ARCH:
        raise RuntimeError(f"{what} requires {REQUIRED_ARCH}, got {_device_arch(device)}")


def call_on(device: torch.device, entry: str, *args) -> None:
    """``entry`` on torch's current stream of ``device``, with that device current
    for the launch."""

    if device.index is None or device.index == torch.cuda.current_device():
        _native.call(entry, *args, _native.stream_handle(device))
        return
    with torch.cuda.device(device):
        _native.call(entry, *args, _native.stream_handle(device))


def aligned(x: torch.Tensor, vector: int = 8) -> torch.Tensor:
    """``x`` with unit stride in its last dimension, every row 16-byte aligned:
    itself where it is so, else a contiguous copy."""

    strides = x.stride()
    if strides[-1] == 1 and x.data_ptr() % 16 == 0 and all(s % vector == 0 for s in strides[:-1]):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def rotate_append(q, k, v, cache, table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps):
    require_device(q.device, "the key/value append")
    q, k, v = aligned(q), aligned(k), aligned(v)
    rows, heads, dim = q.shape
    pages, kv_heads, page, _ = cache.k.shape
    out = torch.empty((rows, heads, dim), device=q.device, dtype=q.dtype)
    call_on(
        q.device, "kq_kv_rotate_append", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
        v.data_ptr(), v.stride(0), v.stride(1), _native.dtype_code(q.dtype), rows, heads, kv_heads, dim,
        cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page,
        table.data_ptr(), table.stride(0), table.shape[1], cu_rows.data_ptr(), lengths.data_ptr(), lengths.shape[0],
        _native.ptr(cos_sin), 0 if cos_sin is None else cos_sin.shape[0], 0 if cos_sin is None else cos_sin.shape[1],
        int(interleaved), _native.ptr(q_norm), _native.ptr(k_norm), eps, out.data_ptr(),
    )
    return out


@lru_cache(maxsize=4096)
def _attention_bytes(device_index: int, *shape: int) -> int:
    return int(_native.library().kq_kv_attention_workspace_size(*shape))


def attention(q, cache, table, cu_rows, lengths, scale, causal, window):
    require_device(q.device, "attention over a key/value cache")
    q = aligned(q)
    rows, heads, dim = q.shape
    pages, kv_heads, page, _ = cache.k.shape
    out = torch.empty((rows, heads, dim), device=q.device, dtype=q.dtype)
    seqs, width = lengths.shape[0], table.shape[1]
    # partial results of split sequences, of the call's own: torch's allocator keeps
    # them to the calling stream and, under capture, to the graph
    need = _attention_bytes(q.device.index or 0, rows, heads, kv_heads, dim, page, width, seqs)
    scratch = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    call_on(
        q.device, "kq_kv_attention", q.data_ptr(), q.stride(0), q.stride(1), _native.dtype_code(q.dtype), rows, heads,
        kv_heads, dim, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages,
        page, table.data_ptr(), table.stride(0), width, cu_rows.data_ptr(), lengths.data_ptr(), seqs, scale, int(causal),
        window, out.data_ptr(), _native.ptr(scratch), need,
    )
    return out
