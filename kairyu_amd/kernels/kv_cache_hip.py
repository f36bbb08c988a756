"""Launches of the paged e4m3 key/value cache's kernels: the rotation and append,
attention, drafted trees, and moves of tokens and pages.  Shapes and types are checked
by the public functions (``kairyu_amd/attention.py``, ``drafts.py``, ``pages.py``);
all launch on torch's current stream of the tensors' device and read lengths and tables
on the device only."""

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


# (torch.cuda.current_device, which this device's tensors have initialised, without its checks)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def call_on(device: torch.device, entry: str, *args) -> None:
    """``entry`` on torch's current stream of ``device``, with that device current
    for the launch."""

    if device.index == _current_device():
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


def rotate_append(q, k, v, shape, cache, cache_shape, table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps,
                  positions):
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
    at = () if positions is None else (positions.data_ptr(),)
    call_on(
        device, "kq_kv_rotate_append_at" if at else "kq_kv_rotate_append", *at, q_at, q_row, q_head, k_at, k_row, k_head, v_at, v_row, v_head,
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


@lru_cache(maxsize=4096)
def _tree_bytes(*shape: int) -> int:
    return int(_native.library().kq_kv_tree_attention_workspace_size(*shape))


def tree_attention(q, shape, cache, cache_shape, table, cu_rows, lengths, scale, tree, words, window):
    device = q.device
    require_device(device, "attention over a key/value cache")
    q, q_at, q_row, q_head = _heads(q)
    rows, heads, dim = shape
    pages, kv_heads, page, _ = cache_shape
    seqs, width = table.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    need = _tree_bytes(rows, heads, kv_heads, dim, page, width, seqs)  # (of the call's own, as attention's)
    scratch = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    call_on(
        device, "kq_kv_tree_attention", q_at, q_row, q_head, _native.dtype_code(q.dtype), rows, heads, kv_heads, dim,
        cache[0].data_ptr(), cache[1].data_ptr(), cache[2].data_ptr(), cache[3].data_ptr(), pages, page, table.data_ptr(),
        _pitch(table, seqs, width), width, cu_rows.data_ptr(), lengths.data_ptr(), seqs, tree[0].data_ptr(), words,
        tree[1].data_ptr(), scale, window, out.data_ptr(), _native.ptr(scratch), need,
    )
    return out


def draft_tree(parents, cu_rows, lengths, most, window):
    device = parents.device
    require_device(device, "a tree of drafts")
    rows, seqs = parents.shape[0], lengths.shape[0]
    mask, positions = parents.new_empty((rows, -(-most // 32))), parents.new_empty(rows)
    call_on(device, "kq_draft_tree", parents.data_ptr(), rows, cu_rows.data_ptr(), lengths.data_ptr(), seqs, most, window,
            mask.data_ptr(), positions.data_ptr())
    return mask, positions


def accept_drafts(tokens, targets, parents, cu_rows, most):
    device = tokens.device
    require_device(device, "the walk along drafts")
    rows, seqs = tokens.shape[0], cu_rows.shape[0] - 1
    kept, counts, following = parents.new_empty((seqs, most)), parents.new_empty(seqs), tokens.new_empty(seqs)
    call_on(device, "kq_draft_accept", tokens.data_ptr(), targets.data_ptr(), tokens.dtype is torch.int64, parents.data_ptr(),
            rows, cu_rows.data_ptr(), seqs, most, kept.data_ptr(), counts.data_ptr(), following.data_ptr())
    return kept, counts, following


def keep_tokens(caches, table, cu_rows, lengths, kept, counts):
    device = table.device
    require_device(device, "the move of kept tokens")
    pages, kv_heads, page, dim = caches.shape
    seqs, width = table.shape
    out = torch.empty_like(lengths)
    call_on(device, "kq_kv_keep_tokens", caches.pointers, len(caches.layers), pages, kv_heads, page, dim, table.data_ptr(),
            _pitch(table, seqs, width), width, cu_rows.data_ptr(), lengths.data_ptr(), seqs, kept.data_ptr(), kept.shape[1],
            counts.data_ptr(), out.data_ptr())
    return out


def copy_pages(caches, sources, targets):
    device = sources.device
    require_device(device, "the copy of pages")
    pages, kv_heads, page, dim = caches.shape
    call_on(device, "kq_kv_copy_pages", caches.pointers, len(caches.layers), pages, kv_heads, page, dim, sources.data_ptr(),
            targets.data_ptr(), sources.shape[0])


@lru_cache(maxsize=4096)
def _fork_bytes(*shape: int) -> int:
    return int(_native.library().kq_kv_fork_workspace_size(*shape))


def fork_sequences(caches, holders, table, lengths, parents, room):
    device = table.device
    require_device(device, "the fork of sequences")
    pages, kv_heads, page, dim = caches.shape
    seqs, width = table.shape
    rows = parents.shape[0]
    new_table, new_lengths, missing = table.new_empty((rows, width)), table.new_empty(rows), table.new_empty(1)
    need = _fork_bytes(seqs, rows, width, page, room)
    scratch = table.new_empty(need // 4)
    call_on(device, "kq_kv_fork_sequences", caches.pointers, len(caches.layers), pages, kv_heads, page, dim, holders.data_ptr(),
            table.data_ptr(), _pitch(table, seqs, width), width, lengths.data_ptr(), seqs, parents.data_ptr(), rows, room,
            new_table.data_ptr(), new_lengths.data_ptr(), missing.data_ptr(), scratch.data_ptr(), need)
    return new_table, new_lengths, missing
