"""A paged 8-bit key/value cache: rotary append, and attention over it.

What a decoder layer runs between its packed q/k/v projection and its output
projection (the reference's ``Attention.forward_decode_tensors``,
kairyu/models/attention.py:315-351, with its rotary and paged-write kernels,
kairyu/kernels/rope_gpu.py and paged_kv_write_gpu.py), over a cache of e4m3
codes with one power-of-two scale per page and head:

* :func:`rotate_append` rotates queries and keys by their positions (after
  Qwen3's per-head norms, if given) and stores keys and values, one launch.
* :func:`paged_attention` attends to the cache: single tokens, prompts, chunks
  of prompts and any mix of them in one ragged batch.
* :func:`tree_attention` attends with drafted tokens that branch, each seeing the
  tokens before all drafts and its own ancestors (``kairyu_amd/drafts.py``).

:meth:`QuantLinearPack.attend` runs them behind a pack's projection.  A batch is
given by ``cu_rows [S + 1]`` (sequence ``s`` has rows ``cu_rows[s]`` up to
``cu_rows[s + 1]``), ``lengths [S]`` (its tokens, the new ones included and last)
and ``block_table [S, W]`` (its pages in order), int32 on the device and never
read by the host, so every call can be captured into a graph and replayed for
other lengths.  Rows past ``cu_rows[S]`` are padding: zero in the outputs, nothing
stored.  Calls on several streams share nothing but the cache itself.

On CPU tensors the same is computed by elementary torch operations.  Like the
rest of the package this is for inference: inputs that require a gradient are
refused.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from kairyu_amd.kernels import kv_cache_hip as hip

__all__ = ["DraftTree", "PagedKvCache", "paged_attention", "rotary_table", "rotate_append", "tree_attention"]

E4M3 = torch.float8_e4m3fn
HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128)
MOST_NODES = 1024  # drafted tokens of one sequence


class PagedKvCache(NamedTuple):
    """Codes ``[pages, kv_heads, page_size, head_dim]`` and fp32 scales
    ``[pages, kv_heads]`` of keys and values; an element is ``code * scale``.  The
    append writes powers of two; scales of the caller's own must be positive and
    finite (a page of zeros too), and values' codes not NaN."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def create(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
               device: torch.device | str = "cuda") -> PagedKvCache:
        """An empty cache: ``pages * page_size`` tokens, ``2 * kv_heads *
        head_dim`` bytes each."""

        codes = [torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(E4M3)
                 for _ in range(2)]
        scales = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        cache = cls(*codes, *scales)
        _check_cache(cache)
        return cache

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


class DraftTree(NamedTuple):
    """Drafted tokens of a batch's rows (:func:`kairyu_amd.drafts.draft_tree`, or the
    caller's own): ``mask [R, words]`` int32, whose bit ``j % 32`` of word ``j // 32``
    says that the row sees its sequence's ``j``-th new token (itself among them), and
    ``positions [R]`` int32, the place of each in its own continuation; a row whose
    position is negative sees nothing."""

    mask: torch.Tensor
    positions: torch.Tensor


def rotary_table(positions: int, rotary_dim: int, theta: float = 10000.0,
                 device: torch.device | str = "cuda") -> torch.Tensor:
    """fp32 ``[positions, rotary_dim]``: each position's ``rotary_dim / 2``
    cosines, then its sines, of angles ``position * theta^(-2i / rotary_dim)``.
    The angles are formed in fp64: in fp32 a position of 100,000 is off by up to
    2^-8 of a radian already.  Scaled variants (other frequencies, a factor on
    the amplitudes) are tables of the caller's own."""

    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    frequency = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * frequency
    return torch.cat((angle.cos(), angle.sin()), dim=-1).to(torch.float32).to(device)


# ------------------------------------------------------------------ checks
# (a decode step's call is bound by this host path: each property is read once)
def _check_cache(cache: PagedKvCache) -> torch.Size:
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"cache keys {tuple(shape)} and values {tuple(v.shape)} must be alike, "
                         "[pages, kv_heads, page_size, head_dim]")
    if k.dtype is not E4M3 or v.dtype is not E4M3:
        raise ValueError(f"cache codes must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
    scales = shape[:2]
    if ks.shape != scales or vs.shape != scales or ks.dtype is not torch.float32 or vs.dtype is not torch.float32:
        raise ValueError(f"cache scales must be float32 {tuple(scales)}")
    if shape[3] not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS}, got {shape[3]}")
    if shape[2] not in PAGE_SIZES:
        raise ValueError(f"page size must be one of {PAGE_SIZES}, got {shape[2]}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError("cache codes must be 16-byte aligned")
    return shape


def _check_batch(q: torch.Tensor, cache: PagedKvCache, cache_shape: torch.Size, table, cu_rows, lengths) -> torch.Size:
    """The queries, the cache and the batch; the queries' shape."""

    shape, device = q.shape, q.device
    if len(shape) != 3 or shape[2] != cache_shape[3]:
        raise ValueError(f"q must be [rows, heads, {cache_shape[3]}], got {tuple(shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if shape[1] < 1 or cache_shape[1] < 1 or shape[1] % cache_shape[1]:
        raise ValueError(f"{shape[1]} query heads are not a multiple of {cache_shape[1]} kv heads")
    table_shape, cu_shape, seqs = table.shape, cu_rows.shape, lengths.shape
    if len(table_shape) != 2 or len(seqs) != 1 or len(cu_shape) != 1:
        raise ValueError("block_table must be [S, W], cu_rows [S + 1] and lengths [S]")
    if table_shape[0] != seqs[0] or cu_shape[0] != seqs[0] + 1:
        raise ValueError(f"block_table {tuple(table_shape)} and cu_rows {tuple(cu_shape)} do not match {seqs[0]} lengths")
    if table.dtype is not torch.int32 or cu_rows.dtype is not torch.int32 or lengths.dtype is not torch.int32:
        raise ValueError(f"block_table, cu_rows and lengths must be int32, got {table.dtype}, {cu_rows.dtype}, {lengths.dtype}")
    if not (cu_rows.is_contiguous() and lengths.is_contiguous() and (table.is_contiguous() or _rows_apart(table))):
        raise ValueError("cu_rows, lengths and the rows of block_table must be contiguous, and its rows not overlap")
    for t in (*cache, table, cu_rows, lengths):
        if t.device != device:
            raise RuntimeError(f"cache and batch tensors must be on {device}; found {t.device}")
    return shape


def _rows_apart(table: torch.Tensor) -> bool:
    (rows, width), (pitch, unit) = table.shape, table.stride()
    return (unit == 1 or width <= 1) and (pitch >= width or rows <= 1)


def _check_keys(x: torch.Tensor, name: str, q: torch.Tensor, q_shape: torch.Size, cache_shape: torch.Size) -> None:
    if x.shape != (q_shape[0], cache_shape[1], q_shape[2]):
        raise ValueError(f"{name} must be [{q_shape[0]}, {cache_shape[1]}, {q_shape[2]}] as the queries' rows and the "
                         f"cache's heads, got {tuple(x.shape)}")
    if x.dtype is not q.dtype or x.device != q.device:
        raise ValueError(f"{name} must have the queries' dtype and device")


def check_scores(scale: float | None, causal: bool, window: int, dim: int) -> float:
    """The factor of the scores; what attention refuses of its own arguments."""

    if window < 0 or window > 1 << 30 or (window and not causal):
        raise ValueError(f"window must be 0, or a positive number of tokens of causal attention, got {window}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 2.0**100:
        raise ValueError(f"scale must be finite and at most 2^100, got {scale}")
    return scale


def _check_positions(positions: torch.Tensor, rows: int, device: torch.device) -> None:
    if positions.shape != (rows,) or positions.dtype is not torch.int32 or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int32 [{rows}], got {positions.dtype} {tuple(positions.shape)}")
    if positions.device != device:
        raise RuntimeError(f"positions must be on {device}; found {positions.device}")


def check_tree(tree: DraftTree, rows: int, device: torch.device) -> int:
    """Words of a row's mask; what attention refuses of a tree."""

    mask, positions = tree
    _check_positions(positions, rows, device)
    if mask.dim() != 2 or mask.shape[0] != rows or mask.dtype is not torch.int32 or not mask.is_contiguous():
        raise ValueError(f"mask must be contiguous int32 [{rows}, words], got {mask.dtype} {tuple(mask.shape)}")
    if not 1 <= mask.shape[1] <= MOST_NODES // 32:
        raise ValueError(f"mask must have 1 to {MOST_NODES // 32} words a row, got {mask.shape[1]}")
    if mask.device != device:
        raise RuntimeError(f"mask must be on {device}; found {mask.device}")
    return mask.shape[1]


def _refuse_grad(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the key/value cache is for inference: an input requires a gradient")


# ------------------------------------------------------------- public calls
def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKvCache, block_table: torch.Tensor,
                  cu_rows: torch.Tensor, lengths: torch.Tensor, cos_sin: torch.Tensor | None = None, *,
                  interleaved: bool = False, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                  eps: float = 1e-6, positions: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate ``q [R, Hq, D]`` and ``k [R, Hkv, D]`` by their positions, store the
    keys and ``v [R, Hkv, D]`` in the cache, and return the rotated queries.

    ``cos_sin`` is a :func:`rotary_table` (or a table of the caller's own) whose
    width, a multiple of 16, is the number of leading elements that rotate; pairs
    lie half that width apart or, ``interleaved``, next to each other.  None
    rotates nothing.  ``q_norm`` / ``k_norm [D]``, if given, are the weights of an
    RMS norm of each head before the rotation.  A position past the table makes
    its queries and keys NaN.  ``positions [R]`` int32, if given, says where rows turn
    instead of their slots (drafted tokens that branch, :class:`DraftTree`; a
    negative one is past the table); keys and values are stored in the slots all the
    same.

    A page's scale is the smallest power of two that holds what this call stores in
    it within e4m3's 448, and no smaller than the scale the page has if it holds
    earlier tokens of the sequence; those then move to the new scale.  A token whose
    key or value is not finite in a head is stored as a key of NaN codes there (with
    zeros for such elements of the value): rows that attend to it become NaN, and
    only they.  Tokens whose table entry is no page, or whose position is past the
    table, are not stored.  No two sequences of a call, nor two slots of one, may
    append to one page.

    Heads may be strided views (``q``, ``k`` and ``v`` of one packed projection);
    rows that are not 16-byte aligned are copied first."""

    cache_shape = _check_cache(cache)
    shape = _check_batch(q, cache, cache_shape, block_table, cu_rows, lengths)
    _check_keys(k, "k", q, shape, cache_shape)
    _check_keys(v, "v", q, shape, cache_shape)
    dim = shape[2]
    if cos_sin is not None:
        angles = cos_sin.shape
        if len(angles) != 2 or cos_sin.dtype is not torch.float32 or cos_sin.device != q.device or not cos_sin.is_contiguous():
            raise ValueError("cos_sin must be a contiguous float32 [positions, rotary] table on the queries' device")
        if angles[1] % 16 or not 16 <= angles[1] <= dim:
            raise ValueError(f"rotary width must be a multiple of 16 up to {dim}, got {angles[1]}")
        if cos_sin.data_ptr() % 16:
            raise ValueError("cos_sin must be 16-byte aligned")
    for norm in (q_norm, k_norm):
        if norm is not None and (norm.shape != (dim,) or norm.dtype != q.dtype or norm.device != q.device):
            raise ValueError(f"head norm weights must be [{dim}] of the queries' dtype and device")
    if positions is not None:
        _check_positions(positions, shape[0], q.device)
    _refuse_grad(q, k, v, q_norm, k_norm)
    if not q.is_cuda:
        return _rotate_append_plain(q, k, v, cache, block_table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps,
                                    positions)
    return hip.rotate_append(q, k, v, shape, cache, cache_shape, block_table, cu_rows, lengths, cos_sin, interleaved, q_norm,
                             k_norm, eps, positions)


def paged_attention(q: torch.Tensor, cache: PagedKvCache, block_table: torch.Tensor, cu_rows: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, causal: bool = True,
                    window: int = 0) -> torch.Tensor:
    """Attention of ``q [R, Hq, D]`` over the cached tokens of each row's sequence:
    query head ``h`` reads kv head ``h // (Hq // Hkv)``, scores times ``scale``
    (``D ** -0.5``).  Causal rows see the tokens up to their own, the last
    ``window`` of them if that is positive; otherwise every token of the sequence.
    Returns ``[R, Hq, D]``; a row that sees no token is zero."""

    cache_shape = _check_cache(cache)
    shape = _check_batch(q, cache, cache_shape, block_table, cu_rows, lengths)
    scale = check_scores(scale, causal, window, shape[2])
    _refuse_grad(q)
    if not q.is_cuda:
        return _paged_attention_plain(q, cache, block_table, cu_rows, lengths, scale, causal, window)
    return hip.attention(q, shape, cache, cache_shape, block_table, cu_rows, lengths, scale, causal, window)


def tree_attention(q: torch.Tensor, cache: PagedKvCache, block_table: torch.Tensor, cu_rows: torch.Tensor,
                   lengths: torch.Tensor, tree: DraftTree, *, scale: float | None = None, window: int = 0) -> torch.Tensor:
    """Attention of drafted tokens ``q [R, Hq, D]``, stored as their sequences' last
    ones: each sees the tokens before its sequence's new ones (from ``position -
    window`` on, exclusive, where ``window`` is positive) and those new ones that its
    mask names.  Heads, scores and the result are :func:`paged_attention`'s; a row that
    sees no token is zero."""

    cache_shape = _check_cache(cache)
    shape = _check_batch(q, cache, cache_shape, block_table, cu_rows, lengths)
    scale = check_scores(scale, True, window, shape[2])
    words = check_tree(tree, shape[0], q.device)
    _refuse_grad(q)
    if not q.is_cuda:
        return _paged_attention_plain(q, cache, block_table, cu_rows, lengths, scale, True, window, tree)
    return hip.tree_attention(q, shape, cache, cache_shape, block_table, cu_rows, lengths, scale, tree, words, window)


# ------------------------------------------------------------- plain forms
def _sequences(rows: int, cache: PagedKvCache, table, cu_rows, lengths):
    """(sequence, first row, rows, position of the first row, tokens that the table
    holds) of each sequence."""

    cu = [min(max(int(c), 0), rows) for c in cu_rows]
    for s, length in enumerate(lengths.tolist()):
        n = max(cu[s + 1] - cu[s], 0)
        length = max(length, 0)
        yield s, cu[s], n, length - n, min(length, table.shape[1] * cache.page_size)


def _head_norm(x, weight, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.to(torch.float32)


def _rotated(x, cos_sin, positions, interleaved):
    r = cos_sin.shape[1]
    inside = ((positions >= 0) & (positions < cos_sin.shape[0]))[:, None, None]
    angles = cos_sin[positions.clamp(0, max(cos_sin.shape[0] - 1, 0))][:, None] if cos_sin.shape[0] else x.new_zeros(1, 1, r)
    cos, sin = angles.chunk(2, -1)
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((torch.where(inside, turned, math.nan), x[..., r:]), -1)


def _power_of_two_scale(amax: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(amax.clamp(min=1e-12))  # 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).to(e.dtype))


def _rotate_append_plain(q, k, v, cache, table, cu_rows, lengths, cos_sin, interleaved, q_norm, k_norm, eps, given=None):
    page, pages = cache.page_size, cache.k.shape[0]
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    for s, row, n, first, tokens in _sequences(q.shape[0], cache, table, cu_rows, lengths):
        skip = max(-first, 0)  # rows before the first token
        if n <= skip:
            continue
        positions = torch.arange(first + skip, first + n) if given is None else given[row + skip: row + n].long()
        part = [x[row + skip: row + n].to(torch.float32) for x in (q, k, v)]
        if q_norm is not None:
            part[0] = _head_norm(part[0], q_norm, eps)
        if k_norm is not None:
            part[1] = _head_norm(part[1], k_norm, eps)
        if cos_sin is not None:
            part[:2] = [_rotated(x, cos_sin, positions, interleaved) for x in part[:2]]
        out[row + skip: row + n] = part[0].to(q.dtype)
        good = part[1].isfinite().all(-1) & part[2].isfinite().all(-1)  # [tokens, heads]
        keys = torch.where(good[..., None], part[1], 0.0)
        values = torch.where(part[2].isfinite(), part[2], 0.0)
        start = first + skip
        for slot in range(start // page, -(-tokens // page)):
            p = int(table[s, slot])
            if not 0 <= p < pages:
                continue
            lo, hi = max(start, slot * page), min(tokens, (slot + 1) * page)
            kept = lo - slot * page
            for codes, scales, x in ((cache.k, cache.k_scale, keys), (cache.v, cache.v_scale, values)):
                x = x[lo - start: hi - start].transpose(0, 1)
                scale = _power_of_two_scale(x.abs().amax((1, 2)))
                if kept:
                    scale = torch.fmax(scale, scales[p])
                    moved = codes[p, :, :kept].to(torch.float32) * (scales[p] / scale)[:, None, None]
                    codes[p, :, :kept] = moved.clamp(-448, 448).to(E4M3)
                scales[p] = scale
                codes[p, :, kept: kept + hi - lo] = (x / scale[:, None, None]).clamp(-448, 448).to(E4M3)
            # (codes of tokens that are not finite)
            bad = (~good)[lo - start: hi - start].transpose(0, 1)
            new = cache.k[p, :, kept: kept + hi - lo].view(torch.uint8)
            new.copy_(torch.where(bad[..., None], torch.full_like(new, 0x7F), new))
    return out


def _tree_seen(tree, row, n, first, tokens, window):
    """Whether each of a sequence's rows sees each of its tokens."""

    positions, words = tree.positions[row: row + n].long()[:, None], tree.mask[row: row + n].long()
    token = torch.arange(tokens)
    node = (token - first).expand(n, -1)
    word = node >> 5
    bit = words.gather(1, word.clamp(0, words.shape[1] - 1)) >> (node & 31) & 1
    drafted = (node >= 0) & (word < words.shape[1]) & (bit == 1)
    context = node < 0
    if window:
        context = context & (token > positions.clamp(min=first) - window)
    return (positions >= 0) & (drafted | context)


def _paged_attention_plain(q, cache, table, cu_rows, lengths, scale, causal, window, tree=None):
    heads, kv_heads, pages, page = q.shape[1], cache.k.shape[1], cache.k.shape[0], cache.page_size
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    for s, row, n, first, tokens in _sequences(q.shape[0], cache, table, cu_rows, lengths):
        if not n or not tokens or not pages:
            continue
        at = table[s, : -(-tokens // page)].long()
        there = ((at >= 0) & (at < pages)).repeat_interleave(page)[:tokens]
        at = at.clamp(0, pages - 1)
        k, v = ((codes.view(torch.uint8)[at].view(E4M3).to(torch.float32) * scales[at][..., None, None])
                .transpose(0, 1).flatten(1, 2)[:, :tokens] for codes, scales in
                ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))  # [kv heads, tokens, dim]
        v = torch.where(there[:, None], v, 0.0)
        position = torch.arange(first, first + n)[:, None]
        token = torch.arange(tokens)
        seen = there.expand(n, -1)
        if tree is not None:
            seen = seen & _tree_seen(tree, row, n, first, tokens, window)
        elif causal:
            seen = seen & (token <= position)
        if window and tree is None:
            seen = seen & (token > position - window)
        x = q[row: row + n].to(torch.float32).unflatten(1, (kv_heads, heads // kv_heads))
        z = torch.einsum("nhgd,htd->hgnt", x, k) * scale
        z = z.masked_fill(~seen, -math.inf)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = torch.einsum("hgnt,htd->nhgd", p / torch.where(total == 0, 1.0, total), v)
        out[row: row + n] = o.flatten(1, 2).to(q.dtype)
    return out
