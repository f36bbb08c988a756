"""64-bit definitions of the paged e4m3 cache's append and attention and of the
norms around a block, with the bounds that the kernels' fp32 arithmetic and single
roundings stay within (numpy / torch on the CPU; none of the package's code).

A batch is ``(table, cu, lengths)`` as the package takes it; a cache is a dict of
``k`` and ``v`` (values the codes stand for, ``[pages, kv heads, page, dim]``
fp64, before their scales) and ``k_scale`` / ``v_scale``.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0**-24
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
#: smallest normal's half step: what a rounding may be off by near zero
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to even), saturated at 448; NaN stays."""

    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-6)))
    step = torch.exp2(e.clamp(min=-6, max=8) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def scale_for(amax: float) -> float:
    """Smallest power of two ``s`` with ``max(amax, 1e-12) <= 448 s``."""

    m, e = math.frexp(max(amax, 1e-12))  # 448 = 0.875 * 2^9
    return math.ldexp(1.0, e - 9 + (m > 0.875))


def sequences(rows, table, cu, lengths, page):
    for s, length in enumerate(lengths.tolist()):
        lo, hi = int(cu[s]), int(cu[s + 1])
        yield s, lo, hi - lo, length - (hi - lo), min(length, table.shape[1] * page)


def rotate(x, cos_sin, position, interleaved):
    """One token's heads ``x [heads, dim]`` turned; fp64."""

    if cos_sin is None:
        return x
    y = x.clone()
    r = cos_sin.shape[1]
    if position >= cos_sin.shape[0]:
        y[:, :r] = math.nan
        return y
    cos, sin = cos_sin[position, : r // 2].double(), cos_sin[position, r // 2:].double()
    one = slice(0, r, 2) if interleaved else slice(0, r // 2)
    two = slice(1, r, 2) if interleaved else slice(r // 2, r)
    y[:, one] = x[:, one] * cos - x[:, two] * sin
    y[:, two] = x[:, two] * cos + x[:, one] * sin
    return y


def head_norm(x, weight, eps):
    return x if weight is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def append(q, k, v, cache, table, cu, lengths, cos_sin=None, interleaved=False, q_norm=None, k_norm=None, eps=1e-6):
    """``(rotated queries, new cache)``, all fp64; padding rows are zero."""

    new = {n: t.clone() for n, t in cache.items()}
    pages, _, page, _ = cache["k"].shape
    out = torch.zeros(q.shape, dtype=torch.float64)
    for s, row, n, first, tokens in sequences(q.shape[0], table, cu, lengths, page):
        groups: dict[int, list] = {}
        for j in range(n):
            position = first + j
            if position < 0:
                continue
            out[row + j] = rotate(head_norm(q[row + j].double(), q_norm, eps), cos_sin, position, interleaved)
            if position >= tokens or not 0 <= int(table[s, position // page]) < pages:
                continue
            key = rotate(head_norm(k[row + j].double(), k_norm, eps), cos_sin, position, interleaved)
            groups.setdefault(position // page, []).append((position % page, key, v[row + j].double()))
        for slot, stored in groups.items():
            p, kept = int(table[s, slot]), stored[0][0]
            for h in range(cache["k"].shape[1]):
                keys = [key[h] if key[h].isfinite().all() and value[h].isfinite().all() else None for _, key, value in stored]
                values = [torch.where(value[h].isfinite(), value[h], 0.0) for _, _, value in stored]
                for name, parts in (("k", keys), ("v", values)):
                    most = max([float(x.abs().max()) for x in parts if x is not None], default=0.0)
                    scale = scale_for(most)
                    if kept:
                        old = float(new[name + "_scale"][p, h])
                        scale = max(scale, old)
                        new[name][p, h, :kept] = to_e4m3(new[name][p, h, :kept] * (old / scale))
                    new[name + "_scale"][p, h] = scale
                    for (at, _, _), x in zip(stored, parts):
                        new[name][p, h, at] = math.nan if x is None else to_e4m3(x / scale)
    return out, new


def attend(q, cache, table, cu, lengths, scale=None, causal=True, window=0):
    """``(o, bound)`` in fp64: attention, and what a kernel may be off by before its
    output's own rounding.

    With weights ``p = exp(z - max)``, ``A = sum p |v| / sum p``:

    * a score's products are exact in fp32 (8- or 11-bit times 4-bit significands)
      and its ``dim`` terms are added with at most ``dim`` roundings of the sum of
      magnitudes; scaling, the maximum's subtraction and the exponential add some
      roundings of ``|w|``, the base-2 exponent.  A weight is thus off by
      ``d = ln 2 * (dim * 2^-24 * sum |q k| scale log2 e + 8 * 2^-24 * max |w|) + 2^-21``
      relative, the numerator and denominator alike: ``2 d A``.
    * a weight enters the product with the values rounded once, ``2^-11`` of it, and
      one far below the largest by no more than ``2^-34`` of that: beside a token that
      takes nearly all of the mass, a million others lose ``2^-14`` of a value together
      at the very most.
    * numerator and denominator add ``n`` terms in fp32 and the parts of a split
      sequence are rescaled: ``(2 n + 64) * 2^-24 A``.
    """

    scale = q.shape[-1] ** -0.5 if scale is None else scale
    pages, kv_heads, page, dim = cache["k"].shape
    rows, heads = q.shape[:2]
    group = heads // kv_heads
    out, bound = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    log2e = math.log2(math.e)
    for s, row, n, first, tokens in sequences(rows, table, cu, lengths, page):
        if n == 0 or tokens <= 0:
            continue
        at = table[s, : -(-tokens // page)].long()
        there = ((at >= 0) & (at < pages)).repeat_interleave(page)[:tokens]
        at = at.clamp(0, pages - 1)
        position, token = torch.arange(first, first + n)[:, None], torch.arange(tokens)[None]
        seen = there[None].expand(n, -1).clone()
        if causal:
            seen &= token <= position
        if window:
            seen &= token > position - window
        seen = seen.repeat_interleave(group, 0)  # [n * group, tokens]
        for h in range(kv_heads):
            code = {x: cache[x][at, h].reshape(-1, dim)[:tokens] for x in "kv"}
            unit = {x: cache[x + "_scale"][at, h].double().repeat_interleave(page)[:tokens] for x in "kv"}
            code["v"] = torch.where(there[:, None], code["v"], 0.0)
            k, v = code["k"] * unit["k"][:, None], code["v"] * unit["v"][:, None]
            x = q[row: row + n, h * group: (h + 1) * group].double().reshape(-1, dim)
            z = torch.where(seen, (x @ k.T) * scale, -math.inf)
            magnitude = torch.where(seen, (x.abs() @ k.abs().T) * abs(scale), 0.0)
            top = z.amax(-1, keepdim=True)
            p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            some = torch.where(total == 0, 1.0, total)
            o = (p @ v) / some
            a = (p @ v.abs()) / some
            w = torch.where(seen, z * log2e + torch.log2(unit["v"])[None], -math.inf)
            high = w.amax(-1, keepdim=True)
            spread = torch.where(seen, (z * log2e).abs() + torch.log2(unit["v"]).abs()[None], 0.0).amax(-1, keepdim=True)
            d = math.log(2) * (dim * U32 * magnitude.amax(-1, keepdim=True) * log2e + 8 * U32 * spread) + 2.0**-21
            # the largest exp2(w) against the denominator, in units of sum p
            unit_p = torch.exp((high - torch.where(top == -math.inf, 0.0, top) * log2e) * math.log(2))
            sub = 2.0**-34 * torch.where(total == 0, 0.0, unit_p / some) * (seen.double() @ code["v"].abs())
            err = a * (2 * d + 2.0**-11 + (2 * tokens + 64) * U32) + sub
            out[row: row + n, h * group: (h + 1) * group] = o.reshape(n, group, dim)
            bound[row: row + n, h * group: (h + 1) * group] = err.reshape(n, group, dim)
    return out, bound


def block_norm(x, residual, weight, post=None, gate=None, residual_scale=1.0, eps=1e-6, unit_offset=False):
    """``(r, y, bound of r, bound of y)`` in fp64 before any rounding of theirs.

    A norm's sum of squares adds at most 64 + ``hidden`` / 64 positive terms in a row
    (a thread's elements, then lanes and waves), so its root is off by half that in
    2^-24 relative, and the products around it by some more."""

    one = 1.0 if unit_offset else 0.0
    hidden = x.shape[-1]
    steps = (64 + hidden / 64 + 16) * U32
    b = x.double()
    if post is not None:
        b = b / torch.sqrt(b.square().mean(-1, keepdim=True) + eps) * (post.double() + one)
    if gate is not None:
        b = b * gate.double()
    b = b * residual_scale
    base = torch.zeros_like(b) if residual is None else residual.double()
    r = base + b
    r_err = steps * b.abs() + 2 * U32 * (base.abs() + b.abs())
    root = torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    w = weight.double() + one
    y = r / root * w
    # d root / root <= sum |r| |dr| / sum r^2, and the sum's own roundings
    d_root = (r.abs() * r_err).mean(-1, keepdim=True) / root.square() + steps
    y_err = (r_err / root * w.abs()) + y.abs() * (d_root + 8 * U32)
    return r, y, r_err, y_err
