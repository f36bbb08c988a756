"""Batches, caches and comparisons shared by the key/value cache's tests."""

from __future__ import annotations

import math

import torch

from kairyu_amd.attention import PagedKvCache
from oracle import attention as oatt

E4M3 = torch.float8_e4m3fn


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def batch(new, total, page, seed=0, pad=0, spare=3, holes=()):
    """(table, cu, lengths, rows, pages): the sequences' pages in random order, the
    table's unused entries -1, ``holes`` (sequence, slot) without a page."""

    g = gen(seed)
    held = [-(-t // page) for t in total]
    pages = max(sum(held) + spare, 1)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(new), max(held + [1])), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = order[at: at + n]
        at += n
    for s, slot in holes:
        table[s, slot] = -1 if slot % 2 else pages
    cu = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
    return table, cu, torch.tensor(total, dtype=torch.int32), sum(new) + pad, pages


def cache(pages, kv_heads, page, dim, seed=0, low=-9, high=-4, stale=0x7F):
    """A cache of random codes and power-of-two scales."""

    g = gen(seed)
    parts = []
    for span in (100.0, 90.0):
        x = torch.randn((pages, kv_heads, page, dim), generator=g) * span
        parts.append(x.clamp(-448, 448).to(E4M3))
    for _ in range(2):
        parts.append(torch.exp2(torch.randint(low, high, (pages, kv_heads), generator=g).float()))
    return PagedKvCache(*parts)


def stain(pool, table, lengths, code=0x7F):
    """Slots past each sequence's end, and every page of no sequence, hold NaN codes."""

    page = pool.page_size
    held = torch.zeros(pool.k.shape[0], page, dtype=torch.bool)
    for s, n in enumerate(lengths.tolist()):
        for slot in range(-(-min(n, table.shape[1] * page) // page)):
            p = int(table[s, slot])
            if 0 <= p < held.shape[0]:
                held[p, : max(0, min(page, n - slot * page))] = True
    for codes in (pool.k, pool.v):
        raw = codes.view(torch.uint8)
        raw.copy_(torch.where(held[:, None, :, None], raw, torch.full_like(raw, code)))


def to(pool, device):
    return PagedKvCache(*(t.to(device) for t in pool))


def values(pool):
    """The cache as the oracle takes it."""

    return {"k": pool.k.cpu().float().double(), "v": pool.v.cpu().float().double(),
            "k_scale": pool.k_scale.cpu().double(), "v_scale": pool.v_scale.cpu().double()}


def assert_within(got, want, bound, dtype, label=""):
    """NaN where the oracle has it; elsewhere within the bound and one rounding."""

    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, label
    assert torch.equal(got.isnan(), want.isnan()), f"{label}: NaN at other places"
    slack = bound + oatt.HALF_STEP[dtype] * (want.abs() + bound) + oatt.TINY[dtype]
    over = torch.where(want.isnan(), 0.0, ((got - want).abs() - slack))
    assert not over.isnan().any(), f"{label}: infinite values"
    worst = over.max().item() if over.numel() else 0.0
    used = torch.where(want.isnan(), 0.0, (got - want).abs() / slack).max().item() if over.numel() else 0.0
    print(f"[kv] {label}: at most {used:.3f} of the bound", flush=True)
    assert worst <= 0, f"{label}: {worst} past the bound ({used:.2f} of it)"


def check_attention(out, q, pool, table, cu, lengths, label="", **how):
    want, bound = oatt.attend(q.cpu(), values(pool), table.cpu(), cu.cpu(), lengths.cpu(), **how)
    assert_within(out, want, bound, out.dtype, label)


def check_append(got_q, pool, before, q, k, v, table, cu, lengths, label="", **how):
    """``before``: the cache's values ahead of the call."""

    want_q, want = oatt.append(q.cpu(), k.cpu(), v.cpu(), before, table, cu, lengths, **how)
    # rotation: two products and a sum in fp32; the norm before it
    normed = how.get("q_norm") is not None
    noise = (64 + 16) * oatt.U32 if normed else 4 * oatt.U32
    pair = want_q.abs().amax(-1, keepdim=True) * math.sqrt(2)  # a pair's length bounds both products
    assert_within(got_q, want_q, torch.where(want_q.isnan(), 0.0, noise * 2 * pair.nan_to_num(0.0)), got_q.dtype, label + " q")
    got = values(pool)
    for name in "kv":
        assert torch.equal(got[name + "_scale"], want[name + "_scale"]), f"{label}: {name} scales"
        x, y = got[name], want[name]
        assert torch.equal(x.isnan(), y.isnan()), f"{label}: {name} NaN codes at other places"
        # the same code, or a neighbour where fp32 noise moved a value over a midpoint: at
        # most a step, 2^-3 of the value or 2^-9, and seldom
        far = torch.where(y.isnan(), 0.0, (x - y).abs())
        assert (far <= torch.where(y.isnan(), 1.0, torch.maximum(x.abs(), y.abs()) * 2.0**-3 + 2.0**-9)).all(), f"{label}: {name} codes"
        moved = (far > 0).double().mean().item()
        assert moved <= 1e-3, f"{label}: {moved} of the {name} codes differ"
