"""Drafted trees on the GPU against their definitions: positions and masks, the walk, the
append at given positions, attention, the move of kept tokens, and whole steps of
speculative decoding as a program runs them, captured and replayed too."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import DraftTree, PagedKvCache, paged_attention, rotary_table, rotate_append, tree_attention
from kairyu_amd.drafts import accept_drafts, draft_tree, keep_tokens
from kairyu_amd.kernels import kv_cache_hip as hip
from kairyu_amd.pages import KvCaches, fork_sequences
from kairyu_amd.quant.packed import QuantLinearPack
from oracle import attention as oatt
from oracle import drafts as odr
from test_gpu_packed import _fp8

pytestmark = pytest.mark.gpu

BATCHES = {
    # (new rows, tokens after them) of each sequence
    "one row": ([1], [1]),
    "one tree": ([12], [300]),
    "trees": ([5, 1, 0, 40, 7, 17, 2], [20, 1, 9, 75, 300, 1100, 66]),
    "more rows than tokens": ([6, 70, 2, 1], [4, 20, 0, 0]),
    "wide": ([100, 33], [130, 1500]),
    "nothing before": ([16, 3, 64], [16, 3, 64]),
}
HEADS = {"8 of 2, 64": (8, 2, 64), "7 of 1, 128": (7, 1, 128), "4 of 4, 128": (4, 4, 128), "3 of 1, 256": (3, 1, 256),
         "32 of 4, 128": (32, 4, 128), "40 of 2, 64": (40, 2, 64)}


def _case(cuda, batch, heads, page, dtype, seed=0, pad=2, kind="tree", window=0, holes=()):
    """Queries, cache, batch, tree and what its rows see."""
    new, total = BATCHES[batch] if isinstance(batch, str) else batch
    hq, hk, dim = HEADS[heads] if isinstance(heads, str) else heads
    table, cu, lengths, rows, pages = kv.batch(new, total, page, seed=seed, pad=pad, holes=holes)
    pool = kv.cache(pages, hk, page, dim, seed=seed + 1)
    kv.stain(pool, table, lengths)
    tree, seen = dh.oracle_tree(dh.parents(new, seed, kind, pad), cu, lengths, max(new), window)
    q = (torch.randn(rows, hq, dim, generator=kv.gen(seed + 2)) * 2).to(dtype).to(cuda)
    tree = DraftTree(*(t.to(cuda) for t in tree))
    return q, kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda), tree, seen


# --------------------------------------------------------------- trees and walks
@pytest.mark.parametrize("window", [0, 3])
@pytest.mark.parametrize("kind", ["tree", "chain", "star", "roots"])
@pytest.mark.parametrize("batch", BATCHES)
def test_tree(cuda, batch, kind, window):
    banner(f"draft tree {batch} {kind} window {window}")
    new, total = BATCHES[batch]
    _, cu, lengths, rows, _ = kv.batch(new, total, 16, pad=3)
    par = dh.parents(new, 1, kind, pad=3)
    par[0] = 5  # (no row before it: a root)
    for most in {max(new), max(1, max(new) - 5), 64}:
        got = draft_tree(par.to(cuda), cu.to(cuda), lengths.to(cuda), most, window=window)
        seen, positions = odr.tree(par, cu, lengths, most, window)
        assert got.positions.tolist() == positions
        assert odr.unpack(got.mask.cpu()) == seen


@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_the_largest_tree(cuda, kind):
    banner(f"largest draft tree {kind}")
    new = [1024, 1030]
    par, cu, lengths = dh.parents(new, 3, kind), dh.ints(0, 1024, 2054), dh.ints(1024, 2000)
    tokens, targets = dh.tokens_for(par, cu, 4, agree=1.0)
    got = draft_tree(par.to(cuda), cu.to(cuda), lengths.to(cuda), 1024)
    seen, positions = odr.tree(par, cu, lengths, 1024)
    assert got.positions.tolist() == positions and torch.equal(got.mask.cpu(), odr.pack(seen, 32))
    kept, counts, following = accept_drafts(tokens.to(cuda), targets.to(cuda), par.to(cuda), cu.to(cuda), 1024)
    for s, (nodes, after) in enumerate(odr.walk(tokens, targets, par, cu, 1024)):
        assert kept[s, : len(nodes)].tolist() == nodes and int(counts[s]) == len(nodes) and int(following[s]) == after


@pytest.mark.parametrize("window", [1, 31, 33, 500, 1 << 30])
@pytest.mark.parametrize("most", [1024, 700, 65])
def test_large_trees_in_windows(cuda, most, window):
    banner(f"large draft trees {most} window {window}")
    cu, lengths = dh.ints(0, 800, 1900, 1903), dh.ints(900, 1090, 3)  # (rows before the first token in the second)
    for kind in ("tree", "chain"):
        par = dh.parents([800, 1100, 3], 5, kind)
        got = draft_tree(par.to(cuda), cu.to(cuda), lengths.to(cuda), most, window=window)
        seen, positions = odr.tree(par, cu, lengths, most, window)
        assert got.positions.tolist() == positions and torch.equal(got.mask.cpu(), odr.pack(seen, -(-most // 32)))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", ["tree", "chain", "star"])
@pytest.mark.parametrize("batch", BATCHES)
def test_walk(cuda, batch, kind, dtype):
    banner(f"draft walk {batch} {kind} {dtype}")
    new, total = BATCHES[batch]
    _, cu, _, _, _ = kv.batch(new, total, 16, pad=3)
    par = dh.parents(new, 2, kind, pad=3)
    tokens, targets = dh.tokens_for(par, cu, 3, dtype=dtype)
    for most in (max(new), max(1, max(new) // 2)):
        kept, counts, following = accept_drafts(tokens.to(cuda), targets.to(cuda), par.to(cuda), cu.to(cuda), most)
        for s, (nodes, after) in enumerate(odr.walk(tokens, targets, par, cu, most)):
            assert kept[s].tolist() == nodes + [-1] * (most - len(nodes)), s
            assert int(counts[s]) == len(nodes) and int(following[s]) == after, s


# ------------------------------------------------------------------- the append
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_at_positions(cuda, dim, interleaved):
    """The same bits as a call without positions whose table holds them in the slots' rows."""
    banner(f"append at positions {dim} {interleaved}")
    n, total, page = 40, 90, 32
    table, cu, lengths, rows, pages = kv.batch([n], [total], page, pad=3)
    q, k, v = (torch.randn(rows, h, dim, generator=kv.gen(h)).to(torch.bfloat16).to(cuda) for h in (8, 2, 2))
    angles = rotary_table(80, dim, device=cuda)
    at = torch.randint(0, 80, (rows,), generator=kv.gen(5)).to(torch.int32).to(cuda)
    slots = torch.zeros(total, dim, device=cuda)
    slots[total - n:] = angles[at[:n].long()]
    batch = [x.to(cuda) for x in (table, cu, lengths)]
    pools = [kv.to(kv.cache(pages, 2, page, dim), cuda) for _ in range(2)]
    norm = (torch.randn(dim, generator=kv.gen(6)) * 0.1 + 1).to(torch.bfloat16).to(cuda)
    how = dict(interleaved=interleaved, q_norm=norm, k_norm=norm)
    got = rotate_append(q, k, v, pools[0], *batch, angles, positions=at, **how)
    want = rotate_append(q, k, v, pools[1], *batch, slots, **how)
    assert torch.equal(got, want)
    for a, b in zip(*pools):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    far = at.clone()
    far[3], far[7] = -1, 80
    out = rotate_append(q, k, v, pools[0], *batch, angles, positions=far, **how)
    assert out[[3, 7]].isnan().all() and not out[[2, 4, 8]].isnan().any()


# -------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", BATCHES)
def test_attention(cuda, batch, heads, dtype):
    page = {64: 16, 128: 64, 256: 32}[HEADS[heads][2]]
    banner(f"tree attention {batch} {heads} page {page} {dtype}")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, batch, heads, page, dtype, seed=1)
    out = tree_attention(q, pool, table, cu, lengths, tree)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, batch)
    assert not out[-2:].any()


@pytest.mark.parametrize("how", [dict(window=1), dict(window=5), dict(window=513), dict(scale=0.02), dict(scale=-0.1),
                                 dict(scale=0.0)], ids=str)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", ["8 of 2, 64", "3 of 1, 256"])
def test_attention_windows_and_pages(cuda, heads, page, how):
    banner(f"tree attention {heads} page {page} {how}")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, "trees", heads, page, torch.float16, seed=4, window=how.get("window", 0))
    out = tree_attention(q, pool, table, cu, lengths, tree, **how)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, **how)


@pytest.mark.parametrize("heads", ["7 of 1, 128", "32 of 4, 128", "8 of 2, 64"])
def test_attention_of_masks_of_the_callers_own(cuda, heads):
    """Rows that see no drafted token, not themselves, all of them, ones behind the sequence's
    rows (which are none), and rows of negative positions, which are zero."""
    banner(f"tree attention own masks {heads}")
    q, pool, table, cu, lengths, tree, _ = _case(cuda, ([9, 70, 20], [9, 200, 1500]), heads, 32, torch.bfloat16, seed=5)
    rows = q.shape[0]
    g = kv.gen(6)
    mask = torch.randint(-2**31, 2**31, (rows, 5), generator=g).to(torch.int32)
    mask[::4] = 0
    mask[1::7] = -1
    positions = torch.where(torch.rand(rows, generator=g) < 0.2, -1, tree.positions.cpu())
    for window in (0, 40):
        out = tree_attention(q, pool, table, cu, lengths, DraftTree(mask.to(cuda), positions.to(cuda)), window=window)
        torch.cuda.synchronize()
        dh.check_attention(out, q, pool, table, cu, lengths, odr.unpack(mask), positions, window=window)
        assert not out[positions.to(cuda) < 0].any()
    assert not out[0].any()  # nothing before it, and no bit


@pytest.mark.parametrize("page", [16, 128])
def test_attention_pages_that_are_none(cuda, page):
    """Tokens of no page are not seen, also by queries that are not finite; a row left with
    none is zero."""
    banner(f"tree attention holes page {page}")
    holes = [(0, 0), (0, 1), (0, 600 // page), (1, 1), *((2, s) for s in range(-(-150 // page)))]
    q, pool, table, cu, lengths, tree, seen = _case(cuda, ([20, 20, 20], [610, 300, 150]), "7 of 1, 128", page, torch.bfloat16,
                                                    seed=6, holes=holes)
    q[41], q[45] = float("inf"), float("nan")
    out = tree_attention(q, pool, table, cu, lengths, tree)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions)
    assert not out[40:].any()


def test_attention_of_nan_keys_and_extreme_scores(cuda):
    """A drafted key of NaN reaches the rows below it and no other; scores of thousands and
    value scales 2^40 apart stay exact."""
    banner("tree attention NaN keys")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, ([30, 30], [420, 300]), "8 of 2, 64", 16, torch.bfloat16, seed=8)
    p = table[0, 395 // 16].long()  # drafted token 5 of the first
    pool.k.view(torch.uint8)[p, 1, 395 % 16] = 0x7F
    pool.v_scale[table[1, 3].long()] = 2.0**-40
    pool.v_scale[table[1, 5].long()] = 2.0**12
    q = q * 20
    out = tree_attention(q, pool, table, cu, lengths, tree)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions)
    assert out[:30, 4:].isnan().all(-1).all(-1).tolist() == [5 in s for s in seen[:30]] and not out[:, :4].isnan().any()


@pytest.mark.parametrize("heads", [(4, 1, 128), (16, 1, 64), (8, 1, 256)], ids=str)
def test_attention_of_long_contexts(cuda, heads):
    banner(f"tree attention long contexts {heads}")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, ([10, 3, 2], [70001, 33000, 5]), heads, 64, torch.bfloat16, seed=9)
    for window in (0, 40000):
        out = tree_attention(q, pool, table, cu, lengths, tree, window=window)
        torch.cuda.synchronize()
        dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, window=window)


def test_attention_of_many_sequences(cuda):
    """More than a wave's lanes hold, some without rows."""
    banner("tree attention 150 sequences")
    new = [(7 * i) % 11 for i in range(150)]
    total = [n + (37 * i) % 300 for i, n in enumerate(new)]
    q, pool, table, cu, lengths, tree, seen = _case(cuda, (new, total), "8 of 2, 64", 32, torch.float16, seed=10)
    out = tree_attention(q, pool, table, cu, lengths, tree)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions)


def test_attention_of_chains_is_causal_attention(cuda):
    banner("tree attention of chains")
    q, pool, table, cu, lengths, tree, _ = _case(cuda, "trees", "32 of 4, 128", 64, torch.bfloat16, seed=11, kind="chain")
    out, want = tree_attention(q, pool, table, cu, lengths, tree), paged_attention(q, pool, table, cu, lengths)
    kv.check_attention(out, q, pool, table, cu, lengths, "chains")
    kv.check_attention(want, q, pool, table, cu, lengths, "causal")


def test_attention_is_the_same_every_time(cuda):
    """Same bits from call to call, on another stream, from strided and misaligned queries."""
    banner("tree attention repeats")
    q, pool, table, cu, lengths, tree, _ = _case(cuda, "trees", "8 of 2, 64", 64, torch.bfloat16, seed=12)
    first = tree_attention(q, pool, table, cu, lengths, tree)
    wide = torch.nn.functional.pad(q, (0, 0, 0, 3))[:, :8]
    odd = torch.empty(q.numel() + 3, dtype=q.dtype, device=cuda)[3:].view(q.shape).copy_(q)
    for same in (q, q, wide, odd):
        assert torch.equal(tree_attention(same, pool, table, cu, lengths, tree), first)
    pitched = torch.nn.functional.pad(table, (0, 3))[:, : table.shape[1]]
    assert torch.equal(tree_attention(q, pool, pitched, cu, lengths, tree), first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = tree_attention(q, pool, table, cu, lengths, tree)
    side.synchronize()
    assert torch.equal(out, first)


def test_lengths_and_bounds_that_are_wrong_stay_in_range(cuda):
    """Row bounds past the tensor or going back, lengths past the table and below zero."""
    banner("tree attention bad bounds")
    q, pool, table, cu, lengths, tree, _ = _case(cuda, ([9, 7, 5], [40, 30, 20]), "8 of 2, 64", 16, torch.bfloat16, seed=13)
    par = dh.parents([9, 7, 5], pad=2).to(cuda)
    tokens = torch.zeros(23, dtype=torch.int64, device=cuda)
    for bad_cu, bad_lengths in (((0, 9, 5, 500), (40, 30, 20)), ((-3, 9, 16, 21), (40, 2**31 - 1, -5)),
                                ((4, 2, 1, 0), (40, 30, 20)), ((0, 9, 16, 21), (-(2**31), 60, 2**31 - 1))):
        c, n = dh.ints(*bad_cu).to(cuda), torch.tensor(bad_lengths, dtype=torch.int32, device=cuda)
        made = draft_tree(par, c, n, 9)
        tree_attention(q, pool, table, c, n, made)
        kept, counts, _ = accept_drafts(tokens, tokens, par, c, 9)
        keep_tokens(PagedKvCache(*(t.clone() for t in pool)), table, c, n, kept, counts)
    torch.cuda.synchronize()
    out = tree_attention(q, pool, table, cu, lengths, tree)
    assert out.isfinite().all()


def _columns(q, pool, table, lengths):
    """Columns of the tiles that a call without a window runs in, from its scratch (0: none)."""
    pages, kv_heads, page, dim = pool.k.shape
    need = hip._tree_bytes(*q.shape[:2], kv_heads, dim, page, table.shape[1], lengths.shape[0])
    return need // (8 * (dim + 4) * kv_heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", BATCHES)
def test_attention_in_wide_tables(cuda, batch, heads, dtype):
    """A table for a million tokens: tiles of as many columns as the trees have, cut along the
    tokens where there are enough, and bounds that say nothing of the lengths."""
    page = {64: 16, 128: 64, 256: 32}[HEADS[heads][2]]
    banner(f"tree attention wide {batch} {heads} page {page} {dtype}")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, batch, heads, page, dtype, seed=21)
    table = torch.nn.functional.pad(table, (0, (1 << 20) // page - table.shape[1]), value=-1)
    out = tree_attention(q, pool, table, cu, lengths, tree)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, batch)
    assert not out[-2:].any()


@pytest.mark.parametrize("group", [1, 3, 8], ids=lambda g: f"group {g}")
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_every_tile(cuda, dim, page, group):
    """Trees of 13 and 40 rows, 13 to 320 rows x heads, in tiles of 16, 32, 64 and 128 columns;
    whole ones, cut ones, holes and NaN queries among them."""
    banner(f"tree attention tiles {dim} page {page} group {group}")
    seen_columns = set()
    for new, holes in (([13, 9], [(0, 1)]), ([40, 33], [(1, 0), (1, 3)])):
        q, pool, table, cu, lengths, tree, seen = _case(cuda, (new, [2500, 700]), (2 * group, 2, dim), page, torch.bfloat16,
                                                        seed=22, holes=holes)
        q[3, 0], q[5, -1] = float("nan"), float("inf")
        table = torch.nn.functional.pad(table, (0, (1 << 20) // page - table.shape[1]), value=-1)
        shares = {64: {16: 768, 32: 512, 64: 512, 128: 512}, 128: {16: 512, 32: 512, 64: 512, 128: 512},
                  256: {16: 512, 32: 256, 64: 256, 128: 256}}[dim]
        need = _columns(q, pool, table, lengths)
        seen_columns |= {c for c, s in shares.items() if c * (s // 2) == need}
        out = tree_attention(q, pool, table, cu, lengths, tree)
        torch.cuda.synchronize()
        dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions)
    assert seen_columns >= {1: {16, 64}, 3: {64, 128}, 8: {128}}[group]


@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 4, 64), (16, 4, 64), (16, 4, 128), (8, 4, 128)], ids=str)
@pytest.mark.parametrize("window", [7, 300, 1500])
def test_attention_windows_in_every_tile(cuda, heads, window):
    """Many trees under a window: tiles whole and cut, from 16 to 128 columns."""
    banner(f"tree attention windows {heads} {window}")
    new = [8 + (5 * i) % 19 for i in range(48)]
    total = [n + (331 * i) % 2000 for i, n in enumerate(new)]
    q, pool, table, cu, lengths, tree, seen = _case(cuda, (new, total), heads, 32, torch.float16, seed=23, window=window)
    out = tree_attention(q, pool, table, cu, lengths, tree, window=window)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, window=window)


@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_positions_far_off(cuda, wide):
    """Under a window, positions before the first drafted slot count as it, and the largest
    leave nothing of the context."""
    banner(f"tree attention far positions {wide}")
    q, pool, table, cu, lengths, tree, seen = _case(cuda, ([12, 40], [90, 400]), "32 of 4, 128", 16, torch.bfloat16, seed=25)
    if wide:
        table = torch.nn.functional.pad(table, (0, 65536 - table.shape[1]), value=-1)
    positions = tree.positions.cpu()
    positions[::3], positions[1::3] = 0, 2**31 - 1
    for window in (1, 50, 1 << 30):
        out = tree_attention(q, pool, table, cu, lengths, DraftTree(tree.mask, positions.to(cuda)), window=window)
        torch.cuda.synchronize()
        dh.check_attention(out, q, pool, table, cu, lengths, seen, positions, window=window)


def test_attention_of_lengths_past_the_table(cuda):
    """Tokens past the table are not there: rows see those of the context that are."""
    banner("tree attention lengths past the table")
    for wide in (6, 4096):
        q, pool, table, cu, lengths, tree, _ = _case(cuda, ([9, 30], [90, 96]), "32 of 4, 128", 16, torch.bfloat16, seed=24)
        table = torch.nn.functional.pad(table, (0, max(wide - table.shape[1], 0)), value=-1)[:, :wide].contiguous()
        long = lengths + torch.tensor([40, 5000], dtype=torch.int32, device=cuda)
        tree, seen = dh.oracle_tree(dh.parents([9, 30], 24, pad=2), cu.cpu(), long.cpu(), 30)
        pool.v.view(torch.uint8).copy_(torch.where((pool.v.view(torch.uint8) & 0x7F) == 0x7F, 0, pool.v.view(torch.uint8)))
        pool.k.view(torch.uint8).copy_(torch.where((pool.k.view(torch.uint8) & 0x7F) == 0x7F, 0, pool.k.view(torch.uint8)))
        out = tree_attention(q, pool, table, cu, long, DraftTree(*(t.to(cuda) for t in tree)))
        torch.cuda.synchronize()
        dh.check_attention(out, q, pool, table, cu, long, seen, tree.positions)


# ------------------------------------------------------------------ kept tokens
def _kept(new, most, seed=0, share=3):
    kept = torch.full((len(new), most), -1, dtype=torch.int32)
    counts = []
    for s, n in enumerate(new):
        take = sorted(torch.randperm(n, generator=kv.gen(seed + s))[: max(1, n // share)].tolist()) if n else []
        kept[s, : len(take)] = torch.tensor(take, dtype=torch.int32)
        counts.append(len(take))
    return kept, torch.tensor(counts, dtype=torch.int32)


@pytest.mark.parametrize("share", [1, 3])
@pytest.mark.parametrize("shape", [(2, 16, 64), (8, 64, 128), (1, 32, 256), (5, 128, 128)], ids=str)
@pytest.mark.parametrize("batch", BATCHES)
def test_keep(cuda, batch, shape, share):
    banner(f"keep {batch} {shape} 1/{share}")
    (kv_heads, page, dim), (new, total) = shape, BATCHES[batch]
    table, cu, lengths, _, pages = kv.batch(new, total, page, seed=3)
    pools = dh.layers(2, pages, kv_heads, page, dim, seed=4)
    kv.stain(pools[1], table, lengths)
    kept, counts = _kept(new, max(new) + 1, 5, share)
    want = [odr.keep(kv.values(p), table, cu, lengths, kept, counts) for p in pools]
    pools = [kv.to(p, cuda) for p in pools]
    got = keep_tokens(KvCaches(pools), *(t.to(cuda) for t in (table, cu, lengths, kept, counts)))
    torch.cuda.synchronize()
    assert got.tolist() == want[0][1]
    dh.same_caches(pools, [w for w, _ in want])


def test_keep_of_the_longest_tree_and_many_layers(cuda):
    """1024 of 1030 rows through small pages; 70 layers, more than one launch takes."""
    banner("keep longest")
    for new, count, heads in (([1030], 1, 2), ([1030], 1, 8), ([9, 14], 70, 2)):  # (the second's scales do not fit in LDS)
        total = [n + 21 for n in new]
        table, cu, lengths, _, pages = kv.batch(new, total, 16, seed=3)
        pools = dh.layers(count, pages, heads, 16, 64, seed=4)
        kept, counts = _kept(new, min(max(new), 1024), 5, 2)
        want = [odr.keep(kv.values(p), table, cu, lengths, kept, counts) for p in pools]
        pools = [kv.to(p, cuda) for p in pools]
        got = keep_tokens(KvCaches(pools), *(t.to(cuda) for t in (table, cu, lengths, kept, counts)))
        torch.cuda.synchronize()
        assert got.tolist() == want[0][1]
        dh.same_caches(pools, [w for w, _ in want])


def test_keep_ends_where_it_has_to(cuda):
    banner("keep ends")
    new, total = [20, 20, 20, 20, 3], [50, 50, 50, 50, 30]
    table, cu, lengths, _, pages = kv.batch(new, total, 16, holes=[(3, 2)])
    kept = torch.stack([dh.ints(*x) for x in ((0, 3, 3, 5), (1, 20, 21, 22), (2, 1, 3, 4), (0, 1, 2, 3), (0, 2, 7, 9))])
    counts = dh.ints(4, 4, 9, 4, -3)
    pools = dh.layers(1, pages, 2, 16, 64)
    want, after = odr.keep(kv.values(pools[0]), table, cu, lengths, kept, counts)
    pool = kv.to(pools[0], cuda)
    got = keep_tokens(pool, *(t.to(cuda) for t in (table, cu, lengths, kept, counts)))
    assert got.tolist() == after
    dh.same_caches([pool], [want])


# ------------------------------------------------------------------ whole steps
HQ, HK, DIM, PAGE, HIDDEN, ROOM = 8, 2, 64, 16, 256, 12


class _Model:
    """Two layers' packed projections, caches for them, and a block table with its books: what a
    program of speculative decoding holds.  Every sequence drafts ROOM rows a step."""

    def __init__(self, cuda, seqs):
        widths = (HQ * DIM, HK * DIM, HK * DIM)
        self.packs = [QuantLinearPack.create([_fp8(HIDDEN, n, 10 * i + j).to(cuda) for j, n in enumerate(widths)]) for i in range(2)]
        self.pools = [PagedKvCache.create(80, HK, DIM, PAGE, device=cuda) for _ in range(2)]
        self.caches = KvCaches(self.pools)
        self.angles = rotary_table(200, DIM, device=cuda)
        self.holders = torch.zeros(80, dtype=torch.int32, device=cuda)
        self.table = torch.full((seqs, 12), -1, dtype=torch.int32, device=cuda)
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=cuda)
        self.rows = torch.arange(seqs, dtype=torch.int32, device=cuda)
        self.cu = self.rows.new_tensor([ROOM * i for i in range(seqs + 1)])

    def step(self, hidden, parents, tokens, targets):
        table, lengths, missing = fork_sequences(self.caches, self.holders, self.table, self.lengths, self.rows, ROOM)
        lengths = lengths + ROOM
        tree = draft_tree(parents, self.cu, lengths, ROOM)
        outs = [pack.attend(hidden, pool, table, self.cu, lengths, self.angles, tree=tree) for pack, pool in zip(self.packs, self.pools)]
        kept, counts, following = accept_drafts(tokens, targets, parents, self.cu, ROOM)
        self.table.copy_(table)
        self.lengths.copy_(keep_tokens(self.caches, table, self.cu, lengths, kept, counts))
        return *outs, following, missing, counts, tree.positions, tree.mask, lengths

    def state(self):
        return [self.holders, self.table, self.lengths, *(t for pool in self.pools for t in pool)]


def _drafts(seqs, seed, cuda):
    par = dh.parents([ROOM] * seqs, seed)
    tokens, targets = dh.tokens_for(par, torch.arange(seqs + 1) * ROOM, seed)
    hidden = torch.randn(seqs * ROOM, HIDDEN, generator=kv.gen(seed)).to(torch.bfloat16)
    return [x.to(cuda) for x in (hidden, par, tokens, targets)]


def test_steps_of_speculative_decoding(cuda):
    """Pages, trees, both layers, the walk and the move, step after step, each against its
    definition on the state before it."""
    banner("speculative steps")
    seqs = 3
    model = _Model(cuda, seqs)
    for step in range(8):
        hidden, par, tokens, targets = _drafts(seqs, 100 + step, cuda)
        before = [t.cpu().clone() for t in (model.holders, model.table, model.lengths)]
        caches = [kv.values(p) for p in model.pools]
        out = model.step(hidden, par, tokens, targets)
        torch.cuda.synchronize()
        table, lengths, holders, copies, missing = odr.fork(*before, model.rows.cpu(), ROOM, PAGE)
        assert missing == 0 and int(out[3]) == 0 and not copies
        assert model.table.tolist() == table and model.holders.tolist() == holders
        table, lengths = torch.tensor(table), torch.tensor(lengths, dtype=torch.int32) + ROOM
        cu = model.cu.cpu()
        seen, positions = odr.tree(par.cpu(), cu, lengths, ROOM)
        assert out[5].tolist() == positions and odr.unpack(out[6].cpu()) == seen
        walks = odr.walk(tokens.cpu(), targets.cpu(), par.cpu(), cu, ROOM)
        assert out[2].tolist() == [after for _, after in walks] and out[4].tolist() == [len(nodes) for nodes, _ in walks]
        # each layer's rows, turned and attending as the definition has it
        kept = torch.tensor([nodes + [-1] * (ROOM - len(nodes)) for nodes, _ in walks], dtype=torch.int32)
        for pack, pool, old, got in zip(model.packs, model.pools, caches, out):
            q, k, v = (x.unflatten(-1, (-1, DIM)) for x in pack(hidden))
            twin = PagedKvCache(*(t.to(cuda) for t in (old["k"].float().to(kv.E4M3), old["v"].float().to(kv.E4M3),
                                                       old["k_scale"].float(), old["v_scale"].float())))
            q = rotate_append(q, k, v, twin, table.int().to(cuda), model.cu, lengths.to(cuda), model.angles, positions=out[5])
            dh.check_attention(got.view(q.shape), q, twin, table, cu, lengths, seen, out[5], f"step {step}")
            angles = model.angles.cpu()
            for row, position in enumerate(positions):
                want = oatt.rotate(pack(hidden)[0].cpu()[row].view(HQ, DIM).double(), angles, position, False)
                assert (q[row].cpu().double() - want).abs().max() <= 2.0**-8 * want.abs().max() + 1e-6
            want, after = odr.keep(kv.values(twin), table, cu, lengths, kept, torch.tensor([len(nodes) for nodes, _ in walks]))
            dh.same_caches([pool], [want])
            assert model.lengths.tolist() == after


def test_steps_captured_and_replayed(cuda):
    """One captured step replayed equals eager steps on a second model, bit for bit, with eager
    work in between."""
    banner("speculative steps captured")
    seqs = 3
    models = [_Model(cuda, seqs) for _ in range(2)]
    static = _drafts(seqs, 1, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        models[0].step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = models[0].step(*static)
    for t, fresh in zip(models[0].state(), _Model(cuda, seqs).state()):
        t.copy_(fresh)
    for step in range(10):
        drafts = _drafts(seqs, 200 + step, cuda)
        for a, b in zip(static, drafts):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        eager = models[1].step(*drafts)
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), step
        for a, b in zip(models[0].state(), models[1].state()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), step


def test_two_graphs_of_attention_side_by_side(cuda):
    """Graphs that replay on two streams at once do not share scratch."""
    banner("tree attention two graphs")
    cases = [_case(cuda, ([14, 9], [9000, 5000]), "32 of 4, 128", 64, torch.bfloat16, seed=20 + i) for i in range(2)]
    eager = [tree_attention(*c[:6]) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tree_attention(*c[:6]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        tree_attention(*cases[0][:6])
        torch.cuda.synchronize()
