"""Drafted trees on the CPU: positions and masks, the walk, the move of kept tokens and
attention against their definitions, and the calls that are refused."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from kairyu_amd import _native
from kairyu_amd.attention import DraftTree, rotary_table, rotate_append, tree_attention
from kairyu_amd.drafts import accept_drafts, draft_tree, keep_tokens
from kairyu_amd.pages import KvCaches
from kairyu_amd.quant.packed import QuantLinearPack
from oracle import drafts as odr
from test_packed import _int8

NEW, TOTAL = [5, 1, 0, 40, 7], [20, 1, 9, 75, 4]  # the last has more rows than tokens


def _batch(page=16, pad=2, new=NEW, total=TOTAL, seed=0, **how):
    return kv.batch(new, total, page, seed=seed, pad=pad, **how)


@pytest.mark.parametrize("window", [0, 1, 3])
@pytest.mark.parametrize("most", [40, 33, 6])
@pytest.mark.parametrize("kind", ["tree", "chain", "star", "roots"])
def test_tree(kind, most, window):
    _, cu, lengths, rows, _ = _batch()
    par = dh.parents(NEW, 1, kind, pad=2)
    par[8] = 500  # (no such row: a root)
    par[9] = -7
    got = draft_tree(par, cu, lengths, most, window=window)
    seen, positions = odr.tree(par, cu, lengths, most, window)
    assert got.mask.shape == (rows, -(-most // 32))
    assert odr.unpack(got.mask) == seen and got.positions.tolist() == positions


def test_a_tree_with_its_top_bit_set():
    cu, lengths = dh.ints(0, 32), dh.ints(40)
    got = draft_tree(dh.parents([32], kind="chain"), cu, lengths, 32)
    assert int(got.mask[31, 0]) == -1 and int(got.mask[30, 0]) == 2**31 - 1
    assert got.positions.tolist() == list(range(8, 40))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("most", [40, 3, 1])
@pytest.mark.parametrize("kind", ["tree", "chain", "star"])
def test_walk(kind, most, dtype):
    _, cu, _, _, _ = _batch()
    par = dh.parents(NEW, 2, kind, pad=2)
    tokens, targets = dh.tokens_for(par, cu, 3, dtype=dtype)
    kept, counts, following = accept_drafts(tokens, targets, par, cu, most)
    assert kept.shape == (len(NEW), most) and following.dtype is dtype
    for s, (nodes, after) in enumerate(odr.walk(tokens, targets, par, cu, most)):
        assert kept[s].tolist() == nodes + [-1] * (most - len(nodes))
        assert int(counts[s]) == len(nodes) and int(following[s]) == after


def test_the_lowest_of_equal_children_is_kept():
    cu, par = dh.ints(0, 6), dh.ints(-1, 0, 0, 0, 2, 3)
    kept, counts, following = accept_drafts(torch.tensor([9, 4, 7, 7, 8, 8]), torch.tensor([7, 1, 8, 8, 3, 2]), par, cu, 6)
    assert kept.tolist() == [[0, 2, 4, -1, -1, -1]] and counts.tolist() == [3] and following.tolist() == [3]


def _kept(new, most, seed=0):
    kept = torch.full((len(new), most), -1, dtype=torch.int32)
    counts = []
    for s, n in enumerate(new):
        take = sorted(torch.randperm(n, generator=kv.gen(seed + s))[: max(1, n // 3)].tolist()) if n else []
        kept[s, : len(take)] = torch.tensor(take, dtype=torch.int32)
        counts.append(len(take))
    return kept, torch.tensor(counts, dtype=torch.int32)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("seed", range(4))
def test_keep(page, seed):
    table, cu, lengths, _, pages = _batch(page, seed=seed)
    pools = dh.layers(2, pages, 2, page, 64, seed=seed)
    kv.stain(pools[1], table, lengths)
    kept, counts = _kept(NEW, 41, seed)
    want = [odr.keep(kv.values(p), table, cu, lengths, kept, counts) for p in pools]
    got = keep_tokens(KvCaches(pools), table, cu, lengths, kept, counts)
    assert got.tolist() == want[0][1]
    dh.same_caches(pools, [w for w, _ in want])


def test_keep_ends_where_it_has_to():
    """Indices that are none, go back or repeat, counts past the width, pages that are none."""
    new, total = [20, 20, 20, 20, 3], [50, 50, 50, 50, 30]
    table, cu, lengths, _, pages = kv.batch(new, total, 16, holes=[(3, 2)])  # (3: tokens 32-47 in no page)
    kept = torch.full((5, 4), -1, dtype=torch.int32)
    kept[0] = dh.ints(0, 3, 3, 5)
    kept[1] = dh.ints(1, 20, 21, 22)
    kept[2] = dh.ints(2, 1, 3, 4)
    kept[3] = dh.ints(0, 1, 2, 3)
    kept[4] = dh.ints(0, 2, 7, 9)
    counts = dh.ints(4, 4, 9, 4, -3)
    pools = dh.layers(1, pages, 2, 16, 64)
    want, after = odr.keep(kv.values(pools[0]), table, cu, lengths, kept, counts)
    assert keep_tokens(pools[0], table, cu, lengths, kept, counts).tolist() == after == [32, 31, 31, 32, 27]
    dh.same_caches(pools, [want])


@pytest.mark.parametrize("kind", ["tree", "roots"])
@pytest.mark.parametrize("how", [dict(), dict(window=9), dict(scale=-0.2)], ids=str)
def test_attention(how, kind):
    table, cu, lengths, rows, pages = _batch(holes=[(3, 1)])
    pool = kv.cache(pages, 2, 16, 64)
    tree, seen = dh.oracle_tree(dh.parents(NEW, 4, kind, pad=2), cu, lengths, 40, how.get("window", 0))
    q = torch.randn(rows, 4, 64, generator=kv.gen(5)).to(torch.bfloat16)
    out = tree_attention(q, pool, table, cu, lengths, tree, **how)
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, **how)


def test_append_at_positions():
    """Rows turn by their positions and are stored in their slots."""
    table, cu, lengths, rows, pages = _batch(new=[4, 6], total=[20, 40])
    q, k, v = (torch.randn(rows, 2, 64, generator=kv.gen(i)).to(torch.bfloat16) for i in range(3))
    angles = rotary_table(30, 64, device="cpu")
    at = torch.arange(rows, dtype=torch.int32) * 3 - 2  # (one before the table, some past it)
    pools = [kv.cache(pages, 2, 16, 64) for _ in range(3)]
    got = rotate_append(q, k, v, pools[0], table, cu, lengths, angles, positions=at)
    still = rotate_append(q, k, v, pools[1], table, cu, lengths)
    assert got[0].isnan().all() and got[10:].eq(0).all() and torch.equal(pools[0].v.view(torch.uint8), pools[1].v.view(torch.uint8))
    slots = torch.cat((torch.arange(16, 20), torch.arange(34, 40))).to(torch.int32)
    rotate_append(q, k, v, pools[2], table, cu, lengths, angles)
    again = kv.cache(pages, 2, 16, 64)
    rotate_append(q, k, v, again, table, cu, lengths, angles, positions=torch.nn.functional.pad(slots, (0, rows - 10)))
    assert torch.equal(again.k.view(torch.uint8), pools[2].k.view(torch.uint8))
    turned = rotate_append(still, k, v, pools[1], table, cu, lengths, angles, positions=at)
    assert torch.equal(turned.nan_to_num(7.0), got.nan_to_num(7.0))


def test_refusals():
    table, cu, lengths, rows, pages = _batch()
    pool = kv.cache(pages, 2, 16, 64)
    par = dh.parents(NEW, pad=2)
    for bad in (dict(most=0), dict(most=1025), dict(window=-1)):
        with pytest.raises(ValueError):
            draft_tree(par, cu, lengths, **{"most": 40, **bad})
    for args in ((par.long(), cu, lengths), (par, cu[:-1], lengths), (par[::2], cu, lengths), (par[None], cu, lengths)):
        with pytest.raises(ValueError):
            draft_tree(*args, 40)
    tokens = torch.zeros(rows, dtype=torch.int64)
    for args in ((tokens.float(), tokens.float(), par, cu), (tokens, tokens.int(), par, cu), (tokens, tokens[1:], par, cu),
                 (tokens, tokens, par[1:], cu), (tokens, tokens, par, cu[:0])):
        with pytest.raises(ValueError):
            accept_drafts(*args, 40)
    q = torch.zeros(rows, 4, 64, dtype=torch.bfloat16)
    tree = draft_tree(par, cu, lengths, 40)
    mask, positions = tree
    for bad in (DraftTree(mask[1:], positions), DraftTree(mask.long(), positions), DraftTree(mask[:, :0], positions),
                DraftTree(mask, positions[1:]), DraftTree(mask, positions.long()), DraftTree(mask[:, ::2], positions),
                DraftTree(torch.zeros(rows, 33, dtype=torch.int32), positions)):
        with pytest.raises(ValueError):
            tree_attention(q, pool, table, cu, lengths, bad)
    for how in (dict(window=-1), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            tree_attention(q, pool, table, cu, lengths, tree, **how)
    with pytest.raises(RuntimeError, match="gradient"):
        tree_attention(q.requires_grad_(), pool, table, cu, lengths, tree)
    k = torch.zeros(rows, 2, 64, dtype=torch.bfloat16)
    for at in (positions.long(), positions[1:], positions.repeat(2)[::2]):
        with pytest.raises(ValueError, match="positions"):
            rotate_append(q.detach(), k, k, pool, table, cu, lengths, positions=at)
    kept, counts = _kept(NEW, 41)
    for args in ((table.long(), cu, lengths, kept, counts), (table, cu[1:], lengths, kept, counts),
                 (table, cu, lengths[1:], kept, counts), (table, cu, lengths, kept[1:], counts),
                 (table, cu, lengths, kept.long(), counts), (table, cu, lengths, kept, counts[1:]),
                 (table[0], cu, lengths, kept, counts), (table, cu, lengths, torch.zeros(5, 1025, dtype=torch.int32), counts)):
        with pytest.raises(ValueError):
            keep_tokens(pool, *args)


def test_a_pack_refuses_before_it_stores():
    table, cu, lengths, rows, pages = kv.batch([2, 1], [20, 3], 16)
    pack = QuantLinearPack.create([_int8(64, n, n) for n in (256, 128, 128)])
    pool = kv.cache(pages, 2, 16, 64)
    before = dh.clones([pool])[0]
    hidden = torch.randn(rows, 64, generator=kv.gen(1)).to(torch.bfloat16)
    tree = draft_tree(dh.parents([2, 1]), cu, lengths, 2)
    for how in (dict(tree=tree, causal=False), dict(tree=DraftTree(tree.mask[1:], tree.positions)),
                dict(tree=DraftTree(tree.mask, tree.positions[1:]))):
        with pytest.raises(ValueError):
            pack.attend(hidden, pool, table, cu, lengths, **how)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, before))
    assert pack.attend(hidden, pool, table, cu, lengths, tree=tree).shape == (rows, 256)


def test_c_entries_refuse_bad_shapes_before_a_launch():
    def attention(**change):
        a = dict(q_ld=256, dtype=1, heads=4, dim=64, words=1, window=0, scale=1.0)
        a.update(change)
        _native.call("kq_kv_tree_attention", None, a["q_ld"], 64, a["dtype"], 1, a["heads"], 2, a["dim"], None, None, None,
                     None, 1, 16, None, 1, 1, None, None, 1, None, a["words"], None, a["scale"], a["window"], None, None, 0, None)

    for change in (dict(heads=3), dict(dim=96), dict(window=-1), dict(words=0), dict(words=33), dict(q_ld=257), dict(scale=1e40)):
        with pytest.raises(ValueError):
            attention(**change)
    for args in ((-1, 1, 4, 0), (1, 1, 0, 0), (1, 1, 1025, 0), (1, 1, 4, -1)):
        with pytest.raises(ValueError):
            _native.call("kq_draft_tree", None, args[0], None, None, args[1], args[2], args[3], None, None, None)
    with pytest.raises(ValueError):
        _native.call("kq_draft_accept", None, None, 1, None, 1, None, 1, 1025, None, None, None, None)
    pool = KvCaches([kv.cache(2, 2, 16, 64)])
    for layers, most, dim in ((0, 4, 64), (1, 1025, 64), (1, 4, 80)):
        with pytest.raises(ValueError):
            _native.call("kq_kv_keep_tokens", pool.pointers, layers, 2, 2, 16, dim, None, 1, 1, None, None, 1, None, most, None,
                         None, None)


def test_empty_calls():
    none, cu = dh.ints(), dh.ints(0)
    tree = draft_tree(none, cu, none, 4)
    assert tree.mask.shape == (0, 1) and tree.positions.shape == (0,)
    kept, counts, following = accept_drafts(none.long(), none.long(), none, cu, 4)
    assert kept.shape == (0, 4) and counts.shape == following.shape == (0,)
    pool = kv.cache(3, 2, 16, 64)
    assert keep_tokens(pool, none.view(0, 1), cu, none, kept, counts).shape == (0,)
    out = tree_attention(torch.zeros(0, 4, 64, dtype=torch.bfloat16), pool, none.view(0, 1), cu, none, tree)
    assert out.shape == (0, 4, 64)
