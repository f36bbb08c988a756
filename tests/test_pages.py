"""Copies of pages and forks of sequences on the CPU against their definition, and the calls
that are refused."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from kairyu_amd import _native
from kairyu_amd.attention import PagedKvCache
from kairyu_amd.pages import KvCaches, copy_pages, fork_sequences
from oracle import drafts as odr

FORKS = {
    "reserve": lambda n: list(range(n)),
    "beams": lambda n: [j // 4 * 4 + (0, 0, 2, 3)[j % 4] for j in range(n)],
    "one": lambda n: [5] * n,
    "backwards": lambda n: list(range(n - 1, -1, -1)),
    "ended": lambda n: [-1 if j % 3 == 0 else j for j in range(n)],
    "fewer": lambda n: [3, 3, 99],
    "more": lambda n: [j % n for j in range(2 * n + 1)],
    "none": lambda n: [],
}


def apply(pools, copies):
    """The oracle's copies, on caches as values."""

    out = [kv.values(p) for p in pools]
    old = [{n: t.clone() for n, t in w.items()} for w in out]
    for w, o in zip(out, old):
        for a, b, tokens in copies:
            for n in "kv":
                w[n][b, :, :tokens] = o[n][a, :, :tokens]
                w[n + "_scale"][b] = o[n + "_scale"][a]
    return out


@pytest.mark.parametrize("room", [0, 1, 17, 40])
@pytest.mark.parametrize("how", FORKS)
def test_fork(how, room):
    page, width = 16, 9
    table, lengths, holders, pages = dh.beams([33, 64, 5], 4, page, width, spare=60)
    pools = dh.layers(2, pages, 2, page, 64)
    par = torch.tensor(FORKS[how](12), dtype=torch.int32)
    new, out, held, copies, missing = odr.fork(holders, table, lengths, par, room, page)
    want = apply(pools, copies)
    got = fork_sequences(KvCaches(pools), holders, table, lengths, par, room)
    assert got[0].tolist() == new and got[1].tolist() == out and got[2].tolist() == [missing]
    assert holders.tolist() == held
    dh.same_caches(pools, want)


def test_a_half_filled_page_shared_and_then_taken_apart():
    """With no room a page is shared; every holder then goes on in a copy, and the page is free."""
    table, lengths, holders, pages = dh.beams([21], 1, 16, 4, spare=6)
    pool = dh.layers(1, pages, 2, 16, 64)
    table, lengths, _ = fork_sequences(pool[0], holders, table, lengths, dh.ints(0, 0, 0), 0)
    shared = int(table[0, 1])
    assert table[:, 1].tolist() == [shared] * 3 and int(holders[shared]) == 3
    table, lengths, missing = fork_sequences(pool[0], holders, table, lengths, dh.ints(0, 1, 2), 1)
    assert len(set(table[:, 1].tolist()) | {shared}) == 4 and int(holders[shared]) == 0 and missing.tolist() == [0]
    table, lengths, _ = fork_sequences(pool[0], holders, table, lengths, dh.ints(-1, -1, -1))
    assert not holders.any() and (table == -1).all() and not lengths.any()


def test_too_few_pages():
    table, lengths, holders, pages = dh.beams([20, 40], 2, 16, 6, spare=1)
    pool = dh.layers(1, pages, 2, 16, 64)
    want = odr.fork(holders, table, lengths, dh.ints(0, 0, 2, 2, 2), 30, 16)
    got = fork_sequences(pool[0], holders, table, lengths, dh.ints(0, 0, 2, 2, 2), 30)
    assert got[0].tolist() == want[0] and got[2].tolist() == [want[4]] and want[4] > 0
    assert holders.tolist() == want[2]


def test_copy():
    pools = dh.layers(3, 9, 2, 16, 64)
    want = [kv.values(p) for p in pools]
    for w in want:
        for t in w.values():
            t[5], t[0] = t[1], t[8]
    copy_pages(KvCaches(pools), dh.ints(1, -1, 3, 3, 8, 9), dh.ints(5, 2, 9, 3, 0, 4))
    dh.same_caches(pools, want)


def test_refusals():
    pool, other = kv.cache(4, 2, 16, 64), kv.cache(5, 2, 16, 64)
    with pytest.raises(ValueError, match="at least one"):
        KvCaches([])
    with pytest.raises(ValueError, match="alike"):
        KvCaches([pool, other])
    with pytest.raises(ValueError, match="different tensors"):
        KvCaches([pool, pool])
    with pytest.raises(ValueError, match="different tensors"):
        KvCaches([PagedKvCache(pool.k, pool.k, pool.k_scale, pool.v_scale)])
    one = dh.ints(0)
    for args in ((one, dh.ints(0, 1)), (one.long(), one), (one[None], one), (dh.ints(0, 1, 2, 3)[::2], dh.ints(1, 2))):
        with pytest.raises(ValueError):
            copy_pages(pool, *args)
    table, lengths, holders = torch.zeros(2, 3, dtype=torch.int32), dh.ints(4, 4), dh.ints(2, 0, 0, 0)
    for args in ((holders[1:], table, lengths, one, 1), (holders.long(), table, lengths, one, 1),
                 (holders, table[0], lengths, one, 1), (holders, table.long(), lengths, one, 1),
                 (holders, table, lengths[1:], one, 1), (holders, table, lengths, one[None], 1),
                 (holders, table, lengths, one, -1), (holders, table, lengths, one, (1 << 24) + 1),
                 (holders, table[:, ::2], lengths, one, 1)):
        with pytest.raises(ValueError):
            fork_sequences(pool, *args)


def test_c_entries_refuse_bad_shapes_before_a_launch():
    pool = KvCaches([kv.cache(2, 2, 16, 64)])
    for layers, dim, count in ((0, 64, 1), (5000, 64, 1), (1, 80, 1), (1, 64, -1), (1, 64, 1 << 24)):
        with pytest.raises(ValueError):
            _native.call("kq_kv_copy_pages", pool.pointers, layers, 2, 2, 16, dim, None, None, count, None)

    def fork(**change):
        a = dict(pages=2, ld=3, width=3, seqs=2, rows=2, room=1, ws=1 << 20)
        a.update(change)
        _native.call("kq_kv_fork_sequences", pool.pointers, 1, a["pages"], 2, 16, 64, None, None, a["ld"], a["width"], None,
                     a["seqs"], None, a["rows"], a["room"], None, None, None, None, a["ws"], None)

    for change in (dict(pages=-1), dict(ld=2), dict(seqs=-1), dict(rows=-1), dict(room=-1), dict(room=1 << 25), dict(rows=1 << 24)):
        with pytest.raises(ValueError):
            fork(**change)
    with pytest.raises(RuntimeError, match="workspace"):
        fork(ws=4)
