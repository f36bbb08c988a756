"""Copies of pages and forks of sequences on the GPU against their definition, and rows that
are sampled apart from one prompt, captured and replayed too."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import PagedKvCache, paged_attention, rotate_append
from kairyu_amd.pages import KvCaches, copy_pages, fork_sequences
from oracle import drafts as odr
from test_pages import FORKS, apply

pytestmark = pytest.mark.gpu


def _fork(cuda, pools, holders, table, lengths, par, room, page):
    """Runs a fork and checks all that it leaves; the new table and lengths."""
    new, out, held, copies, missing = odr.fork(holders.cpu(), table.cpu(), lengths.cpu(), par, room, page)
    want = apply(pools, copies)
    got = fork_sequences(KvCaches(pools), holders, table, lengths, par.to(cuda), room)
    torch.cuda.synchronize()
    assert got[0].tolist() == new and got[1].tolist() == out and got[2].tolist() == [missing]
    assert holders.tolist() == held
    dh.same_caches(pools, want)
    return got[:2]


@pytest.mark.parametrize("room", [0, 1, 17, 40])
@pytest.mark.parametrize("shape", [(2, 16, 64), (3, 64, 128), (1, 32, 256)], ids=str)
@pytest.mark.parametrize("how", FORKS)
def test_fork(cuda, how, shape, room):
    banner(f"fork {how} {shape} room {room}")
    kv_heads, page, dim = shape
    table, lengths, holders, pages = dh.beams([2 * page + 1, 4 * page, 5, page - 1], 4, page, 9, spare=90)
    pools = dh.layers(2, pages, kv_heads, page, dim, device=cuda)
    par = torch.tensor(FORKS[how](16), dtype=torch.int32)
    _fork(cuda, pools, holders.to(cuda), table.to(cuda), lengths.to(cuda), par, room, page)


def test_fork_after_fork(cuda):
    """A batch that forks, shrinks, ends and grows again, page books and all."""
    banner("forks in a row")
    page = 16
    table, lengths, holders, pages = dh.beams([40, 23], 3, page, 12, spare=70)
    pools = dh.layers(2, pages, 2, page, 64, device=cuda)
    table, lengths, holders = table.to(cuda), lengths.to(cuda), holders.to(cuda)
    for i, (par, room, grow) in enumerate([([0, 0, 1, 4, 4, 4], 1, 1), ([0, 1, 2, 3, 4, 5], 20, 18), ([5, 4, 3, 2, 1, 0, 0], 0, 0),
                                           ([0, 1, 2, 3, 4, 5, 6], 1, 1), ([-1, 1, 2], 3, 3), ([2, 2, 2, 2], 5, 5), ([-1] * 4, 1, 0)]):
        table, lengths = _fork(cuda, pools, holders, table, lengths, dh.ints(*par), room, page)
        lengths = lengths + grow
    assert not holders.any()


@pytest.mark.parametrize("rows", [1, 700, 1500])
def test_fork_of_many_rows_and_pages(cuda, rows):
    """More rows, slots and pages than one round of the plan holds, few free pages among many."""
    banner(f"fork {rows} rows")
    page, width = 16, 5
    pages = 9000
    g = kv.gen(rows)
    holders = (torch.rand(pages, generator=g) < 0.4).to(torch.int32)
    free = (holders == 0).nonzero()[:, 0]
    table = torch.full((rows, width), -1, dtype=torch.int32)
    order = free[torch.randperm(len(free), generator=g)]
    table[:, 0] = order[:rows].to(torch.int32)
    holders[order[:rows]] += 1
    lengths = torch.randint(0, 17, (rows,), generator=g).to(torch.int32)
    pools = dh.layers(1, pages, 1, page, 64, device=cuda)
    par = torch.randint(-1, rows + 1, (rows + 3,), generator=g).to(torch.int32)
    _fork(cuda, pools, holders.to(cuda), table.to(cuda), lengths.to(cuda), par, 40, page)


@pytest.mark.parametrize("spare", [0, 1, 5])
def test_too_few_pages(cuda, spare):
    banner(f"fork with {spare} pages")
    table, lengths, holders, pages = dh.beams([20, 40], 2, 16, 6, spare=spare)
    pools = dh.layers(1, pages, 2, 16, 64, device=cuda)
    _fork(cuda, pools, holders.to(cuda), table.to(cuda), lengths.to(cuda), dh.ints(0, 0, 2, 2, 2), 30, 16)


def test_entries_and_lengths_that_are_wrong_stay_in_range(cuda):
    """Entries past the cache, lengths past the table and below zero, books that do not add up."""
    banner("fork of bad tables")
    table, lengths, holders, pages = dh.beams([33, 20, 9], 1, 16, 4, spare=9)
    table[0, 0], table[1, 1], table[2, 3] = pages, 2**31 - 1, -(2**31)
    lengths = torch.tensor([33, -4, 2**31 - 1], dtype=torch.int32)
    holders = torch.bincount(table[(table >= 0) & (table < pages)].long(), minlength=pages).to(torch.int32)
    holders[table[0, 1].long()] = 0
    pools = dh.layers(1, pages, 2, 16, 64, device=cuda)
    _fork(cuda, pools, holders.to(cuda), table.to(cuda), lengths.to(cuda), dh.ints(0, 0, 1, 2, 2), 20, 16)


def test_more_layers_than_a_launch_takes(cuda):
    banner("fork and copy of 70 layers")
    table, lengths, holders, pages = dh.beams([20], 3, 16, 4)
    pools = dh.layers(70, pages, 1, 16, 64, device=cuda)
    _fork(cuda, pools, holders.to(cuda), table.to(cuda), lengths.to(cuda), dh.ints(0, 0, 0, 1), 1, 16)
    want = [kv.values(p) for p in pools]
    for w in want:
        for t in w.values():
            t[2] = t[1]
    copy_pages(KvCaches(pools), dh.ints(1).to(cuda), dh.ints(2).to(cuda))
    dh.same_caches(pools, want)


@pytest.mark.parametrize("shape", [(2, 16, 64), (8, 64, 128), (3, 32, 256), (5, 128, 128), (1, 16, 64)], ids=str)
def test_copy(cuda, shape):
    banner(f"copy pages {shape}")
    kv_heads, page, dim = shape
    pools = dh.layers(3, 40, kv_heads, page, dim, device=cuda)
    want = [kv.values(p) for p in pools]
    sources, targets = [1, -1, 3, 3, 8, 40, 2**31 - 1, *range(10, 24)], [5, 2, 40, 3, 0, 4, 6, *range(39, 25, -1)]
    for w in want:
        for t in w.values():
            for a, b in zip(sources, targets):
                if 0 <= a < 40 and 0 <= b < 40:
                    t[b] = t[a].clone()
    copy_pages(KvCaches(pools), dh.ints(*sources).to(cuda), dh.ints(*targets).to(cuda))
    torch.cuda.synchronize()
    dh.same_caches(pools, want)


def test_refusals(cuda):
    banner("pages refusals")
    pool = dh.layers(1, 4, 2, 16, 64, device=cuda)[0]
    one = dh.ints(0)
    with pytest.raises(RuntimeError, match="must be on"):
        copy_pages(pool, one, one)
    with pytest.raises(RuntimeError, match="must be on"):
        fork_sequences(pool, torch.zeros(4, dtype=torch.int32), one.view(1, 1).to(cuda), one.to(cuda), one.to(cuda))
    with pytest.raises(RuntimeError, match="must be on"):
        KvCaches([pool, dh.layers(1, 4, 2, 16, 64)[0]])


def _samples(pool, holders, table, lengths, par, q, k, v):
    """One step of rows that go on as others: their pages, one token appended, attention."""
    table, lengths, missing = fork_sequences(pool, holders, table, lengths, par)
    lengths = lengths + 1
    cu = torch.arange(par.shape[0] + 1, dtype=torch.int32, device=q.device)
    q = rotate_append(q, k, v, pool, table, cu, lengths)
    return paged_attention(q, pool, table, cu, lengths), table, lengths, missing


def test_samples_of_one_prompt(cuda):
    """Four rows that share a prompt and go on apart hold what a cache of their own would: the
    same attention, bit for bit, as rows that never shared a page; eager, and replayed."""
    banner("samples of one prompt")
    page, dim, kv_heads, heads, rows = 16, 64, 2, 4, 4
    g = kv.gen(3)
    pool, own = (PagedKvCache.create(64, kv_heads, dim, page, device=cuda) for _ in range(2))
    holders = torch.zeros(64, dtype=torch.int32, device=cuda)
    prompt = [torch.randn(37, h, dim, generator=g).to(torch.bfloat16).to(cuda) for h in (heads, kv_heads, kv_heads)]
    table = torch.full((1, 8), -1, dtype=torch.int32, device=cuda)
    table, lengths, _ = fork_sequences(pool, holders, table, dh.ints(0).to(cuda), dh.ints(0).to(cuda), 37)
    rotate_append(*prompt, pool, table, dh.ints(0, 37).to(cuda), lengths + 37)
    lengths = lengths + 37
    apart = torch.arange(rows * 8, dtype=torch.int32, device=cuda).view(rows, 8)
    for r in range(rows):
        rotate_append(*prompt, own, apart[r: r + 1], dh.ints(0, 37).to(cuda), dh.ints(37).to(cuda))
    cu = torch.arange(rows + 1, dtype=torch.int32, device=cuda)

    table, lengths, _ = fork_sequences(pool, holders, table, lengths, dh.ints(0, 0, 0, 0).to(cuda), 0)
    static = [torch.zeros(rows, h, dim, dtype=torch.bfloat16, device=cuda) for h in (heads, kv_heads, kv_heads)]
    par = cu[:rows].clone()
    state = [holders, table, lengths, *pool]
    kept = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _samples(pool, holders, table, lengths, par, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _samples(pool, holders, table, lengths, par, *static)
    for t, k in zip(state, kept):
        t.copy_(k)
    for step in range(40):
        for t in static:
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        if step % 2:
            out, new_table, new_lengths, missing = _samples(pool, holders, table, lengths, par, *static)
        else:
            graph.replay()
            out, new_table, new_lengths, missing = captured
        torch.cuda.synchronize()
        q = rotate_append(*static, own, apart, cu, lengths + 1)
        want = paged_attention(q, own, apart, cu, lengths + 1)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and missing.tolist() == [0], step
        table.copy_(new_table)
        lengths.copy_(new_lengths)
        named = torch.bincount(table[table >= 0].long(), minlength=64).to(torch.int32)
        assert torch.equal(named, holders), step
    full = table[:, : 37 // page]
    assert (full == full[0]).all() and int(holders[full[0, 0].long()]) == rows
