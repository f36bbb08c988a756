"""Trees, block tables and comparisons shared by the tests of drafts and shared pages."""

from __future__ import annotations

import random

import torch

import kv_helpers as kv
from kairyu_amd.attention import DraftTree, PagedKvCache
from oracle import drafts as odr


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def parents(new, seed=0, kind="tree", pad=0):
    """Parents of each sequence's rows, one after the other."""

    rng = random.Random(seed)
    out = []
    for n in new:
        for i in range(n):
            p = {"chain": i - 1, "star": 0 if i else -1, "roots": -1}.get(kind)
            if p is None:
                p = rng.randrange(max(0, i - 9), i) if i else -1
            out.append(p)
    return torch.tensor(out + [0] * pad, dtype=torch.int32)


def oracle_tree(par, cu, lengths, most, window=0):
    """A tree as the oracle defines it: (tree, seen)."""

    seen, positions = odr.tree(par, cu, lengths, most, window)
    return DraftTree(odr.pack(seen, -(-most // 32)), torch.tensor(positions, dtype=torch.int32)), seen


def check_attention(out, q, pool, table, cu, lengths, seen, positions, label="", window=0, **how):
    how["seen_by"] = odr.seen_by(seen, positions.cpu(), window)
    kv.check_attention(out, q, pool, table, cu, lengths, label, **how)


def tokens_for(par, cu, seed=0, agree=0.7, dtype=torch.int64):
    """Tokens and targets: most nodes with children have one of them as their target."""

    rng = random.Random(seed)
    rows = par.shape[0]
    tokens, targets = [rng.randrange(5) for _ in range(rows)], [rng.randrange(5, 9) for _ in range(rows)]
    for row, n in odr.spans(rows, cu):
        for i in range(n):
            p = int(par[row + i])
            if 0 <= p < i and rng.random() < agree:
                targets[row + p] = tokens[row + i]
    return torch.tensor(tokens, dtype=dtype), torch.tensor(targets, dtype=dtype)


def same_caches(pools, want):
    """Every layer's codes (as values) and scales are the oracle's, NaN where it has it."""

    for layer, (pool, w) in enumerate(zip(pools, want)):
        got = kv.values(pool)
        for name in w:
            assert torch.equal(got[name].isnan(), w[name].isnan()), (layer, name)
            assert torch.equal(got[name].nan_to_num(0.0), w[name].nan_to_num(0.0)), (layer, name)


def layers(count, pages, kv_heads, page, dim, seed=0, device="cpu"):
    return [kv.to(kv.cache(pages, kv_heads, page, dim, seed=seed + i), device) for i in range(count)]


def clones(pools):
    return [PagedKvCache(*(t.clone() for t in pool)) for pool in pools]


def beams(requests, count, page, width, seed=0, spare=20, ended=()):
    """(table, lengths, holders, pages): ``count`` rows for each request's tokens that share full
    pages and hold their last alone; the requests in ``ended`` have no pages."""

    order = torch.randperm(sum(t // page + count for t in requests) + spare, generator=kv.gen(seed)).tolist()
    pages, table, lengths = len(order), [], []
    for r, tokens in enumerate(requests):
        full = [order.pop() for _ in range(tokens // page)]
        for _ in range(count):
            row = full + ([order.pop()] if tokens % page else [])
            row = [] if r in ended else row
            table.append(row + [-1] * (width - len(row)))
            lengths.append(0 if r in ended else tokens)
    table = torch.tensor(table, dtype=torch.int32)
    holders = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
    return table, torch.tensor(lengths, dtype=torch.int32), holders, pages
