"""Attention of drafted trees in batches of more than 64 sequences, whose bounds a wave no longer
holds: tiles cut into parts of one length and into runs, and joined, against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import DraftTree, tree_attention
from kairyu_amd.kernels import kv_cache_hip as hip

pytestmark = pytest.mark.gpu

FORMS = {
    # sequences, most rows of one, (query heads, kv heads, head dim), page, columns of a tile, parts of one length
    "32 columns, parts": (150, 11, (4, 1, 128), 32, 32, True),
    "32 columns, parts, 65 sequences": (65, 9, (8, 2, 64), 16, 32, True),
    "64 columns, parts": (130, 27, (4, 1, 64), 64, 64, True),
    "64 columns, parts, dim 256": (100, 13, (16, 1, 256), 32, 64, True),
    "128 columns, parts": (128, 40, (8, 2, 128), 64, 128, True),
    "128 columns, parts, 200 sequences": (200, 33, (8, 1, 64), 16, 128, True),
    "16 columns, runs": (150, 5, (8, 2, 64), 32, 16, False),
    "16 columns, runs, dim 256": (90, 3, (12, 3, 256), 16, 16, False),
    "32 columns, runs": (150, 11, (32, 8, 128), 64, 32, False),
    "64 columns, runs": (130, 27, (32, 8, 64), 32, 64, False),
    "128 columns, runs": (300, 40, (16, 2, 128), 16, 128, False),
}


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("form", FORMS)
def test_attention_of_many_sequences(cuda, form, window):
    banner(f"tree attention many sequences {form} window {window}")
    seqs, most, (hq, hk, dim), page, columns, alike = FORMS[form]
    new = [most if i == 3 else (7 * i) % (most + 1) for i in range(seqs)]  # (some without rows)
    total = [n + ((37 * i) % 300 if i % 29 else 2500 + 40 * i) for i, n in enumerate(new)]
    table, cu, lengths, rows, pages = kv.batch(new, total, page, seed=1, pad=2, holes=[(29, 1), (58, 0), (58, 2)])
    pool = kv.cache(pages, hk, page, dim, seed=2)
    kv.stain(pool, table, lengths)
    tree, seen = dh.oracle_tree(dh.parents(new, 3, pad=2), cu, lengths, most, window)
    q = (torch.randn(rows, hq, dim, generator=kv.gen(4)) * 2).to(torch.bfloat16)
    table = torch.nn.functional.pad(table, (0, (1 << 20) // page - table.shape[1]), value=-1)
    # the form, from the scratch of a call without a window: a place for every workgroup and column, twice
    shares = (3 if columns * dim == 1024 else 1 if columns > 16 and dim == 256 else 2) * 256 // hk
    assert hip._tree_bytes(rows, hq, hk, dim, page, table.shape[1], seqs) == 8 * (dim + 4) * hk * shares * columns
    assert (columns > 16 and rows * (hq // hk) // columns + seqs <= shares) == alike
    out = tree_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda),
                         DraftTree(*(t.to(cuda) for t in tree)), window=window)
    torch.cuda.synchronize()
    dh.check_attention(out, q, pool, table, cu, lengths, seen, tree.positions, form, window=window)
    assert not out[-2:].any()
