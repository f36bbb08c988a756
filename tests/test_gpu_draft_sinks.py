"""Attention of drafted trees where one token holds nearly all of the softmax's mass and has
a value of zero, so that the output is what the many tokens of tiny weight add up to: tiles
of every width against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

import draft_helpers as dh
import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import DraftTree, tree_attention
from oracle import drafts as odr
from test_gpu_kv_sinks import HEADS, sink_case

pytestmark = pytest.mark.gpu

FORMS = {
    # (drafted rows, tokens after them), the share of the mass that is not the sink's, the
    # sink's position, whether the table is for a million tokens
    "read whole": ([3, 2, 5], [1000, 900, 1024], 2.0**-15, 5, False),
    "small tiles, one context": ([4], [33000], 2.0**-10, 0, False),
    "few rows": ([6, 5], [1900, 1500], 2.0**-14, 70, True),
    "more rows": ([16, 12], [1900, 1500], 2.0**-14, 5, True),
    "many rows": ([50, 40], [1900, 1500], 2.0**-14, 5, True),
    "many rows, the sink late": ([50, 40], [1900, 1500], 2.0**-14, 1203, True),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("form", FORMS)
def test_the_tail_beside_a_sink(cuda, form, heads, dtype):
    banner(f"tree sink {form} {heads} {dtype}")
    new, total, share, at, wide = FORMS[form]
    q, pool, table, cu, lengths = sink_case(new, total, share, at, HEADS[heads], dtype, 71)
    tree, seen = dh.oracle_tree(dh.parents(new, 72), cu, lengths, max(new))
    want, bound = kv.oatt.attend(q, kv.values(pool), table, cu, lengths, seen_by=odr.seen_by(seen, tree.positions))
    # (values of one sign: what the test can miss is a fiftieth of the answer at the most)
    assert (bound <= 0.02 * want.abs()).all() and want.abs().min() > 0
    if wide:
        table = torch.nn.functional.pad(table, (0, (1 << 20) // pool.page_size - table.shape[1]), value=-1)
    out = tree_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda),
                         DraftTree(*(t.to(cuda) for t in tree)))
    torch.cuda.synchronize()
    kv.assert_within(out, want, bound, dtype, form)
