"""Attention where one token holds nearly all of the softmax's mass and a value of zero,
so that the output is what the many tokens of tiny weight add up to: each of the kernels'
forms against the 64-bit oracle."""

from __future__ import annotations

import math

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import paged_attention

pytestmark = pytest.mark.gpu

HEADS = {"8 of 2, 64": (8, 2, 64), "7 of 1, 128": (7, 1, 128), "3 of 1, 256": (3, 1, 256)}
FORMS = {
    # (new rows, tokens after them), the share of the mass that is not the sink's, the sink's position
    "tiles of 16, read whole": ([1, 1, 1], [1000, 900, 1024], 2.0**-15, 5),
    "tiles of 16, shared out": ([1] * 40, [1500] * 40, 2.0**-14, 70),
    "tiles of 16, one context": ([1], [33000], 2.0**-10, 0),
    "tiles of 128": ([50, 200], [1900, 1500], 2.0**-14, 5),
    "tiles of 128, the sink late": ([50, 200], [1900, 1500], 2.0**-14, 1203),
    "tiles of 128, cut": ([90], [5000], 2.0**-13, 0),
}


def sink_case(new, total, share, at, heads, dtype, seed):
    """(q, pool, table, cu, lengths) on the CPU: queries alike but for some noise, keys of
    small scores with values of 64 to 128 steps, and at position ``at`` of each sequence
    a key that takes all but ``share`` of the mass, with a value of zero."""

    hq, hk, dim = heads
    page = 32
    table, cu, lengths, rows, pages = kv.batch(new, total, page, seed=seed)
    g = kv.gen(seed + 1)
    pool = kv.cache(pages, hk, page, dim, seed=seed + 2)
    side = torch.randn(dim, generator=g).sign()
    q = (side + 0.1 * torch.randn(rows, hq, dim, generator=g)).to(dtype)
    pool.k.copy_((torch.randn(pool.k.shape, generator=g) * 4).to(kv.E4M3))
    pool.v.copy_((64 + 64 * torch.rand(pool.v.shape, generator=g)).to(kv.E4M3))
    pool.k_scale.fill_(2.0**-6)
    pool.v_scale.copy_(torch.exp2(torch.randint(0, 3, pool.v_scale.shape, generator=g).float()))
    for s, n in enumerate(total):
        p = int(table[s, at // page])
        score = math.log(n / share)  # over keys of scores around 0
        pool.k[p, :, at % page] = (side * score / (dim**0.5 * 2.0**-6)).to(kv.E4M3)
        pool.v.view(torch.uint8)[p, :, at % page] = 0
    kv.stain(pool, table, lengths)
    return q, pool, table, cu, lengths


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("form", FORMS)
def test_the_tail_beside_a_sink(cuda, form, heads, dtype):
    banner(f"kv sink {form} {heads} {dtype}")
    new, total, share, at = FORMS[form]
    q, pool, table, cu, lengths = sink_case(new, total, share, at, HEADS[heads], dtype, 61)
    want, bound = kv.oatt.attend(q, kv.values(pool), table, cu, lengths)
    # (values of one sign: what the test can miss is a fiftieth of the answer at the most)
    assert (bound <= 0.02 * want.abs()).all() and want.abs().min() > 0
    out = paged_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda))
    torch.cuda.synchronize()
    kv.assert_within(out, want, bound, dtype, form)
