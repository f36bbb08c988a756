"""The paged 8-bit key/value cache on the CPU where it is easily wrong: what the oracle
allows beside a dominant token, angles without positions, caches without pages, calls
that are refused."""

from __future__ import annotations

import math

import pytest
import torch

import kv_helpers as kv
from kairyu_amd.attention import PagedKvCache, paged_attention, rotary_table, rotate_append
from kairyu_amd.quant.packed import QuantLinearPack
from oracle import attention as oatt
from test_packed import _int8


def test_the_oracles_bound_beside_a_sink():
    """Where one token holds nearly all of the mass and has a value of zero, the output is
    the others' tail, and the bound is far below it."""

    n, dim = 32768, 64
    table, cu, lengths, rows, pages = kv.batch([1], [n], 128, spare=0)
    pool = kv.cache(pages, 1, 128, dim)
    pool.k.view(torch.uint8).zero_()
    pool.v.view(torch.uint8).fill_(0x38)  # 1.0
    pool.k_scale.fill_(1.0)
    pool.v_scale.fill_(1.0)
    sink = int(table[0, 0])
    pool.k[sink, 0, 0] = torch.tensor(2.0).to(kv.E4M3)
    pool.v.view(torch.uint8)[sink, 0, 0] = 0
    score = math.log(n * 999.0)
    q = torch.full((1, 1, dim), score / (dim**0.5 * 2.0))
    o, bound = oatt.attend(q, kv.values(pool), table, cu, lengths)
    assert (o - 1e-3).abs().max() <= 1e-5
    assert (bound <= 0.01 * o).all()


def test_angles_without_positions():
    """Every position is past a table that has none: NaN where heads would turn."""

    table, cu, lengths, rows, pages = kv.batch([3, 1], [20, 7], 16, pad=1)
    pool = kv.cache(pages, 2, 16, 64)
    q, k, v = (torch.randn(rows, h, 64, generator=kv.gen(h)).to(torch.bfloat16) for h in (4, 2, 2))
    before = kv.values(pool)
    cos_sin = rotary_table(0, 32, device="cpu")
    out = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    assert out[:4, :, :32].isnan().all() and not out[:4, :, 32:].isnan().any()
    kv.check_append(out, pool, before, q, k, v, table, cu, lengths, cos_sin=cos_sin)


def test_caches_without_pages():
    """No token is there: zero outputs, turned queries."""

    pool = PagedKvCache.create(0, 2, 64, 16, device="cpu")
    table, cu, lengths, rows, _ = kv.batch([3, 1], [20, 7], 16, pad=1)
    q, k = (torch.randn(rows, h, 64, generator=kv.gen(h)).to(torch.bfloat16) for h in (4, 2))
    out = paged_attention(q, pool, table, cu, lengths)
    assert out.shape == q.shape and not out.any()
    some = kv.cache(9, 2, 16, 64)
    where = (table, cu, lengths, rotary_table(32, 64, device="cpu"))
    assert torch.equal(rotate_append(q, k, k, pool, *where), rotate_append(q, k, k, some, *where))


@pytest.mark.parametrize("how", [dict(window=-1), dict(window=8, causal=False), dict(scale=math.nan)], ids=str)
def test_attend_refuses_before_it_stores(how):
    table, cu, lengths, rows, pages = kv.batch([2, 1], [20, 3], 16)
    pack = QuantLinearPack.create([_int8(64, n, n) for n in (256, 128, 128)])
    pool = kv.cache(pages, 2, 16, 64)
    before = [t.clone() for t in pool]
    hidden = torch.randn(rows, 64, generator=kv.gen(1)).to(torch.bfloat16)
    with pytest.raises(ValueError):
        pack.attend(hidden, pool, table, cu, lengths, **how)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, before))
    assert pack.attend(hidden, pool, table, cu, lengths).shape == (rows, 256)
