"""The paged 8-bit key/value cache on the GPU where it is easily wrong: angles without
positions, caches without pages, queries that are not finite, prompts in wide tables,
pages that nobody holds, value scales far apart."""

from __future__ import annotations

import math

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import PagedKvCache, paged_attention, rotary_table, rotate_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows", [[20, 1], [900, 700]])
def test_angles_without_positions(cuda, rows, interleaved):
    """Every position is past a table that has none: NaN where heads would turn."""
    banner(f"kv append no positions {rows} {interleaved}")
    table, cu, lengths, n, pages = kv.batch(rows, [r + 9 for r in rows], 32, seed=71, pad=1)
    pool = kv.cache(pages, 2, 32, 128, seed=72)
    g = kv.gen(73)
    q, k, v = (torch.randn(n, h, 128, generator=g).to(torch.bfloat16) for h in (8, 2, 2))
    before, on = kv.values(pool), kv.to(pool, cuda)
    where = (table.to(cuda), cu.to(cuda), lengths.to(cuda))
    cos_sin = rotary_table(0, 64, device=cuda)
    out = rotate_append(q.to(cuda), k.to(cuda), v.to(cuda), on, *where, cos_sin, interleaved=interleaved)
    torch.cuda.synchronize()
    assert out[: sum(rows), :, :64].isnan().all() and not out[: sum(rows), :, 64:].isnan().any()
    kv.check_append(out, on, before, q, k, v, table, cu, lengths, cos_sin=cos_sin.cpu(), interleaved=interleaved)


def test_caches_without_pages(cuda):
    """No token is there: zero outputs, turned queries."""
    banner("kv no pages")
    pool = PagedKvCache.create(0, 2, 64, 16, device=cuda)
    table, cu, lengths, rows, _ = kv.batch([40, 1], [70, 7], 16, pad=1)
    q, k = (torch.randn(rows, h, 64, generator=kv.gen(h)).to(torch.bfloat16).to(cuda) for h in (4, 2))
    where = (table.to(cuda), cu.to(cuda), lengths.to(cuda))
    out = paged_attention(q, pool, *where)
    cos_sin = rotary_table(80, 64, device=cuda)
    turned = rotate_append(q, k, k, pool, *where, cos_sin)
    torch.cuda.synchronize()
    assert out.shape == q.shape and not out.any()
    some = kv.to(kv.cache(9, 2, 16, 64), cuda)
    assert torch.equal(turned, rotate_append(q, k, k, some, *where, cos_sin))
    torch.cuda.synchronize()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (3, 1, 256)], ids=str)
@pytest.mark.parametrize("new,total", [([1, 1, 1], [600, 300, 150]), ([1, 1, 1], [3000, 2000, 150]),
                                       ([150, 150, 150], [600, 300, 150]), ([150, 150, 150], [5000, 2300, 150])], ids=str)
def test_queries_that_are_not_finite_over_tokens_of_no_page(cuda, new, total, heads, value):
    """A row that sees no token is zero whatever its query holds; one that sees a token
    is NaN then; and no other row is touched."""
    banner(f"kv attention queries {value} {new} {total} {heads}")
    hq, hk, dim = heads
    page = 32
    holes = [(0, s) for s in range(-(-total[0] // page))] + [(1, 0)]
    table, cu, lengths, n, pages = kv.batch(new, total, page, seed=74, holes=holes)
    pool = kv.cache(pages, hk, page, dim, seed=75)
    kv.stain(pool, table, lengths)
    q = torch.randn(n, hq, dim, generator=kv.gen(76)).to(torch.bfloat16)
    clean = q.clone()
    rows = [0, new[0] - 1, new[0], n - 1]  # the first two in a sequence without pages
    for r in rows:
        q[r, 1, 5] = value
    on, where = kv.to(pool, cuda), (table.to(cuda), cu.to(cuda), lengths.to(cuda))
    out = paged_attention(q.to(cuda), on, *where).cpu()
    assert not out[: new[0]].any()
    assert out[new[0], 1].isnan().all() and out[n - 1, 1].isnan().all()
    want, bound = kv.oatt.attend(clean, kv.values(pool), table, cu, lengths)
    out[rows, 1], want[rows, 1] = 0, 0
    kv.assert_within(out, want, bound, q.dtype, "the others")


@pytest.mark.parametrize("seqs", [1, 2])
def test_many_rows_in_a_wide_table(cuda, seqs):
    """Prompts of many rows and heads in a table for a million tokens, whose pages repeat."""
    banner(f"kv attention many rows in a wide table, {seqs}")
    rows, heads, dim, page, window = 65536, 64, 64, 16, 40
    pool = kv.to(kv.cache(40, 1, page, dim, seed=77), cuda)
    slots = (1 << 20) // page
    table = (torch.arange(slots, device=cuda) % 40).to(torch.int32).expand(seqs, -1).contiguous()
    bounds = [0, rows - 30, rows] if seqs == 2 else [0, rows]
    cu = torch.tensor(bounds, dtype=torch.int32, device=cuda)
    lengths = torch.tensor([bounds[s + 1] - bounds[s] + 70 for s in range(seqs)], dtype=torch.int32, device=cuda)
    row = torch.randn(1, heads, dim, generator=kv.gen(78)).to(torch.bfloat16).to(cuda)
    out = paged_attention(row.expand(rows, -1, -1), pool, table, cu, lengths, window=window)
    torch.cuda.synchronize()
    # a row by itself, as a sequence of that length
    for r in (0, 1000, rows - 31, rows - 30, rows - 1):
        s = seqs - 1 if r >= rows - 30 else 0
        length = int(lengths[s]) - (bounds[s + 1] - r) + 1
        near = (length - 64) // page if length > 64 else 0  # pages that the window touches, and their tokens
        kv.check_attention(out[r: r + 1], row, pool, table[:1, near: near + 8], torch.tensor([0, 1], dtype=torch.int32),
                           torch.tensor([length - near * page], dtype=torch.int32), f"row {r}", window=window)


@pytest.mark.parametrize("page,heads", [(16, (8, 2, 64)), (32, (8, 2, 64)), (64, (8, 2, 64)), (16, (7, 1, 128)), (32, (4, 4, 128)),
                                        (128, (7, 1, 128)), (16, (3, 1, 256)), (32, (3, 1, 256))], ids=str)
@pytest.mark.parametrize("new,total", [([1, 1, 2], [600, 303, 1100]), ([150, 1, 70], [600, 303, 2100]), ([90, 9], [5000, 133])],
                         ids=str)
def test_a_first_page_that_nobody_holds(cuda, new, total, page, heads):
    """Loads for tokens that are not there must not take the cache's first page, all NaN."""
    banner(f"kv attention first page {page} {heads} {new}")
    hq, hk, dim = heads
    table, cu, lengths, n, pages = kv.batch(new, total, page, seed=79)
    table = torch.where(table >= 0, table + 1, table)
    table[0, 1], table[0, total[0] // page - 1], table[1, 0] = -1, pages + 1, -5
    pool = kv.cache(pages + 1, hk, page, dim, seed=80)
    kv.stain(pool, table, lengths)
    for scales in pool[2:]:
        scales[0] = math.nan
    q = torch.randn(n, hq, dim, generator=kv.gen(81)).to(torch.bfloat16)
    out = paged_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda))
    torch.cuda.synchronize()
    pool.k_scale[0], pool.v_scale[0] = 1, 1
    kv.check_attention(out, q, pool, table, cu, lengths)


@pytest.mark.parametrize("new,total", [([1, 1], [600, 303]), ([1, 1], [3000, 1303]), ([150, 70], [600, 303]), ([90], [5000])], ids=str)
def test_value_scales_far_apart(cuda, new, total):
    """Pages whose value scales lie 2^98 apart: those of small values add nothing to the
    output and count in its denominator."""
    banner(f"kv attention value scales {new} {total}")
    table, cu, lengths, n, pages = kv.batch(new, total, 32, seed=82)
    pool = kv.cache(pages, 2, 32, 128, seed=83)
    pool.v_scale.copy_(torch.where(torch.rand(pool.v_scale.shape, generator=kv.gen(84)) < 0.5, 2.0**-48, 2.0**50))
    q = (0.25 * torch.randn(n, 8, 128, generator=kv.gen(85))).to(torch.bfloat16)
    out = paged_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda))
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)


@pytest.mark.parametrize("size", [10, 20, 24, 25, 26, 27, 28, 40, 100])
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (3, 1, 256)], ids=str)
@pytest.mark.parametrize("new,total", [([1, 1], [600, 303]), ([1, 1], [3000, 1303]), ([150, 70], [600, 303]), ([90], [5000])], ids=str)
def test_scores_of_any_size(cuda, new, total, heads, size):
    """Rows whose largest score, times 2^size, stands far above the others take its value,
    or the mean of two in one page, however coarse fp32 is up there."""
    banner(f"kv attention scores of 2^{size} {heads} {new}")
    hq, hk, dim = heads
    table, cu, lengths, n, pages = kv.batch(new, total, 32, seed=86)
    pool = kv.cache(pages, hk, 32, dim, seed=87)
    g = kv.gen(88)
    pool.k.view(torch.uint8).zero_()
    pool.k[..., 3] = (torch.rand(pool.k.shape[:3], generator=g) * 300 - 200).to(kv.E4M3)  # at most 104
    pool.k_scale.fill_(1.0)
    want = torch.zeros(n, hq, dim, dtype=torch.float64)
    for s, (rows, length) in enumerate(zip(new, total)):
        first = length - rows  # token 40 for the first row, then 72 and 73 of one page, alike
        for token, code in ((40, 384.0), (72, 448.0), (73, 448.0)):
            pool.k[int(table[s, token // 32]), :, token % 32, 3] = torch.tensor(code).to(kv.E4M3)
        for r in range(rows):
            at = [72, 73] if first + r >= 73 else [72] if first + r == 72 else [40] if first + r >= 40 else None
            assert at is not None
            value = torch.stack([pool.v[int(table[s, t // 32]), :, t % 32].double()
                                 * pool.v_scale[int(table[s, t // 32])].double()[:, None] for t in at]).mean(0)
            want[int(cu[s]) + r] = value.repeat_interleave(hq // hk, 0)
    q = torch.zeros(n, hq, dim, dtype=torch.bfloat16)
    q[..., 3] = 2.0 ** size
    kv.stain(pool, table, lengths)
    out = paged_attention(q.to(cuda), kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda))
    torch.cuda.synchronize()
    # one weight or two alike, exact but for the weights' and the quotient's roundings
    kv.assert_within(out, want, 2.0**-10 * want.abs(), q.dtype)
