"""The paged 8-bit key/value cache on the GPU against the 64-bit oracle: the
append's pages, scales and codes, attention over every shape of batch, and the two
in a row as decode steps and prompts run them, captured and replayed too."""

from __future__ import annotations

import math

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import PagedKvCache, paged_attention, rotary_table, rotate_append

pytestmark = pytest.mark.gpu

BATCHES = {
    # (new rows, tokens after them) of each sequence
    "one token": ([1], [1]),
    "decode": ([1] * 9, [1, 15, 16, 17, 63, 64, 65, 300, 1029]),
    "prompts": ([5, 33, 64, 129], [5, 33, 64, 129]),
    "chunks": ([7, 100, 64], [90, 421, 1000]),
    "mixed": ([1, 130, 0, 3, 1, 0], [50, 200, 30, 66, 700, 0]),
    "more rows than tokens": ([6, 70, 2, 1], [4, 20, 0, 0]),
}
HEADS = {"8 of 2, 64": (8, 2, 64), "7 of 1, 128": (7, 1, 128), "4 of 4, 128": (4, 4, 128), "3 of 1, 256": (3, 1, 256),
         "40 of 2, 64": (40, 2, 64)}


def _case(cuda, batch, heads, page, dtype, seed=0, pad=0, stale=True, holes=()):
    new, total = BATCHES[batch] if isinstance(batch, str) else batch
    hq, hk, dim = HEADS[heads] if isinstance(heads, str) else heads
    table, cu, lengths, rows, pages = kv.batch(new, total, page, seed=seed, pad=pad, holes=holes)
    pool = kv.cache(pages, hk, page, dim, seed=seed + 1)
    if stale:
        kv.stain(pool, table, lengths)
    g = kv.gen(seed + 2)
    packed = torch.randn(rows, (hq + 2 * hk) * dim, generator=g)
    packed[:, : hq * dim] *= 2
    packed = packed.to(dtype).to(cuda)
    q, k, v = (x.unflatten(-1, (-1, dim)) for x in packed.split((hq * dim, hk * dim, hk * dim), -1))
    return q, k, v, kv.to(pool, cuda), table.to(cuda), cu.to(cuda), lengths.to(cuda)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", BATCHES)
def test_attention(cuda, batch, heads, dtype):
    page = {64: 16, 128: 64, 256: 32}[HEADS[heads][2]]
    banner(f"kv attention {batch} {heads} page {page} {dtype}")
    q, _, _, pool, table, cu, lengths = _case(cuda, batch, heads, page, dtype, seed=1, pad=2)
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, batch)


@pytest.mark.parametrize("how", [dict(causal=False), dict(window=1), dict(window=70), dict(window=513), dict(scale=0.02),
                                 dict(scale=-0.1), dict(scale=0.0)], ids=str)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("batch", ["decode", "chunks", "mixed"])
def test_attention_masks_and_pages(cuda, batch, page, how):
    banner(f"kv attention {batch} page {page} {how}")
    q, _, _, pool, table, cu, lengths = _case(cuda, batch, "8 of 2, 64", page, torch.float16, seed=4)
    out = paged_attention(q, pool, table, cu, lengths, **how)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, batch, **how)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("new", [1, 150])
def test_attention_pages_that_are_none(cuda, page, new):
    """Table entries outside the cache hold no tokens; a row left with none is zero."""
    banner(f"kv attention holes page {page} new {new}")
    batch = ([new, new, new], [600, 300, 150])
    holes = [(0, 0), (0, 1), (0, 600 // page), (1, 1), *((2, s) for s in range(-(-150 // page)))]
    q, _, _, pool, table, cu, lengths = _case(cuda, batch, "7 of 1, 128", page, torch.bfloat16, seed=6, holes=holes)
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)
    assert not out[2 * new:].any()


@pytest.mark.parametrize("new", [1, 17, 200])
def test_attention_of_nan_keys_and_extreme_scores(cuda, new):
    """A NaN key reaches the rows that see it and no other; scores of thousands, and
    pages whose value scales lie 2^40 apart, stay exact."""
    banner(f"kv attention NaN keys, new {new}")
    q, _, _, pool, table, cu, lengths = _case(cuda, ([new, new], [420, 300]), "8 of 2, 64", 16, torch.bfloat16, seed=8)
    p = table[0, 410 // 16].long()
    pool.k.view(torch.uint8)[p, 1, 410 % 16] = 0x7F
    pool.v_scale[table[1, 3].long()] = 2.0**-40
    pool.v_scale[table[1, 5].long()] = 2.0**12
    q = q * 40
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)
    seen = [420 - new + j >= 410 for j in range(new)]
    assert out[:new, 4:].isnan().all(-1).all(-1).tolist() == seen and not out[:, :4].isnan().any()


def test_attention_of_long_contexts(cuda):
    banner("kv attention long contexts")
    q, _, _, pool, table, cu, lengths = _case(cuda, ([1, 1, 2], [70001, 33000, 5]), (4, 1, 128), 64, torch.bfloat16, seed=9)
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)
    out = paged_attention(q, pool, table, cu, lengths, window=40000)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, window=40000)


def test_attention_of_a_long_prompt(cuda):
    banner("kv attention long prompt")
    q, _, _, pool, table, cu, lengths = _case(cuda, ([1500], [2100]), (4, 1, 128), 32, torch.float16, seed=10)
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)


def test_attention_is_the_same_every_time(cuda):
    """Same bits from call to call, in a wider table and next to other sequences."""
    banner("kv attention repeats")
    q, _, _, pool, table, cu, lengths = _case(cuda, "decode", "7 of 1, 128", 64, torch.bfloat16, seed=11)
    first = paged_attention(q, pool, table, cu, lengths)
    for _ in range(3):
        assert torch.equal(paged_attention(q, pool, table, cu, lengths), first)


@pytest.mark.parametrize("rows", ["packed", "odd offset", "head-major", "one head repeated"])
def test_strides(cuda, rows):
    banner(f"kv strides {rows}")
    new, total = BATCHES["mixed"]
    q, k, v, pool, table, cu, lengths = _case(cuda, "mixed", "8 of 2, 64", 32, torch.float16, seed=12, pad=1)
    if rows == "odd offset":  # 2-byte aligned rows
        q, k, v = (torch.empty(x.numel() + 3, dtype=x.dtype, device=cuda)[3:].view(x.shape).copy_(x) for x in (q, k, v))
    elif rows == "head-major":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    elif rows == "one head repeated":
        q = q[:, :1].expand(-1, 8, -1)
    wide = torch.full((len(new), table.shape[1] + 5), -1, dtype=torch.int32, device=cuda)
    wide[:, : table.shape[1]] = table
    table = wide[:, : table.shape[1]]
    before = kv.values(pool)
    cos_sin = rotary_table(1100, 64, device=cuda)
    turned = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    torch.cuda.synchronize()
    kv.check_append(turned, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(), cos_sin=cos_sin.cpu())
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)


def test_offsets_past_32_bits(cuda):
    """Pages whose codes start more than 2^32 bytes into a cache."""
    banner("kv cache past 4 GB")
    hk, dim, page = 2, 128, 64
    pages = (1 << 32) // (hk * dim * page) + 40
    pool = PagedKvCache.create(pages, hk, dim, page, device=cuda)
    table = torch.tensor([[pages - 1, 3, pages - 17], [pages - 2, pages - 9, 0]], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 180, 310], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([180, 130], dtype=torch.int32, device=cuda)
    g = kv.gen(13)
    q, k, v = (torch.randn(310, h, dim, generator=g).to(torch.bfloat16).to(cuda) for h in (4, 2, 2))
    cos_sin = rotary_table(200, dim, device=cuda)
    turned = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    torch.cuda.synchronize()
    picked = table.flatten().long()
    small = PagedKvCache(*(t.view(torch.uint8)[picked].view(t.dtype) if t.dtype == kv.E4M3 else t[picked] for t in pool))
    small_table = torch.arange(6, dtype=torch.int32).view(2, 3)
    empty = kv.values(PagedKvCache.create(6, hk, dim, page, device="cpu"))
    kv.check_append(turned, small, empty, q, k, v, small_table, cu.cpu(), lengths.cpu(), cos_sin=cos_sin.cpu())
    for rows in (slice(0, 310), slice(179, 180)):
        one = rows.start != 0
        part = cu if not one else torch.tensor([0, 1, 1], dtype=torch.int32, device=cuda)
        out = paged_attention(turned[rows], pool, table, part, lengths)
        torch.cuda.synchronize()
        kv.check_attention(out, turned[rows], small, small_table, part, lengths)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", BATCHES)
def test_append(cuda, batch, heads, dtype):
    hq, hk, dim = HEADS[heads]
    page = {64: 32, 128: 16, 256: 128}[dim]
    banner(f"kv append {batch} {heads} page {page} {dtype}")
    q, k, v, pool, table, cu, lengths = _case(cuda, batch, heads, page, dtype, seed=21, pad=3)
    before = kv.values(pool)
    cos_sin = rotary_table(1100, dim, theta=500000.0, device=cuda)
    out = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    torch.cuda.synchronize()
    kv.check_append(out, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(), batch, cos_sin=cos_sin.cpu())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("interleaved,share,normed", [(False, 2, True), (True, 1, False), (True, 4, True), (False, 0, True)])
def test_append_rotations(cuda, dim, page, interleaved, share, normed):
    """Partial and interleaved rotations, head norms, no rotation at all."""
    banner(f"kv append dim {dim} page {page} {interleaved} {share} {normed}")
    q, k, v, pool, table, cu, lengths = _case(cuda, "mixed", (6, 3, dim), page, torch.bfloat16, seed=22)
    before = kv.values(pool)
    g = kv.gen(23)
    norms = [(torch.randn(dim, generator=g) * 0.1 + 1).to(q.dtype).to(cuda) if normed else None for _ in "qk"]
    cos_sin = rotary_table(1100, dim // share, device=cuda) if share else None
    out = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin, interleaved=interleaved, q_norm=norms[0],
                        k_norm=norms[1], eps=1e-5)
    torch.cuda.synchronize()
    kv.check_append(out, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(),
                    cos_sin=None if cos_sin is None else cos_sin.cpu(), interleaved=interleaved, eps=1e-5,
                    q_norm=None if not normed else norms[0].cpu(), k_norm=None if not normed else norms[1].cpu())


def test_append_one_token_at_a_time(cuda):
    """Pages filled by single tokens of growing and shrinking size end with the scale
    that the prompt as a whole has, their codes within the roundings of the moves."""
    banner("kv append token by token")
    n, page, hk, dim = 70, 32, 2, 128
    g = kv.gen(24)
    size = torch.exp2(torch.randint(-6, 7, (n, hk, 1), generator=g).float())
    k, v = ((torch.randn(n, hk, dim, generator=g) * size).to(torch.bfloat16).to(cuda) for _ in range(2))
    q = torch.zeros(n, hk, dim, dtype=torch.bfloat16, device=cuda)
    table = torch.tensor([[4, 0, 2]], dtype=torch.int32, device=cuda)
    whole, steps = (PagedKvCache.create(5, hk, dim, page, device=cuda) for _ in range(2))

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device=cuda)

    rotate_append(q, k, v, whole, table, ints(0, n), ints(n))
    for i in range(n):
        before = kv.values(steps)
        out = rotate_append(q[i: i + 1], k[i: i + 1], v[i: i + 1], steps, table, ints(0, 1), ints(i + 1))
        if i in (0, 1, 31, 32, 69):
            torch.cuda.synchronize()
            kv.check_append(out, steps, before, q[i: i + 1], k[i: i + 1], v[i: i + 1], table.cpu(), ints(0, 1).cpu(),
                            ints(i + 1).cpu(), f"token {i}")
    torch.cuda.synchronize()
    assert torch.equal(whole.k_scale, steps.k_scale) and torch.equal(whole.v_scale, steps.v_scale)
    for a, b, s in ((whole.k, steps.k, whole.k_scale), (whole.v, steps.v, whole.v_scale)):
        a, b = a.float(), b.float()
        # the moves are exact but below 2^-6, where each may round by half of 2^-9
        assert ((a - b).abs() <= torch.where(a.abs() < 2.0**-5, 7 * 2.0**-10 + 2.0**-9, 0.0)).all()
    # appending what is there again changes nothing
    again = PagedKvCache(*(t.clone() for t in whole))
    rotate_append(q, k, v, again, table, ints(0, n), ints(n))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(again, whole))


def test_append_of_values_that_are_not_finite(cuda):
    banner("kv append NaN and infinity")
    q, k, v, pool, table, cu, lengths = _case(cuda, ([40, 1], [50, 20]), (4, 2, 128), 16, torch.float16, seed=25)
    k, v = k.clone(), v.clone()
    k[3, 0, 100], k[17, 1, 0], v[20, 0, 9], v[39, 1, 127], k[40, 0, 1] = math.nan, math.inf, -math.inf, math.nan, math.nan
    before = kv.values(pool)
    cos_sin = rotary_table(45, 64, device=cuda)  # and positions past the table
    out = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    torch.cuda.synchronize()
    kv.check_append(out, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(), cos_sin=cos_sin.cpu())


def test_append_leaves_everything_else(cuda):
    """Pages of other sequences, slots past the end, padding rows, positions past the
    table and entries that are no page."""
    banner("kv append leaves the rest")
    q, k, v, pool, table, cu, lengths = _case(cuda, ([30, 1, 20], [70, 64, 90]), (4, 2, 64), 16, torch.bfloat16, seed=26,
                                              pad=4, holes=[(0, 3), (2, 5)])
    table = table[:, :5]  # sequence 2's last positions are past it
    before, codes = kv.values(pool), [t.clone() for t in pool]
    rotate_append(q, k, v, pool, table, cu, lengths)
    torch.cuda.synchronize()
    out = rotate_append(q, k, v, pool, table, cu, lengths)  # (and once more: the same)
    torch.cuda.synchronize()
    kv.check_append(out, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu())
    written = {int(table[s, t // 16]) * 16 + t % 16 for s, (n, total) in enumerate(((30, 70), (1, 64), (20, 90)))
               for t in range((total - n) // 16 * 16, min(total, 80)) if 0 <= int(table[s, t // 16]) < pool.k.shape[0]}
    left = torch.ones(pool.k.shape[0] * 16, dtype=torch.bool)
    left[list(written)] = False
    for now, was in zip(pool[:2], codes[:2]):
        x, y = (t.cpu().view(torch.uint8).transpose(1, 2).reshape(-1, 2, 64)[left] for t in (now, was))
        assert torch.equal(x, y)


# ------------------------------------------------------------------ together
def _step(x, pool, table, cu, lengths, cos_sin, hq, hk, dim):
    q, k, v = (t.unflatten(-1, (-1, dim)) for t in x.split((hq * dim, hk * dim, hk * dim), -1))
    q = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    return paged_attention(q, pool, table, cu, lengths)


def test_prompt_then_decode_steps(cuda):
    """A prompt in chunks, then tokens one by one: every step against the oracle on the
    cache as it is, and the last against attention in 64 bits over the unquantized keys
    and values, within e4m3's rounding."""
    banner("kv prompt then decode")
    hq, hk, dim, page, n = 8, 2, 128, 32, 150
    g = kv.gen(31)
    x = torch.randn(n, (hq + 2 * hk) * dim, generator=g).to(torch.bfloat16).to(cuda)
    pool = PagedKvCache.create(8, hk, dim, page, device=cuda)
    table = torch.tensor([[6, 1, 3, 0, 7]], dtype=torch.int32, device=cuda)
    cos_sin = rotary_table(n, dim, device=cuda)
    at = 0
    for size in (100, 33, *[1] * 17):
        cu = torch.tensor([0, size], dtype=torch.int32, device=cuda)
        length = torch.tensor([at + size], dtype=torch.int32, device=cuda)
        out = _step(x[at: at + size], pool, table, cu, length, cos_sin, hq, hk, dim)
        at += size
    torch.cuda.synchronize()
    rot = kv.oatt.rotate
    q, k, v = (t.unflatten(-1, (-1, dim)).cpu().double() for t in x.split((hq * dim, hk * dim, hk * dim), -1))
    k = torch.stack([rot(k[t], cos_sin.cpu(), t, False) for t in range(n)])
    z = rot(q[-1], cos_sin.cpu(), n - 1, False)
    want = torch.stack([torch.softmax(k[:, h // 4] @ z[h] * dim**-0.5, 0) @ v[:, h // 4] for h in range(hq)])
    got = out[0].cpu().double()
    # independent roundings of up to 2^-4 (rms 2^-4 / sqrt 3 at the most) of every key element move a score by
    # less than 2^-4 |q| |k| dim^-1/2 / sqrt(dim) ~ 2^-4, a weight by that share, and values likewise
    assert ((got - want).norm() / want.norm()).item() < 2 * 2.0**-4
    for label, parts in (("q", z), ("v", v)):
        assert parts.isfinite().all(), label


def test_captured_step_replays_for_other_lengths(cuda):
    """One decode step captured once: replays with other rows, lengths and tables, with
    eager work between them, equal the eager step bit for bit; the graph's padding rows
    store nothing."""
    banner("kv captured step")
    hq, hk, dim, page, seqs = 8, 2, 64, 16, 6
    g = kv.gen(32)
    pools = [PagedKvCache.create(60, hk, dim, page, device=cuda) for _ in range(2)]
    cos_sin = rotary_table(200, dim, device=cuda)
    x = torch.zeros(seqs, (hq + 2 * hk) * dim, dtype=torch.bfloat16, device=cuda)
    table = torch.full((seqs, 10), -1, dtype=torch.int32, device=cuda)
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device=cuda)
    lengths = torch.zeros(seqs, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(x, pools[0], table, cu, lengths, cos_sin, hq, hk, dim)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(x, pools[0], table, cu, lengths, cos_sin, hq, hk, dim)
    order = torch.randperm(60, generator=g).to(torch.int32)
    held = [0] * seqs
    for i, live in enumerate((6, 5, 2, 6, 1, 4)):
        x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
        table.copy_(order.view(seqs, 10))
        for s in range(live):
            held[s] += 1
        lengths.copy_(torch.tensor([h if s < live else 0 for s, h in enumerate(held)], dtype=torch.int32))
        cu.copy_(torch.tensor([min(s, live) for s in range(seqs + 1)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = _step(x, pools[1], table, cu, lengths, cos_sin, hq, hk, dim)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager), i
        assert not captured[live:].any()
        for a, b in zip(*pools):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        kv.check_attention(captured, _turned(x, lengths, cu, cos_sin, hq, dim), pools[0], table, cu, lengths, f"replay {i}")


def _turned(x, lengths, cu, cos_sin, hq, dim):
    """The rotated queries of a decode step, by the oracle, rounded as stored."""
    q = x[:, : hq * dim].cpu().unflatten(-1, (-1, dim)).double()
    out = torch.zeros_like(q)
    for s, n in enumerate(lengths.tolist()):
        if int(cu[s + 1]) > int(cu[s]):
            out[int(cu[s])] = kv.oatt.rotate(q[int(cu[s])], cos_sin.cpu(), n - 1, False)
    return out.to(torch.bfloat16)


def test_calls_on_two_streams(cuda):
    """Steps of two batches on two streams at once, on one cache's different pages."""
    banner("kv two streams")
    parts = [_case(cuda, ([1] * 20, [300 + 7 * s for s in range(20)]), (16, 2, 128), 64, torch.bfloat16, seed=40 + i)
             for i in range(2)]
    want = [paged_attention(p[0], *p[3:]) for p in parts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    got = [[] for _ in parts]
    for _ in range(6):
        for stream, part, out in zip(streams, parts, got):
            with torch.cuda.stream(stream):
                out.append(paged_attention(part[0], *part[3:]))
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(torch.equal(o, w) for o in out)


def test_no_pages_or_sequences(cuda):
    banner("kv nothing to do")
    pool = PagedKvCache.create(2, 2, 64, 16, device=cuda)
    q = torch.randn(3, 4, 64, device=cuda).to(torch.bfloat16)
    k = torch.randn(3, 2, 64, device=cuda).to(torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    table, cu = torch.zeros(0, 1, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    assert not rotate_append(q, k, k, pool, table, cu, none).any()
    assert not paged_attention(q, pool, table, cu, none).any()
    assert paged_attention(q[:0], pool, table, cu, none).shape == (0, 4, 64)
    # sequences whose table has no columns hold no tokens
    seq = torch.tensor([3], dtype=torch.int32, device=cuda)
    bounds = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    empty = torch.zeros(1, 0, dtype=torch.int32, device=cuda)
    rotate_append(q, k, k, pool, empty, bounds, seq)
    assert not paged_attention(q, pool, empty, bounds, seq).any()
    torch.cuda.synchronize()
    assert not pool.k.view(torch.uint8).any()


@pytest.mark.parametrize("heads", ["8 of 2, 64", "7 of 1, 128", "3 of 1, 256"])
@pytest.mark.parametrize("new,total", [([1, 1], [200, 1300]), ([120, 200], [200, 900]), ([300], [4200])])
def test_attention_over_pages_of_small_values(cuda, heads, new, total):
    """Pages whose values are zero or far smaller than the others' count in the
    denominator as much as any."""
    banner(f"kv attention small values {heads} {new} {total}")
    q, _, _, pool, table, cu, lengths = _case(cuda, (new, total), heads, 32, torch.bfloat16, seed=41)
    g = kv.gen(42)
    pick = torch.randint(0, 4, (pool.k.shape[0],), generator=g).to(cuda)
    pool.v.view(torch.uint8)[pick == 0] = 0
    pool.v_scale[pick == 0] = 2.0**-48
    pool.v_scale[pick == 1] *= 2.0**-18
    out = paged_attention(q * 0.25, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q * 0.25, pool, table, cu, lengths)


MANY = {  # more sequences than a wave has lanes
    "decode": ([1] * 131, [1 + 37 * s % 211 for s in range(131)]),
    "padded decode": ([1] * 70 + [0] * 60, [40 + s for s in range(70)] + [0] * 60),
    "mixed": ([1, 40, 0, 3, 17] * 14, [90, 60, 33, 3, 200] * 14),
}


@pytest.mark.parametrize("heads", ["8 of 2, 64", "7 of 1, 128"])
@pytest.mark.parametrize("batch", MANY)
def test_many_sequences(cuda, batch, heads):
    banner(f"kv many sequences {batch} {heads}")
    q, k, v, pool, table, cu, lengths = _case(cuda, MANY[batch], heads, 16, torch.bfloat16, seed=43, pad=5)
    before = kv.values(pool)
    cos_sin = rotary_table(250, q.shape[2], device=cuda)
    turned = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin)
    torch.cuda.synchronize()
    kv.check_append(turned, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(), batch, cos_sin=cos_sin.cpu())
    out = paged_attention(turned, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, turned, pool, table, cu, lengths, batch)


@pytest.mark.parametrize("slots", [64, 65])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 70]])
def test_attention_around_one_block_of_tokens(cuda, slots, new):
    """Tables of 1024 tokens, where no sequence's tokens are split, and one page more."""
    banner(f"kv attention {slots} pages, new {new}")
    q, _, _, pool, table, cu, lengths = _case(cuda, (new, [slots * 16, 1017, 100]), "8 of 2, 64", 16, torch.float16, seed=44)
    assert table.shape[1] == slots
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)


@pytest.mark.parametrize("heads", ["8 of 2, 64", "4 of 4, 128", "3 of 1, 256"])
@pytest.mark.parametrize("how", [dict(), dict(causal=False), dict(window=1500)], ids=str)
def test_attention_of_few_rows_over_many_tokens(cuda, heads, how):
    """Tiles whose tokens are cut into parts."""
    banner(f"kv attention cut tokens {heads} {how}")
    q, _, _, pool, table, cu, lengths = _case(cuda, ([90, 1], [5000, 4000]), heads, 64, torch.bfloat16, seed=45, pad=1)
    out = paged_attention(q, pool, table, cu, lengths, **how)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, **how)


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("how", [dict(), dict(window=40), dict(causal=False)], ids=str)
@pytest.mark.parametrize("past", [30, 100_000, 2**31 - 1])
def test_lengths_past_the_table(cuda, past, how, new):
    """Only the tokens that the table has room for are there."""
    banner(f"kv lengths past the table {past} {how} new {new}")
    q, k, v, pool, table, cu, lengths = _case(cuda, ([new, new], [96, 60]), "8 of 2, 64", 16, torch.bfloat16, seed=46)
    lengths[0] = min(96 + past, 2**31 - 1)
    before = kv.values(pool)
    turned = rotate_append(q, k, v, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_append(turned, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu())
    out = paged_attention(q, pool, table, cu, lengths, **how)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, **how)


def test_row_bounds_outside_the_rows(cuda):
    """Rows before the first bound are padding, bounds past the rows end with them."""
    banner("kv row bounds")
    q, k, v, pool, table, _, lengths = _case(cuda, ([4, 1, 30], [40, 33, 70]), "8 of 2, 64", 32, torch.float16, seed=47)
    cu = torch.tensor([2, 6, 7, 500], dtype=torch.int32, device=cuda)
    within = cu.clamp(max=35)
    before = kv.values(pool)
    turned = rotate_append(q, k, v, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_append(turned, pool, before, q, k, v, table.cpu(), within.cpu(), lengths.cpu())
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, within, lengths)
    assert not out[:2].any() and not turned[:2].any()


@pytest.mark.parametrize("window", [900, 1024, 1700, 2100])
@pytest.mark.parametrize("new", [[1] * 33, [2, 1, 60] * 11])
def test_windows_of_many_sequences(cuda, new, window):
    """Windows that one workgroup reads whole, and larger ones."""
    banner(f"kv attention many windows {window} new {max(new)}")
    total = [60 + 97 * s * s % 2600 for s in range(33)]
    q, _, _, pool, table, cu, lengths = _case(cuda, (new, total), (8, 8, 64), 32, torch.float16, seed=48, pad=1)
    out = paged_attention(q, pool, table, cu, lengths, window=window)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, window=window)


@pytest.mark.parametrize("batch", [([1] * 5, [900, 20, 333, 64, 1]), ([20] + [0] * 23, [700] + [30] * 23), ([3, 40], [60, 500])])
@pytest.mark.parametrize("heads", [(200, 1, 64), (48, 2, 128)])
def test_attention_of_large_groups(cuda, batch, heads):
    """More query heads to a kv head than a tile has rows; one sequence with all the rows."""
    banner(f"kv attention large groups {batch} {heads}")
    q, _, _, pool, table, cu, lengths = _case(cuda, batch, heads, 32, torch.bfloat16, seed=49, pad=1)
    out = paged_attention(q, pool, table, cu, lengths)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths)


def test_misaligned_head_norms(cuda):
    banner("kv append misaligned head norms")
    q, k, v, pool, table, cu, lengths = _case(cuda, "mixed", (6, 3, 64), 16, torch.bfloat16, seed=50)
    g = kv.gen(51)
    wide = (torch.randn(2 * 64 + 1, generator=g) * 0.1 + 1).to(q.dtype).to(cuda)
    norms = [wide[1:65], wide[:128:2]]  # 2-byte aligned, and not contiguous
    before = kv.values(pool)
    out = rotate_append(q, k, v, pool, table, cu, lengths, q_norm=norms[0], k_norm=norms[1])
    torch.cuda.synchronize()
    kv.check_append(out, pool, before, q, k, v, table.cpu(), cu.cpu(), lengths.cpu(), q_norm=norms[0].cpu(), k_norm=norms[1].cpu())


def test_captured_batches_replay_beside_each_other(cuda):
    """Two graphs, prompts whose tokens are cut and ragged single tokens, replayed in turn on
    two streams for changing lengths: each equals the eager call bit for bit."""
    banner("kv captured prompts and decode")
    parts = [_case(cuda, ([90, 1], [5000, 4000]), "4 of 4, 128", 64, torch.bfloat16, seed=52, pad=2),
             _case(cuda, ([1] * 9, [3000 - 300 * s for s in range(9)]), "7 of 1, 128", 32, torch.float16, seed=53)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in parts], [], []
    for stream, (q, _, _, pool, table, cu, lengths) in zip(streams, parts):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            paged_attention(q, pool, table, cu, lengths)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, pool, table, cu, lengths))
        graphs.append(graph)
    full = [p[6].clone() for p in parts]
    for less in (0, 700, 33, 1500, 0):
        for part, most in zip(parts, full):
            part[6].copy_((most - less).clamp(min=1))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for part, out in zip(parts, outs):
            assert torch.equal(out, paged_attention(part[0], *part[3:])), less
            torch.cuda.synchronize()


BESIDE = {  # mostly single tokens, so that they and the prompts' tiles are two launches
    "short": ([1] * 40 + [45, 3, 9, 130], [30 + 19 * s for s in range(40)] + [300, 900, 9, 130]),
    "joined": ([1] * 40 + [45, 3, 9, 130], [30 + 37 * s for s in range(40)] + [300, 1900, 9, 130]),
    "long": ([1] * 5 + [50, 2, 70, 90], [2600, 1, 700, 2049, 64, 900, 2300, 70, 1700]),
    "many": ([1, 1, 1, 1, 1, 1, 8, 36] * 10, [700, 33, 1500, 64, 65, 1024, 1100, 400] * 10),
}


@pytest.mark.parametrize("how", [dict(), dict(causal=False), dict(window=300)], ids=str)
@pytest.mark.parametrize("heads", ["8 of 2, 64", "7 of 1, 128", "3 of 1, 256"])
@pytest.mark.parametrize("batch", BESIDE)
def test_single_tokens_beside_prompts(cuda, batch, heads, how):
    banner(f"kv attention beside {batch} {heads} {how}")
    q, _, _, pool, table, cu, lengths = _case(cuda, BESIDE[batch], heads, 32, torch.bfloat16, seed=54, pad=2)
    out = paged_attention(q, pool, table, cu, lengths, **how)
    torch.cuda.synchronize()
    kv.check_attention(out, q, pool, table, cu, lengths, batch, **how)
