"""The paged 8-bit key/value cache on the CPU: its plain forms against the 64-bit
oracle, the table of angles, the oracle's own properties, and what the public
functions refuse (before any launch)."""

from __future__ import annotations

import math

import pytest
import torch

import kv_helpers as kv
from kairyu_amd.attention import PagedKvCache, paged_attention, rotary_table, rotate_append
from oracle import attention as oatt

PATTERNS = {
    "decode": ([1, 1, 1, 1], [1, 17, 64, 130]),
    "prompts": ([5, 33, 70], [5, 40, 131]),
    "mixed": ([1, 40, 0, 2], [50, 40, 30, 66]),
    "more rows than tokens": ([6, 3, 2], [4, 0, 2]),
}


def test_power_of_two_scales():
    for amax, scale in ((448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (1.0, 2.0**-8), (1.75, 2.0**-8), (1.76, 2.0**-7)):
        assert oatt.scale_for(amax) == scale
        assert scale * 448 >= amax > scale * 224
    assert oatt.scale_for(0.0) == oatt.scale_for(1e-12) == 2.0**-48


def test_oracle_rounding_is_the_formats():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    codes = codes[codes.isfinite()]
    assert torch.equal(oatt.to_e4m3(codes), codes)
    x = torch.randn(20000, generator=kv.gen(1)).double() * torch.exp2(torch.randint(-12, 9, (20000,), generator=kv.gen(2)))
    x = x.float().clamp(-448, 448)
    assert torch.equal(oatt.to_e4m3(x.double()), x.to(torch.float8_e4m3fn).float().double())


def test_rotary_table_of_far_positions():
    table = rotary_table(131072, 64, theta=500000.0, device="cpu")
    for position in (0, 1, 4095, 131071):
        for i in (0, 7, 31):
            angle = position * 500000.0 ** (-2 * i / 64)
            assert abs(table[position, i].item() - math.cos(angle)) <= 2.0**-24
            assert abs(table[position, 32 + i].item() - math.sin(angle)) <= 2.0**-24
    with pytest.raises(ValueError, match="even"):
        rotary_table(4, 7, device="cpu")


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("interleaved,rotary,normed", [(False, 64, False), (True, 32, True)])
def test_plain_append(pattern, interleaved, rotary, normed):
    new, total = PATTERNS[pattern]
    table, cu, lengths, rows, pages = kv.batch(new, total, 16, seed=3, pad=2)
    pool = kv.cache(pages, 2, 16, 64, seed=4)
    g = kv.gen(5)
    q, k, v = (torch.randn(rows, h, 64, generator=g).to(torch.bfloat16) for h in (4, 2, 2))
    norms = [(torch.randn(64, generator=g) * 0.1 + 1).to(torch.bfloat16) if normed else None for _ in "qk"]
    cos_sin = rotary_table(140, rotary, device="cpu")
    before = kv.values(pool)
    how = dict(interleaved=interleaved, q_norm=norms[0], k_norm=norms[1])
    out = rotate_append(q, k, v, pool, table, cu, lengths, cos_sin, **how)
    kv.check_append(out, pool, before, q, k, v, table, cu, lengths, cos_sin=cos_sin, **how)


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("how", [dict(causal=True), dict(causal=False), dict(causal=True, window=20), dict(scale=0.3)])
def test_plain_attention(pattern, how):
    new, total = PATTERNS[pattern]
    table, cu, lengths, rows, pages = kv.batch(new, total, 16, seed=6, pad=2)
    pool = kv.cache(pages, 2, 16, 64, seed=7)
    kv.stain(pool, table, lengths)
    q = torch.randn(rows, 6, 64, generator=kv.gen(8)).to(torch.float16)
    out = paged_attention(q, pool, table, cu, lengths, **how)
    kv.check_attention(out, q, pool, table, cu, lengths, pattern, **how)


def test_a_token_that_is_not_finite_is_stored_as_a_nan_key():
    table, cu, lengths, rows, pages = kv.batch([4], [4], 16, seed=9)
    pool = kv.cache(pages, 2, 16, 64, seed=10)
    kv.stain(pool, table, lengths)
    q, k, v = (torch.randn(rows, 2, 64, generator=kv.gen(11)).to(torch.bfloat16) for _ in range(3))
    v[1, 0, 5] = math.nan
    k[2, 1, 3] = math.inf
    before = kv.values(pool)
    out = rotate_append(q, k, v, pool, table, cu, lengths)
    kv.check_append(out, pool, before, q, k, v, table, cu, lengths)
    o = paged_attention(out, pool, table, cu, lengths)
    assert o[:, 0].isnan().all(-1).tolist() == [False, True, True, True]
    assert o[:, 1].isnan().all(-1).tolist() == [False, False, True, True]
    assert not o[0].isnan().any() and not o[1, 1].isnan().any()


# ------------------------------------------------------------------ refusals
def _call(**change):
    table, cu, lengths, rows, pages = kv.batch([2, 1], [20, 3], 16)
    q, k, v = (torch.zeros(rows, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    a = dict(q=q, k=k, v=v, cache=kv.cache(pages, 2, 16, 64), block_table=table, cu_rows=cu, lengths=lengths,
             cos_sin=rotary_table(32, 32, device="cpu"))
    a.update(change)
    return rotate_append(**a)


BAD_APPEND = [
    ("kv heads", dict(k=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ValueError),
    ("rows", dict(v=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), ValueError),
    ("dtype", dict(q=torch.zeros(3, 4, 64)), RuntimeError),
    ("mixed dtypes", dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), ValueError),
    ("query heads", dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), ValueError),
    ("head dim", dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), ValueError),
    ("rank", dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), ValueError),
    ("lengths' type", dict(lengths=torch.tensor([20, 3])), ValueError),
    ("bounds", dict(cu_rows=torch.tensor([0, 2, 3, 3], dtype=torch.int32)), ValueError),
    ("table", dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError),
    ("table's order", dict(block_table=torch.zeros(2, 2, dtype=torch.int32).t()), ValueError),
    ("angles' type", dict(cos_sin=torch.zeros(32, 32, dtype=torch.float64)), ValueError),
    ("rotary width", dict(cos_sin=torch.zeros(32, 24)), ValueError),
    ("rotary past the head", dict(cos_sin=torch.zeros(32, 128)), ValueError),
    ("norm", dict(q_norm=torch.zeros(32, dtype=torch.bfloat16)), ValueError),
    ("norm's type", dict(k_norm=torch.zeros(64)), ValueError),
    ("gradient", dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16, requires_grad=True)), RuntimeError),
]


@pytest.mark.parametrize("name,change,error", BAD_APPEND, ids=[b[0] for b in BAD_APPEND])
def test_append_refuses(name, change, error):
    assert _call().shape == (3, 4, 64)
    with pytest.raises(error):
        _call(**change)


def _bad_caches():
    good = kv.cache(4, 2, 16, 64)
    return {
        "page size": kv.cache(4, 2, 8, 64), "head dim": kv.cache(4, 2, 16, 96),
        "code type": good._replace(k=good.k.float()), "shapes": good._replace(v=good.v[:3]),
        "scale shape": good._replace(k_scale=good.k_scale[:, :1]), "scale type": good._replace(v_scale=good.v_scale.double()),
        "strides": good._replace(k=good.k.transpose(0, 1).contiguous().transpose(0, 1)),
        "alignment": good._replace(k=torch.zeros(good.k.numel() + 1, dtype=torch.uint8)[1:].view(good.k.shape).view(kv.E4M3)),
    }


@pytest.mark.parametrize("name", list(_bad_caches()))
def test_calls_refuse_other_caches(name):
    table, cu, lengths, rows, _ = kv.batch([2, 1], [20, 3], 16, spare=1)
    pool = _bad_caches()[name]
    q = torch.zeros(rows, 4, pool.k.shape[3], dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, cu, lengths)
    k = torch.zeros(rows, 2, pool.k.shape[3], dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        rotate_append(q, k, k, pool, table, cu, lengths)


@pytest.mark.parametrize("how", [dict(window=-1), dict(window=4, causal=False), dict(window=(1 << 30) + 1)])
def test_attention_refuses(how):
    table, cu, lengths, rows, pages = kv.batch([2], [20], 16)
    with pytest.raises(ValueError, match="window"):
        paged_attention(torch.zeros(rows, 2, 64, dtype=torch.bfloat16), kv.cache(pages, 2, 16, 64), table, cu, lengths, **how)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e40])
def test_attention_refuses_scales(scale):
    from kairyu_amd import _native

    table, cu, lengths, rows, pages = kv.batch([2], [20], 16)
    with pytest.raises(ValueError, match="scale"):
        paged_attention(torch.zeros(rows, 2, 64, dtype=torch.bfloat16), kv.cache(pages, 2, 16, 64), table, cu, lengths, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        _native.call("kq_kv_attention", None, 256, 64, 1, 1, 4, 2, 64, None, None, None, None, 1, 16, None, 1, 1, None, None, 1,
                     scale, 1, 0, None, None, 0, None)


def test_create():
    pool = PagedKvCache.create(5, 2, 64, 32, device="cpu")
    assert pool.k.shape == pool.v.shape == (5, 2, 32, 64) and pool.page_size == 32
    assert pool.k_scale.shape == (5, 2)
    with pytest.raises(ValueError, match="page size"):
        PagedKvCache.create(5, 2, 64, 48, device="cpu")
    with pytest.raises(ValueError, match="head dim"):
        PagedKvCache.create(5, 2, 80, 32, device="cpu")


def test_empty_calls():
    pool = kv.cache(3, 2, 16, 64)
    none = torch.zeros(0, dtype=torch.int32)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16)
    out = paged_attention(q, pool, torch.zeros(0, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), none)
    assert out.shape == (0, 4, 64)


def test_c_entries_refuse_bad_shapes_before_a_launch():
    from kairyu_amd import _native

    def append(**change):
        a = dict(dtype=1, rows=1, heads=4, kv_heads=2, dim=64, pages=1, page=16, ld=1, width=1, seqs=1, rotary=0)
        a.update(change)
        _native.call("kq_kv_rotate_append", None, 256, 64, None, 256, 64, None, 256, 64, a["dtype"], a["rows"], a["heads"],
                     a["kv_heads"], a["dim"], None, None, None, None, a["pages"], a["page"], None, a["ld"], a["width"], None,
                     None, a["seqs"], a.get("table"), 8, a["rotary"], 0, None, None, 1e-6, None, None)

    for change in (dict(heads=3), dict(dim=80), dict(page=48), dict(rows=-1), dict(pages=-1), dict(ld=0), dict(seqs=-1),
                   dict(table=256, rotary=24), dict(rows=1 << 25), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            append(**change)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        append(dtype=2)

    def attention(**change):
        a = dict(q_ld=256, dtype=1, heads=4, dim=64, causal=1, window=0)
        a.update(change)
        _native.call("kq_kv_attention", None, a["q_ld"], 64, a["dtype"], 1, a["heads"], 2, a["dim"], None, None, None, None, 1,
                     16, None, 1, 1, None, None, 1, 1.0, a["causal"], a["window"], None, None, 0, None)

    for change in (dict(heads=3), dict(dim=96), dict(window=-1), dict(causal=0, window=4), dict(q_ld=257)):
        with pytest.raises(ValueError):
            attention(**change)
