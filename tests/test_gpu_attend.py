"""``QuantLinearPack.attend``: the projections, the append to a paged 8-bit cache and
attention of a decoder layer, and the norms around it, run together as a layer runs
them: prompts, decode steps, and a step captured into a graph."""

from __future__ import annotations

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import PagedKvCache, paged_attention, rotary_table, rotate_append
from kairyu_amd.norm import block_norm
from kairyu_amd.quant.packed import QuantLinearPack
from test_block_norm import check as check_norm
from test_gpu_packed import _fp8, _int8
from test_gpu_w4a16 import _awq_module, _gptq_module

pytestmark = pytest.mark.gpu

K, HQ, HK, DIM, PAGE = 512, 8, 2, 64, 16
WIDTHS = (HQ * DIM, HK * DIM, HK * DIM)


def _modules(scheme, cuda):
    make = {"fp8": _fp8, "int8": _int8, "awq": lambda k, n, s: _awq_module(k, n, group=128, seed=s),
            "gptq": lambda k, n, s: _gptq_module(k, n, group=128, seed=s)}[scheme]
    return [make(K, n, 50 + i).to(cuda) for i, n in enumerate(WIDTHS)]


def _ints(cuda, *x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("scheme", ["fp8", "int8", "awq", "gptq"])
def test_attend_is_the_three_in_a_row(cuda, scheme):
    banner(f"attend {scheme}")
    mods = _modules(scheme, cuda)
    dtype = torch.float16 if scheme in ("awq", "gptq") else torch.bfloat16
    pack = QuantLinearPack.create(mods)
    assert pack is not None
    pools = [PagedKvCache.create(20, HK, DIM, PAGE, device=cuda) for _ in range(2)]
    cos_sin = rotary_table(100, DIM, device=cuda)
    norms = [(torch.randn(DIM, generator=kv.gen(i)) * 0.1 + 1).to(dtype).to(cuda) for i in range(2)]
    table = torch.randperm(20, generator=kv.gen(3)).to(torch.int32)[:12].view(3, 4).to(cuda)
    held = [0, 0, 0]
    for new in ([20, 7, 33], [1, 1, 1], [1, 0, 1], [5, 17, 1]):
        held = [h + n for h, n in zip(held, new)]
        cu, lengths = _ints(cuda, 0, new[0], sum(new[:2]), sum(new)), _ints(cuda, *held)
        x = torch.randn(sum(new), K, generator=kv.gen(sum(held))).to(dtype).to(cuda)
        out = pack.attend(x, pools[0], table, cu, lengths, cos_sin, q_norm=norms[0], k_norm=norms[1])
        q, k, v = (t.unflatten(-1, (-1, DIM)) for t in pack(x))
        q = rotate_append(q, k, v, pools[1], table, cu, lengths, cos_sin, q_norm=norms[0], k_norm=norms[1])
        want = paged_attention(q, pools[1], table, cu, lengths)
        torch.cuda.synchronize()
        assert out.shape == (sum(new), HQ * DIM)
        assert torch.equal(out, want.flatten(1))
        for a, b in zip(*pools):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        kv.check_attention(want, q, pools[0], table, cu, lengths, f"{scheme} {new}")


def test_attend_refuses(cuda):
    banner("attend refusals")
    mods = _modules("int8", cuda)
    pack, pair = QuantLinearPack.create(mods), QuantLinearPack.create(_modules("int8", cuda)[1:])
    x = torch.zeros(2, K, dtype=torch.bfloat16, device=cuda)
    args = (_ints(cuda, 0, 1).view(1, 2), _ints(cuda, 0, 2), _ints(cuda, 2))
    pool = PagedKvCache.create(2, HK, DIM, PAGE, device=cuda)
    for bad_pack, bad_pool in ((pair, pool), (pack, PagedKvCache.create(2, 4, DIM, PAGE, device=cuda)),
                               (pack, PagedKvCache.create(2, HK, 128, PAGE, device=cuda))):
        with pytest.raises(ValueError, match="attend needs"):
            bad_pack.attend(x, bad_pool, *args)
    with pytest.raises(RuntimeError, match="gradient"):
        pack.attend(x.clone().requires_grad_(), pool, *args)
    with pytest.raises(RuntimeError, match="must be on"):
        pack.attend(x, pool, *(a.cpu() for a in args))
    assert pack.attend(x[None], pool, *args).shape == (1, 2, HQ * DIM)


def _layer(x, residual, pack, o_proj, pool, table, cu, lengths, cos_sin, w):
    """Attention half of a decoder layer with norms before and after it."""
    attended = pack.attend(x, pool, table, cu, lengths, cos_sin)
    return block_norm(o_proj(attended), residual, w[0], post_weight=w[1], residual_scale=0.5)


def test_layer_captured_and_replayed(cuda):
    """Norm, packed projection, append, attention, output projection and norms of a
    decode step in one graph: replays equal the eager step on a second cache."""
    banner("decoder layer step captured")
    pack = QuantLinearPack.create(_modules("fp8", cuda))
    o_proj = _fp8(HQ * DIM, K, 60).to(cuda)
    cos_sin = rotary_table(100, DIM, device=cuda)
    w = [(torch.randn(K, generator=kv.gen(61 + i)) * 0.1 + 1).to(torch.bfloat16).to(cuda) for i in range(2)]
    pools = [PagedKvCache.create(24, HK, DIM, PAGE, device=cuda) for _ in range(2)]
    seqs = 4
    table = torch.randperm(24, generator=kv.gen(62)).to(torch.int32).view(4, 6).to(cuda)
    x, residual = (torch.zeros(seqs, K, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    cu, lengths = _ints(cuda, *range(seqs + 1)), _ints(cuda, *[1] * seqs)
    args = (table, cu, lengths, cos_sin, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(x, residual, pack, o_proj, pools[0], *args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _layer(x, residual, pack, o_proj, pools[0], *args)
    g = kv.gen(63)
    for step in range(1, 41):
        x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
        residual.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
        lengths.fill_(step)
        graph.replay()
        torch.cuda.synchronize()
        eager = _layer(x, residual, pack, o_proj, pools[1], *args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), step
    attended = pack.attend(x, pools[1], *args[:4])
    block = o_proj(attended)
    out = block_norm(block, residual, w[0], post_weight=w[1], residual_scale=0.5)
    check_norm(out, block, residual, w[0], dict(post_weight=w[1], residual_scale=0.5))
    assert all(torch.equal(a, b) for a, b in zip(out, captured))
