"""The norms around a block on the GPU against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.norm import block_norm
from test_block_norm import check, make

pytestmark = pytest.mark.gpu


def _on(cuda, x, res, weight, how):
    move = lambda t: t.to(cuda) if torch.is_tensor(t) else t  # noqa: E731
    return move(x), move(res), move(weight), {k: move(v) for k, v in how.items()}


@pytest.mark.parametrize("quantize", [None, "fp8", "int8", "fp8_block"])
@pytest.mark.parametrize("rows,hidden", [(1, 4096), (1, 1), (3, 200), (2, 129), (5, 2048), (300, 3584), (257, 8192), (2, 8200),
                                         (2, 32768), (300, 12288), (4, 77)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_shapes(cuda, rows, hidden, quantize, dtype):
    banner(f"block norm {rows} x {hidden} {quantize} {dtype}")
    x, res, weight, how = _on(cuda, *make((rows,), hidden, dtype, 3))
    how |= dict(residual_scale=0.7)
    out = block_norm(x, res, weight, quantize=quantize, **how)
    torch.cuda.synchronize()
    check(out, x, res, weight, how, quantize, f"{rows}x{hidden}")


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "channels", "rows"])
@pytest.mark.parametrize("residual", ["none", "same", "fp32"])
@pytest.mark.parametrize("quantize", [None, "fp8_block"])
def test_forms(cuda, post, gate, residual, quantize):
    banner(f"block norm {post} {gate} {residual}")
    x, res, weight, how = _on(cuda, *make((2, 9), 640, torch.bfloat16, 4, post, gate, residual))
    how |= dict(residual_scale=-1.25, unit_offset=True, eps=1e-3)
    out = block_norm(x, res, weight, quantize=quantize, **how)
    torch.cuda.synchronize()
    check(out, x, res, weight, how, quantize)


@pytest.mark.parametrize("quantize", [None, "fp8", "fp8_block"])
def test_strided_and_misaligned_rows(cuda, quantize):
    banner(f"block norm strides {quantize}")
    x, res, weight, how = _on(cuda, *make((7,), 384, torch.float16, 5, residual="fp32"))
    want = block_norm(x, res, weight, quantize=quantize, **how)
    wide = torch.zeros(7, 800, dtype=x.dtype, device=cuda)
    wide[:, 8:392] = x
    odd = torch.zeros(7, 801, dtype=x.dtype, device=cuda)
    odd[:, 3:387] = x
    flipped = x.t().contiguous().t()
    spread = torch.zeros(7, 1000, dtype=torch.float32, device=cuda)
    spread[:, 5:389] = res
    for rows in (wide[:, 8:392], odd[:, 3:387], flipped):
        for stream in (res, spread[:, 5:389]):
            got = block_norm(rows, stream, weight, quantize=quantize, **how)
            torch.cuda.synchronize()
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    gate = torch.zeros(7, 500, dtype=x.dtype, device=cuda)
    gate[:, 2:386] = how["gate"]
    got = block_norm(x, res, weight, quantize=quantize, post_weight=how["post_weight"], gate=gate[:, 2:386])
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    # one row repeated
    one = x[:1].expand(7, -1)
    got = block_norm(one, None, weight, quantize=quantize)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, block_norm(one.contiguous(), None, weight, quantize=quantize)))


@pytest.mark.parametrize("quantize", [None, "fp8", "fp8_block"])
def test_rows_of_zeros_and_values_that_are_not_finite(cuda, quantize):
    """Zero rows stay zero; a row with NaN or infinity is its own affair."""
    banner(f"block norm special rows {quantize}")
    x, res, weight, how = _on(cuda, *make((5,), 512, torch.bfloat16, 6, gate="none"))
    want = block_norm(x, res, weight, quantize=quantize, **how)
    x, res = x.clone(), res.clone()
    x[0], res[0] = 0, 0
    x[2, 7] = float("nan")
    res[3, 500] = float("inf")
    got = block_norm(x, res, weight, quantize=quantize, **how)
    torch.cuda.synchronize()
    assert not got[0][0].float().any() and not got[1][0].float().any()
    assert got[0][2].isnan().all() and got[1][2].float().isnan().all()
    for a, b in zip(got, want):
        assert torch.equal(a[1].float(), b[1].float()) and torch.equal(a[4].float(), b[4].float())


def test_rows_feed_the_quantized_projections(cuda):
    """A quantized row times its scales is the 16-bit row within the two's roundings,
    and the GEMM takes rows and scales as its own quantizer's."""
    from kairyu_amd import _native
    from kairyu_amd.quant.fp8 import quantize_fp8

    banner("block norm into the FP8 GEMM")
    m, k, n = 64, 1024, 512
    x, res, weight, how = _on(cuda, *make((m,), k, torch.bfloat16, 7))
    _, y = block_norm(x, res, weight, **how)
    _, yq, scales = block_norm(x, res, weight, quantize="fp8", **how)
    far = (yq.float() * scales - y.float()).abs()
    assert (far <= (2.0**-4 + 2.0**-8) * 1.01 * y.float().abs() + 2.0**-10 * 1.01 * scales).all()
    w, ws = quantize_fp8(torch.randn(n, k, generator=kv.gen(8)) * 0.02, per_channel=True)
    w, ws = w.to(cuda), ws.reshape(-1).float().to(cuda)
    out = torch.empty(m, n, device=cuda, dtype=torch.bfloat16)
    _native.call("kq_w8a8_fp8_gemm", yq.data_ptr(), scales.data_ptr(), w.data_ptr(), ws.data_ptr(), 1, None, -1, out.data_ptr(),
                 _native.dtype_code(out.dtype), m, n, k, None, 0, _native.stream_handle(cuda))
    want = (yq.float().double() * scales.double()).cpu() @ (w.float().double().cpu() * ws.double().cpu()[:, None]).t()
    terms = (yq.float().double().abs() * scales.double()).cpu() @ (w.float().double().abs().cpu() * ws.double().cpu()[:, None]).t()
    assert ((out.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + k * 2.0**-22 * terms).all()


def test_captured_norm_replays(cuda):
    banner("block norm captured")
    x, res, weight, how = _on(cuda, *make((33,), 2048, torch.bfloat16, 9))
    static = x.clone()
    block_norm(static, res, weight, quantize="fp8", **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block_norm(static, res, weight, quantize="fp8", **how)
    for i in range(4):
        static.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = block_norm(static, res, weight, quantize="fp8", **how)
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(captured, eager)), i
