"""Quantized rows of the block norm in the library's GEMM entries that take rows and
scales (``kq_w8a8_i8_gemm``, ``kq_block_fp8_gemm``), against 64 bits."""

from __future__ import annotations

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd import _native
from kairyu_amd.norm import block_norm
from kairyu_amd.quant.int8 import quantize_int8_weight
from test_block_norm import make
from test_gpu_block_norm import _on

pytestmark = pytest.mark.gpu

N, K = 512, 1024


@pytest.mark.parametrize("m", [1, 20, 200])
def test_int8_rows(cuda, m):
    banner(f"block norm into the INT8 GEMM, {m}")
    x, res, weight, how = _on(cuda, *make((m,), K, torch.bfloat16, 31))
    _, rows, scales = block_norm(x, res, weight, quantize="int8", **how)
    w, ws = quantize_int8_weight(torch.randn(N, K, generator=kv.gen(32)))
    w, ws = w.to(cuda), ws.reshape(-1).float().to(cuda)
    out = torch.empty(m, N, device=cuda, dtype=torch.bfloat16)
    need = int(_native.library().kq_w8a8_workspace_size(m, N, K))
    scratch = torch.empty(max(need, 1), device=cuda, dtype=torch.uint8)
    _native.call("kq_w8a8_i8_gemm", rows.data_ptr(), scales.data_ptr(), w.data_ptr(), ws.data_ptr(), None, -1, out.data_ptr(),
                 _native.dtype_code(out.dtype), None, m, N, K, scratch.data_ptr(), need, _native.stream_handle(cuda))
    torch.cuda.synchronize()
    want = (rows.cpu().double() @ w.cpu().double().t()) * scales.cpu().double() * ws.cpu().double()
    # exact sums, two products in fp32, one rounding to bf16
    assert ((out.cpu().double() - want).abs() <= (2.0**-8 + 2.0**-20) * want.abs()).all()


@pytest.mark.parametrize("m", [1, 20, 200])
def test_block_rows(cuda, m):
    banner(f"block norm into the block FP8 GEMM, {m}")
    x, res, weight, how = _on(cuda, *make((m,), K, torch.bfloat16, 33))
    _, rows, scales = block_norm(x, res, weight, quantize="fp8_block", **how)
    g = kv.gen(34)
    w = (torch.randn(N, K, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).to(cuda)
    ws = (torch.rand(N // 128, K // 128, generator=g) * 1e-3 + 1e-4).to(cuda)
    out = torch.empty(m, N, device=cuda, dtype=torch.bfloat16)
    _native.call("kq_block_fp8_gemm", rows.data_ptr(), scales.data_ptr(), w.data_ptr(), ws.data_ptr(), None, -1, out.data_ptr(),
                 _native.dtype_code(out.dtype), m, N, K, _native.stream_handle(cuda))
    torch.cuda.synchronize()
    y = rows.float().cpu().double() * scales.cpu().double().repeat_interleave(128, 1)
    full = w.float().cpu().double() * ws.cpu().double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    want, terms = y @ full.t(), y.abs() @ full.abs().t()
    # sums of the matrix cores in fp32, as for the FP8 rows
    assert ((out.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + K * 2.0**-22 * terms).all()
