"""The norms around a block on the CPU: the plain form against the 64-bit oracle,
and refusals."""

from __future__ import annotations

import pytest
import torch

import kv_helpers as kv
from kairyu_amd.norm import block_norm
from oracle import attention as oatt


def make(rows, hidden, dtype, seed=0, post=True, gate="rows", residual="same"):
    g = kv.gen(seed)
    x = (torch.randn(*rows, hidden, generator=g) * (1 + 9 * (torch.randn(hidden, generator=g) > 2))).to(dtype)
    res = None if residual == "none" else (torch.randn(*rows, hidden, generator=g) * 4).to(
        torch.float32 if residual == "fp32" else dtype)
    weight, after = ((torch.randn(hidden, generator=g) * 0.1 + 1).to(dtype) for _ in range(2))
    gates = {"none": None, "channels": torch.randn(hidden, generator=g).to(dtype),
             "rows": torch.randn(*rows, hidden, generator=g).to(dtype)}[gate]
    return x, res, weight, dict(post_weight=after if post else None, gate=gates)


def check(out, x, res, weight, how, quantize=None, label=""):
    """Outputs of a call against the oracle."""

    names = {"post_weight": "post"}
    r, y, r_err, y_err = oatt.block_norm(x.cpu(), None if res is None else res.cpu(), weight.cpu(), **{
        names.get(k, k): v.cpu() if torch.is_tensor(v) else v for k, v in how.items()})
    kv.assert_within(out[0], r, r_err, out[0].dtype, label + " r")
    if quantize is None:
        kv.assert_within(out[1], y, y_err, out[1].dtype, label + " y")
        return
    most = 127.0 if quantize == "int8" else 448.0
    hidden = y.shape[-1]
    wide = hidden if quantize != "fp8_block" else 128
    blocks = -(-hidden // wide)
    scale = out[2].cpu().double().reshape(*y.shape[:-1], blocks)
    amax = torch.stack([y[..., wide * i: wide * (i + 1)].abs().amax(-1) for i in range(blocks)], -1)
    err = torch.stack([y_err[..., wide * i: wide * (i + 1)].amax(-1) for i in range(blocks)], -1)
    assert ((scale - amax.clamp(min=1e-12) / most).abs() <= (err + 4 * oatt.U32 * amax) / most + 1e-30).all(), f"{label}: scales"
    # a code's value: half a step of its format, and the noise of y and of its scale
    full = scale.repeat_interleave(wide, -1)[..., :hidden]
    got = out[1].cpu().double() * full
    step = 0.5 * full if quantize == "int8" else 2.0**-4 * y.abs() + 2.0**-10 * full
    noise = 2 * y_err + 2 * err.repeat_interleave(wide, -1)[..., :hidden] + 8 * oatt.U32 * y.abs()
    assert ((got - y).abs() <= step + noise * 1.1).all(), f"{label}: codes"


@pytest.mark.parametrize("quantize", [None, "fp8", "int8", "fp8_block"])
@pytest.mark.parametrize("rows,hidden", [((1,), 8), ((3, 2), 200), ((5,), 1)])
@pytest.mark.parametrize("residual,gate,post", [("same", "rows", True), ("fp32", "channels", False), ("none", "none", True)])
def test_plain_form(quantize, rows, hidden, residual, gate, post):
    x, res, weight, how = make(rows, hidden, torch.bfloat16, 1, post, gate, residual)
    how |= dict(residual_scale=0.5, unit_offset=True)
    check(block_norm(x, res, weight, quantize=quantize, **how), x, res, weight, how, quantize)


def test_refusals():
    x, res, weight, _ = make((4,), 64, torch.float16, 2)
    good = block_norm(x, res, weight)
    assert good[0].shape == good[1].shape == (4, 64)
    for bad, error in (
            (dict(x=x.float()), RuntimeError), (dict(weight=weight[:32]), ValueError), (dict(weight=weight.bfloat16()), ValueError),
            (dict(residual=res[:3]), ValueError), (dict(residual=res.bfloat16()), ValueError),
            (dict(gate=res[:1]), ValueError), (dict(post_weight=res), ValueError), (dict(quantize="int4"), ValueError),
            (dict(x=x.clone().requires_grad_()), RuntimeError), (dict(x=x[:, :0]), ValueError)):
        a = dict(x=x, residual=res, weight=weight)
        a.update(bad)
        with pytest.raises(error):
            block_norm(**a)
    wide = torch.zeros(1, 40000, dtype=torch.float16)
    with pytest.raises(ValueError, match="32768"):
        block_norm(wide, None, torch.zeros(40000, dtype=torch.float16))
    assert block_norm(x[:0], res[:0], weight)[1].shape == (0, 64)


def test_c_entry_refuses_bad_shapes_before_a_launch():
    from kairyu_amd import _native

    def call(dtype=1, rows=1, hidden=64, ld=64, res_dtype=1, mode=0):
        _native.call("kq_block_norm", None, dtype, rows, hidden, ld, None, res_dtype, 0, None, None, 0, 1.0, None, 0.0, 1e-6,
                     mode, None, None, None, None)

    for bad in (dict(rows=-1), dict(hidden=0), dict(hidden=40000, ld=40000), dict(ld=63), dict(mode=4)):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(dtype=2), dict(res_dtype=0)):
        with pytest.raises(RuntimeError):
            call(**bad)
