"""The paged 8-bit key/value cache on the GPU where it is easily wrong: angles without
positions."""

from __future__ import annotations

import pytest
import torch

import kv_helpers as kv
from gpu_helpers import banner
from kairyu_amd.attention import rotary_table, rotate_append

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
