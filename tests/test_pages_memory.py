"""What the caches of a model's layers stand for when their tensors change afterwards."""

from __future__ import annotations

import ctypes
import gc

import torch

import draft_helpers as dh
from kairyu_amd.pages import KvCaches, copy_pages


def test_the_memory_behind_the_addresses_stays():
    """Tensors that get other memory leave the old, which a launch goes by, to the caches: it holds
    what it held, whatever is allocated then."""
    pools = dh.layers(2, 500, 2, 16, 64)
    caches = KvCaches(pools)
    sizes = [t.numel() * t.element_size() for pool in pools for t in pool]
    held = [ctypes.string_at(at, n) for at, n in zip(caches.pointers, sizes)]
    for i, pool in enumerate(pools):
        for t in pool:
            if i:
                t.set_(torch.zeros_like(t))
            else:
                t.data = torch.zeros_like(t)
    gc.collect()
    others = [torch.full((n,), 0x55, dtype=torch.uint8) for n in sizes for _ in range(4)]
    taken = {t.data_ptr() for t in others} | {t.data_ptr() for pool in pools for t in pool}
    assert not taken & set(caches.pointers)
    assert [ctypes.string_at(at, n) for at, n in zip(caches.pointers, sizes)] == held


def test_one_layers_cache_is_taken_as_it_is():
    """A cache handed to a call is looked at in that call."""
    pool, other = dh.layers(2, 5, 2, 16, 64)
    copy_pages(pool, dh.ints(1), dh.ints(3))
    pool.k.data = other.k.clone()
    copy_pages(pool, dh.ints(1), dh.ints(3))
    assert torch.equal(pool.k.view(torch.uint8)[3], other.k.view(torch.uint8)[1])
