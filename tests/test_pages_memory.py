"""What the caches of a model's layers stand for when their tensors change afterwards."""

from __future__ import annotations

import torch

import draft_helpers as dh
import kv_helpers as kv
from kairyu_amd.pages import KvCaches, copy_pages


def test_caches_stay_with_the_memory_they_were_made_over():
    """Tensors that get other memory leave the old to the caches, alive and the same for the
    addresses that a launch takes and the tensors."""
    pools = dh.layers(2, 5, 2, 16, 64)
    caches = KvCaches(pools)
    old = [tuple(t.detach() for t in pool) for pool in pools]
    want = [kv.values(p) for p in pools]
    for w in want:
        for t in w.values():
            t[3] = t[1]
    others = dh.layers(2, 5, 2, 16, 64, seed=9)
    for pool, other in zip(pools, others):
        pool.k.data = other.k.clone()
        pool.v_scale.set_(other.v_scale.clone())
    assert list(caches.pointers) == [t.data_ptr() for cache in old for t in cache]
    assert list(caches.pointers) == [t.data_ptr() for cache in caches.layers for t in cache]
    copy_pages(caches, dh.ints(1), dh.ints(3))
    dh.same_caches(caches.layers, want)
    for pool, other in zip(pools, others):
        assert torch.equal(pool.k.view(torch.uint8), other.k.view(torch.uint8)) and torch.equal(pool.v_scale, other.v_scale)


def test_one_layers_cache_is_taken_as_it_is():
    """A cache handed to a call is looked at in that call."""
    pool, other = dh.layers(2, 5, 2, 16, 64)
    copy_pages(pool, dh.ints(1), dh.ints(3))
    pool.k.data = other.k.clone()
    copy_pages(pool, dh.ints(1), dh.ints(3))
    assert torch.equal(pool.k.view(torch.uint8)[3], other.k.view(torch.uint8)[1])
