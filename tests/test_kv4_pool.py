"""CPU: a 4-bit pool whose tensors are replaced is what its new tensors are."""
from __future__ import annotations

import pytest
import torch

from flexengine_amd import ops
from flexengine_amd.kv_cache import CacheLayout, PagedKVCache

F16, BF16 = torch.float16, torch.bfloat16


def pool(nb=4, bs=16, hkv=2, d=64, lead=(), dt=F16):
    return ops.Kv4Pool.empty((*lead, nb, bs, hkv, d), dt, "cpu")


def test_layers_follow_the_tensors_that_a_cache_is_given():
    cache = PagedKVCache(CacheLayout(3, 4, 16, 2, 64), device="cpu", bits=4)
    before = [cache.k[i] for i in range(3)]
    assert [p.layout() for p in before] == [(4, 16, 2, 64)] * 3
    restored = [cache.k.codes.clone(), cache.k.scales.clone()]
    cache.k.codes, cache.k.scales = restored
    for i in range(3):
        assert cache.k[i].codes.data_ptr() == restored[0][i].data_ptr()
        assert cache.k[i].scales.data_ptr() == restored[1][i].data_ptr()
        assert before[i].codes.data_ptr() != restored[0][i].data_ptr()   # a pool of its own tensors
    assert ops._kv4_ptrs(cache.k[1], cache.v[1])[:2] == (restored[0][1].data_ptr(), restored[1][1].data_ptr())


def test_replaced_tensors_are_checked_and_their_layout_is_taken():
    p, other = pool(), pool(nb=9)
    assert p.layout() == (4, 16, 2, 64)
    p.codes = other.codes
    with pytest.raises(ValueError):       # codes of nine blocks beside the scales of four
        p.layout()
    p.scales = other.scales
    assert p.layout() == (9, 16, 2, 64) and p.shape == (9, 16, 2, 64)
    p.codes = torch.zeros(9, 16, 2, 32, dtype=torch.uint8).transpose(1, 2)
    assert p.layout() == (9, 16, 2, 64)
    with pytest.raises(ValueError):       # the other pool's strides are the dense ones
        ops._check_pool4(p, other)
    p.codes = other.codes
    assert ops._check_pool4(p, other) == (9, 16, 2, 64)
    for bad in (other.codes.float(), other.codes[..., ::2], other.codes[0]):
        p.codes = bad
        with pytest.raises(ValueError):
            p.layout()
    p.codes = other.codes
    p.dtype = torch.float32
    with pytest.raises(ValueError):
        p.layout()
    p.dtype = BF16
    assert p.layout() == (9, 16, 2, 64)
    with pytest.raises(ValueError):       # rows of another type
        ops._check_pool4(p, other)
