"""Host side of the 8-bit paged KV cache: the pool's bookkeeping, argument checks that need no GPU, and the plain
64-bit statement's own properties."""

from __future__ import annotations

import math

import kv8_ref as ref
import numpy as np
import pytest
import torch

from torch2vk_b200 import kernels
from torch2vk_b200.paged_kv import PagedKVCache, PagedKVCacheQ8


def _pool(**kw):
    args = dict(layers=2, num_pages=8, page_size=32, kv_heads=2, head_dim=64, max_seqs=3, max_pages_per_seq=4, device="cpu")
    return PagedKVCacheQ8(**{**args, **kw})


def test_pool_shapes_and_bytes():
    pool = _pool(block=16, keep_weights=True)
    assert pool.k[1].shape == (8, 2, 32, 64) and pool.k[0].dtype == torch.int8
    assert pool.v_scale[0].shape == (8, 2, 2) and pool.v_scale[0].dtype == torch.float16
    assert pool.weights[0].shape == (3, 2, 128) and pool.weights[0].dtype == torch.float32
    assert _pool().weights == []
    fp16 = PagedKVCache(layers=1, num_pages=8, page_size=32, kv_heads=2, head_dim=64, max_seqs=3, max_pages_per_seq=4, device="cpu")
    assert pool.k[0].nbytes * 2 == fp16.k[0].nbytes


def test_pool_grows_shrinks_and_releases():
    pool = _pool()
    pool.reserve(0, 100)
    pool.reserve(1, 33)
    assert pool.pages(0) == [0, 1, 2, 3] and pool.free_pages == 2
    pool.shrink(0, 33)
    assert pool.pages(0) == [0, 1] and pool.free_pages == 4
    assert pool.block_table[0].tolist() == [0, 1, 0, 0]
    pool.shrink(0, 64)  # nothing to give back
    assert pool.pages(0) == [0, 1]
    pool.reserve(0, 65)
    assert len(pool.pages(0)) == 3 and pool.block_table[0, 2] == pool.pages(0)[2]
    pool.release(0)
    assert pool.free_pages == 6


@pytest.mark.parametrize("block", [8, 24, 128])
def test_pool_refuses_blocks(block):
    with pytest.raises(ValueError, match="block"):
        _pool(block=block)


def test_pages_need_the_gpu_and_one_layout():
    k = torch.zeros(2, 2, 32, 64, dtype=torch.int8)
    s = torch.zeros(2, 2, 2, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.Q8Pages(k, k, s, s)
    with pytest.raises(ValueError, match="one layout"):
        kernels.Q8Pages(k, k.transpose(1, 2).contiguous().transpose(1, 2), s, s)
    with pytest.raises(ValueError, match="page_size / block"):
        kernels.Q8Pages(k, k, s[:, :, :1].repeat(1, 1, 3), s[:, :, :1].repeat(1, 1, 3))


def test_statement_scales_are_least():
    rng = np.random.default_rng(1)
    for top in np.concatenate([np.float16(rng.random(500) * 100), np.float16(2.0) ** np.arange(-24, 16)]).astype(np.float64):
        s = float(ref.scale_for(top))
        assert 127 * s >= min(top, 127 * 515.5)
        if 0 < s < 515.5:
            assert 127 * float(np.nextafter(np.float16(s), np.float16(0))) < top
    assert math.isnan(ref.scale_for(math.inf)) and float(ref.scale_for(0.0)) == 0.0


def test_statement_round_trip_is_half_a_step():
    cache, table = ref.pool(3, 1, 32, 64, 16, seed=2), ref.tables(1, 3, 0, seed=3)
    x = torch.randn(1, 70, 1, 64, generator=torch.Generator().manual_seed(4)).half()
    ref.write(cache, x[:, :50], x[:, :50], [0], table)
    for t in range(50, 70):  # appended one by one: a grown scale moves earlier codes at most half a step each time
        ref.write(cache, x[:, t: t + 1], x[:, t: t + 1], [t], table)
    back = ref.rows(cache, table[0], 70)[0][0]
    for start in range(0, 70, 16):
        part, got = x[0, start: start + 16, 0].double(), back[start: start + 16]
        step = float(cache["ks"][int(table[0, start // 32]), 0, start % 32 // 16])
        whole = start + 16 <= 50
        assert float((got - part).abs().max()) <= step * (0.5 if whole else 4.0) + 1e-12
