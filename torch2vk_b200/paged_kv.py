"""Paged KV cache: a pool of fixed-size pages shared by the sequences of a
runner, with per-sequence block tables (logical page -> physical page).

Each layer has one K and one V pool [num_pages, page_size, kv_heads, head_dim]
fp16; page p of sequence s holds positions [p * page_size, (p + 1) * page_size).
Pages are handed out from a free list as sequences grow and returned when a
sequence is released; the device block table [max_seqs, max_pages_per_seq]
int32 is what the paged kernels (t2c_attn_decode_paged,
t2c_kv_cache_write_paged) read.  Host code owns the bookkeeping: reserve()
before a step needs the positions, shrink() after a sequence was cut,
release() when it ends.  PagedKVCacheQ8 keeps the pool in 8 bits.
"""

from __future__ import annotations

import torch

from torch2vk_b200 import kernels


class PagedKVCache:
    def __init__(self, *, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: int, device: torch.device | str = "cuda") -> None:
        if page_size <= 0 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} must be a power of two")
        self.page_size, self.num_pages = page_size, num_pages
        self.max_pages_per_seq = max_pages_per_seq
        self.device = torch.device(device)
        self._allocate(layers, num_pages, page_size, kv_heads, head_dim)
        self.block_table = torch.zeros(max_seqs, max_pages_per_seq, dtype=torch.int32, device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}

    def _allocate(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int) -> None:
        shape = (num_pages, page_size, kv_heads, head_dim)
        self.k = [torch.zeros(shape, dtype=torch.float16, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.float16, device=self.device) for _ in range(layers)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, seq: int) -> list[int]:
        return list(self._pages.get(seq, []))

    def reserve(self, seq: int, positions: int) -> None:
        """Grows sequence `seq` to hold `positions` positions (pages from the free list)."""
        have = self._pages.setdefault(seq, [])
        need = -(-positions // self.page_size)
        if need > self.max_pages_per_seq:
            raise ValueError(f"{positions} positions exceed {self.max_pages_per_seq} pages of {self.page_size}")
        if need - len(have) > len(self._free):
            raise RuntimeError(f"KV pool exhausted: {need - len(have)} pages wanted, {len(self._free)} free")
        new = [self._free.pop() for _ in range(max(0, need - len(have)))]
        if new:
            row = torch.tensor(new, dtype=torch.int32)
            self.block_table[seq, len(have):len(have) + len(new)].copy_(row, non_blocking=False)
            have.extend(new)

    def shrink(self, seq: int, positions: int) -> None:
        """Returns the pages of `seq` past `positions` positions to the free list."""
        have = self._pages.get(seq, [])
        keep = -(-positions // self.page_size)
        if keep >= len(have):
            return
        self.block_table[seq, keep:len(have)].zero_()
        while len(have) > keep:
            self._free.append(have.pop())

    def release(self, seq: int) -> None:
        """Returns the pages of `seq` to the free list."""
        for p in reversed(self._pages.pop(seq, [])):
            self._free.append(p)
        self.block_table[seq].zero_()


class PagedKVCacheQ8(PagedKVCache):
    """The pool in 8 bits: per layer int8 codes k / v [num_pages, kv_heads, page_size, head_dim] and one fp16 scale for
    each `block` consecutive tokens of a KV head (half the fp16 pool's bytes, plus one scale per block * head_dim
    codes).  layer(i) is what the kernels take.  keep_weights: per layer the running attention weight of each cached
    key, fp32 [max_seqs, kv_heads, positions], which attention adds to and eviction goes by."""

    def __init__(self, *, block: int = 16, keep_weights: bool = False, **pool) -> None:
        if block not in (16, 32, 64) or pool["page_size"] < block:
            raise ValueError(f"block {block} must be 16, 32 or 64, at most page_size")
        self.block = block
        super().__init__(**pool)
        positions = self.max_pages_per_seq * self.page_size
        shape = (pool["max_seqs"], pool["kv_heads"], positions)
        self.weights = [torch.zeros(shape, dtype=torch.float32, device=self.device) for _ in range(pool["layers"])] \
            if keep_weights else []

    def _allocate(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int) -> None:
        shape, scales = (num_pages, kv_heads, page_size, head_dim), (num_pages, kv_heads, page_size // self.block)
        self.k, self.v = ([torch.zeros(shape, dtype=torch.int8, device=self.device) for _ in range(layers)] for _ in range(2))
        self.k_scale, self.v_scale = ([torch.zeros(scales, dtype=torch.float16, device=self.device) for _ in range(layers)]
                                      for _ in range(2))
        self._layers: dict[int, kernels.Q8Pages] = {}

    def layer(self, i: int) -> kernels.Q8Pages:
        if i not in self._layers:
            self._layers[i] = kernels.Q8Pages(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])
        return self._layers[i]
