"""Paged KV cache, fp16 or 4 bits (the reference has none: runners/engine.py:90-91 hold
one token's k/v and seq_len is fixed at 1, engine.py:64).

Layout in HBM: K and V are each one tensor fp16
[n_layers, n_pages, n_kv_heads, page_size, head_dim]; a page holds
``page_size`` consecutive positions of one KV head of one sequence, so the
attention kernel reads a (page, head) tile as one contiguous 16 KB block
(page_size 64 x 128 x 2 bytes).  ``block_table`` int32 [max_batch,
pages_per_seq] maps page j of sequence slot b to a pool page.  Row i of the
reference's implied [T, n_kv_heads*128] cache (kernels/attention.metal:33)
is position i here.

:class:`PagedKVCacheQ4` holds the same pages in 4 bits: uint8 [n_layers,
n_pages, n_kv_heads, page_size * 72], 72 bytes a row instead of 256 (format
in include/llamamps_b200.h).
"""
from __future__ import annotations

from typing import List, Optional

import torch

from .config import ModelConfig
from .quant import KV_ROW_BYTES, dequantise_kv_rows, quantise_kv_rows


class PagedKVCache:
    def __init__(self, cfg: ModelConfig, n_layers: int, max_batch: int, max_seq_len: int,
                 page_size: int = 64, device="cuda", n_pages: Optional[int] = None,
                 page_order: Optional[List[int]] = None):
        if max_seq_len <= 0 or page_size <= 0 or max_batch <= 0:
            raise ValueError("max_seq_len, page_size and max_batch must be positive")
        self.cfg = cfg
        self.n_layers = n_layers
        self.page_size = page_size
        self.max_batch = max_batch
        self.pages_per_seq = (max_seq_len + page_size - 1) // page_size
        self.max_seq_len = self.pages_per_seq * page_size
        self.n_pages = n_pages if n_pages is not None else max_batch * self.pages_per_seq
        if self.n_pages < self.pages_per_seq:
            raise ValueError("pool smaller than one sequence")
        self.device = torch.device(device)
        self._allocate_pools()
        self.block_table = torch.zeros(max_batch, self.pages_per_seq, dtype=torch.int32, device=self.device)
        order = list(page_order) if page_order is not None else list(range(self.n_pages))
        if sorted(order) != list(range(self.n_pages)):
            raise ValueError("page_order must be a permutation of the pool's pages")
        self._free: List[int] = order[::-1]
        self._owned: List[List[int]] = [[] for _ in range(max_batch)]

    def _allocate_pools(self) -> None:
        cfg = self.cfg
        shape = (self.n_layers, self.n_pages, cfg.n_kv_heads, self.page_size, cfg.head_dim)
        self.k = torch.zeros(shape, dtype=torch.float16, device=self.device)
        self.v = torch.zeros(shape, dtype=torch.float16, device=self.device)

    # -- page allocation ----------------------------------------------------
    def reserve(self, slot: int, n_positions: int) -> None:
        """Make positions [0, n_positions) of ``slot`` addressable."""
        need = (n_positions + self.page_size - 1) // self.page_size
        if need > self.pages_per_seq:
            raise ValueError(f"{n_positions} positions exceed the cache capacity {self.max_seq_len}")
        owned = self._owned[slot]
        new = []
        while len(owned) < need:
            if not self._free:
                raise MemoryError("KV page pool exhausted")
            owned.append(self._free.pop())
            new.append(len(owned) - 1)
        if new:
            idx = torch.tensor(new, dtype=torch.long)
            vals = torch.tensor([owned[j] for j in new], dtype=torch.int32)
            self.block_table[slot, idx.to(self.device)] = vals.to(self.device)

    def release(self, slot: int) -> None:
        self._free.extend(reversed(self._owned[slot]))
        self._owned[slot] = []

    def release_all(self) -> None:
        for s in range(self.max_batch):
            self.release(s)

    def pages(self, slot: int) -> List[int]:
        return list(self._owned[slot])

    # -- views ---------------------------------------------------------------
    def layer(self, layer: int):
        return self.k[layer], self.v[layer]

    def write_positions(self, slot: int, layer: int, start: int, k_rows: torch.Tensor,
                        v_rows: torch.Tensor) -> None:
        """Scatter rows [T, n_kv_heads*head_dim] into positions start.. of ``slot``."""
        cfg = self.cfg
        T = k_rows.shape[0]
        self.reserve(slot, start + T)
        kr = k_rows.to(self.device, torch.float16).reshape(T, cfg.n_kv_heads, cfg.head_dim)
        vr = v_rows.to(self.device, torch.float16).reshape(T, cfg.n_kv_heads, cfg.head_dim)
        pos = torch.arange(start, start + T, device=self.device)
        pages = self.block_table[slot, (pos // self.page_size)].long()
        off = pos % self.page_size
        for h in range(cfg.n_kv_heads):
            self.k[layer, pages, h, off] = kr[:, h]
            self.v[layer, pages, h, off] = vr[:, h]

    def read_positions(self, slot: int, layer: int, n: int):
        """Rows [n, n_kv_heads*head_dim] of positions 0..n-1 (a copy)."""
        cfg = self.cfg
        pos = torch.arange(n, device=self.device)
        pages = self.block_table[slot, (pos // self.page_size)].long()
        off = pos % self.page_size
        k = torch.stack([self.k[layer, pages, h, off] for h in range(cfg.n_kv_heads)], dim=1)
        v = torch.stack([self.v[layer, pages, h, off] for h in range(cfg.n_kv_heads)], dim=1)
        return k.reshape(n, -1), v.reshape(n, -1)


class PagedKVCacheQ4(PagedKVCache):
    """The paged cache in 4 bits: the kernels' ``*_q4`` entry points read and
    write it.  head_dim 128, page_size a multiple of 16."""

    def _allocate_pools(self) -> None:
        cfg = self.cfg
        if cfg.head_dim != 128:
            raise ValueError(f"the 4-bit KV cache holds heads of 128, not {cfg.head_dim}")
        if self.page_size % 16:
            raise ValueError(f"the 4-bit KV cache needs a page_size that is a multiple of 16, not {self.page_size}")
        shape = (self.n_layers, self.n_pages, cfg.n_kv_heads, self.page_size * KV_ROW_BYTES)
        # (zero bytes: codes of -8 with scale 0, the value 0)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=self.device)

    def rows(self, pool: torch.Tensor):
        """Views of the code rows [..., page_size, 64] and scale rows [..., page_size, 4] of pool blocks."""
        split = self.page_size * 64
        return (pool[..., :split].unflatten(-1, (self.page_size, 64)),
                pool[..., split:].view(torch.float16).unflatten(-1, (self.page_size, 4)))

    def _places(self, slot: int, pos: torch.Tensor):
        return self.block_table[slot, (pos // self.page_size)].long(), pos % self.page_size

    def write_positions(self, slot: int, layer: int, start: int, k_rows: torch.Tensor,
                        v_rows: torch.Tensor) -> None:
        """Quantises rows [T, n_kv_heads*128] into positions start.. of ``slot``."""
        T = k_rows.shape[0]
        self.reserve(slot, start + T)
        pages, off = self._places(slot, torch.arange(start, start + T, device=self.device))
        for pool, rows in ((self.k, k_rows), (self.v, v_rows)):
            x = rows.to(self.device, torch.float16).reshape(T, self.cfg.n_kv_heads, 128)
            codes, scales = self.rows(pool[layer])
            codes[pages, :, off], scales[pages, :, off] = quantise_kv_rows(x)

    def read_positions(self, slot: int, layer: int, n: int):
        """The fp16 values [n, n_kv_heads*128] that positions 0..n-1 hold."""
        pages, off = self._places(slot, torch.arange(n, device=self.device))
        out = []
        for pool in (self.k, self.v):
            codes, scales = self.rows(pool[layer])
            out.append(dequantise_kv_rows(codes[pages, :, off], scales[pages, :, off]).reshape(n, -1))
        return tuple(out)
