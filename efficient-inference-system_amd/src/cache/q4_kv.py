"""Block pools of 4-bit pages for the paged KV cache, and eviction by accumulated attention weight.

Q4BlockPool is a LayerBlockPool (allocation order, growth, free list, release as there) whose blocks are 4-bit
pages, uint8 [num_blocks, kv_heads, page_bytes] for K and for V: 4.5 bits a value, 3.6 times less than bf16 and
7.1 times less than fp32. With track_weights it keeps a float32 [num_blocks, kv_heads, 16] tensor beside
them, the attention weight that each slot's key has had so far, which attention adds to and
BatchedPagedKVCache.evict goes by. No reference counterpart: the reference's pools hold the model's dtype and
keep every key.
"""
from __future__ import annotations

import numpy as np
import torch

from src.cache.paged_kv import KVStorage, LayerBlockPool
from src.kernels import reference_q4


class Q4BlockPool(LayerBlockPool):
    is_q4 = True

    def __init__(self, block_size: int, initial_blocks: int, growth_factor: float, track_weights: bool = False,
                 storage: KVStorage | None = None):
        if block_size != reference_q4.BLOCK:
            raise ValueError(f"4-bit pages hold {reference_q4.BLOCK} tokens, got block_size {block_size}")
        super().__init__(block_size, initial_blocks, growth_factor, dtype=torch.uint8, storage=storage)
        self.track_weights = track_weights
        self.weights: torch.Tensor | None = None

    def _block_shape(self) -> tuple:
        return (self.num_heads, reference_q4.page_bytes(self.head_dim))

    def _grow(self, min_extra_blocks: int) -> None:
        super()._grow(min_extra_blocks)
        if self.track_weights:
            old = self.weights
            self.weights = torch.zeros(self.capacity_blocks, self.num_heads, self.block_size, device=self.device)
            if old is not None:
                self.weights[:old.shape[0]] = old

    def release_block(self, block_id: int) -> None:
        super().release_block(block_id)
        if self.weights is not None:
            self.weights[block_id].zero_()

    def release_blocks(self, block_ids: list[int]) -> None:
        if self.k_blocks is None or self.v_blocks is None or not block_ids:
            return
        if self.k_blocks.is_cuda:
            from src.kernels.hip_paged_attention import zero_blocks_hip
            from src.kernels.staging import upload

            ids = upload(np.asarray(block_ids, dtype=np.int32), self.k_blocks.device)
            # pages as float32 tiles of the same bytes: zeroed in one launch
            zero_blocks_hip(*(t.view(torch.float32).unflatten(-1, (self.block_size, -1)) for t in (self.k_blocks, self.v_blocks)),
                            ids)
        else:
            ids = torch.tensor(block_ids, dtype=torch.long)
            self.k_blocks[ids] = 0
            self.v_blocks[ids] = 0
        if self.weights is not None:
            self.weights.index_fill_(0, ids.long(), 0.0)
        self.free_block_ids.extend(block_ids)
        self.mutations += 1

    def put_rows(self, blocks: torch.Tensor, offsets: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        reference_q4.put_rows(self.k_blocks, blocks, offsets, k, True)
        reference_q4.put_rows(self.v_blocks, blocks, offsets, v, False)
        if self.weights is not None:
            self.weights[blocks, :, offsets] = 0.0

    def tiles(self, ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return (reference_q4.values(self.k_blocks.index_select(0, ids), self.head_dim, True),
                reference_q4.values(self.v_blocks.index_select(0, ids), self.head_dim, False))

    def bytes_per_block(self) -> int:
        pages = super().bytes_per_block()
        return pages + (4 * self.num_heads * self.block_size if self.weights is not None else 0)

    def token_bytes(self) -> int:
        kb = self.k_blocks
        return kb.shape[1] * (2 * kb.shape[2] // self.block_size + (4 if self.weights is not None else 0))

    def evict_rows(self, old: list[list[int]], lengths: list[int], new: list[list[int]], keep: int,
                   window: int) -> list[torch.Tensor]:
        """Move the kept keys of requests with blocks old[i] and lengths[i] > keep keys to blocks new[i];
        returns their old indices, int32 [heads, keep] each."""
        dev = self.k_blocks.device
        if self.k_blocks.is_cuda:
            from src.kernels.hip_q4_attention import evict_q4_hip
            from src.kernels.staging import upload

            n, width, fresh = len(old), max(map(len, old)), len(new[0])
            host = np.full((n, 1 + width + fresh), -1, dtype=np.int32)
            for row, blocks, length, to in zip(host, old, lengths, new):
                row[0], row[1:1 + len(blocks)], row[1 + width:] = length, blocks, to
            packed = upload(host.reshape(-1), dev).view(n, -1)
            kept, _ = evict_q4_hip(self.k_blocks, self.v_blocks, self.weights, packed[:, 1:1 + width].contiguous(),
                                   packed[:, 0].contiguous(), packed[:, 1 + width:].contiguous(), keep=keep, window=window)
            return list(kept)
        out = []
        for blocks, length, to in zip(old, lengths, new):
            ids, at = torch.tensor(blocks), torch.tensor(to)
            totals = self.weights[ids].transpose(0, 1).flatten(1)[:, :length]
            index = reference_q4.choose(totals, keep, window)
            src = ids[index // self.block_size], index % self.block_size
            place = torch.arange(keep).expand_as(index)
            dst = at[place // self.block_size], place % self.block_size
            for pool, is_key in ((self.k_blocks, True), (self.v_blocks, False)):
                reference_q4.move_rows(pool, src, dst, self.head_dim, is_key)
            head = torch.arange(self.num_heads)[:, None]
            self.weights[dst[0], head, dst[1]] = self.weights[src[0], head, src[1]]
            out.append(index.to(torch.int32))
        return out
