"""Physical block pool of the paged KV cache on one MI355X.

Same API and tensor layout as the reference's PagedKVCachePool
(src/mini_infra/worker/paged_kv_cache.py:14-95): ``kv_pools[layer] = (key_pool, value_pool)``,
each ``[num_blocks, block_size, num_kv_heads, head_dim]``, zero-filled, block 0 the null block,
``slot = block_id * block_size + offset``.

MI355X layout: all layers live in ONE allocation ``[num_layers, 2, num_blocks, bs, H, D]`` (a
90 GB pool is a single HBM3E range), and ``kv_pools`` are views of it, so the per-layer tensors
the reference's callers index are unchanged.  ``gather_blocks`` and ``write_prefill`` are single
HIP launches over all layers (kernels 2 and 1) instead of per-layer advanced indexing.

``PagedKVCachePoolFp4`` holds the same blocks in 4 bits (17/64 of the bf16 bytes), with the same calls.
"""

from __future__ import annotations

import math

import torch

from mini_infra_qwen3_amd import data_plane
from mini_infra_qwen3_amd.worker.kv_cache import KVCache


class PagedKVCachePool:
    """Per-layer physical K/V block pools, GPU only (there is no CPU data plane)."""

    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device | str,
    ):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCachePool needs a GPU device, got {device} (no CPU data plane)")
        if num_layers < 1 or num_blocks < 1 or block_size < 1 or num_kv_heads < 1 or head_dim < 1:
            raise ValueError("PagedKVCachePool: every dimension must be positive")
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.storage = torch.zeros(
            (num_layers, 2, num_blocks, block_size, num_kv_heads, head_dim), dtype=dtype, device=device
        )
        self.kv_pools: list[tuple[torch.Tensor, torch.Tensor]] = [
            (self.storage[layer, 0], self.storage[layer, 1]) for layer in range(num_layers)
        ]

    @property
    def row_dtype(self) -> torch.dtype:
        """dtype of the K/V rows that go in and come out."""
        return self.storage.dtype

    @property
    def device(self) -> torch.device:
        return self.storage.device

    @property
    def bytes_per_block(self) -> int:
        """K+V bytes of one physical block across all layers."""
        key_pool, _ = self.kv_pools[0]
        return 2 * len(self.kv_pools) * math.prod(key_pool.shape[1:]) * key_pool.element_size()

    @property
    def total_bytes(self) -> int:
        """Bytes of the whole pool, null block included."""
        return self.num_blocks * self.bytes_per_block

    def gather_blocks(self, block_ids: torch.Tensor) -> tuple[tuple[torch.Tensor, torch.Tensor], ...]:
        """History K/V by block table, every layer in one kernel launch.

        block_ids: ``[B, nb]`` int64 on the pool's device, right-padded with the null block.
        Returns per layer ``(key, value)``, each ``[B, H_kv, nb * block_size, D]`` -- non-contiguous
        ``transpose(1, 2)`` views of a contiguous ``[B, nb * block_size, H_kv, D]`` gather, exactly
        as the reference returns them (whole blocks, null block and stale tails included).
        """
        return self._gather(block_ids, data_plane.gather_blocks)

    def _gather(self, block_ids: torch.Tensor, gather) -> tuple[tuple[torch.Tensor, torch.Tensor], ...]:
        if block_ids.ndim != 2:
            raise ValueError(f"block_ids must be [batch, num_blocks], got {tuple(block_ids.shape)}")
        block_ids = block_ids.to(device=self.device, dtype=torch.long)
        batch, nb = block_ids.shape
        num_layers = len(self.kv_pools)
        out = torch.empty(
            (num_layers, 2, batch, nb * self.block_size, self.num_kv_heads, self.head_dim),
            dtype=self.row_dtype, device=self.device,
        )
        keys = [out[layer, 0] for layer in range(num_layers)]
        values = [out[layer, 1] for layer in range(num_layers)]
        gather(
            [k for k, _ in self.kv_pools], [v for _, v in self.kv_pools], block_ids, keys, values
        )
        return tuple((k.transpose(1, 2), v.transpose(1, 2)) for k, v in zip(keys, values))

    def _block_id_tensor(self, block_ids, unique: bool) -> torch.Tensor:
        if isinstance(block_ids, torch.Tensor):
            return block_ids.to(device=self.device, dtype=torch.long).reshape(-1)
        ids = [int(b) for b in block_ids]
        if any(not 0 <= b < self.num_blocks for b in ids):
            raise ValueError(f"block ids must lie in [0, {self.num_blocks})")
        if unique and len(set(ids)) != len(ids):
            raise ValueError("block ids written by one call must be unique")
        return torch.tensor(ids, dtype=torch.long).to(self.device, non_blocking=True)

    def pack_blocks(self, block_ids) -> torch.Tensor:
        """Blocks ``block_ids`` of every layer as contiguous KV block records
        ``[n, num_layers, 2, bs, H, D]`` (the swap / wire format), one kernel launch."""
        return data_plane.pack_blocks([k for k, _ in self.kv_pools], [v for _, v in self.kv_pools],
                                      self._block_id_tensor(block_ids, unique=False))

    def unpack_blocks(self, records: torch.Tensor, block_ids) -> None:
        """Writes KV block records into blocks ``block_ids`` (unique) of every layer, one kernel launch."""
        data_plane.unpack_blocks(records, [k for k, _ in self.kv_pools], [v for _, v in self.kv_pools],
                                 self._block_id_tensor(block_ids, unique=True))

    def copy_blocks(self, src_blocks, dst_blocks) -> None:
        """Block ``dst_blocks[i]`` of every layer becomes block ``src_blocks[i]``, K and V, in one kernel launch on the
        current stream (for ``KVCacheManager.fork`` and ``compact``).

        Destinations are unique and none is a source; lists are checked, tensors are taken as they are.
        """
        if not isinstance(src_blocks, torch.Tensor) and not isinstance(dst_blocks, torch.Tensor):
            if set(map(int, src_blocks)) & set(map(int, dst_blocks)):
                raise ValueError("a block that one call writes cannot be its source as well")
        src = self._block_id_tensor(src_blocks, unique=False)
        dst = self._block_id_tensor(dst_blocks, unique=True)
        data_plane.copy_blocks([k for k, _ in self.kv_pools], [v for _, v in self.kv_pools], src, dst)

    def write_prefill(
        self,
        prefill_cache: KVCache,
        token_rows: torch.Tensor,
        token_positions: torch.Tensor,
        slot_mapping: torch.Tensor,
    ) -> None:
        """Scatters the valid prefill tokens of every layer into their slots (one kernel launch).

        prefill_cache: per layer ``(key, value)``, each ``[B, H_kv, L, D]`` (any strides, D contiguous).
        token_rows / token_positions / slot_mapping: ``[N]`` int64; slots must be unique.
        """
        self._write(prefill_cache, token_rows, token_positions, slot_mapping, data_plane.reshape_and_cache)

    def _write(self, prefill_cache: KVCache, token_rows: torch.Tensor, token_positions: torch.Tensor,
               slot_mapping: torch.Tensor, scatter) -> None:
        caches = list(prefill_cache)
        if len(caches) != len(self.kv_pools):
            raise ValueError(f"prefill_cache has {len(caches)} layers, pool has {len(self.kv_pools)}")
        scatter(
            [k for k, _ in caches],
            [v for _, v in caches],
            slot_mapping,
            [k for k, _ in self.kv_pools],
            [v for _, v in self.kv_pools],
            token_rows=token_rows,
            token_positions=token_positions,
        )


class PagedKVCachePoolFp4(PagedKVCachePool):
    """A ``PagedKVCachePool`` in 4 bits (MXFP4, ``data_plane.fp4_pool_shape``): groups of 32 dims with a
    power-of-two scale byte, 4.25 bits a value, so a block takes 17/64 of its bf16 bytes.

    ``kv_pools[layer]``: (key, value) pools, uint8 ``[num_blocks, block_size / 16, H_kv, 1088]``.  K/V rows are
    quantised when they are written (bf16, fp16 or fp32) and come back as the bf16 values that they stand for; the
    attention kernels read the pool as it is.  Block records are its bytes: pools of one geometry exchange blocks
    exactly.
    """

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device: torch.device | str):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCachePoolFp4 needs a GPU device, got {device} (no CPU data plane)")
        if num_layers < 1 or num_blocks < 1:
            raise ValueError("PagedKVCachePoolFp4: every dimension must be positive")
        shape = data_plane.fp4_pool_shape(num_blocks, block_size, num_kv_heads, head_dim)
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.storage = torch.zeros((num_layers, 2, *shape), dtype=torch.uint8, device=device)
        self.kv_pools = [(self.storage[layer, 0], self.storage[layer, 1]) for layer in range(num_layers)]

    @property
    def row_dtype(self) -> torch.dtype:
        return torch.bfloat16

    def gather_blocks(self, block_ids: torch.Tensor) -> tuple[tuple[torch.Tensor, torch.Tensor], ...]:
        """``PagedKVCachePool.gather_blocks``, the values as bf16."""
        return self._gather(block_ids, data_plane.gather_blocks_fp4)

    def write_prefill(self, prefill_cache: KVCache, token_rows: torch.Tensor, token_positions: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
        """``PagedKVCachePool.write_prefill``, quantising."""
        self._write(prefill_cache, token_rows, token_positions, slot_mapping, data_plane.reshape_and_cache_fp4)


__all__ = ["PagedKVCachePool", "PagedKVCachePoolFp4"]
