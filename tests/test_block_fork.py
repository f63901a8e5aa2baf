"""Forks and compaction of the block tables (no counterpart in the reference), on the CPU: a pool of token ids that obeys
the returned block pairs keeps every request's tokens through random sequences of both."""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd.core import NULL_BLOCK_ID, KVCacheManager, PagedCacheConfig
from mini_infra_qwen3_amd.worker.block_tables import DeviceBlockTables


class Pool:
    """Blocks of token ids, written slot by slot, copied by pairs as ``copy_blocks`` copies them."""

    def __init__(self, manager):
        self.manager = manager
        self.blocks = np.full((manager.free_block_queue.num_blocks, manager.block_size), -1, dtype=np.int64)
        self.tokens = {}  # request: its token ids

    def append(self, request, ids):
        if not self.manager.allocate_slots(request, len(ids)):
            return False
        have = self.tokens.setdefault(request, [])
        table, bs = self.manager.block_table(request), self.manager.block_size
        for i, token in enumerate(ids, start=len(have)):
            self.blocks[table[i // bs], i % bs] = token
        self.tokens[request] = have + list(ids)
        return True

    def copy(self, pairs):
        sources = {s for s, _ in pairs}
        targets = [d for _, d in pairs]
        assert len(set(targets)) == len(targets) and not sources & set(targets)
        assert all(0 < b < self.blocks.shape[0] for pair in pairs for b in pair)
        for source, target in pairs:
            self.blocks[target] = self.blocks[source]

    def check(self):
        manager = self.manager
        held = {}
        for request, want in self.tokens.items():
            table, bs = manager.block_table(request), manager.block_size
            assert manager.num_tokens(request) == len(want) and len(table) == -(-len(want) // bs)
            assert [int(self.blocks[table[i // bs], i % bs]) for i in range(len(want))] == want
            for b in table:
                held[b] = held.get(b, 0) + 1
        queue = manager.free_block_queue
        at = (queue._head + np.arange(queue.num_free_blocks)) % queue._ring.shape[0]
        free = queue._ring[at].tolist()
        assert sorted(free + list(held)) == list(range(1, queue.num_blocks))  # each id once, never the null block
        assert NULL_BLOCK_ID not in held and manager.num_used_blocks == len(held)


def test_fork_shares_full_blocks_and_copies_the_last():
    manager = KVCacheManager(block_size=4, num_blocks=8)
    pool = Pool(manager)
    assert pool.append(0, range(10, 19))  # 9 tokens: blocks 1, 2 full, 3 with one
    assert manager.fork(0, 5) == [(3, 4)]
    pool.copy([(3, 4)])
    pool.tokens[5] = list(pool.tokens[0])
    assert manager.block_table(5) == [1, 2, 4] and manager.num_used_blocks == 4
    assert pool.append(0, [70]) and pool.append(5, [80, 81])  # both go on in their own block
    pool.check()
    manager.free(0)
    del pool.tokens[0]
    assert manager.num_used_blocks == 3 and manager.block_release_count == 1
    pool.check()
    manager.free(5)
    assert manager.num_used_blocks == 0 and manager.block_release_count == 4


@pytest.mark.parametrize("tokens,table,pairs", [(0, [], []), (3, [4], [(1, 4)]), (4, [1], []), (8, [1, 2], []), (None, [1, 2, 4], [(3, 4)])])
def test_fork_of_a_prefix(tokens, table, pairs):
    manager = KVCacheManager(block_size=4, num_blocks=8)
    assert manager.allocate_slots(0, 9)
    assert manager.fork(0, 1, tokens) == pairs
    assert manager.block_table(1) == table and manager.num_tokens(1) == (9 if tokens is None else tokens)
    manager.free(0)
    assert manager.num_used_blocks == len(table)


def test_fork_without_a_free_block_leaves_no_trace():
    manager = KVCacheManager(block_size=4, num_blocks=4)
    assert manager.allocate_slots(0, 9)
    manager.take_deltas()
    assert manager.fork(0, 1) is None
    with pytest.raises(KeyError):
        manager.block_table(1)
    assert manager.take_deltas()[0].shape == (0,)
    assert manager.fork(0, 1, 8) == []  # full blocks need none
    manager.free(0)
    assert manager.num_used_blocks == 2


def test_fork_refusals():
    manager = KVCacheManager(block_size=4, num_blocks=8)
    assert manager.allocate_slots(0, 5)
    with pytest.raises(KeyError):
        manager.fork(3, 4)
    with pytest.raises(ValueError, match="already"):
        manager.fork(0, 0)
    for tokens in (-1, 6):
        with pytest.raises(ValueError, match="cannot fork"):
            manager.fork(0, 1, tokens)
    assert manager.num_used_blocks == 2


def test_compact_moves_the_upper_blocks_down():
    manager = KVCacheManager(block_size=4, num_blocks=10)
    for request in range(4):
        assert manager.allocate_slots(request, 8)  # blocks 1..8
    manager.free(0)
    manager.free(2)  # 1, 2, 5, 6 free behind 9
    assert manager.compact() == [(7, 1), (8, 2)]
    assert manager.block_table(1) == [3, 4] and manager.block_table(3) == [1, 2]
    assert manager.compact() == []
    assert manager.free_block_queue.allocate(5) == [9, 7, 8, 5, 6]  # each moved block in its target's place


def test_compact_refuses_blocks_taken_around_it():
    manager = KVCacheManager(block_size=4, num_blocks=10)
    manager.free_block_queue.allocate(2)
    with pytest.raises(RuntimeError, match="tables hold 0"):
        manager.compact()


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_and_compactions(seed):
    rng = np.random.default_rng(seed)
    bs = int(rng.choice([1, 3, 4, 16]))
    manager = KVCacheManager(block_size=bs, num_blocks=int(rng.integers(20, 60)))
    pool = Pool(manager)
    device = DeviceBlockTables(manager, 64, 64, torch.device("cpu"))
    serial = 0
    for step in range(400):
        live = list(pool.tokens)
        op = rng.choice(["new", "append", "fork", "free", "compact"], p=[0.2, 0.3, 0.2, 0.2, 0.1])
        if op == "new" and len(live) < 40:
            pool.append(step, [serial + i for i in range(int(rng.integers(1, 4 * bs + 1)))])
        elif op == "append" and live:
            pool.append(int(rng.choice(live)), [serial + i for i in range(int(rng.integers(1, bs + 2)))])
        elif op == "fork" and live and len(live) < 40:
            parent = int(rng.choice(live))
            n = int(rng.integers(0, len(pool.tokens[parent]) + 1)) if rng.random() < 0.5 else None
            pairs = manager.fork(parent, step, n)
            if pairs is not None:
                pool.copy(pairs)
                pool.tokens[step] = pool.tokens[parent][:n]
        elif op == "free" and live:
            request = int(rng.choice(live))
            manager.free(request)
            del pool.tokens[request]
        elif op == "compact":
            pool.copy(manager.compact())
            in_use = [b for r in pool.tokens for b in manager.block_table(r)]
            assert max(in_use, default=0) == manager.num_used_blocks
        serial += 1000
        pool.check()
        if step % 7 == 0:
            device.sync()
            for request in pool.tokens:
                table = manager.block_table(request)
                assert device.tensor[manager.row_of(request), :len(table)].tolist() == table


def test_cache_config_bits():
    assert PagedCacheConfig().kv_bits == 16 and PagedCacheConfig(kv_bits=4).block_size == 16
    with pytest.raises(ValueError, match="kv_bits"):
        PagedCacheConfig(kv_bits=8)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCacheConfig(block_size=24, kv_bits=4)
