"""Logical block allocator of the paged KV cache: FIFO free-block queue and per-request block tables.

The reference's API and observable behaviour (src/mini_infra/core/block_manager.py:17-149): block
ids 1..num_blocks-1 handed out first-freed-first-reused (block 0 is the null block that pads
tables), the cold / reuse / release / peak counters, all-or-nothing slot allocation and FCFS
admission under a reservation.  The state behind it is a few preallocated int64 arrays instead
of Python containers:

* The free queue is a ring over an array holding every allocatable id once.  ``allocate`` takes
  a slice at the head and ``free`` writes at the tail.  The queue starts as 1, 2, ..., n - 1 and
  freed ids always queue behind the never-used ones, so the first n - 1 ids ever handed out are
  exactly the cold allocations and every later one is a reuse: two counters replace a set of
  every id ever allocated.
* Block tables are the rows of one int64 matrix, grown by doubling, null-padded.  A request owns
  a row for its lifetime; freed rows are reused.  Every entry ``allocate_slots`` writes is also
  logged as a ``(row, column, block id)`` delta, so a device copy of the matrix
  (``worker.block_tables.DeviceBlockTables``) stays current by uploading the deltas alone:
  one id per request whenever a decode step crosses a block boundary, instead of re-packing
  every table every step.

Beyond the reference, a request can be forked (``KVCacheManager.fork``: the full blocks of the parent
are shared and counted, the block that both would go on writing is copied) and the live blocks can be
moved to the lowest ids (``KVCacheManager.compact``).  Both return block pairs for
``PagedKVCachePool.copy_blocks``, which has to run before anything else writes those blocks.
"""

from __future__ import annotations

from collections.abc import Iterable, Sequence

import numpy as np

NULL_BLOCK_ID = 0


def num_blocks_for_tokens(num_tokens: int, block_size: int) -> int:
    """Blocks needed to hold ``num_tokens`` tokens (ceil). Reference block_manager.py:20-22."""
    return -(-num_tokens // block_size)


def required_pool_blocks(requests: Iterable, max_running_requests: int, block_size: int) -> int:
    """Pool size (null block included) that no ``max_running_requests`` concurrent requests can exhaust.

    A request holds at most ``prompt_len + max_new_tokens - 1`` tokens (its last generated token is
    never fed back), so the bound is the blocks of the largest ``max_running_requests`` of those.
    Reference block_manager.py:25-32.
    """
    peaks = np.sort(np.fromiter((r.prompt_len + r.max_new_tokens - 1 for r in requests), dtype=np.int64))[::-1]
    top = peaks[:max_running_requests]
    return 1 + int(np.sum(-(-top // block_size)))


class FreeKVCacheBlockQueue:
    """FIFO queue of the free physical block ids 1..num_blocks-1 on a ring buffer.

    Reference block_manager.py:35-76: ``allocate(n)`` returns the n oldest free ids (RuntimeError
    when fewer are free), ``free(ids)`` queues ids behind the rest; counters ``num_free_blocks``,
    ``num_used_blocks`` (null block excluded), ``peak_used_blocks``, ``block_cold_allocation_count``
    (first allocations of an id), ``reuse_count`` and ``release_count``.  Only ids this queue handed
    out may be freed, once each (as the reference assumes); freeing more ids than are allocated
    raises RuntimeError instead of corrupting the queue.
    """

    def __init__(self, num_blocks: int):
        if num_blocks < 2:
            raise ValueError("num_blocks must be at least 2 (block 0 is the null block)")
        self.num_blocks = num_blocks
        self._ring = np.arange(NULL_BLOCK_ID + 1, num_blocks, dtype=np.int64)
        self._head = 0            # ring position of the oldest free id
        self._count = num_blocks - 1
        self._handed_out = 0      # ids ever handed out
        self.release_count = 0
        self.peak_used_blocks = 0

    @property
    def num_free_blocks(self) -> int:
        return self._count

    @property
    def num_used_blocks(self) -> int:
        """Allocated blocks, null block excluded."""
        return self.num_blocks - 1 - self._count

    @property
    def block_cold_allocation_count(self) -> int:
        return min(self._handed_out, self._ring.shape[0])

    @property
    def reuse_count(self) -> int:
        return self._handed_out - self.block_cold_allocation_count

    def allocate(self, num_blocks: int) -> list[int]:
        """The ``num_blocks`` oldest free ids, in queue order."""
        if num_blocks > self._count:
            raise RuntimeError(f"not enough free blocks: need {num_blocks}, have {self._count}")
        cap = self._ring.shape[0]
        start, end = self._head, self._head + num_blocks
        if end <= cap:
            taken = self._ring[start:end].tolist()
        else:
            taken = self._ring[start:].tolist() + self._ring[:end - cap].tolist()
        self._head = end % cap if cap else 0
        self._count -= num_blocks
        self._handed_out += num_blocks
        self.peak_used_blocks = max(self.peak_used_blocks, self.num_used_blocks)
        return taken

    def free(self, block_ids: Sequence[int]) -> None:
        """Queues ids behind every free one (freed blocks keep their stale contents)."""
        ids = np.asarray(block_ids, dtype=np.int64).reshape(-1)
        n = ids.shape[0]
        cap = self._ring.shape[0]
        if self._count + n > cap:
            raise RuntimeError(f"freeing {n} blocks with only {cap - self._count} allocated")
        tail = (self._head + self._count) % cap
        first = min(n, cap - tail)
        self._ring[tail:tail + first] = ids[:first]
        self._ring[:n - first] = ids[first:]
        self._count += n
        self.release_count += n

    def relabel(self, old_ids: np.ndarray, new_ids: np.ndarray) -> None:
        """Puts ``new_ids[i]`` in the place of the free id ``old_ids[i]``: the allocated block ``new_ids[i]`` has been
        moved there.  The queue's order and counters stay (a moved-out block counts as the id it stands in for)."""
        names = np.arange(self.num_blocks, dtype=np.int64)
        names[old_ids] = new_ids
        cap = self._ring.shape[0]
        at = (self._head + np.arange(self._count)) % cap
        self._ring[at] = names[self._ring[at]]


class KVCacheManager:
    """Per-request block tables grown block by block. Reference block_manager.py:79-149.

    ``block_table(idx)`` returns a request's table as a list (logical block -> physical id); the
    same tables are the rows of ``table_matrix`` (``row_of(idx)``), and ``take_deltas()`` hands out
    the entries written since the previous call.
    """

    def __init__(self, block_size: int, num_blocks: int):
        if block_size < 1:
            raise ValueError("block_size must be positive")
        self.block_size = block_size
        self.free_block_queue = FreeKVCacheBlockQueue(num_blocks)
        self._row_of: dict[int, int] = {}
        self._spare_rows: list[int] = []
        self._matrix = np.zeros((8, 8), dtype=np.int64)   # rows x blocks, null-padded
        self._blocks = np.zeros(8, dtype=np.int64)         # blocks per row
        self._tokens = np.zeros(8, dtype=np.int64)         # tokens per row
        self._refs = np.zeros(num_blocks, dtype=np.int64)  # tables that hold a block
        self._rows_used = 0
        self._delta_rows: list[np.ndarray] = []
        self._delta_cols: list[np.ndarray] = []
        self._delta_ids: list[np.ndarray] = []

    # -- counters (reference block_manager.py:97-115) -----------------------------------------
    @property
    def num_used_blocks(self) -> int:
        return self.free_block_queue.num_used_blocks

    @property
    def block_cold_allocation_count(self) -> int:
        return self.free_block_queue.block_cold_allocation_count

    @property
    def block_reuse_count(self) -> int:
        return self.free_block_queue.reuse_count

    @property
    def block_release_count(self) -> int:
        return self.free_block_queue.release_count

    @property
    def peak_used_blocks(self) -> int:
        return self.free_block_queue.peak_used_blocks

    # -- tables --------------------------------------------------------------------------------
    def block_table(self, request_idx: int) -> list[int]:
        """Logical block index -> physical block id of one request (KeyError if unknown)."""
        row = self._row_of[request_idx]
        return self._matrix[row, :self._blocks[row]].tolist()

    def row_of(self, request_idx: int) -> int:
        """The table-matrix row of a live request (KeyError if unknown)."""
        return self._row_of[request_idx]

    @property
    def table_matrix(self) -> np.ndarray:
        """``[rows, width]`` int64: row r holds its request's table, then stale ids or the null block."""
        return self._matrix

    def num_tokens(self, request_idx: int) -> int:
        return int(self._tokens[self._row_of[request_idx]])

    def take_deltas(self) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """(rows, columns, ids) of every table entry written since the last call."""
        if not self._delta_rows:
            empty = np.zeros(0, dtype=np.int64)
            return empty, empty, empty
        out = (np.concatenate(self._delta_rows), np.concatenate(self._delta_cols), np.concatenate(self._delta_ids))
        self._delta_rows, self._delta_cols, self._delta_ids = [], [], []
        return out

    def _new_row(self) -> int:
        if self._spare_rows:
            return self._spare_rows.pop()
        row = self._rows_used
        if row == self._matrix.shape[0]:
            grown = self._matrix.shape[0] * 2
            self._matrix = np.pad(self._matrix, ((0, grown - self._matrix.shape[0]), (0, 0)))
            self._blocks = np.pad(self._blocks, (0, grown - self._blocks.shape[0]))
            self._tokens = np.pad(self._tokens, (0, grown - self._tokens.shape[0]))
        self._rows_used += 1
        return row

    # -- admission and allocation (reference block_manager.py:117-149) ----------------------
    def num_admissible(self, prompt_lens: Sequence[int], num_reserved_blocks: int) -> int:
        """How many requests, in FCFS order, fit into the free blocks left after the reservation:
        the longest prefix whose block needs add up to at most that budget."""
        budget = self.free_block_queue.num_free_blocks - num_reserved_blocks
        need = -(-np.asarray(prompt_lens, dtype=np.int64) // self.block_size)
        return int(np.searchsorted(np.cumsum(need), budget, side="right"))

    def allocate_slots(self, request_idx: int, num_new_tokens: int) -> bool:
        """Adds room for ``num_new_tokens`` tokens; all-or-nothing (False leaves no trace)."""
        row = self._row_of.get(request_idx)
        have_blocks = int(self._blocks[row]) if row is not None else 0
        total = (int(self._tokens[row]) if row is not None else 0) + num_new_tokens
        extra = num_blocks_for_tokens(total, self.block_size) - have_blocks
        if extra > self.free_block_queue.num_free_blocks:
            return False
        if row is None:
            row = self._new_row()
            self._row_of[request_idx] = row
        if extra > 0:
            ids = np.asarray(self.free_block_queue.allocate(extra), dtype=np.int64)
            self._refs[ids] = 1
            self._write_table(row, have_blocks, ids)
        self._tokens[row] = total
        return True

    def _write_table(self, row: int, column: int, ids: np.ndarray) -> None:
        """Writes table entries ``[column, column + len(ids))``, the last of the row, and logs them."""
        end = column + ids.shape[0]
        if end > self._matrix.shape[1]:
            width = max(end, 2 * self._matrix.shape[1])
            self._matrix = np.pad(self._matrix, ((0, 0), (0, width - self._matrix.shape[1])))
        self._matrix[row, column:end] = ids
        self._blocks[row] = end
        self._log(np.full(ids.shape[0], row, dtype=np.int64), np.arange(column, end, dtype=np.int64), ids)

    def _log(self, rows: np.ndarray, cols: np.ndarray, ids: np.ndarray) -> None:
        self._delta_rows.append(rows)
        self._delta_cols.append(cols)
        self._delta_ids.append(ids)

    def free(self, request_idx: int) -> None:
        """Returns the request's blocks to the free queue, those that no other table holds, and its row to the spare rows."""
        row = self._row_of.pop(request_idx)
        ids = self._matrix[row, :int(self._blocks[row])].copy()
        self._refs[ids] -= 1
        self.free_block_queue.free(ids[self._refs[ids] == 0])
        self._blocks[row] = 0
        self._tokens[row] = 0
        self._spare_rows.append(row)

    # -- forks and compaction (not in the reference) ------------------------------------------
    def fork(self, parent_idx: int, child_idx: int, num_tokens: int | None = None) -> list[tuple[int, int]] | None:
        """Starts request ``child_idx`` with the parent's first ``num_tokens`` tokens (default: all of them).

        Their K/V must be in the pool already.  Full blocks are shared: nobody writes them again, and each goes back to
        the free queue with its last holder.  A block that the tokens fill in part is copied, so that parent and child
        each go on in their own.  Returns the ``(source, destination)`` pairs to copy (none or one), or None, without a
        trace, when the copy finds no free block.
        """
        parent = self._row_of[parent_idx]
        if child_idx in self._row_of:
            raise ValueError(f"request {child_idx} has a block table already")
        have = int(self._tokens[parent])
        tokens = have if num_tokens is None else int(num_tokens)
        if not 0 <= tokens <= have:
            raise ValueError(f"request {parent_idx} has {have} tokens, cannot fork {tokens}")
        full, rest = divmod(tokens, self.block_size)
        if rest and self.free_block_queue.num_free_blocks < 1:
            return None
        ids = self._matrix[parent, :full + (rest > 0)].copy()
        self._refs[ids[:full]] += 1
        pairs = []
        if rest:
            own = self.free_block_queue.allocate(1)[0]
            self._refs[own] = 1
            pairs.append((int(ids[full]), own))
            ids[full] = own
        row = self._row_of[child_idx] = self._new_row()
        if ids.shape[0]:
            self._write_table(row, 0, ids)
        self._tokens[row] = tokens
        return pairs

    def compact(self) -> list[tuple[int, int]]:
        """Gives the ``n`` blocks in use the ids ``1..n``: those above move to the free ids below.

        Tables (and their deltas) and the free queue are up to date on return.  Returns the ``(source, destination)``
        pairs; no destination is a source, and the copy has to be enqueued before the next step.
        """
        live = np.flatnonzero(self._refs)
        n = live.shape[0]
        if n != self.num_used_blocks:
            raise RuntimeError(f"{self.num_used_blocks} blocks are in use, tables hold {n}: compact() moves only blocks "
                               "of this manager's tables")
        src = live[live > n]
        if src.shape[0] == 0:
            return []
        dst = 1 + np.flatnonzero(self._refs[1:n + 1] == 0)
        moved = np.arange(self._refs.shape[0], dtype=np.int64)
        moved[src] = dst
        for row in self._row_of.values():
            ids = self._matrix[row, :int(self._blocks[row])]
            cols = np.flatnonzero(moved[ids] != ids)
            if cols.shape[0]:
                ids[cols] = moved[ids[cols]]  # a view: the matrix itself
                self._log(np.full(cols.shape[0], row, dtype=np.int64), cols, ids[cols])
        self._refs[dst] = self._refs[src]
        self._refs[src] = 0
        self.free_block_queue.relabel(dst, src)
        return list(zip(src.tolist(), dst.tolist()))


__all__ = [
    "FreeKVCacheBlockQueue",
    "KVCacheManager",
    "NULL_BLOCK_ID",
    "num_blocks_for_tokens",
    "required_pool_blocks",
]
