"""The 4-bit pool under the model and the runner: whole runs of prefill chunks, decode steps, forks, compactions, swaps and
graphs.

Runs that should not differ are compared bit for bit: the same launches on the same values, only block ids, tables' device
copies or the way blocks got their contents differ.  What the attention computes is checked against 64 bits elsewhere; here
each form of the layer is compared with the same operators called one by one."""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import data_plane
from mini_infra_qwen3_amd.core import KVCacheManager, PagedCacheConfig
from mini_infra_qwen3_amd.core.scheduler import SchedulePhase
from mini_infra_qwen3_amd.engine import PagedScheduleBackend, run_scheduler
from mini_infra_qwen3_amd.model import (PagedAttentionMetadata, PagedMixedMetadata, PagedPrefillMetadata, Qwen3Config,
                                        Qwen3ForCausalLM, init_random_)
from mini_infra_qwen3_amd.worker import (DeviceBlockTables, HostSwapPool, KVCache, PagedKVCachePool, PagedKVCachePoolFp4,
                                         PagedRunner, load_kv_blocks, save_kv_blocks)
from mini_infra_qwen3_amd.workloads import serving_requests
from oracle import fp4_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    config = Qwen3Config(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=3,
                         num_attention_heads=16, num_key_value_heads=8, head_dim=128)
    net = Qwen3ForCausalLM(config, exact=False)
    init_random_(net, seed=0, std=0.05, untied_head_seed=1234)
    return net.to(torch.bfloat16).to("cuda:0").eval()


def prompt(seed, n):
    return np.random.default_rng(seed).integers(0, 1000, n).tolist()


class Session:
    """A manager, a 4-bit pool and a runner; every token that a step needs is given, so runs can be compared."""

    def __init__(self, model, num_blocks=64, block_size=16, tables=False):
        config = model.config
        self.manager = KVCacheManager(block_size, num_blocks)
        self.pool = PagedKVCachePoolFp4(config.num_hidden_layers, num_blocks, block_size, 8, 128, "cuda:0")
        self.runner = PagedRunner(model)
        self.tables = DeviceBlockTables(self.manager, 8, 32, "cuda:0") if tables else None
        self.log = []

    def prefill(self, request, ids, chunk=20):
        for start in range(0, len(ids), chunk):
            part = ids[start:start + chunk]
            assert self.manager.allocate_slots(request, len(part))
            table = [self.manager.block_table(request)]
            out = self.runner.run_prefill_chunk_step([part], [start], table, self.pool)
            self.runner.store_prefill(self.pool, out.prefill_cache, table, [len(part)], [start])
        self.log.append(out.next_tokens)

    def decode(self, requests, tokens):
        positions = [self.manager.num_tokens(r) for r in requests]
        for r in requests:
            assert self.manager.allocate_slots(r, 1)
        if self.tables is not None:
            step = self.runner.prepare_decode_from_tables(self.tables, requests, tokens, positions)
        else:
            step = self.runner.prepare_decode_inputs([self.manager.block_table(r) for r in requests], tokens, positions,
                                                     self.manager.block_size)
        self.log.append(self.runner.run_decode_step(*step, self.pool).next_tokens)

    def fork(self, parent, child, n=None):
        pairs = self.manager.fork(parent, child, n)
        self.pool.copy_blocks([s for s, _ in pairs], [d for _, d in pairs])

    def compact(self):
        pairs = self.manager.compact()
        self.pool.copy_blocks([s for s, _ in pairs], [d for _, d in pairs])
        return len(pairs)

    def contents(self, request):
        """The request's K and V of every layer, as stored: [layers, 2, tokens, heads, 128] bf16."""
        ids = torch.tensor([self.manager.block_table(request)])
        n = self.manager.num_tokens(request)
        return torch.stack([torch.stack((k[0, :, :n], v[0, :, :n])) for k, v in self.pool.gather_blocks(ids)]).cpu()


def same(a, b, requests):
    assert a.log == b.log
    for r in requests:
        assert torch.equal(a.contents(r), b.contents(r))


@pytest.mark.parametrize("block_size", [16, 48])
def test_a_fork_is_a_request_of_its_own(native_lib, model, block_size):
    """A forked request against one that was prefilled with the same tokens, decoding in the same batches."""
    ids, a, b = prompt(0, 53), Session(model, block_size=block_size), Session(model, block_size=block_size)
    for s in (a, b):
        s.prefill(0, ids)
    a.prefill(1, ids)
    b.fork(0, 1)
    b.log.append(b.log[-1])
    same(a, b, (0, 1))
    for step in range(14):
        for s in (a, b):
            s.decode([0, 1], [step, 500 + step])
    same(a, b, (0, 1))
    for s in (a, b):
        s.manager.free(0)
        s.decode([1], [7])
    same(a, b, (1,))
    assert b.manager.num_used_blocks == a.manager.num_used_blocks


def test_a_forked_prefix(native_lib, model):
    ids = prompt(1, 60)
    a, b = Session(model), Session(model)
    for s in (a, b):
        s.prefill(0, ids, chunk=20)
    a.prefill(1, ids[:40], chunk=20)
    a.log.pop()
    b.fork(0, 1, 40)
    same(a, b, (0, 1))
    for s in (a, b):
        s.decode([1, 0], [3, 4])
    same(a, b, (0, 1))


@pytest.mark.parametrize("tables", [False, True])
def test_compaction_changes_nothing(native_lib, model, tables):
    a, b = Session(model, tables=tables), Session(model, tables=tables)
    for s in (a, b):
        for r in range(4):
            s.prefill(r, prompt(r, 30 + 11 * r))
        s.decode([0, 1, 2, 3], [1, 2, 3, 4])
        s.manager.free(0)
        s.manager.free(2)
    assert b.compact() > 0
    assert max(max(b.manager.block_table(r)) for r in (1, 3)) == b.manager.num_used_blocks
    same(a, b, (1, 3))
    for step in range(20):
        for s in (a, b):
            s.decode([3, 1], [10 + step, 60 + step])
            if step == 9:
                s.prefill(7, prompt(9, 50))
    same(a, b, (1, 3, 7))


def test_graphs_replay_the_eager_steps(native_lib, model):
    """Decode graphs of the step's own batch over device tables; the host goes on with its own work between replays."""
    a, b = Session(model, tables=True), Session(model, tables=True)
    for s in (a, b):
        s.prefill(0, prompt(3, 33))
        s.prefill(1, prompt(4, 47))
    b.runner.enable_decode_graphs(b.pool, max_batch=2, max_blocks=32, batch_buckets=[2], tables=b.tables)
    for step in range(20):
        for s in (a, b):
            s.decode([0, 1], [step, 999 - step])
            if step == 7:
                s.fork(1, 5)
            if step == 12:
                s.manager.free(0)
                s.compact()
                s.fork(5, 0)
        same(a, b, (0, 1))
        torch.cuda.synchronize()


def test_prefill_graphs_write_the_same_rows(native_lib, model):
    """Chunks in a graph's padded width: every row of the chunk goes into its slot, and nowhere else."""
    s = Session(model)
    s.runner.enable_prefill_graphs(s.pool, max_rows=1, max_width=32, max_history_blocks=8, width_quantum=32)
    before = s.pool.storage.clone()
    s.prefill(0, prompt(5, 50), chunk=32)
    t = s.manager.block_table(0)
    untouched = [b for b in range(s.pool.num_blocks) if b not in t]
    assert torch.equal(s.pool.storage[:, :, untouched], before[:, :, untouched])
    e = Session(model)
    e.prefill(0, prompt(5, 50), chunk=32)
    assert s.log == e.log
    # One padded width more or less changes a matrix product's shape, so later layers may differ by roundings, but the first
    # layer's rows depend on nothing but their token.
    assert torch.equal(s.contents(0)[0], e.contents(0)[0])


def qkv(model, tokens, seed):
    gen = torch.Generator().manual_seed(seed)
    config = model.config
    return [torch.randn(1, tokens, heads * 128, generator=gen).to(torch.bfloat16).cuda()
            for heads in (config.num_attention_heads, 8, 8)]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("block_size", [16, 32])
def test_mixed_step_is_its_two_parts(native_lib, model, ragged, block_size):
    """Chunk rows of 0, 1 and 29 tokens and four decode rows, one of them padding."""
    layer = model.model.layers[0].self_attn
    rng = np.random.default_rng(2)
    sub = block_size // 16
    pools = [fp4_ref.to_torch(fp4_ref.random_pool(rng, 40 * sub, 8), sub).cuda() for _ in range(2)]
    again = [p.clone() for p in pools]
    rows, width, decode_rows = 3, 29, 4
    lens, starts = [29, 0, 1], [3 * block_size + 5, 0, 17]
    c = 34 if ragged else rows * width
    first = [3, 0, 33]
    total = c + decode_rows
    history = torch.zeros(rows, 4, dtype=torch.long)
    history[0], history[2, :2] = torch.tensor([9, 4, 30, 31]), torch.tensor([12, 13])
    tables = torch.tensor([[1, 2, 3], [0, 0, 0], [5, 0, 0], [6, 7, 8]])
    contexts = torch.tensor([2 * block_size + 1, 0, 1, 3 * block_size])
    slots = torch.tensor([3 * block_size, -1, 5 * block_size, 8 * block_size + block_size - 1])
    q, k, v = qkv(model, total, 3)
    cos, sin = model.model.rotary_emb(torch.arange(total, device="cuda").unsqueeze(0), torch.bfloat16)
    dev = lambda x: (torch.tensor(x) if isinstance(x, list) else x).cuda()  # noqa: E731
    meta = PagedMixedMetadata(
        prefill=PagedPrefillMetadata(dev(history), dev(starts), dev(lens)),
        decode=PagedAttentionMetadata(dev(slots), dev(tables), dev(contexts)),
        prefill_rows=rows, prefill_width=width, chunk_first=dev(first) if ragged else None, chunk_tokens=c if ragged else 0)
    with torch.inference_mode():
        got, present = layer._fp4(q, k, v, cos, sin, pools, meta, None)
        q_rot, k_rot, v_rows = data_plane.qk_norm_rope(q, k, v, layer.q_norm.weight, layer.k_norm.weight, cos, sin,
                                                       layer.q_norm.eps)
        data_plane.reshape_and_cache_fp4([k_rot[c:].unsqueeze(2)], [v_rows[c:].unsqueeze(2)], dev(slots), [again[0]], [again[1]])
        padded = [torch.zeros(rows, width, t.shape[1], 128, dtype=torch.bfloat16, device="cuda") for t in (q_rot, k_rot, v_rows)]
        for r, n in enumerate(lens):
            at = first[r] if ragged else (r + 1) * width - n
            for p, t in zip(padded, (q_rot, k_rot, v_rows)):
                p[r, width - n:] = t[at:at + n]
        chunk = data_plane.chunked_prefill_attention_fp4(*(p.transpose(1, 2) for p in padded), *again, dev(history), dev(starts),
                                                         dev(lens), layer.scaling)
        want = torch.zeros(1, total, 2048, dtype=torch.bfloat16, device="cuda")
        for r, n in enumerate(lens):
            at = first[r] if ragged else (r + 1) * width - n
            want[0, at:at + n] = chunk[r, width - n:]
        want[0, c:] = data_plane.paged_decode_attention_fp4(q_rot[c:], *again, dev(tables), dev(contexts), layer.scaling)
        assert float(want[0, c:].float().abs().amax()) > 0
        want = layer.o_proj(want)
    assert torch.equal(pools[0], again[0]) and torch.equal(pools[1], again[1])
    assert torch.equal(got, want)
    shape = (1, 8, c, 128) if ragged else (rows, 8, width, 128)
    for t, flat in zip(present, (k_rot, v_rows)):
        assert t.shape == shape and torch.equal(t.transpose(1, 2).reshape(c, 8, 128), flat[:c])


@pytest.mark.parametrize("heads,kv_heads,block_size", [(16, 8, 16), (5, 1, 32), (6, 3, 48), (8, 8, 16)])
@pytest.mark.parametrize("tokens", [1, 37])
def test_norm_rope_stores_what_the_two_calls_store(native_lib, heads, kv_heads, block_size, tokens):
    """Slots -1, past the pool and unwritten tokens' bytes included; a row with an infinity is stored as NaN."""
    gen = torch.Generator().manual_seed(tokens + heads)
    randn = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    qkv = randn(tokens, (heads + 2 * kv_heads) * 128)
    q, k, v = qkv[:, :heads * 128], qkv[:, heads * 128:(heads + kv_heads) * 128], qkv[:, (heads + kv_heads) * 128:]
    if tokens > 1:
        v[3, 40], k[4, 7] = float("inf"), float("nan")
    weights, cos, sin = (1 + 0.1 * randn(128), 1 + 0.1 * randn(128)), randn(tokens, 128), randn(tokens, 128)
    sub, blocks = block_size // 16, 4
    slots = torch.randperm(blocks * block_size, generator=gen)[:tokens]
    if tokens > 1:
        slots[5], slots[9], slots[11] = -1, blocks * block_size, -7
    table = torch.stack((slots, slots), 1).cuda()[:, 0]  # a stride of 2
    rng = np.random.default_rng(tokens)
    before = [fp4_ref.to_torch(fp4_ref.random_pool(rng, blocks * sub, kv_heads), sub).cuda() for _ in range(2)]
    want = [p.clone() for p in before]
    rows = data_plane.qk_norm_rope(q, k, v, *weights, cos, sin, 1e-6)
    data_plane.reshape_and_cache_fp4([rows[1].unsqueeze(2)], [rows[2].unsqueeze(2)], table, [want[0]], [want[1]])
    for keep in (True, False):
        pools = [p.clone() for p in before]
        got = data_plane.qk_norm_rope(q, k, v, *weights, cos, sin, 1e-6, slot_mapping=table, key_pool=pools[0],
                                      value_pool=pools[1], rows=keep)
        assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
        for a, b in zip(got, rows if keep else (rows[0], None, None)):
            assert a is b is None or torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert not torch.equal(want[0], before[0])
    with pytest.raises(ValueError, match="KV heads"):
        data_plane.qk_norm_rope(q, k, v, *weights, cos, sin, 1e-6, slot_mapping=table,
                                key_pool=torch.zeros(2, 1, kv_heads + 1, 1088, dtype=torch.uint8, device="cuda"),
                                value_pool=torch.zeros(2, 1, kv_heads + 1, 1088, dtype=torch.uint8, device="cuda"))
    odd = torch.zeros(tokens, heads * 128 + 8, dtype=torch.bfloat16, device="cuda")[:, 1:heads * 128 + 1]
    with pytest.raises(ValueError, match="aligned"):
        data_plane.qk_norm_rope(odd, k, v, *weights, cos, sin, 1e-6, slot_mapping=table, key_pool=pools[0], value_pool=pools[1])


def test_swap_and_files_keep_the_bytes(native_lib, tmp_path):
    pool = PagedKVCachePoolFp4(2, 12, 32, 3, 128, "cuda:0")
    gen = torch.Generator().manual_seed(0)
    pool.storage.copy_(torch.randint(0, 255, pool.storage.shape, generator=gen, dtype=torch.uint8))
    want = pool.storage.clone()
    assert pool.bytes_per_block * 12 == pool.total_bytes == pool.storage.numel()
    swap = HostSwapPool(6, pool)
    slots = swap.swap_out(pool, [3, 7, 1])
    save_kv_blocks(tmp_path / "blocks", pool, [5, 2])
    swap.swap_in(pool, slots, [8, 9, 10])
    load_kv_blocks(tmp_path / "blocks", pool, [4, 11])
    want[:, :, [8, 9, 10, 4, 11]] = want[:, :, [3, 7, 1, 5, 2]]
    assert torch.equal(pool.storage, want)
    other = PagedKVCachePool(2, 12, 32, 3, 128, torch.bfloat16, "cuda:0")
    with pytest.raises(ValueError, match="geometry"):
        swap.swap_out(other, [1])
    with pytest.raises(ValueError, match="does not match"):
        load_kv_blocks(tmp_path / "blocks", other, [1, 2])


def test_copy_blocks_of_pools(native_lib):
    for pool in (PagedKVCachePool(3, 10, 16, 2, 128, torch.float16, "cuda:0"), PagedKVCachePoolFp4(3, 10, 16, 2, 128, "cuda:0")):
        gen = torch.Generator().manual_seed(1)
        flat = pool.storage.view(torch.uint8)
        flat.copy_(torch.randint(0, 255, flat.shape, generator=gen, dtype=torch.uint8))
        want = flat.clone()
        pool.copy_blocks([1, 1, 9], [4, 5, 2])
        pool.copy_blocks([], [])
        pool.copy_blocks(torch.tensor([7]), torch.tensor([8]))
        want[:, :, [4, 5, 2, 8]] = want[:, :, [1, 1, 9, 7]]
        assert torch.equal(flat, want)
        for src, dst, what in (([1], [1], "source as well"), ([1, 2], [3, 2], "source as well"), ([1, 2], [3, 3], "unique"),
                               ([10], [1], "lie in"), ([1], [-1], "lie in"), ([1, 2], [3], "destinations")):
            with pytest.raises(ValueError, match=what):
                pool.copy_blocks(src, dst)
        assert torch.equal(flat, want)


def test_write_and_gather_of_the_pool(native_lib):
    """write_prefill into scattered slots, gather_blocks by table: the quantised values of each row."""
    pool = PagedKVCachePoolFp4(2, 6, 32, 3, 128, "cuda:0")
    gen = torch.Generator().manual_seed(2)
    layers = [tuple(torch.randn(2, 3, 9, 128, generator=gen).to(torch.bfloat16) for _ in range(2)) for _ in range(2)]
    rows, positions = torch.tensor([0, 1, 1, 0]), torch.tensor([8, 0, 4, 3])
    slots = torch.tensor([2 * 32 + 31, 5 * 32, 5 * 32 + 17, 32 + 3])
    pool.write_prefill(KVCache([(k.cuda(), v.cuda()) for k, v in layers]), rows.cuda(), positions.cuda(), slots.cuda())
    got = pool.gather_blocks(torch.tensor([[1, 2, 5]]))
    place = {1: 0, 2: 1, 5: 2}
    for (key, value), sources in zip(got, layers):
        for tensor, source in ((key, sources[0]), (value, sources[1])):
            assert tensor.shape == (1, 3, 96, 128) and tensor.dtype == torch.bfloat16
            want = np.zeros((96, 3, 128))
            for r, p, s in zip(rows.tolist(), positions.tolist(), slots.tolist()):
                for h in range(3):
                    want[place[s // 32] * 32 + s % 32, h] = fp4_ref.values_of(*fp4_ref.quantize_row(source[r, h, p].double().numpy()))
            assert np.array_equal(tensor[0].transpose(0, 1).double().cpu().numpy(), want)


@pytest.mark.parametrize("mixed", [False, True])
def test_scheduled_run(native_lib, model, mixed):
    """The serving loop on a 4-bit pool: chunked prompts, forty decode steps and, when asked, mixed steps; a compaction after
    every tenth step changes no token."""
    requests = [type(r)(r.request_idx, tuple(t % 1000 for t in r.token_ids), r.max_new_tokens, r.arrival_ms)
                for r in serving_requests(seed=3, num_requests=8, min_prompt=20, max_prompt=200, max_new_tokens=40)]
    clock = lambda out: 10.0 if out.phase is SchedulePhase.PREFILL else 5.0  # noqa: E731

    def run(compacting):
        backend = PagedScheduleBackend(model, requests, 4, PagedCacheConfig(kv_bits=4), decode_graphs=True, mixed_graphs=mixed,
                                       mixed_graph_rows=2, mixed_graph_tokens=64, mixed_graph_decode_rows=4)
        assert isinstance(backend.pool, PagedKVCachePoolFp4)
        moved, steps, execute = 0, 0, backend.execute_decode

        def decode(states):
            nonlocal moved, steps
            steps += 1
            if compacting and steps % 10 == 0:
                moved += backend.compact_cache()
            return execute(states)

        backend.execute_decode = decode
        result = run_scheduler(backend, requests, token_budget=64, max_running_requests=4, eos_token_id=-1, stop_on_eos=False,
                               step_clock=clock, mixed_batching=mixed)
        assert backend.kv_cache_manager.num_used_blocks == 0
        return result, moved

    plain, _ = run(False)
    moving, moved = run(True)
    assert moved > 0
    assert (plain.num_steps(SchedulePhase.MIXED) > 0) == mixed
    assert all(len(t) == 40 for t in plain.tokens.values()) and plain.tokens == moving.tokens
