"""Pools of 4-bit pages, their backend in torch and eviction, on the CPU."""
import numpy as np
import pytest
import torch

from oracle import q4
from src.cache.paged_kv import BatchedPagedKVCache, LayerBlockPool, PagedKVCacheState
from src.cache.q4_kv import Q4BlockPool
from src.config import KVEviction
from src.inference.generate_with_cache import generate_with_cache
from src.kernels import reference_q4
from src.kernels.paged_attention import paged_attention
from src.model.transformer import TinyTransformerLM


def _cache(B, track=True, blocks=4):
    pool = Q4BlockPool(16, blocks, 2.0, track_weights=track)
    return BatchedPagedKVCache([PagedKVCacheState(pool=pool) for _ in range(B)], pool)


@pytest.mark.parametrize("hd", [64, 128])
def test_pages_in_torch_are_the_oracles(hd):
    rng = np.random.default_rng(hd)
    for is_key in (True, False):
        pool = torch.from_numpy(rng.integers(0, 256, (3, 2, q4.page_bytes(hd)), dtype=np.uint8))
        want = pool.numpy().copy()
        rows = torch.randn(12, 2, hd)
        rows[3] = 1.5
        rows[4, 0, 3] = float("nan")
        rows[5, 1, 9] = float("inf")
        rows[6] *= 1e-7
        rows[7] = rows[7].mul(4).round() / 4
        slots = torch.randperm(48)[:12]
        reference_q4.put_rows(pool, slots // 16, slots % 16, rows, is_key)
        for i, s in enumerate(slots.tolist()):
            for h in range(2):
                q4.put(want, s // 16, h, s % 16, rows[i, h].numpy(), is_key)
        assert np.array_equal(pool.numpy(), want)
        got = reference_q4.values(pool, hd, is_key).numpy()
        assert np.array_equal(got, q4.values(want, hd, is_key).astype(np.float32), equal_nan=True)


def test_pool_follows_the_block_pools_order_and_accounting():
    plain, q = LayerBlockPool(16, 3, 2.0), Q4BlockPool(16, 3, 2.0, track_weights=True)
    for pool in (plain, q):
        pool.ensure_initialized(2, 64, torch.float32, torch.device("cpu"))
    assert [q.allocate_block() for _ in range(7)] == [plain.allocate_block() for _ in range(7)]
    for pool in (plain, q):
        pool.release_blocks([4, 1])
        pool.release_block(2)
    assert q.free_block_ids == plain.free_block_ids and q.capacity_blocks == plain.capacity_blocks
    assert q.k_blocks.shape == (q.capacity_blocks, 2, 576) and q.weights.shape == (q.capacity_blocks, 2, 16)
    assert q.bytes_per_block() == 2 * 2 * 576 + 2 * 16 * 4
    state = PagedKVCacheState(pool=q, block_ids=[0, 3], seq_len=20)
    assert state.live_bytes() == 20 * 2 * (2 * 36 + 4)
    with pytest.raises(ValueError, match="block_size"):
        Q4BlockPool(32, 3, 2.0)
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        Q4BlockPool(16, 3, 2.0).ensure_initialized(2, 80, torch.float32, torch.device("cpu"))


def test_reference_backend_attends_to_the_pages_values_and_keeps_their_weights():
    torch.manual_seed(0)
    cache = _cache(3)
    H, hd, T = 2, 64, 21
    cur = torch.tensor([21, 9, 0])
    for _ in range(2):
        k, v = torch.randn(3, H, T, hd), torch.randn(3, H, T, hd)
        cache.append_batch(k, v, current_lengths=cur)
        q = torch.randn(3, 2 * H, T, hd)  # two query heads per KV head
        before = cache.pool.weights.clone()
        out = paged_attention("paged_reference", q, cache, cur)
        table = cache.page_table_tensor().numpy()
        lens = [s.seq_len for s in cache.states]
        want, added = q4.attention(q.double().numpy(), q4.values(cache.pool.k_blocks.numpy(), hd, True),
                                   q4.values(cache.pool.v_blocks.numpy(), hd, False), table, lens, cur.tolist())
        # fp32 products and softmax of a few dozen keys: 64 roundings of 2^-24 of the scores' and values' size
        assert np.abs(out.double().numpy() - want).max() < 64 * 2.0 ** -24 * 16
        assert np.abs((cache.pool.weights - before).double().numpy() - added).max() < 64 * 2.0 ** -24 * 42
    assert not paged_attention("paged_reference", q, cache, cur)[2].any()


def test_eviction_moves_rows_and_releases_blocks():
    torch.manual_seed(1)
    cache = _cache(3, blocks=2)
    H, hd = 2, 64
    lens = torch.tensor([70, 33, 12])
    cache.append_batch(torch.randn(3, H, 70, hd), torch.randn(3, H, 70, hd), current_lengths=lens)
    pool = cache.pool
    pool.weights.copy_(torch.rand(pool.weights.shape))
    pool.weights[cache.states[0].block_ids[1]] = 0.5  # equal ones
    before = (pool.k_blocks.clone(), pool.v_blocks.clone(), pool.weights.clone())
    old = [list(s.block_ids) for s in cache.states]
    kept = cache.evict(keep=24, window=6, limit=32)
    assert [s.seq_len for s in cache.states] == [24, 24, 12] and kept[2] is None and cache.states[2].block_ids == old[2]
    want = q4.evict(before[2].numpy(), [old[0], old[1]], [70, 33], 24, 6)
    k, v = pool.tiles(torch.arange(pool.capacity_blocks))
    k0, v0 = reference_q4.values(before[0], hd, True), reference_q4.values(before[1], hd, False)
    for b in (0, 1):
        assert kept[b].tolist() == want[b]
        ids = cache.states[b].block_ids
        assert len(ids) == 2 and not set(ids) & set(old[b]) and not set(ids) & set(pool.free_block_ids)
        assert set(old[b]) <= set(pool.free_block_ids)
        for h in range(H):
            for i, t in enumerate(want[b][h]):
                src, dst = (old[b][t // 16], h, t % 16), (ids[i // 16], h, i % 16)
                assert torch.equal(k[dst], k0[src]) and torch.equal(v[dst], v0[src])
                assert pool.weights[dst] == before[2][src]
    for blk in old[0] + old[1]:
        assert not pool.k_blocks[blk].any() and not pool.v_blocks[blk].any() and not pool.weights[blk].any()
    assert cache.evict(keep=24, window=6) == [None] * 3  # nothing left to cut


def test_eviction_refusals():
    cache = _cache(1, track=False)
    with pytest.raises(ValueError, match="attention weights"):
        cache.evict(4, 1)
    plain = BatchedPagedKVCache([PagedKVCacheState(pool=LayerBlockPool(16, 2, 2.0))])
    with pytest.raises(ValueError, match="attention weights"):
        plain.evict(4, 1)
    cache = _cache(1)
    for keep, window in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            cache.evict(keep, window)
    cache.append_batch(torch.randn(1, 2, 20, 64), torch.randn(1, 2, 20, 64))
    twice = BatchedPagedKVCache([cache.states[0]] * 2, cache.pool)
    with pytest.raises(ValueError, match="twice"):
        twice.evict(4, 1)
    for bad in (dict(limit=4, keep=5, window=1), dict(limit=4, keep=4, window=5), dict(limit=4, keep=0, window=0)):
        with pytest.raises(ValueError):
            KVEviction(**bad)


def _model(**kw):
    torch.manual_seed(3)
    return TinyTransformerLM(vocab_size=50, d_model=128, num_heads=2, num_layers=2, d_ff=64, max_seq_len=96,
                             attention_backend="paged_reference", kv_pool_initial_blocks=2, **kw).eval()


def test_model_over_4_bit_pages_with_eviction():
    ids = torch.randint(0, 50, (2, 40), generator=torch.Generator().manual_seed(0))
    lengths = torch.tensor([40, 23])
    model = _model(kv_cache_dtype="int4", track_attention_weights=True)
    full = generate_with_cache(model, ids, [12, 9], lengths)
    model.reset_paged_cache_pools()
    # a budget that nothing reaches leaves the run as it was
    same = generate_with_cache(model, ids, [12, 9], lengths, eviction=KVEviction(limit=64, keep=32, window=8))
    assert all(torch.equal(a, b) for a, b in zip(full["generated_ids"], same["generated_ids"]))
    model.reset_paged_cache_pools()
    cut = generate_with_cache(model, ids, [12, 9], lengths, eviction=KVEviction(limit=30, keep=20, window=8))
    assert cut["generated_tokens_per_request"] == [12, 9]
    for cache in cut["kv_caches"]:
        assert all(s.seq_len <= 30 for s in cache.states)
        assert [s.seq_len for s in cache.states] == [s.seq_len for s in cut["kv_caches"][0].states]
    assert torch.equal(full["generated_ids"][0][:41], cut["generated_ids"][0][:41])  # the prompt's token came first


def test_model_refusals():
    with pytest.raises(ValueError, match="int4"):
        _model(kv_cache_dtype="int8")
    with pytest.raises(ValueError, match="track_attention_weights"):
        _model(track_attention_weights=True)


def test_step_events_count_4_bit_bytes():
    from src.serving.continuous_generate import run_prefill_chunk
    from src.serving.request import InferenceRequest

    model = _model(kv_cache_dtype="int4", track_attention_weights=True)
    requests = [InferenceRequest(i, 0.0, n, 4, torch.arange(n)) for i, n in enumerate((12, 7))]
    event = run_prefill_chunk(model, requests, 16, "cpu", 0.0, 0)
    # 5 padded rows; a token takes 2 x 36 bytes and its total in each of 2 heads and 2 layers
    assert event["padding_waste_tokens"] == 5
    assert event["padding_waste_bytes_est"] == 5 * 2 * 2 * (2 * 36 + 4)
