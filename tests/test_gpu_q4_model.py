"""The 4-bit cache through the framework on the GPU: pools, the attention dispatch, the model, eviction and the
continuous-batching executors, against the torch backend on the same pages."""
import numpy as np
import pytest
import torch

from oracle import q4
from src.cache.paged_kv import BatchedPagedKVCache, PagedKVCacheState
from src.cache.q4_kv import Q4BlockPool
from src.config import KVEviction
from src.inference.generate_with_cache import generate_with_cache
from src.kernels.paged_attention import paged_attention
from src.model.transformer import TinyTransformerLM
from src.serving.continuous_generate import StepExecutor, run_decode_step, run_prefill_chunk
from src.serving.request import InferenceRequest
from src.serving.scheduler import ContinuousBatchingScheduler

pytestmark = pytest.mark.gpu


def _caches(device, B):
    pools = [Q4BlockPool(16, 4, 2.0, track_weights=True) for _ in range(2)]
    return [BatchedPagedKVCache([PagedKVCacheState(pool=p) for _ in range(B)], p) for p in pools]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd, H, Hk", [(64, 8, 8), (128, 6, 2)])
def test_steps_and_eviction_as_the_cpu_pool_does_them(device, dtype, hd, H, Hk):
    """Chunks, single tokens and evictions in turn: equal pages and choices, and attention over them."""
    g = torch.Generator().manual_seed(hd)
    rng = np.random.default_rng(0)
    gpu, cpu = _caches(device, 3)
    for step, T in enumerate([37, 1, 24, 1, 1, 50, 1]):
        cur = [T, max(T // 2, 1), 0 if T > 1 else 1]
        k, v = (torch.randn(3, Hk, T, hd, generator=g).to(dtype) for _ in range(2))
        lens = torch.tensor(cur)
        assert torch.equal(gpu.append_batch(k.to(device), v.to(device), lens).cpu(), cpu.append_batch(k, v, lens))
        assert [s.block_ids for s in gpu.states] == [s.block_ids for s in cpu.states]
        assert torch.equal(gpu.pool.k_blocks.cpu(), cpu.pool.k_blocks)
        assert torch.equal(gpu.pool.v_blocks.cpu(), cpu.pool.v_blocks)
        q = torch.randn(3, H, T, hd, generator=g).to(dtype)
        out = paged_attention("hip_paged", q.to(device), gpu, lens)
        # bf16: the torch backend's products round to bf16, so it gets the fp32 values of the same q
        want = paged_attention("paged_reference", q.float(), cpu, lens)
        tol = 1e-4 if dtype == torch.float32 else 2.0 ** -8 * 4 + 2.0 ** -7
        assert float((out.float().cpu() - want).abs().max()) < tol
        # the same sums of the same weights, rounded in another order
        assert float((gpu.pool.weights.cpu() - cpu.pool.weights).abs().max()) < (1e-3 if dtype == torch.float32 else 2e-2)
        if step % 2:
            w = torch.from_numpy(rng.random(cpu.pool.weights.shape, dtype=np.float32))
            gpu.pool.weights.copy_(w)
            cpu.pool.weights.copy_(w)
            a, b = gpu.evict(20, 5), cpu.evict(20, 5)
            assert [x is None for x in a] == [x is None for x in b]
            assert all(x is None or torch.equal(x.cpu(), y) for x, y in zip(a, b))
            assert torch.equal(gpu.pool.k_blocks.cpu(), cpu.pool.k_blocks)
            assert torch.equal(gpu.pool.weights.cpu(), cpu.pool.weights)
            assert gpu.pool.free_block_ids == cpu.pool.free_block_ids


def _model(device, dtype=torch.float32, layers=2, **kw):
    torch.manual_seed(7)
    m = TinyTransformerLM(vocab_size=200, d_model=256, num_heads=4, num_layers=layers, d_ff=256, max_seq_len=256,
                          attention_backend="hip_paged", kv_cache_dtype="int4", **kw)
    return m.to(device=device, dtype=dtype).eval()


def test_model_steps_equal_the_torch_backends(device):
    """One layer, whose keys and values do not depend on attention: equal pages, and logits that differ by
    what the attention outputs do (some 1e-6 of values of size 1, through weights of norm below 10)."""
    ids = torch.randint(0, 200, (3, 50), generator=torch.Generator().manual_seed(1)).to(device)
    models = [_model(device, layers=1) for _ in range(2)]
    models[1].set_attention_backend("paged_reference")
    caches, pos = [None, None], 0
    for T in (40, 1, 1, 6, 1):
        logits = [None, None]
        for i, m in enumerate(models):
            with torch.no_grad():
                logits[i], caches[i] = m(ids[:, pos:pos + T], kv_caches=caches[i], use_cache=True, position_offset=pos)
        assert float((logits[0] - logits[1]).abs().max()) < 1e-3
        assert torch.equal(models[0].layer_block_pools[0].k_blocks, models[1].layer_block_pools[0].k_blocks)
        assert torch.equal(models[0].layer_block_pools[0].v_blocks, models[1].layer_block_pools[0].v_blocks)
        pos += T
    # 4.5 bits a value
    assert caches[0][0].live_bytes() == 4 * 72 * 3 * pos


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_generation_with_eviction_holds_its_budget(device, dtype):
    ids = torch.randint(0, 200, (3, 60), generator=torch.Generator().manual_seed(2)).to(device)
    model = _model(device, dtype, track_attention_weights=True)
    free = generate_with_cache(model, ids, 4)
    model.reset_paged_cache_pools()
    cut = generate_with_cache(model, ids, 40, eviction=KVEviction(limit=48, keep=32, window=12))
    assert cut["generated_tokens_per_request"] == [40] * 3
    for cache in cut["kv_caches"]:
        assert all(s.seq_len <= 48 and len(s.block_ids) == -(-s.seq_len // 16) for s in cache.states)
        live = torch.tensor(sorted(b for s in cache.states for b in s.block_ids), device=device)
        rest = torch.ones(cache.pool.capacity_blocks, dtype=torch.bool, device=device)
        rest[live] = False
        assert not cache.pool.weights[rest].any() and bool((cache.pool.weights[live] >= 0).all())
    assert torch.equal(free["generated_ids"][0][:61], cut["generated_ids"][0][:61])


def test_continuous_batching_with_eviction(device):
    model = _model(device, track_attention_weights=True)
    g = torch.Generator().manual_seed(5)
    requests = [InferenceRequest(i, 0.0, n, new, torch.randint(0, 200, (n,), generator=g))
                for i, (n, new) in enumerate([(90, 10), (33, 20), (64, 5), (120, 12)])]
    executor = StepExecutor(model, device, eviction=KVEviction(limit=56, keep=40, window=10))
    seen = []
    executor.observer = lambda plan, tokens, logits, event: seen.append(
        max(s.seq_len for r in plan.requests for s in r.kv_caches))
    sched = ContinuousBatchingScheduler(max_batch_size=3, prefill_chunk_size=32, max_tokens_per_iteration=128)
    done, _ = sched.run(requests, lambda rs, n, t, e: run_prefill_chunk(model, rs, n, device, t, e, executor),
                        lambda rs, t, e: run_decode_step(model, rs, device, t, e, executor),
                        release_request_cache=lambda r: model.release_request_caches(r.kv_caches))
    assert [r.num_generated_tokens for r in done] == [10, 20, 5, 12]
    assert max(seen) <= 56
    for pool in model.layer_block_pools:
        assert len(pool.free_block_ids) == pool.capacity_blocks
        assert not pool.k_blocks.any() and not pool.weights.any()
