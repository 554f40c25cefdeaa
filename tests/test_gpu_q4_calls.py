"""How calls on the 4-bit cache reach the library: the native front and the checked Python path give the same,
a growing context's workspaces, calls of nothing."""
import numpy as np
import pytest
import torch

from q4_cases import filled_pools, tables
from src.kernels import hip_paged_attention as hpa
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


def _state(device, lens, hd=64, heads=2, blocks=64):
    rng = np.random.default_rng(len(lens))
    kp, vp = filled_pools(rng, blocks, heads, hd)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    totals = torch.from_numpy(rng.uniform(0, 1, (blocks, heads, 16)).astype(np.float32)).to(device)
    return torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device), totals, i32(tables(rng, lens, blocks)), i32(lens), i32


def _everything(device, dtype):
    lens = [200, 33, 90]
    k, v, totals, table, L, i32 = _state(device, lens)
    g = torch.Generator().manual_seed(0)
    rows = lambda *shape: torch.randn(*shape, generator=g).to(dtype).to(device)  # noqa: E731
    # rows in the layout that projections leave, and a pair whose strides differ
    new_k, new_v = rows(3, 5, 2, 64).transpose(1, 2), rows(3, 2, 5, 64)
    slots = i32([int(table[b, (n - 5 + t) // 16]) * 16 + (n - 5 + t) % 16 for b, n in enumerate(lens) for t in range(5)])
    out = []
    kq.kv_append_q4_hip(new_k, new_k, k, v, slots, weights=totals)
    kq.kv_append_q4_hip(new_k, new_v, k, v, slots)
    out += [k.clone(), v.clone(), totals.clone()]
    out += kq.kv_read_q4_hip(k, v, slots, batch=3, dtype=dtype)
    for T, fn in ((1, kq.paged_attention_decode_q4_hip), (5, kq.paged_attention_prefill_q4_hip)):
        q = rows(3, 8, T, 64)
        cur = L * 0 + T
        dest = torch.empty_like(q)
        assert fn(q, k, v, table, L, cur, weights=totals, out=dest) is dest
        out += [dest, fn(q, k, v, table, L, cur), totals.clone()]
    free = sorted(set(range(64)) - set(table.flatten().tolist()))
    fresh = i32(np.array(free[:9]).reshape(3, 3))
    out += kq.evict_q4_hip(k, v, totals, table, L, fresh, keep=40, window=8)
    return out + [k, v, totals]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_python_path_gives_what_the_native_front_gives(device, dtype, monkeypatch):
    if hpa.native_call() is None:
        pytest.skip("the native front is not built")
    want = _everything(device, dtype)
    monkeypatch.setattr(kq, "native_call", lambda: None)
    for a, b in zip(_everything(device, dtype), want):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float32 else a,
                           b.view(torch.uint8) if b.dtype == torch.float32 else b)


def test_a_growing_context_allocates_a_few_workspaces(device):
    """Decode steps with totals, the page table one page wider each time, on the default stream, which keeps
    every workspace that it outgrew."""
    k, v, totals, _, _, i32 = _state(device, [1], blocks=8)
    q = torch.randn(16, 16, 1, 64, device=device)
    lens, cur = i32([40] * 16), i32([1] * 16)
    before = len(hpa._retired_workspaces)
    key = (torch.cuda.current_device(), "q4")
    for pages in range(64, 512, 4):  # 1 to 8 MiB of scores
        table = torch.zeros(16, pages, dtype=torch.int32, device=device)
        kq.paged_attention_decode_q4_hip(q, k, v, table, lens, cur, weights=totals)
    kept = [w.numel() for w in hpa._retired_workspaces[before:]]
    assert len(kept) <= 5 and sum(kept) <= hpa._workspaces[key].numel()


@pytest.mark.parametrize("native", [True, False])
def test_calls_of_nothing(device, native, monkeypatch):
    if not native:
        monkeypatch.setattr(kq, "native_call", lambda: None)
    k, v, totals, table, L, i32 = _state(device, [20, 30])
    was = [x.clone() for x in (k, v, totals)]
    none = torch.empty(0, dtype=torch.int32, device=device)
    kq.kv_append_q4_hip(torch.empty(2, 2, 0, 64, device=device), torch.empty(2, 2, 0, 64, device=device), k, v, none, weights=totals)
    assert kq.kv_read_q4_hip(k, v, none, batch=2)[0].shape == (2, 2, 0, 64)
    q = torch.empty(2, 4, 0, 64, device=device)
    assert kq.paged_attention_prefill_q4_hip(q, k, v, table, L, L * 0, weights=totals).shape == q.shape
    kept, lens = kq.evict_q4_hip(k, v, totals, table, none, torch.empty(0, 1, dtype=torch.int32, device=device), keep=4, window=1)
    assert kept.shape == (0, 2, 4) and lens.shape == (0,)
    assert all(torch.equal(a, b) for a, b in zip(was, (k, v, totals)))


@pytest.mark.parametrize("native", [True, False])
def test_output_over_the_queries_is_refused(device, native, monkeypatch):
    if not native:
        monkeypatch.setattr(kq, "native_call", lambda: None)
    k, v, totals, table, L, _ = _state(device, [20, 30])
    q = torch.randn(2, 4, 3, 64, device=device)
    with pytest.raises(ValueError, match="out must not be q"):
        kq.paged_attention_prefill_q4_hip(q, k, v, table, L, L * 0 + 3, weights=totals, out=q)


def test_captured_eviction_of_long_tables(device):
    """More totals than a kernel's default LDS holds, captured and replayed with other totals."""
    n, keep = 20000, 500
    k, v, totals, table, L, i32 = _state(device, [n], blocks=1300)
    free = sorted(set(range(1300)) - set(table.flatten().tolist()))[:32]
    fresh = i32([free])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kq.evict_q4_hip(k, v, totals, table, L, fresh, keep=keep, window=10)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept, lens = kq.evict_q4_hip(k, v, totals, table, L, fresh, keep=keep, window=10)
    for seed in range(3):
        totals.copy_(torch.rand(totals.shape, generator=torch.Generator().manual_seed(seed)))
        state = [x.clone() for x in (k, v, totals)]
        graph.replay()
        torch.cuda.synchronize()
        want, want_lens = kq.evict_q4_hip(*state, table, L, fresh, keep=keep, window=10)
        assert torch.equal(kept, want) and torch.equal(lens, want_lens)
        assert all(torch.equal(a, b) for a, b in zip(state, (k, v, totals)))
