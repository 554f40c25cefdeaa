"""Eviction by accumulated weight against the oracle: the choice and the moved bits, exactly."""
import numpy as np
import pytest
import torch

from oracle import q4
from q4_cases import filled_pools, tables
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


def _run(device, rng, lens, Hk, hd, keep, window, weights=None, table=None, spare=4):
    width = -(-max(lens) // 16)
    fresh_pages = [-(-min(max(n, 0), keep) // 16) for n in lens]
    blocks = sum(-(-max(n, 0) // 16) for n in lens) + sum(fresh_pages) + spare
    kp, vp = filled_pools(rng, blocks, Hk, hd)
    if table is None:
        both = tables(rng, list(lens) + [16 * n for n in fresh_pages], blocks, width=width)
        table, fresh = both[:len(lens), :width].copy(), both[len(lens):, :max(max(fresh_pages), 1)].copy()
    else:
        table, fresh = table
    w = weights(blocks) if weights is not None else np.exp(2 * rng.normal(0, 1, (blocks, Hk, 16))).astype(np.float32)
    dk, dv, dw = (torch.from_numpy(x.copy()).to(device) for x in (kp, vp, w))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    kept, new_lens = kq.evict_q4_hip(dk, dv, dw, i32(table), i32(lens), i32(fresh), keep=keep, window=window)
    want = q4.evict(w, table, lens, keep, window)
    N = kp.shape[0]
    for b in range(len(lens)):
        assert int(new_lens[b]) == min(max(lens[b], 0), keep, 16 * table.shape[1])
        for h in range(Hk):
            row = kept[b, h].cpu().tolist()
            n = len(want[b][h])
            assert row[:n] == want[b][h] and all(x == -1 for x in row[n:])
    # the moved rows, value by value of their bits, and everything else as it was
    codes = [_token_bits(p, hd, is_k) for p, is_k in ((kp, True), (vp, False))]
    ek, ev = codes[0].copy(), codes[1].copy()
    ew = w.copy()
    for b in range(len(lens)):
        for h in range(Hk):
            for i, t in enumerate(want[b][h]):
                src, dst = int(table[b, t // 16]), int(fresh[b, i // 16])
                if not 0 <= dst < N:
                    continue
                ok = 0 <= src < N
                for e, c in ((ek, codes[0]), (ev, codes[1])):
                    e[dst, h, i % 16] = c[src, h, t % 16] if ok else 0
                ew[dst, h, i % 16] = w[src, h, t % 16] if ok else 0
    assert np.array_equal(_token_bits(dk.cpu().numpy(), hd, True), ek)
    assert np.array_equal(_token_bits(dv.cpu().numpy(), hd, False), ev)
    assert np.array_equal(dw.cpu().numpy(), ew, equal_nan=True)


def _token_bits(pool, hd, is_k):
    """[N, H, 16, hd + 4 groups]: a token's codes and the bytes of its pairs."""
    n = q4._nibbles(hd, is_k)
    c = pool[:, :, n // 2] >> (4 * (n % 2)) & 15
    meta = pool[:, :, 16 * hd // 2:].reshape(*pool.shape[:2], hd // 64, 16, 4).swapaxes(2, 3).reshape(*pool.shape[:2], 16, -1)
    return np.concatenate([c, meta], -1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keep, window", [(1, 0), (1, 1), (16, 4), (50, 0), (50, 50), (100, 17), (128, 64), (700, 3)])
def test_choice_and_move(device, hd, keep, window):
    rng = np.random.default_rng(keep + window)
    _run(device, rng, [1, 17, 64, 129, 640, 333], 3, hd, keep, window)


def test_equal_totals_go_to_the_lower_index(device):
    rng = np.random.default_rng(0)
    for few in (1, 2, 5):
        _run(device, rng, [200, 555], 2, 64, 61, 7,
             weights=lambda n: rng.integers(0, few, (n, 2, 16)).astype(np.float32))


def test_special_totals(device):
    rng = np.random.default_rng(1)

    def weights(n):
        w = rng.normal(0, 1, (n, 2, 16)).astype(np.float32)
        pick = rng.integers(0, 9, w.shape)
        for i, x in enumerate((0.0, -0.0, np.nan, np.inf, -np.inf, 1e-45, 3e38)):
            w[pick == i] = x
        return w

    _run(device, rng, [300, 410], 2, 64, 96, 5, weights=weights)


def test_longer_than_what_lds_holds(device):
    _run(device, np.random.default_rng(2), [33000 + 777], 1, 64, 1000, 100)


def test_pages_that_are_not_there(device):
    rng = np.random.default_rng(3)
    table = np.array([[5, -1, 9, 40, 2], [7, 6, 1, -1, -1]], dtype=np.int32)  # the pool has 21 blocks
    fresh = np.array([[10, 11], [12, -1]], dtype=np.int32)
    _run(device, rng, [75, 45], 2, 64, 24, 20, table=(table, fresh), spare=9)


def test_lengths_past_the_table_and_empty_requests(device):
    rng = np.random.default_rng(4)
    table = np.array([[5, 3], [7, 6], [-1, -1]], dtype=np.int32)
    fresh = np.array([[8], [9], [10]], dtype=np.int32)
    _run(device, rng, [40, 20, 0], 2, 128, 16, 2, table=(table, fresh))


def test_captured_replays(device):
    rng = np.random.default_rng(5)
    lens, keep, window = [500, 70, 900], 64, 16
    kp, vp = filled_pools(rng, 110, 2, 64)
    both = tables(rng, lens + [64] * 3, 110)
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    args = (i32(both[:3]), i32(lens), i32(both[3:, :4]))
    w = torch.zeros(110, 2, 16, device=device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kq.evict_q4_hip(dk, dv, w, *args, keep=keep, window=window)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept, new_lens = kq.evict_q4_hip(dk, dv, w, *args, keep=keep, window=window)
    for i in range(4):
        w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = kept.clone()
        want = q4.evict(w.cpu().numpy(), both[:3], lens, keep, window)
        assert [[[t for t in row if t >= 0] for row in heads] for heads in got.tolist()] == want
        again, _ = kq.evict_q4_hip(dk, dv, w, *args, keep=keep, window=window)
        assert torch.equal(again, got)
        assert new_lens.tolist() == [64, 64, 64]


def test_refusals(device):
    pool = torch.zeros(8, 2, kq.page_bytes(64), dtype=torch.uint8, device=device)
    w = torch.zeros(8, 2, 16, device=device)
    table = torch.zeros(1, 4, dtype=torch.int32, device=device)
    fresh = torch.ones(1, 2, dtype=torch.int32, device=device)
    lens = torch.full((1,), 50, dtype=torch.int32, device=device)
    kq.evict_q4_hip(pool, pool, w, table, lens, fresh, keep=32, window=8)
    for kw in (dict(keep=0, window=0), dict(keep=8, window=9), dict(keep=8, window=-1), dict(keep=33, window=8)):
        with pytest.raises(ValueError):
            kq.evict_q4_hip(pool, pool, w, table, lens, fresh, **kw)
    for args in ((pool, pool, None, table, lens, fresh), (pool, pool, w, table, lens, fresh.long()),
                 (pool, pool, w, table[0], lens, fresh), (pool, pool, w, table, lens.cpu(), fresh),
                 (pool, pool, w.cpu(), table, lens, fresh), (pool, pool, w[:4], table, lens, fresh),
                 (pool, pool, w, table, lens, fresh[:0])):
        with pytest.raises(ValueError):
            kq.evict_q4_hip(*args, keep=32, window=8)


@pytest.mark.parametrize("cluster", [1, 2, 63, 64, 65, 200])
@pytest.mark.parametrize("kinds", [1, 3, 1 << 16])
def test_totals_that_share_their_high_bits(device, cluster, kinds):
    """The border falls among `cluster` totals whose low 16 bits alone differ, in `kinds` ways; 100 are larger."""
    rng = np.random.default_rng(cluster + kinds)

    def weights(n):
        w = rng.uniform(0, 0.5, (n, 2, 16)).astype(np.float32)
        for h in range(2):
            flat = rng.permutation(n * 16)
            view = np.empty(n * 16, dtype=np.float32)
            view[:] = w[:, h].reshape(-1)
            view[flat[:100]] = rng.uniform(2, 90, 100)
            view[flat[100:100 + cluster]] = (0x3f800000 + rng.integers(0, kinds, cluster)).astype(np.uint32).view(np.float32)
            w[:, h] = view.reshape(n, 16)
        return w

    _run(device, rng, [600], 2, 64, 100 + cluster // 2 + 9, 9, weights=weights, spare=0)
