"""Attention over 4-bit pages against the oracle in 64 bits: head layouts, lengths, masks, garbage in what
a row does not see, running totals, streams and captured graphs."""
import numpy as np
import pytest
import torch

from oracle import q4
from q4_cases import bounds, filled_pools, poison, tables, to_q
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


def _call(device, q, kp, vp, table, lens, cur, weights=None, out=None, prefill=None):
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    fn = kq.paged_attention_prefill_q4_hip if (prefill if prefill is not None else q.shape[2] > 1) \
        else kq.paged_attention_decode_q4_hip
    return fn(q.to(device) if not q.is_cuda else q, kp, vp, i32(table), i32(lens), i32(cur), weights=weights, out=out)


def _check(device, rng, dtype, H, Hk, hd, T, lens, cur, kp, vp, table, prefill=None):
    q, qd = to_q(rng, (len(lens), H, T, hd), dtype)
    dk, dv = (torch.from_numpy(x).to(device) for x in (kp, vp))
    start = rng.uniform(0, 1, (kp.shape[0], Hk, 16)).astype(np.float32)
    want, added = q4.attention(qd, q4.values(kp, hd, True), q4.values(vp, hd, False), table, lens, cur)
    tol, rel = bounds(qd, kp, vp, hd, want, dtype)
    for weights in (None, torch.from_numpy(start.copy()).to(device)):
        got = _call(device, q, dk, dv, table, lens, cur, weights, prefill=prefill)
        off = np.abs(got.double().cpu().numpy() - want)
        assert not np.isnan(off).any()
        assert (off <= tol).all(), (off - tol).max()
        if weights is not None:
            sums = weights.double().cpu().numpy()
            # an addition in fp32, the sum over at most 2^10 rows and the weights' own error
            assert (np.abs(sums - start - added) <= 2.0 ** -23 * (start + added) + added * (rel + 2.0 ** -14)).all()


HEADS = [(2, 2), (6, 2), (8, 1), (12, 1), (20, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_decode_head_layouts(device, dtype, hd, heads):
    rng = np.random.default_rng(hd + heads[0])
    lens = [1, 16, 17, 47, 128, 300]
    kp, vp = filled_pools(rng, 48, heads[1], hd)
    _check(device, rng, dtype, *heads, hd, 1, lens, [1] * len(lens), kp, vp, tables(rng, lens, 48))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length", [15, 31, 32, 33, 255, 1025, 2100])
def test_decode_lengths(device, dtype, hd, length):
    rng = np.random.default_rng(length)
    lens = [length, max(1, length // 3)]
    blocks = 2 * (length // 16 + 2)
    kp, vp = filled_pools(rng, blocks, 2, hd)
    _check(device, rng, dtype, 4, 2, hd, 1, lens, [1, 1], kp, vp, tables(rng, lens, blocks))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_rows_without_keys_and_padding(device, dtype):
    rng = np.random.default_rng(3)
    # no keys at all; more new tokens than keys; a padded request (attends, adds nothing); a wide table
    lens, cur = [0, 2, 20, 33], [1, 5, 0, 1]
    kp, vp = filled_pools(rng, 12, 2, 64)
    _check(device, rng, dtype, 4, 2, 64, 1, lens, cur, kp, vp, tables(rng, lens, 12, width=70))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_unseen_pages_and_tails_may_hold_anything(device, dtype, T):
    """NaN in every slot that no row sees: behind the last key, in unused blocks, and in block 0, which
    stands in for pages that are not there."""
    rng = np.random.default_rng(T)
    lens = [70, 45, 131]
    kp, vp = filled_pools(rng, 24, 2, 64)
    table = 1 + tables(rng, lens, 23)
    table[table == 0] = -1
    table[2, 3] = -1  # a page missing in the middle
    table[0, 1] = 24  # one that is none of the pool's
    for pool in (kp, vp):
        used = set(table[(table > 0) & (table < 24)].tolist())
        for blk in range(24):
            if blk not in used:
                poison(pool, 64, blk, slice(None))
        for b, n in enumerate(lens):
            if n % 16 and table[b, n // 16] < 24:
                poison(pool, 64, table[b, n // 16], slice(n % 16, None))
    _check(device, rng, dtype, 4, 2, 64, T, lens, [min(T, 5)] * 3, kp, vp, table)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads", [(2, 2), (6, 2), (16, 1)], ids=str)
@pytest.mark.parametrize("T", [2, 7, 19, 80])
def test_prefill(device, dtype, hd, heads, T):
    rng = np.random.default_rng(T + hd + heads[0])
    cur = [T, max(1, T // 2), 1, T]
    lens = [T + 100, T // 2 + 16, 1, T]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], hd)
    _check(device, rng, dtype, *heads, hd, T, lens, cur, kp, vp, tables(rng, lens, blocks))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_over_a_long_context(device, dtype, hd):
    rng = np.random.default_rng(hd)
    lens, cur = [1400, 700], [33, 20]
    kp, vp = filled_pools(rng, 140, 1, hd)
    _check(device, rng, dtype, 3, 1, hd, 33, lens, cur, kp, vp, tables(rng, lens, 140))


def test_prefill_of_one_row_and_rows_without_keys(device):
    rng = np.random.default_rng(8)
    kp, vp = filled_pools(rng, 12, 2, 64)
    lens, cur = [40, 3, 0], [1, 1, 1]
    _check(device, rng, torch.float32, 2, 2, 64, 1, lens, cur, kp, vp, tables(rng, lens, 12), prefill=True)
    lens, cur = [40, 3, 0], [20, 9, 4]  # the second has rows before its first key
    _check(device, rng, torch.float32, 2, 2, 64, 20, lens, cur, kp, vp, tables(rng, lens, 12))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_key_that_is_nan_stays_with_the_rows_that_see_it(device, dtype):
    rng = np.random.default_rng(1)
    T, L = 24, 60
    kp, vp = filled_pools(rng, 6, 1, 64)
    table = tables(rng, [L], 6)
    clean = kp.copy(), vp.copy()
    at = L - T + 10  # the chunk's 11th row
    for pool in (kp, vp):
        poison(pool, 64, table[0, at // 16], at % 16)
    q, qd = to_q(rng, (1, 2, T, 64), dtype)
    got = _call(device, q, torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device), table, [L], [T]).cpu()
    want, _ = q4.attention(qd, q4.values(clean[0], 64, True), q4.values(clean[1], 64, False), table, [L], [T])
    tol, _ = bounds(qd, *clean, 64, want, dtype)
    assert (np.abs(got.double().numpy() - want)[:, :, :10] <= tol[:, :, :10]).all()
    assert got[:, :, 10:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_scale, kv_scale", [(1e-6, 1.0), (300.0, 1.0), (1.0, 1e-3), (1.0, 100.0), (0.0, 1.0)])
def test_magnitudes(device, dtype, q_scale, kv_scale):
    """Scores from flat to one-hot, values from small to large: the error stays relative to the values."""
    rng = np.random.default_rng(2)
    lens = [90, 640]
    kp, vp = filled_pools(rng, 50, 2, 64, kv_scale)
    table = tables(rng, lens, 50)
    q, _ = to_q(rng, (2, 4, 1, 64), torch.float32)
    q = (q * q_scale).to(dtype)
    qd = q.double().numpy()
    got = _call(device, q, torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device), table, lens, [1, 1])
    want, _ = q4.attention(qd, q4.values(kp, 64, True), q4.values(vp, 64, False), table, lens, [1, 1])
    tol, _ = bounds(qd, kp, vp, 64, want, dtype)
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


def test_scales_that_grow_along_the_context(device):
    """V's scales from 2^-12 to 2^12 and K's scores rising: the accumulators are rescaled on the way."""
    rng = np.random.default_rng(5)
    n = 640
    for dtype in (torch.float32, torch.bfloat16):
        kp, vp = filled_pools(rng, 40, 1, 128)
        table = np.arange(40, dtype=np.int32)[None]
        meta = vp[:, :, 1024:].view(np.float16).reshape(40, 1, 2, 16, 2)
        grow = 2.0 ** np.linspace(-12, 12, 40)
        meta[...] = (meta.astype(np.float64) * grow[:, None, None, None, None]).astype(np.float16)
        q, qd = to_q(rng, (1, 2, 1, 128), dtype)
        got = _call(device, q, torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device), table, [n], [1])
        want, _ = q4.attention(qd, q4.values(kp, 128, True), q4.values(vp, 128, False), table, [n], [1])
        tol, _ = bounds(qd, kp, vp, 128, want, dtype)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


def test_strided_and_unaligned_q_and_out(device):
    rng = np.random.default_rng(4)
    B, H, T, hd = 2, 4, 6, 64
    lens, cur = [50, 33], [6, 4]
    kp, vp = filled_pools(rng, 10, 2, hd)
    table = tables(rng, lens, 10)
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    for dtype in (torch.float32, torch.bfloat16):
        q, _ = to_q(rng, (B, H, T, hd), dtype)
        want = _call(device, q.contiguous(), dk, dv, table, lens, cur)
        big = torch.zeros(B, T, H, hd + 3, dtype=dtype, device=device)
        view = big[..., 1:hd + 1].transpose(1, 2)
        view.copy_(q)
        assert torch.equal(_call(device, view, dk, dv, table, lens, cur), want)
        dest = torch.full((B, T, H, hd + 3), 7.0, dtype=dtype, device=device)
        out = dest[..., 1:hd + 1].transpose(1, 2)
        assert _call(device, view, dk, dv, table, lens, cur, out=out) is out
        assert torch.equal(out, want)
        assert (dest[..., 0] == 7).all() and (dest[..., hd + 1:] == 7).all()
        last = torch.empty(B, H, hd, T, dtype=dtype, device=device).transpose(2, 3)  # head_dim not innermost
        last.copy_(q)
        assert torch.equal(_call(device, last, dk, dv, table, lens, cur), want)


def test_a_block_of_two_requests_gets_both_weights(device):
    """Two requests over the same pages (a shared prefix): the totals hold the sum of both."""
    rng = np.random.default_rng(6)
    kp, vp = filled_pools(rng, 6, 2, 64)
    table = np.array([[1, 2, 3], [1, 2, 4]], dtype=np.int32)
    _check(device, rng, torch.float32, 4, 2, 64, 1, [40, 45], [1, 1], kp, vp, table)
    _check(device, rng, torch.float32, 4, 2, 64, 9, [40, 45], [9, 7], kp, vp, table)


def test_offsets_past_32_bits(device):
    """Blocks behind the first 4 GiB of a pool."""
    hd, Hk = 128, 8
    per = Hk * kq.page_bytes(hd)
    blocks = (1 << 32) // per + 40
    rng = np.random.default_rng(7)
    kp, vp = filled_pools(rng, 24, Hk, hd)
    dk, dv = (torch.zeros(blocks, Hk, kq.page_bytes(hd), dtype=torch.uint8, device=device) for _ in range(2))
    dk[-24:] = torch.from_numpy(kp).to(device)
    dv[-24:] = torch.from_numpy(vp).to(device)
    lens = [100, 150]
    table = tables(rng, lens, 24)
    far = np.where(table >= 0, table + blocks - 24, -1).astype(np.int32)
    near = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    for T in (1, 30):
        q, _ = to_q(rng, (2, 16, T, hd), torch.bfloat16)
        assert torch.equal(_call(device, q, dk, dv, far, lens, [T, T]), _call(device, q, *near, table, lens, [T, T]))
    rows = torch.randn(1, Hk, 4, hd, device=device)
    slots = torch.tensor([(blocks - 3) * 16 + i for i in (0, 5, 9, 15)], dtype=torch.int32, device=device)
    kq.kv_append_q4_hip(rows, rows, dk, dv, slots)
    back = kq.kv_read_q4_hip(dk, dv, slots)[0]
    assert float((back - rows).abs().max()) < 0.5 and bool(dk[-3].any())


def test_empty_batches_and_tables(device):
    pool = torch.zeros(2, 2, kq.page_bytes(64), dtype=torch.uint8, device=device)
    q = torch.empty(0, 4, 1, 64, device=device)
    none = torch.empty(0, dtype=torch.int32, device=device)
    assert kq.paged_attention_decode_q4_hip(q, pool, pool, none.view(0, 3), none, none).shape == q.shape
    q = torch.randn(2, 4, 1, 64, device=device)
    zero = torch.zeros(2, dtype=torch.int32, device=device)
    totals = torch.ones(2, 2, 16, device=device)
    out = kq.paged_attention_decode_q4_hip(q, pool, pool, torch.empty(2, 0, dtype=torch.int32, device=device), zero + 5, zero + 1,
                                           weights=totals)
    assert not out.any() and (totals == 1).all()


def test_refusals(device):
    pool = torch.zeros(4, 2, kq.page_bytes(64), dtype=torch.uint8, device=device)
    q = torch.zeros(2, 4, 1, 64, device=device)
    table = torch.zeros(2, 3, dtype=torch.int32, device=device)
    lens = torch.ones(2, dtype=torch.int32, device=device)
    good = dict(q=q, k_pool=pool, v_pool=pool, page_table=table, seq_lens=lens, current_lengths=lens)
    kq.paged_attention_decode_q4_hip(**good)
    for change in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=torch.zeros(2, 4, 1, 128, device=device)), dict(q=q.cpu()),
                   dict(q=q[0]), dict(q=torch.zeros(2, 4, 2, 64, device=device)), dict(k_pool=pool[:2]),
                   dict(k_pool=pool.int(), v_pool=pool.int()), dict(page_table=table.long()), dict(page_table=table[:1]),
                   dict(page_table=table.cpu()), dict(page_table=table[0]), dict(seq_lens=lens[:1]), dict(seq_lens=lens.float()),
                   dict(current_lengths=lens.cpu()), dict(weights=torch.zeros(4, 2, 8, device=device)),
                   dict(weights=torch.zeros(4, 2, 16, device=device).half()), dict(out=torch.zeros(2, 4, 1, 64, device=device).half()),
                   dict(out=torch.zeros(2, 4, 2, 64, device=device)), dict(weights=torch.zeros(4, 2, 16))):
        with pytest.raises((ValueError, TypeError)):
            kq.paged_attention_decode_q4_hip(**{**good, **change})


@pytest.mark.parametrize("T", [1, 24])
def test_captured_replays_and_two_streams(device, T):
    """A captured call with totals, replayed between eager calls; then two streams at once."""
    rng = np.random.default_rng(T)
    lens = [700, 90, 300, 33]
    kp, vp = filled_pools(rng, 80, 2, 64)
    table = torch.from_numpy(tables(rng, lens, 80)).to(device)
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    L = torch.tensor(lens, dtype=torch.int32, device=device)
    C = torch.full((4,), T, dtype=torch.int32, device=device)
    fn = kq.paged_attention_decode_q4_hip if T == 1 else kq.paged_attention_prefill_q4_hip
    q = torch.empty(4, 4, T, 64, device=device)
    totals = torch.zeros(80, 2, 16, device=device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fn(q.zero_(), dk, dv, table, L, C, weights=totals)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = fn(q, dk, dv, table, L, C, weights=totals)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        totals.zero_()
        graph.replay()
        torch.cuda.synchronize()
        mine = torch.zeros_like(totals)
        want = fn(q, dk, dv, table, L, C, weights=mine)
        assert torch.equal(out, want)
        assert torch.equal(totals, mine)
    qs = [torch.randn(4, 4, T, 64, device=device) for _ in range(2)]
    wants = [fn(x, dk, dv, table, L, C) for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    gots = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                gots[i].append(fn(qs[i], dk, dv, table, L, C, weights=torch.zeros_like(totals)))
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        assert all(torch.equal(g, want) for g in got)


# Sizes on both sides of the launch rules' borders (rows of a KV head, width of the page table, units).
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads, T, width", [
    ((2, 2), 1, 6200),    # a row, many pages
    ((8, 1), 1, 40),      # five rows and more of a decode step, 512 keys and more
    ((8, 1), 1, 4200),    # the same, totals by the scores
    ((16, 2), 3, 31),     # a short chunk, few pages
    ((16, 2), 3, 260),    # two tiles
    ((6, 2), 1, 4200),
    ((4, 2), 10, 4200),   # totals: pages of its own for a wavefront, four at a time
    ((8, 2), 16, 300),    # up to 32 tiles
    ((8, 1), 80, 20),     # more, few pages
    ((8, 1), 80, 300),    # more, four pages at a time
    ((2, 2), 70, 8),      # eight wavefronts to four tiles
    ((2, 2), 70, 260),    # ranges of keys
], ids=str)
def test_launch_rules(device, dtype, hd, heads, T, width):
    rng = np.random.default_rng(T + width)
    cur = [T, max(1, T // 2), 1, T]
    lens = [T + 37, T // 2 + 90, 1, T]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], hd)
    _check(device, rng, dtype, *heads, hd, T, lens, cur, kp, vp, tables(rng, lens, blocks, width=width))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [1, 3, 12])
def test_groups_over_long_contexts(device, dtype, hd, T):
    rng = np.random.default_rng(hd + T)
    lens, cur = [2100, 905, 33], [T, T, min(T, 2)]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, 2, hd)
    _check(device, rng, dtype, 16, 2, hd, T, lens, cur, kp, vp, tables(rng, lens, blocks))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads, T", [((4, 2), 3), ((4, 2), 12), ((8, 1), 80)], ids=str)
def test_padded_rows_may_hold_anything(device, dtype, garbage, heads, T):
    """NaN and infinities in q's rows behind a request's last new token: its real rows and the totals are those of
    any other padding."""
    rng = np.random.default_rng(T)
    lens, cur = [T + 60, 40, 5], [T, 2, 0]
    kp, vp = filled_pools(rng, 20, heads[1], 64)
    table = tables(rng, lens, 20)
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    q, _ = to_q(rng, (3, heads[0], T, 64), dtype)
    outs, sums = [], []
    for fill in (0.0, garbage):
        for b, n in enumerate(cur):
            q[b, :, n:] = fill
        totals = torch.zeros(20, heads[1], 16, device=device)
        outs.append(_call(device, q, dk, dv, table, lens, cur, totals))
        sums.append(totals)
    assert torch.equal(sums[0], sums[1])
    for b, n in enumerate(cur):
        assert torch.equal(outs[0][b, :, :n], outs[1][b, :, :n])
