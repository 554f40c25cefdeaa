"""Running totals of 4-bit attention where they can go wrong: workspaces full of rubbish, rows that see nothing beside
long requests, keys that no row sees, rows that are NaN."""
import numpy as np
import pytest
import torch

from oracle import q4
from q4_cases import bounds, filled_pools, poison, tables, to_q
from src.kernels import hip_paged_attention as hpa
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


def _call(device, q, kp, vp, table, lens, cur, totals):
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    fn = kq.paged_attention_prefill_q4_hip if q.shape[2] > 1 else kq.paged_attention_decode_q4_hip
    return fn(q.to(device), kp, vp, i32(table), i32(lens), i32(cur), weights=totals)


def _fill_workspace(device):
    """0x7f in every byte of the default stream's workspace: halves that are NaN, floats of 3.4e38, lengths past all keys."""
    ws = hpa._workspaces.get((torch.device(device).index or 0, "q4"))
    if ws is not None:
        ws.fill_(0x7F)


def _check(device, q, qd, kp, vp, table, lens, cur, hd, bound_pools=None):
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    want, added = q4.attention(qd, q4.values(kp, hd, True), q4.values(vp, hd, False), table, lens, cur)
    tol, rel = bounds(qd, *(bound_pools or (kp, vp)), hd, want, q.dtype)
    for _ in range(2):  # (the first call may allocate the workspace, the second finds it full of rubbish)
        totals = torch.zeros(kp.shape[0], kp.shape[1], 16, device=device)
        _fill_workspace(device)
        got = _call(device, q, dk, dv, table, lens, cur, totals).double().cpu().numpy()
        sums = totals.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isnan(sums), np.isnan(added))
    there = ~np.isnan(want)
    assert (np.abs(got - want) <= tol)[there].all()
    there = ~np.isnan(added)
    # as for finite totals: an addition in fp32 and the weights' own error
    assert (np.abs(sums - added) <= 2.0 ** -23 * added + added * (rel + 2.0 ** -14))[there].all()


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
# Few rows (the kernel of a tile of rows), and more than two tiles (a tile per wavefront), over few and over
# several ranges of keys.
SHAPES = pytest.mark.parametrize("heads, T, width", [((4, 2), 3, 8), ((4, 2), 3, 300), ((2, 2), 40, 8), ((2, 2), 40, 130),
                                                     ((8, 1), 80, 130)], ids=str)


@DTYPES
@SHAPES
def test_rows_that_see_no_key_beside_a_long_request(device, dtype, heads, T, width):
    """Some requests claim more new tokens than they have keys and rows: all, or all but a few, of their rows
    see nothing."""
    rng = np.random.default_rng(T + width)
    L = min(width * 16 - 5, 1900)
    lens, cur = [T, L, T, 7], [2 * T + 5, T, 2 * T - 2, 3 * T]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], 64)
    q, qd = to_q(rng, (4, heads[0], T, 64), dtype)
    _check(device, q, qd, kp, vp, tables(rng, lens, blocks, width=width), lens, cur, 64)


@DTYPES
@pytest.mark.parametrize("heads, T", [((32, 1), 2), ((4, 2), 12), ((2, 2), 40)], ids=str)
def test_the_largest_claim(device, dtype, heads, T):
    """current_lengths of 2^31 - 1: no row sees a key, and nothing is read in front of the first row."""
    rng = np.random.default_rng(T)
    lens, cur = [100, 2000], [2 ** 31 - 1, T]
    kp, vp = filled_pools(rng, 140, heads[1], 64)
    q, qd = to_q(rng, (2, heads[0], T, 64), dtype)
    _check(device, q, qd, kp, vp, tables(rng, lens, 140), lens, cur, 64)


@DTYPES
@SHAPES
def test_keys_behind_the_last_rows_view_may_hold_anything(device, dtype, heads, T, width):
    """A request that claims more new tokens than the call has rows: the keys that its last row does not see are
    NaN, and nothing of them reaches the totals."""
    rng = np.random.default_rng(T + width)
    lens, over = [T + 60, T + 30], [21, 4]
    cur = [T + n for n in over]  # row i sees L - over - T + 1 + i keys
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], 64)
    table = tables(rng, lens, blocks, width=width)
    clean = kp.copy(), vp.copy()
    for b, n in enumerate(lens):
        for t in range(n - over[b], n):
            for pool in (kp, vp):
                poison(pool, 64, table[b, t // 16], t % 16)
    q, qd = to_q(rng, (2, heads[0], T, 64), dtype)
    _check(device, q, qd, kp, vp, table, lens, cur, 64, clean)


@DTYPES
@pytest.mark.parametrize("heads, T, width", [((4, 2), 1, 8), ((4, 2), 1, 300), ((16, 2), 1, 300), ((40, 1), 1, 40), ((4, 2), 3, 8),
                                             ((4, 2), 3, 300), ((2, 2), 40, 8), ((2, 2), 40, 130), ((8, 1), 80, 130)], ids=str)
def test_a_row_that_is_nan_makes_the_totals_of_its_keys_nan(device, dtype, heads, T, width):
    rng = np.random.default_rng(T + width)
    lens, cur = [T + 50, T + 30], [T, T]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], 64)
    table = tables(rng, lens, blocks, width=width)
    q, _ = to_q(rng, (2, heads[0], T, 64), dtype)
    q[0, 1, T // 2, 5] = float("nan")
    clean = q.clone()
    clean[0, 1, T // 2, 5] = 0
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    want, added = q4.attention(q.double().numpy(), q4.values(kp, 64, True), q4.values(vp, 64, False), table, lens, cur)
    _, rel = bounds(clean.double().numpy(), kp, vp, 64, np.nan_to_num(want), dtype)
    totals = torch.zeros(blocks, heads[1], 16, device=device)
    got = _call(device, q, dk, dv, table, lens, cur, totals).double().cpu().numpy()
    sums = totals.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(added).any() and np.array_equal(np.isnan(sums), np.isnan(added))
    there = ~np.isnan(added)
    assert (np.abs(sums - added) <= 2.0 ** -23 * added + added * (rel + 2.0 ** -14))[there].all()


@DTYPES
@pytest.mark.parametrize("heads, T, width", [((4, 2), 1, 8), ((4, 2), 1, 300), ((4, 2), 5, 8), ((2, 2), 40, 130)], ids=str)
def test_a_key_that_is_nan_makes_its_rows_totals_nan(device, dtype, heads, T, width):
    rng = np.random.default_rng(T + width)
    lens, cur = [T + 50, T + 30], [T, T]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], 64)
    table = tables(rng, lens, blocks, width=width)
    clean = kp.copy(), vp.copy()
    at = lens[0] - max(T // 2, 1)  # seen by the chunk's later rows only
    for pool in (kp, vp):
        poison(pool, 64, table[0, at // 16], at % 16)
    q, qd = to_q(rng, (2, heads[0], T, 64), dtype)
    _check(device, q, qd, kp, vp, table, lens, cur, 64, clean)
