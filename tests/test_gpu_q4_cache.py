"""Append and read of the 4-bit cache against the oracle, bit for bit, and the wrappers' refusals."""
import numpy as np
import pytest
import torch

from oracle import q4
from q4_cases import filled_pools
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


def _rows(rng, B, H, T, hd, dtype, layout):
    x = rng.normal(0, 1, (B, T, H, hd)).astype(np.float32)
    x *= (10.0 ** rng.integers(-3, 4, (B, T, H, 1))).astype(np.float32)
    x.flat[::97] = 0
    flat = x.reshape(-1, hd)
    flat[:: 5] = np.round(flat[:: 5] * 4) / 4  # ties between codes
    flat[1:: 11] = 3.0  # constant rows
    flat[2:: 13, 7] = 1e5  # beyond half's range
    flat[3:: 17, 1] = -np.inf
    flat[4:: 19, 2] = np.nan
    flat[5:: 23] *= np.float32(1e-7)
    t = torch.from_numpy(x).to(dtype)
    if layout == "heads":
        return t.transpose(1, 2).contiguous(), t.float().numpy().swapaxes(1, 2)
    if layout == "offset":  # rows off the 16-byte grid
        big = torch.zeros(B, T, H, hd + 1, dtype=dtype)
        big[..., 1:] = t
        return big[..., 1:].transpose(1, 2), t.float().numpy().swapaxes(1, 2)
    return t.transpose(1, 2), t.float().numpy().swapaxes(1, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 5), (2, 8, 37)], ids=str)
@pytest.mark.parametrize("layout", ["rows", "heads", "offset"])
def test_append_and_read_bit_exact(device, dtype, hd, shape, layout):
    B, H, T = shape
    rng = np.random.default_rng(B * T + hd)
    (kt, kx), (vt, vx) = (_rows(rng, B, H, T, hd, dtype, layout) for _ in range(2))
    blocks = B * T // 16 + 3
    kp, vp = filled_pools(rng, blocks, H, hd)
    slots = rng.permutation(blocks * 16)[: B * T].astype(np.int32)
    slots[1:: 7] = -1
    slots[2:: 11] = blocks * 16 + 5  # past the pool: skipped
    totals = rng.uniform(0.5, 1, (blocks, H, 16)).astype(np.float32)
    dk, dv, dw = (torch.from_numpy(x.copy()).to(device) for x in (kp, vp, totals))
    ds = torch.from_numpy(slots).to(device)
    kq.kv_append_q4_hip(_dev(kt, device), _dev(vt, device), dk, dv, ds, weights=dw)
    for i, s in enumerate(slots):
        if 0 <= s < blocks * 16:
            for h in range(H):
                q4.put(kp, s // 16, h, s % 16, kx[i // T, h, i % T], True)
                q4.put(vp, s // 16, h, s % 16, vx[i // T, h, i % T], False)
                totals[s // 16, h, s % 16] = 0
    assert np.array_equal(dk.cpu().numpy(), kp)
    assert np.array_equal(dv.cpu().numpy(), vp)
    assert np.array_equal(dw.cpu().numpy(), totals)

    for out_dtype in (torch.float32, torch.bfloat16):
        got = kq.kv_read_q4_hip(dk, dv, ds, batch=B, dtype=out_dtype)
        for g, pool, is_k in zip(got, (kp, vp), (True, False)):
            val = q4.values(pool, hd, is_k)
            want = np.zeros((B, T, H, hd))
            for i, s in enumerate(slots):
                if 0 <= s < blocks * 16:
                    want[i // T, i % T] = val[s // 16, :, s % 16]
            want = torch.from_numpy(want).float().to(out_dtype).transpose(1, 2)
            assert torch.equal(g.cpu().nan_to_num(9e9), want.nan_to_num(9e9))


def _dev(t, device):
    """A copy on the device with the same strides."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
    return out.copy_(t)


def test_append_of_nothing(device):
    pool = torch.zeros(2, 2, kq.page_bytes(64), dtype=torch.uint8, device=device)
    none = torch.empty(0, 2, 3, 64, device=device)
    kq.kv_append_q4_hip(none, none, pool, pool, torch.empty(0, dtype=torch.int32, device=device))
    k, v = kq.kv_read_q4_hip(pool, pool, torch.empty(0, dtype=torch.int32, device=device))
    assert k.shape == (1, 2, 0, 64) and not pool.any()


def test_refusals(device):
    pool = torch.zeros(4, 2, kq.page_bytes(64), dtype=torch.uint8, device=device)
    slots = torch.zeros(3, dtype=torch.int32, device=device)
    rows = torch.zeros(1, 2, 3, 64, device=device)
    bad = [
        (rows.half(), rows.half(), pool, pool, slots, None), (rows[:, :1], rows[:, :1], pool, pool, slots, None),
        (rows, rows[:, :, :2], pool, pool, slots, None), (rows, rows, pool, pool, slots[:2], None),
        (rows, rows, pool, pool, slots.long(), None), (rows, rows, pool, pool[:2], slots, None),
        (rows, rows, pool.float(), pool.float(), slots, None), (rows, rows, pool[:, :, :-1], pool[:, :, :-1], slots, None),
        (rows.cpu(), rows.cpu(), pool, pool, slots, None), (rows, rows, pool, pool, slots, torch.zeros(4, 2, 8, device=device)),
        (rows, rows, pool, pool, slots, torch.zeros(4, 2, 16, device=device, dtype=torch.float64)),
        (rows, rows, pool, pool.cpu(), slots, None), (rows, rows, pool, pool, slots.cpu(), None),
    ]
    for k, v, kp, vp, s, w in bad:
        with pytest.raises((ValueError, TypeError)):
            kq.kv_append_q4_hip(k, v, kp, vp, s, weights=w)
    with pytest.raises(ValueError):
        kq.kv_read_q4_hip(pool, pool, slots, batch=2)
    with pytest.raises(TypeError):
        kq.kv_read_q4_hip(pool, pool, slots, dtype=torch.float16)
    assert not pool.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("centre", [0.0, 1.0, 30.0, 3000.0, -60000.0])
def test_values_at_borders_and_a_step_beside_them(device, dtype, centre):
    """Groups full of values at z + m s, m whole (a tie between two codes where that is exact), and of the next
    number of the type on either side, about centres of 0 to 60000 steps and more."""
    rng = np.random.default_rng(int(abs(centre)))
    rows = 160
    k = np.empty((rows, 64), dtype=np.float32)
    for i in range(rows):
        half = np.float32(2.0 ** rng.integers(-3, 4) * rng.uniform(4, 8))
        ends = torch.tensor([centre * half / 7.5 + half, centre * half / 7.5 - half]).clamp(-65000, 65000).to(dtype).float().numpy()
        s, z = (np.float64(np.float16(x)) for x in ((ends[0] - ends[1]) * np.float32(1 / 15), (ends[0] + ends[1]) * np.float32(0.5)))
        at = torch.from_numpy(z + rng.integers(-7, 8, 62) * s).float().to(dtype)
        step = torch.from_numpy(rng.integers(-1, 2, 62).astype(np.int32))
        if dtype == torch.float32:
            at = (at.view(torch.int32) + step).view(torch.float32)
        else:
            at = (at.view(torch.int16) + step.to(torch.int16)).view(torch.bfloat16)
        k[i] = np.concatenate([ends, at.float().numpy()]).clip(ends.min(), ends.max())
    t = torch.from_numpy(k).to(dtype).view(1, rows, 1, 64).transpose(1, 2).to(device)
    pool = np.zeros((rows // 16, 1, q4.page_bytes(64)), dtype=np.uint8)
    dk, dv = torch.from_numpy(pool.copy()).to(device), torch.from_numpy(pool.copy()).to(device)
    kq.kv_append_q4_hip(t, t, dk, dv, torch.arange(rows, dtype=torch.int32, device=device))
    vp = pool.copy()
    for i in range(rows):
        q4.put(pool, i // 16, 0, i % 16, k[i], True)
        q4.put(vp, i // 16, 0, i % 16, k[i], False)
    assert np.array_equal(dk.cpu().numpy(), pool)
    assert np.array_equal(dv.cpu().numpy(), vp)
