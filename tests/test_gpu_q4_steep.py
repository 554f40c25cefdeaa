"""4-bit attention at scores so large that they are whole numbers in fp32, and past them: finite inputs give finite
outputs, which lie between the values of the keys that may have any weight."""
import math

import numpy as np
import pytest
import torch

from oracle import q4
from q4_cases import filled_pools, tables
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu

SHAPES = {  # heads, KV heads, rows, width of the table
    "decode": (4, 2, 1, 0),
    "decode, ranges of keys": (4, 2, 1, 300),
    "decode, a tile of heads": (12, 1, 1, 0),
    "chunk, a tile": (4, 2, 5, 0),
    "chunk, wide": (2, 2, 40, 0),
    "chunk, wide, ranges of keys": (2, 2, 40, 130),
}


def make(name, hd, dtype, magnitude, v_scale=1.0):
    H, Hk, T, width = SHAPES[name]
    rng = np.random.default_rng(hd + T)
    lens = [T + 200, T + 60]
    kp, vp = filled_pools(rng, 60, Hk, hd)
    if v_scale != 1.0:
        vp = filled_pools(rng, 60, Hk, hd, v_scale)[1]
    table = tables(rng, lens, 60, width=width)
    q = torch.from_numpy(rng.normal(0, 1, (2, H, T, hd)) * magnitude).to(dtype)
    return q, kp, vp, table, lens


def call(device, q, kp, vp, table, lens, totals=None):
    T = q.shape[2]
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    fn = kq.paged_attention_prefill_q4_hip if T > 1 else kq.paged_attention_decode_q4_hip
    return fn(q.to(device), torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device), i32(table), i32(lens),
              i32([T] * len(lens)), weights=totals)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("v_scale", [1.0, 2.0 ** -13])
@pytest.mark.parametrize("name", SHAPES)
def test_outputs_stay_between_the_values(device, dtype, hd, v_scale, name):
    for magnitude in (1e4, 1e6, 2e7, 6e7, 1e8, 3e8, 1e9, 1e12, 1e20, 1e30, 1e35):
        q, kp, vp, table, lens = make(name, hd, dtype, magnitude, v_scale)
        got = call(device, q, kp, vp, table, lens).double().cpu().numpy()
        k, v = q4.values(kp, hd, True), q4.values(vp, hd, False)
        meta = np.ascontiguousarray(kp[:, :, 8 * hd:]).view(np.float16).astype(np.float64).reshape(-1, 2)
        reach = (np.abs(meta[:, 1]) + 15 * meta[:, 0]).max()
        qd = q.double().numpy()
        B, H, T, _ = qd.shape
        one_hot = 0
        for b, L in enumerate(lens):
            blk, tok = np.array([(p, t) for p in table[b] for t in range(16)][:L]).T
            for h in range(H):
                kh = h // (H // k.shape[1])
                for i in range(T):
                    n = L - T + 1 + i
                    s = k[blk[:n], kh, tok[:n]] @ qd[b, h, i] / math.sqrt(hd)
                    # a score is off by 2^-13 (2^-19) of its terms' sizes at the most; keys 40 below the largest
                    # weigh 2^-57
                    off = 2.0 ** (-13 if dtype == torch.bfloat16 else -19) * np.abs(qd[b, h, i]).sum() * reach / math.sqrt(hd)
                    near = v[blk[:n], kh, tok[:n]][s >= s.max() - 2 * off - 40]
                    one_hot += len(near) == 1
                    # bf16's roundings: 2^-8 of the output, 2^-11 of the values' parts; fp32's far less
                    slack = (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18) * np.abs(v).max()
                    assert (got[b, h, i] >= near.min(0) - slack).all() and (got[b, h, i] <= near.max(0) + slack).all(), (
                        magnitude, b, h, i, len(near))
        if magnitude >= 1e6:
            assert one_hot > 0.4 * B * H * T  # (most rows have one key that counts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("name", SHAPES)
def test_a_rows_weights_add_up_to_one(device, dtype, hd, name):
    """The totals of a request's keys add up to the rows that gave weights, at every size of the scores."""
    for magnitude in (0.0, 1.0, 30.0, 300.0, 1e4, 1e5, 1e6, 2e7, 1e8, 3e8, 1e9, 1e12, 1e20, 1e30, 1e35):
        q, kp, vp, table, lens = make(name, hd, dtype, magnitude)
        totals = torch.zeros(60, kp.shape[1], 16, device=device)
        call(device, q, kp, vp, table, lens, totals)
        totals = totals.double().cpu().numpy()
        for b in range(2):
            got = totals[table[b][table[b] >= 0]].sum((0, 2))
            want = q.shape[1] // kp.shape[1] * q.shape[2]
            # exponents of up to 2^8 rounded to fp32, a few sums of a few hundred terms
            assert (np.abs(got - want) <= 2.0 ** -14 * want).all(), (magnitude, got, want)
