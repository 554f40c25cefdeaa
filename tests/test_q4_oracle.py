"""The 4-bit page's definition and the wrappers' refusals, on the CPU."""
import numpy as np
import pytest
import torch

from oracle import q4
from src.kernels import _lib, hip_q4_attention as kq


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("is_k", [True, False])
def test_rows_come_back_within_half_a_step(hd, is_k):
    rng = np.random.default_rng(hd)
    pool = rng.integers(0, 256, (2, 3, q4.page_bytes(hd)), dtype=np.uint8)
    rows = (rng.normal(0, 1, (3, 16, hd)) * 10.0 ** rng.integers(-2, 3, (3, 16, 1))).astype(np.float32)
    rows[0, 3] = 2.5  # a constant row: its centre
    for h in range(3):
        for t in rng.permutation(16):
            q4.put(pool, 1, h, t, rows[h, t], is_k)
    got = q4.values(pool, hd, is_k)[1]
    groups = rows.reshape(3, 16, -1, 64).astype(np.float64)
    step = (groups.max(-1) - groups.min(-1)) / 15
    # half a step, and the roundings of s (15 of them end to end) and z to 11 bits
    tol = step * (0.5 + 15 * 2.0 ** -11) + np.abs(groups).max(-1) * 2.0 ** -11
    assert (np.abs(got.reshape(groups.shape) - groups).max(-1) <= tol).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("is_k", [True, False])
def test_every_nibble_belongs_to_one_value(hd, is_k):
    n = q4._nibbles(hd, is_k)
    assert sorted(n.flatten().tolist()) == list(range(16 * hd))


def test_page_sizes():
    for hd in (64, 128):
        assert kq.page_bytes(hd) == q4.page_bytes(hd) == _lib.load().pa_q4_page_bytes(hd)
    assert _lib.load().pa_q4_page_bytes(96) == 0
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        kq.page_bytes(96)


def test_header_and_signatures_agree():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "paged_hip_q4.h").read_text()
    names = sorted(set(re.findall(r"\b(pa_q4_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))))
    assert names == sorted(_lib.SIGNATURES_Q4)


def test_host_tensors_are_refused():
    pool = torch.zeros(4, 2, kq.page_bytes(64), dtype=torch.uint8)
    i32 = torch.zeros(1, dtype=torch.int32)
    rows = torch.zeros(1, 2, 1, 64)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: kq.kv_append_q4_hip(rows, rows, pool, pool, i32),
                 lambda: kq.kv_read_q4_hip(pool, pool, i32),
                 lambda: kq.paged_attention_decode_q4_hip(rows, pool, pool, table, i32, i32),
                 lambda: kq.evict_q4_hip(pool, pool, torch.zeros(4, 2, 16), table, i32, table, keep=1, window=0)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def _evict(keep=4, window=1, new_pages=1, hd=64):
    return _lib.load().pa_q4_evict(256, 256, 256, 4, 256, 1, 1, 256, 256, max(new_pages, 1), new_pages, keep, window, 256,
                                   256, 1, 2, hd, None)


def _attention(heads=4, kv=2, hd=64, scale=0.125, dtype=0, pages=1, batch=1, ws=None, ws_bytes=0, k=256):
    return _lib.load().pa_q4_attention(256, 1, 1, 1, 256, 1, 1, 1, dtype, k, 256, 4, 256, pages, pages, 256, 256, None, batch,
                                       heads, kv, 1, hd, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("call, status", [
    (lambda: _evict(keep=0), 1), (lambda: _evict(window=5), 1), (lambda: _evict(window=-1), 1),
    (lambda: _evict(new_pages=0), 1), (lambda: _evict(hd=96), 2),
    (lambda: _attention(heads=3), 1), (lambda: _attention(hd=80), 2), (lambda: _attention(scale=0.0), 1),
    (lambda: _attention(scale=float("nan")), 1), (lambda: _attention(dtype=2), 1), (lambda: _attention(k=8), 1),
    (lambda: _attention(pages=4096), 3), (lambda: _attention(batch=-1), 1), (lambda: _attention(batch=0), 0),
])
def test_the_library_refuses_before_it_launches(call, status):
    assert call() == status
    assert bool(_lib.load().pa_last_error_message()) == (status != 0)
