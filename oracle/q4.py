"""ORACLE — test infrastructure only.

The 4-bit paged KV cache in numpy and 64 bits, from its definition: every value's bits are looked up by
their place in the page, and attention and eviction are loops over requests and heads.
"""
from __future__ import annotations

import math

import numpy as np

BLOCK, GROUP = 16, 64


def page_bytes(hd: int) -> int:
    return BLOCK * hd // 2 + BLOCK * (hd // GROUP) * 4


def _nibbles(hd: int, is_k: bool) -> np.ndarray:
    """[16, hd] nibble index of value d of token t."""
    t, d = np.arange(BLOCK)[:, None], np.arange(hd)[None]
    if is_k:
        j = d % 8
        word = (t * 4 + d // 8 % 4) * (hd // 32) + d // 32
        return word * 8 + np.where(j % 2 == 0, j // 2, 4 + j // 2)
    word = ((t // 4 * 16 + d % GROUP // 4) * 2 + t % 4 // 2) * (hd // GROUP) + d // GROUP
    return word * 8 + t % 2 * 4 + d % 4


def quantise(x: np.ndarray):
    """x [..., hd] (float32 values) -> codes, s, z; a group with a NaN gets NaN for both and codes 0."""
    x = np.asarray(x, dtype=np.float32)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    bad = np.isnan(g).any(-1)
    g = np.clip(np.where(np.isnan(g), np.float32(0), g), np.float32(-65504), np.float32(65504))
    hi, lo = g.max(-1), g.min(-1)
    s = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
    z = ((hi + lo) * np.float32(0.5)).astype(np.float16) + np.float16(0)  # a centre of zero is +0
    sd, zd = s.astype(np.float64)[..., None], z.astype(np.float64)[..., None]
    c = np.rint((g.astype(np.float64) - zd) / np.where(sd > 0, sd, 1) + 7.5).clip(0, 15)
    c = np.where((sd > 0) & ~bad[..., None], c, 0).astype(np.int64)
    return (c.reshape(x.shape), np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(np.nan), z))


def put(pool: np.ndarray, block: int, head: int, token: int, row: np.ndarray, is_k: bool) -> None:
    hd = row.shape[-1]
    c, s, z = quantise(row)
    page = pool[block, head]
    for n, code in zip(_nibbles(hd, is_k)[token], c):
        shift = 4 * (int(n) % 2)
        page[n // 2] = (int(page[n // 2]) & (0xF0 >> shift)) | (int(code) << shift)
    meta = page[BLOCK * hd // 2:].view(np.float16).reshape(hd // GROUP, BLOCK, 2)
    meta[:, token, 0], meta[:, token, 1] = s, z


def values(pool: np.ndarray, hd: int, is_k: bool) -> np.ndarray:
    """Pool [N, H, bytes] -> float64 [N, H, 16, hd]."""
    pool = np.ascontiguousarray(pool)
    n = _nibbles(hd, is_k)
    c = pool[:, :, n // 2] >> (4 * (n % 2)) & 15
    meta = np.ascontiguousarray(pool[:, :, BLOCK * hd // 2:]).view(np.float16).astype(np.float64)
    meta = meta.reshape(*pool.shape[:2], hd // GROUP, BLOCK, 2).swapaxes(2, 3).repeat(GROUP, axis=3)
    return meta[..., 1] + meta[..., 0] * (c - 7.5)


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, page_table, seq_lens, cur_lens):
    """q [B, H, T, hd] float64, k / v values [N, Hk, 16, hd] -> (out, weight added per slot [N, Hk, 16])."""
    B, H, T, hd = q.shape
    N, Hk = k.shape[:2]
    out = np.zeros(q.shape)
    added = np.zeros((N, Hk, BLOCK))
    for b in range(B):
        L, C = int(seq_lens[b]), int(cur_lens[b])
        pages = [int(p) for p in page_table[b]]
        slots = [(p, t) for p in pages for t in range(BLOCK)][:max(L, 0)]
        for h in range(H):
            kh = h // (H // Hk)
            for i in range(T):
                n = max(min(len(slots), L - C + 1 + i), 0)
                at = [s for s in slots[:n] if 0 <= s[0] < N]
                if not at:
                    continue
                blk, tok = np.array(at).T
                a = k[blk, kh, tok] @ q[b, h, i] / math.sqrt(hd)
                p = np.exp(a - a.max())
                p /= p.sum()
                out[b, h, i] = p @ v[blk, kh, tok]
                if i < C:
                    np.add.at(added, (blk, kh, tok), p)
    return out, added


def evict(weights: np.ndarray, page_table, seq_lens, keep: int, window: int):
    """kept [B][Hk] lists of ascending indices."""
    N, Hk = weights.shape[:2]
    out = []
    for row, L in zip(page_table, seq_lens):
        L = min(int(L), BLOCK * len(row))
        heads = []
        for h in range(Hk):
            def rank(t):
                p = int(row[t // BLOCK])
                if not 0 <= p < N:
                    return (0, 0.0)
                w = float(weights[p, h, t % BLOCK])
                return (2, 0.0) if math.isnan(w) else (1, w)
            old = list(range(max(L - window, 0))) if L > keep else []
            best = sorted(old, key=lambda t: (rank(t), -t), reverse=True)[:keep - window]
            heads.append(sorted(best) + list(range(L - window, L)) if L > keep else list(range(max(L, 0))))
        out.append(heads)
    return out
