"""How far bf16 attention over 4-bit pages may be off, row by row from the row's own weights."""
import math

import numpy as np

from oracle import q4

BLOCK = 16
KEYS = 32  # of a matrix instruction of the second product


def _pairs(pool, hd):
    """[blocks, heads, 16, groups, 2] scales and centres."""
    n, heads = pool.shape[:2]
    m = np.ascontiguousarray(pool[:, :, BLOCK * hd // 2:]).view(np.float16).astype(np.float64)
    return m.reshape(n, heads, hd // 64, BLOCK, 2).swapaxes(2, 3)


def attention(q, k_pool, v_pool, hd, table, lens, cur):
    """(out, totals added, bound of out, bound of the totals) for q [B, H, T, hd] whose values are bf16's.

    Scores. The codes enter the matrix cores as fp16 subnormals, whose products they align by their nominal
    exponent, 2^10 above that of code 1, to 24 bits: a product of code 1's unit and q keeps 2^-13 of the
    row's largest |q|, each of the 64 of a group, the start and the join of the two instructions: 66 s 2^-13
    max|q|. The centres' part is fp32, 2^-22 of its terms. The exponent's argument is below 2^5 in size, its
    roundings and the exponential's are below 2^-18. All times a key's weight is e^E off, and, the denominator
    likewise, an output by e^2E - 1 times sum p |v - out|.
    Second product. w = p s rounds to fp16, 2^-11 of w (and 2^-25 of 2^4, what the heaviest key's w is held
    near, where w is subnormal), beside a code within 7.5 of the middle: 2^-11 sum p |v - z|. Its products
    align as those above, in instructions of 32 keys: 2^-14 of an instruction's largest w each. The sums so far
    round to 2^-24 per product: n 2^-24 of 15 sum w + 7.5 sum w + sum p |z|.
    Output: bf16, 2^-8."""
    B, H, T, _ = q.shape
    N, Hk = k_pool.shape[:2]
    kv, vv = q4.values(k_pool, hd, True), q4.values(v_pool, hd, False)
    km, vm = _pairs(k_pool, hd), _pairs(v_pool, hd)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    added, off = np.zeros((N, Hk, BLOCK)), np.zeros((N, Hk, BLOCK))
    for b in range(B):
        L, C = int(lens[b]), int(cur[b])
        slots = [(int(p), t) for p in table[b] for t in range(BLOCK)][:max(L, 0)]
        if not slots:
            continue
        blk, tok = np.array(slots).T
        blocks32 = np.arange(len(slots)) // KEYS
        for h in range(H):
            kh = h // (H // Hk)
            k, v, ks, vs = kv[blk, kh, tok], vv[blk, kh, tok], km[blk, kh, tok], vm[blk, kh, tok]
            for i in range(T):
                n = max(min(L, L - C + 1 + i), 0)
                if n == 0:
                    continue
                x = q[b, h, i]
                s = k[:n] @ x / math.sqrt(hd)
                p = np.exp(s - s.max())
                p /= p.sum()
                o = p @ v[:n]
                out[b, h, i] = o
                terms = np.abs(x).reshape(-1, 64).sum(1)
                e = (66 * 2.0 ** -13 * np.abs(x).max() * ks[:n, :, 0].sum(1)
                     + 2.0 ** -22 * (np.abs(ks[:n, :, 1]) + 8 * ks[:n, :, 0]) @ terms) / math.sqrt(hd)
                grow = math.expm1(2 * (e.max() + 2.0 ** -18))
                scale = np.repeat(vs[:n, :, 0], 64, axis=1)
                centre = np.repeat(vs[:n, :, 1], 64, axis=1)
                w = p[:, None] * scale
                largest = np.zeros((blocks32[n - 1] + 1, hd))
                np.maximum.at(largest, blocks32[:n], w)
                err = (grow * (p @ np.abs(v[:n] - o)) + 2.0 ** -11 * (p @ np.abs(v[:n] - centre))
                       + n * 7.5 * 2.0 ** -25 * 2.0 ** -4 * scale.max() + KEYS * 2.0 ** -14 * largest.sum(0)
                       + n * 2.0 ** -24 * (22.5 * w.sum(0) + p @ np.abs(centre)))
                tol[b, h, i] = err + 2.0 ** -8 * (np.abs(o) + err)
                if i < C:
                    np.add.at(added, (blk[:n], kh, tok[:n]), p)
                    np.add.at(off, (blk[:n], kh, tok[:n]), p * grow)
    return out, added, tol, off
