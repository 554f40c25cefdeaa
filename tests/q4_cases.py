"""Pools, tables and tolerances of the 4-bit cache's tests."""
import math

import numpy as np
import torch

from oracle import q4

BLOCK = 16


def filled_pools(rng, blocks, heads, hd, scale=1.0):
    """K and V pools (numpy) whose every slot holds random codes, scales and centres."""
    out = []
    for _ in range(2):
        pool = rng.integers(0, 256, (blocks, heads, q4.page_bytes(hd)), dtype=np.uint8)
        meta = pool[:, :, BLOCK * hd // 2:].reshape(blocks, heads, -1)
        pairs = np.empty((blocks, heads, hd // 64, BLOCK, 2), dtype=np.float16)
        pairs[..., 0] = scale * rng.uniform(0.2, 0.45, pairs.shape[:-1])
        pairs[..., 1] = scale * rng.normal(0, 0.2, pairs.shape[:-1])
        meta[...] = pairs.reshape(blocks, heads, -1).view(np.uint8)
        out.append(pool)
    return out


def poison(pool, hd, block, tokens):
    """NaN scales and centres in a block's tokens, for every head."""
    meta = pool[block][:, BLOCK * hd // 2:].view(np.float16).reshape(pool.shape[1], hd // 64, BLOCK, 2)
    meta[:, :, tokens] = np.nan


def tables(rng, lens, blocks, width=0):
    """Shuffled block lists for requests of these lengths, -1 padded."""
    need = [-(-max(n, 0) // BLOCK) for n in lens]
    ids = rng.permutation(blocks)[:sum(need)]
    table = np.full((len(lens), max(need + [width, 1])), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def bounds(q, k_pool, v_pool, hd, out, dtype):
    """Absolute bound of an output's error, elementwise, and the relative one of a weight.

    A score's terms add up to at most A = scale * sum_d |q_d| (|z| + 15 s). fp32 q: both operands hold
    their values to 2^-22, the products' sum, the two fp32 corrections and the exponent's argument round
    some 8 times at 2^-23 of A, so a score is off by at most 2^-19 A; a weight by that and the exponent's and
    the denominator's 2^-21, and an output by twice a weight's relative error (numerator and
    denominator), and the accumulators' 2^-20, of the largest value |z| + 15 s. bf16 q: the codes enter as
    fp16 subnormals, whose products align with 10 bits fewer: 2^-13 of A in place of 2^-19 A at the very
    most; weights round to fp16 (2^-12, both ways); the output rounds to bf16, 2^-8 of itself."""
    def largest(pool):
        m = np.ascontiguousarray(pool[:, :, BLOCK * hd // 2:]).view(np.float16).astype(np.float64).reshape(-1, 2)
        m = m[~np.isnan(m).any(1)]
        return float((np.abs(m[:, 1]) + 15 * m[:, 0]).max())
    a = float(np.abs(q).sum(-1).max()) / math.sqrt(hd) * largest(k_pool)
    if dtype == torch.float32:
        rel = a * 2.0 ** -19 + 2.0 ** -20
        return 2 * (rel + 2.0 ** -20) * largest(v_pool) + 2.0 ** -23 * np.abs(out), rel
    rel = a * 2.0 ** -13
    return 2 * (rel + 2.0 ** -12) * largest(v_pool) + 2.0 ** -8 * np.abs(out), rel


def to_q(rng, shape, dtype):
    """q on the host in `dtype` and its values in float64."""
    q = torch.from_numpy(rng.normal(0, 1, shape).astype(np.float32)).to(dtype)
    return q, q.double().numpy()
