"""The cases of the bf16 precision tests, on the CPU (mistakes planted in the oracle) and on the GPU."""
import numpy as np
import torch

from q4_cases import filled_pools, tables

# heads, KV heads, rows, lengths, width of the table: on both sides of the launch rules' borders (a row; up to four;
# a tile; two tiles; more), few and many keys
SHAPES = {
    "decode": (4, 2, 1, [300, 47], 0),
    "decode, long": (2, 2, 1, [1025, 700], 0),
    "decode, ranges of keys": (2, 2, 1, [1025, 90], 300),
    "decode, four columns": (2, 2, 1, [1025, 300], 12400),
    "decode, eight heads": (8, 1, 1, [600, 300], 40),
    "decode, three heads": (6, 2, 1, [300, 1025], 0),
    "chunk, a tile": (4, 2, 7, [300, 47], 0),
    "chunk, a tile, long": (8, 2, 3, [700, 300], 40),
    "chunk, two tiles": (6, 2, 7, [400, 90], 0),
    "chunk, wide": (2, 2, 40, [300, 200], 0),
    "chunk, wide, ranges of keys": (3, 1, 33, [900, 300], 260),
}
FLAT, ORDINARY = 0.05, 1.0  # of q: weights that are nearly equal, and those of normal activations


def make(name, hd, q_scale):
    H, Hk, T, lens, width = SHAPES[name]
    rng = np.random.default_rng(sum(map(ord, name)) + hd)
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, Hk, hd)
    q = torch.from_numpy((q_scale * rng.normal(0, 1, (len(lens), H, T, hd))).astype(np.float32)).bfloat16()
    cur = [T] * len(lens)
    return dict(q=q, qd=q.double().numpy(), kp=kp, vp=vp, table=tables(rng, lens, blocks, width=width), lens=lens, cur=cur, hd=hd)
