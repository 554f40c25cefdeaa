"""The 4-bit page format in torch, on whatever device the tensors live: what the "paged_reference" backend and
pools on the CPU use. The device path (src/kernels/hip_q4_attention.py) writes and reads the same bytes.

A page holds 16 tokens of one KV head. 64 consecutive values of a row share a half-precision scale s and
centre z, and a code c in 0..15 stands for z + s (c - 7.5). A page's bytes are its codes, then the pairs (s, z)
as [group][token]; the codes' places are those that the matrix instructions' lanes take them from
(csrc/pa_q4.h).
"""
from __future__ import annotations

import functools

import torch

BLOCK = 16
GROUP = 64
HEAD_DIMS = (64, 128)
HALF_MAX = 65504.0


def page_bytes(head_dim: int) -> int:
    """Bytes of one page of one KV head."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"4-bit pages hold head_dim 64 or 128, got {head_dim}")
    return BLOCK * (head_dim // 2 + 4 * (head_dim // GROUP))


@functools.lru_cache(maxsize=None)
def _places(head_dim: int, is_key: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """([16, head_dim] nibble of each token's values, [16, 4 * groups] byte of each token's pairs)."""
    t, d = torch.arange(BLOCK)[:, None], torch.arange(head_dim)[None]
    if is_key:  # word (token, d / 8 % 4, d / 32); its even values in the low nibbles, the odd ones above
        word = (4 * t + d // 8 % 4) * (head_dim // 32) + d // 32
        nibble = 8 * word + d % 8 // 2 + 4 * (d % 2)
    else:  # word (token / 4, d % 64 / 4, token / 2 % 2, d / 64); the odd token in the high half
        word = ((t // 4 * 16 + d % GROUP // 4) * 2 + t // 2 % 2) * (head_dim // GROUP) + d // GROUP
        nibble = 8 * word + 4 * (t % 2) + d % 4
    at = torch.arange(4 * (head_dim // GROUP))
    return nibble, BLOCK * head_dim // 2 + at // 4 * (4 * BLOCK) + 4 * t + at % 4


def quantise(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Rows [..., head_dim] -> codes (uint8, same shape), s and z (float16 [..., groups])."""
    x = rows.float().unflatten(-1, (-1, GROUP))
    bad = x.isnan().any(-1)
    x = x.nan_to_num(0.0, HALF_MAX, -HALF_MAX).clamp(-HALF_MAX, HALF_MAX)
    hi, lo = x.amax(-1), x.amin(-1)
    s = ((hi - lo) * (1.0 / 15.0)).half()
    z = ((hi + lo) * 0.5).half() + 0.0  # a centre of zero is +0
    step = s.double()[..., None]
    # in 64 bits, so that a value next to a border between two codes goes to its own side
    c = (x.double() - z.double()[..., None]) / torch.where(step > 0, step, 1.0) + 7.5
    c = torch.where((step > 0) & ~bad[..., None], c.round().clamp(0, 15), 0.0)
    nan = torch.full_like(s, float("nan"))
    return c.to(torch.uint8).flatten(-2), torch.where(bad, nan, s), torch.where(bad, nan, z)


def put_rows(pool: torch.Tensor, blocks: torch.Tensor, offsets: torch.Tensor, rows: torch.Tensor, is_key: bool) -> None:
    """Quantise rows [n, heads, head_dim] into token offsets[i] of block blocks[i]."""
    c, s, z = quantise(rows)
    nibble, pair = (p.to(pool.device)[offsets] for p in _places(rows.shape[-1], is_key))
    order = nibble.argsort(-1)  # two values to a byte: the even nibble's, then the odd one's
    c = c.gather(-1, order[:, None].expand_as(c))
    head = torch.arange(pool.shape[1], device=pool.device)[None, :, None]
    at = nibble.gather(-1, order)[:, ::2] // 2
    pool[blocks[:, None, None], head, at[:, None]] = c[..., ::2] | c[..., 1::2] << 4
    both = torch.stack([s, z], -1).flatten(-2).contiguous().view(torch.uint8)
    pool[blocks[:, None, None], head, pair[:, None]] = both


def values(pages: torch.Tensor, head_dim: int, is_key: bool) -> torch.Tensor:
    """Pages [n, heads, bytes] -> the float32 values that they stand for, [n, heads, 16, head_dim]."""
    nibble, _ = _places(head_dim, is_key)
    nibble = nibble.to(pages.device)
    c = (pages[:, :, nibble // 2] >> (4 * (nibble % 2)).to(torch.uint8)) & 15
    pairs = pages[:, :, BLOCK * head_dim // 2:].contiguous().view(torch.float16).float()
    pairs = pairs.unflatten(-1, (head_dim // GROUP, BLOCK, 2)).transpose(2, 3)  # [n, heads, token, group, 2]
    x = c.float().unflatten(-1, (-1, GROUP)) - 7.5
    return (pairs[..., 1:] + pairs[..., :1] * x).flatten(-2)


def choose(weights: torch.Tensor, keep: int, window: int) -> torch.Tensor:
    """Totals [heads, n] of n > keep keys -> the kept keys' indices [heads, keep], ascending: the newest
    `window` and, of the others, those of the largest totals (the lower index where they are equal)."""
    old = weights.shape[1] - window
    best = torch.sort(weights[:, :old], dim=1, descending=True, stable=True).indices[:, :keep - window]
    newest = torch.arange(old, old + window, device=weights.device).expand(weights.shape[0], window)
    return torch.cat([best, newest], 1).sort(1).values


def move_rows(pool: torch.Tensor, src: tuple, dst: tuple, head_dim: int, is_key: bool) -> None:
    """Move tokens bit for bit: src and dst are (blocks, offsets), each [heads, n]."""
    nibble, pair = (p.to(pool.device) for p in _places(head_dim, is_key))
    place = torch.cat([nibble.sort(-1).values[:, ::2] // 2, pair], 1)  # a token's bytes, in one order for all tokens
    head = torch.arange(pool.shape[1], device=pool.device)[:, None, None]
    pool[dst[0][..., None], head, place[dst[1]]] = pool[src[0][..., None], head, place[src[1]]]
