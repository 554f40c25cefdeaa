"""torch-facing wrappers of the 4-bit paged KV cache of libpaged_hip.

  kv_append_q4_hip              new K/V rows quantised into their pool slots            (pa_q4_append)
  kv_read_q4_hip                slots read back as the values that they stand for       (pa_q4_read)
  paged_attention_decode_q4_hip   one query row per request over 4-bit pages         (pa_q4_attention)
  paged_attention_prefill_q4_hip  causal chunks over 4-bit pages                     (pa_q4_attention)
  evict_q4_hip                  keys cut back to the newest and the heaviest ones        (pa_q4_evict)

Pools are uint8 [num_blocks, kv_heads, page_bytes(head_dim)], one for K and one for V, 16 tokens a page,
head_dim 64 or 128 (4.5 bits a value: 64 values share a half-precision scale and centre); query heads
may be a multiple of the KV heads. `weights` is a float32 [num_blocks, kv_heads, 16] tensor beside the
pools, the running total of the attention weight that each slot's key has had: the append clears a
written slot's, attention adds to it, the eviction goes by it.

No reference counterpart (its pools hold the model's dtype). All work is enqueued on the current stream
of the tensors' device; nothing here synchronises, and there is no CPU path.
"""
from __future__ import annotations

import contextlib
import math

import torch

from src.kernels import _lib
from src.kernels.hip_paged_attention import _call_workspace, _check_out, _require_i32, _stream_ptr, native_call
from src.kernels.reference_q4 import BLOCK, HEAD_DIMS, page_bytes

def _on_device(device: torch.device):
    """The device of the operands as the current one, for a launch on its stream."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check_device(name: str, device: torch.device, **tensors: torch.Tensor | None) -> None:
    for what, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name}: {what} is on {t.device}, expected {device}")


def _check_q4_pools(name: str, k_pool: torch.Tensor, v_pool: torch.Tensor, weights: torch.Tensor | None) -> int:
    """Checks the pools and returns their head_dim."""
    for t in (k_pool, v_pool):
        if not t.is_cuda:
            raise ValueError(f"{name}: the pools must be on a HIP device, got {t.device}")
    if k_pool.dtype != torch.uint8 or k_pool.dim() != 3 or v_pool.dtype != torch.uint8 or v_pool.shape != k_pool.shape:
        raise ValueError(f"{name}: K/V pools must be uint8 [num_blocks, kv_heads, page_bytes] of one shape")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError(f"{name}: K/V pools must be contiguous")
    head_dim = next((hd for hd in HEAD_DIMS if page_bytes(hd) == k_pool.shape[2]), None)
    if head_dim is None:
        raise ValueError(f"{name}: pages of {k_pool.shape[2]} bytes are no 4-bit pages (head_dim 64: {page_bytes(64)}, "
                         f"128: {page_bytes(128)})")
    _check_device(name, k_pool.device, v_pool=v_pool, weights=weights)
    if weights is not None and (weights.dtype != torch.float32 or not weights.is_contiguous()
                                or tuple(weights.shape) != (*k_pool.shape[:2], BLOCK)):
        raise ValueError(f"{name}: weights must be a contiguous float32 {(*k_pool.shape[:2], BLOCK)} tensor")
    return head_dim


def _check_table(name: str, table: torch.Tensor, batch: int) -> tuple[int, int]:
    """(row stride, width) of an int32 page table of at least `batch` rows."""
    _require_i32(name, table)
    if table.dim() != 2 or table.shape[0] < batch:
        raise ValueError(f"{name} must be [requests, pages] with a row for each of {batch} requests, got {tuple(table.shape)}")
    return max(table.stride(0), table.shape[1]), table.shape[1]


def _check_lens(name: str, t: torch.Tensor, batch: int) -> None:
    _require_i32(name, t)
    if t.numel() < batch:
        raise ValueError(f"{name} has {t.numel()} entries for {batch} requests")


def kv_append_q4_hip(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     slot_mapping: torch.Tensor, *, weights: torch.Tensor | None = None) -> None:
    """Quantise k_new/v_new [B, kv_heads, T, head_dim] (float32 or bfloat16) into their slots (slot_mapping int32
    [B * T]; -1 = skip). weights: the written slots' totals are cleared."""
    native = native_call()
    if native is not None and native.q4_append(k_new, v_new, k_pool, v_pool, slot_mapping, weights) is not None:
        return
    name = "kv_append_q4_hip"
    head_dim = _check_q4_pools(name, k_pool, v_pool, weights)
    _check_device(name, k_pool.device, k_new=k_new, v_new=v_new, slot_mapping=slot_mapping)
    _require_i32("slot_mapping", slot_mapping)
    if k_new.dim() != 4 or v_new.shape != k_new.shape or v_new.dtype != k_new.dtype:
        raise ValueError(f"{name}: k_new and v_new must be [B, kv_heads, T, head_dim] of one shape and dtype")
    B, H, T, Hd = k_new.shape
    if (H, Hd) != (k_pool.shape[1], head_dim):
        raise ValueError(f"{name}: pool heads/head_dim {k_pool.shape[1]}/{head_dim} do not match new rows {H}/{Hd}")
    if slot_mapping.numel() != B * T:
        raise ValueError(f"slot_mapping has {slot_mapping.numel()} entries, expected {B * T}")
    dtype = _lib.dtype_code(k_new.dtype)
    if k_new.stride() != v_new.stride() or k_new.stride(3) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    with _on_device(k_pool.device):
        status = _lib.load().pa_q4_append(
            k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1), k_new.stride(2), dtype,
            k_pool.data_ptr(), v_pool.data_ptr(), k_pool.shape[0], weights.data_ptr() if weights is not None else None,
            slot_mapping.data_ptr(), B, H, T, Hd, _stream_ptr(k_pool.device),
        )
    _lib.check(status, "pa_q4_append")


def kv_read_q4_hip(k_pool: torch.Tensor, v_pool: torch.Tensor, slot_mapping: torch.Tensor, *, batch: int = 1,
                   dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The values that slots stand for: (k, v), each [batch, kv_heads, T, head_dim], for slot_mapping int32
    [batch * T]; zeros where a slot is negative or outside the pool. The tensors are views of [batch, T,
    kv_heads, head_dim] memory, the layout that the model's projections leave."""
    code = _lib.dtype_code(dtype)
    native = native_call()
    if native is not None:
        done = native.q4_read(k_pool, v_pool, slot_mapping, batch, code)
        if done is not None:
            return done
    name = "kv_read_q4_hip"
    head_dim = _check_q4_pools(name, k_pool, v_pool, None)
    _check_device(name, k_pool.device, slot_mapping=slot_mapping)
    _require_i32("slot_mapping", slot_mapping)
    if batch < 1 or slot_mapping.numel() % batch:
        raise ValueError(f"{name}: {slot_mapping.numel()} slots are no whole rows of {batch} requests")
    H, T = k_pool.shape[1], slot_mapping.numel() // batch
    k = torch.empty((batch, T, H, head_dim), dtype=dtype, device=k_pool.device).transpose(1, 2)
    v = torch.empty((batch, T, H, head_dim), dtype=dtype, device=k_pool.device).transpose(1, 2)
    with _on_device(k_pool.device):
        status = _lib.load().pa_q4_read(
            k_pool.data_ptr(), v_pool.data_ptr(), k_pool.shape[0], slot_mapping.data_ptr(),
            k.data_ptr(), v.data_ptr(), T * H * head_dim, head_dim, H * head_dim, code, batch, H, T, head_dim,
            _stream_ptr(k_pool.device),
        )
    _lib.check(status, "pa_q4_read")
    return k, v


def paged_attention_decode_q4_hip(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    current_lengths: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention for q [B, H, 1, head_dim] over 4-bit pages; returns a tensor shaped and strided like q.
    weights: every key's softmax weight, summed over the query heads of its KV head, is added to its
    slot's total (requests with current_lengths 0 add nothing)."""
    if q.dim() == 4 and q.shape[2] != 1:
        raise ValueError(f"decode expects query_len 1, got {q.shape[2]}")
    return _attention("paged_attention_decode_q4_hip", q, k_pool, v_pool, page_table, seq_lens, current_lengths, weights, out)


def paged_attention_prefill_q4_hip(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    current_lengths: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Chunked causal prefill attention for q [B, H, T, head_dim] over 4-bit pages (the chunk's keys appended
    before); returns a tensor shaped like q. weights: as in decode, summed over the chunk's real rows
    (i < current_lengths[b])."""
    return _attention("paged_attention_prefill_q4_hip", q, k_pool, v_pool, page_table, seq_lens, current_lengths, weights, out)


def _attention(name, q, k_pool, v_pool, page_table, seq_lens, current_lengths, weights, out):
    native = native_call()
    if native is not None:
        done = native.q4_attention(q, k_pool, v_pool, page_table, seq_lens, current_lengths, weights, out)
        if done is not None:
            return done
    head_dim = _check_q4_pools(name, k_pool, v_pool, weights)
    _check_device(name, k_pool.device, q=q, page_table=page_table, seq_lens=seq_lens, current_lengths=current_lengths)
    if q.dim() != 4:
        raise ValueError(f"{name}: q must be [B, H, T, head_dim], got {tuple(q.shape)}")
    B, H, T, Hd = q.shape
    heads = k_pool.shape[1]
    if Hd != head_dim or H % heads or H == 0:
        raise ValueError(f"{name}: q heads/head_dim {H}/{Hd} do not go with the pools' {heads}/{head_dim}")
    dtype = _lib.dtype_code(q.dtype)
    if q.stride(3) != 1:
        q = q.contiguous()
    stride, max_pages = _check_table("page_table", page_table, B)
    _check_lens("seq_lens", seq_lens, B)
    _check_lens("current_lengths", current_lengths, B)
    if out is None:
        out = torch.empty_like(q)
    _check_out(name, out, q)
    lib = _lib.load()
    with _on_device(q.device):
        need = lib.pa_q4_attention_workspace_size(dtype, B, H, heads, T, Hd, max_pages, weights is not None)
        ws = _call_workspace(q.device, need, "q4") if need else None
        status = lib.pa_q4_attention(
            q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
            out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), dtype,
            k_pool.data_ptr(), v_pool.data_ptr(), k_pool.shape[0],
            page_table.data_ptr() if max_pages else None, stride, max_pages,
            seq_lens.data_ptr(), current_lengths.data_ptr(), weights.data_ptr() if weights is not None else None,
            B, H, heads, T, Hd, 1.0 / math.sqrt(Hd), ws.data_ptr() if need else None, need, _stream_ptr(q.device),
        )
    _lib.check(status, "pa_q4_attention")
    return out


def evict_q4_hip(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    weights: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    new_page_table: torch.Tensor,
    *,
    keep: int,
    window: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cut every request back to at most `keep` keys per KV head: the newest `window` and, of the others, those
    of the largest totals (the lower index where totals are equal). The kept rows and totals move, in their
    order, into the pages of new_page_table (int32 [B, pages], none of them an old page of the batch).
    Returns (kept int32 [B, kv_heads, keep], the kept keys' old indices, -1 behind the last; new lengths int32
    [B]). Old pages stay as they are, for the caller to release."""
    native = native_call()
    if native is not None:
        done = native.q4_evict(k_pool, v_pool, weights, page_table, seq_lens, new_page_table, keep, window)
        if done is not None:
            return done
    name = "evict_q4_hip"
    head_dim = _check_q4_pools(name, k_pool, v_pool, weights)
    if weights is None:
        raise ValueError(f"{name} goes by the slots' totals: weights is missing")
    _check_device(name, k_pool.device, page_table=page_table, seq_lens=seq_lens, new_page_table=new_page_table)
    B = seq_lens.numel()
    stride, max_pages = _check_table("page_table", page_table, B)
    new_stride, new_pages = _check_table("new_page_table", new_page_table, B)
    _check_lens("seq_lens", seq_lens, B)
    if keep < 1 or not 0 <= window <= keep:
        raise ValueError(f"{name}: keep ({keep}) must be positive and hold the window ({window})")
    heads = k_pool.shape[1]
    kept = torch.empty((B, heads, keep), dtype=torch.int32, device=k_pool.device)
    lens = torch.empty((B,), dtype=torch.int32, device=k_pool.device)
    with _on_device(k_pool.device):
        status = _lib.load().pa_q4_evict(
            k_pool.data_ptr(), v_pool.data_ptr(), weights.data_ptr(), k_pool.shape[0],
            page_table.data_ptr(), stride, max_pages, seq_lens.data_ptr(),
            new_page_table.data_ptr(), new_stride, new_pages, keep, window, kept.data_ptr(), lens.data_ptr(),
            B, heads, head_dim, _stream_ptr(k_pool.device),
        )
    _lib.check(status, "pa_q4_evict")
    return kept, lens
