"""torch-facing wrappers of the C ABI: shape checks, output allocation and a per-device workspace.

Each function launches on the current CUDA stream and never synchronises. Inputs must be CUDA
tensors (or device views of pinned host memory); there is no CPU path.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from lazykv_b200 import _lib as L
from lazykv_b200._lib import call, dtype_code, ptr, require_cuda, stream_handle

_WS: dict[tuple[int, int], torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int, slot: int = 0) -> torch.Tensor:
    """A reusable device buffer of at least `nbytes` (grown on demand), one per (device, slot).

    Calls on one stream run in order, so reusing the buffer between them is safe; work on another
    stream must use another slot.
    """
    key = (device.index if device.index is not None else torch.cuda.current_device(), slot)
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        # Zeroed once: the selection keeps counters at the start of its workspace that must read
        # zero on entry and that its kernels leave zero.
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WS[key] = buf
    return buf


def current_workspace(device: torch.device, slot: int = 0) -> torch.Tensor | None:
    """The buffer workspace() would hand out now for (device, slot), without growing it (None if
    there is none yet): a caller holding an earlier buffer compares identities to see a regrowth."""
    return _WS.get((device.index if device.index is not None else torch.cuda.current_device(), slot))


def packed_pair_bytes(block_size: int, head_dim: int) -> int:
    return int(L.lib().lkv_packed_pair_bytes(block_size, head_dim))


def block_minmax(keys: torch.Tensor, block_size: int, kmin: torch.Tensor, kmax: torch.Tensor, first_block: int = 0) -> None:
    """kmin/kmax[j, first_block + b] = channel min/max of block b of `keys`: [h, n*bs, d] or
    [h, n, bs, d] (any strides; the 4-D form reads blocks that are not evenly spaced tokens, such as
    the keys of a store in its [n, h, 2, bs, d] layout)."""
    require_cuda(keys, kmin, kmax)
    if keys.dim() == 4:
        h, n, bs, d = keys.shape
        if bs != block_size:
            raise ValueError(f"block_minmax: blocks of {bs} tokens, block_size {block_size}")
        s_head, s_blk, s_tok = keys.stride(0), keys.stride(1), keys.stride(2)
    else:
        h, t, d = keys.shape
        n = t // block_size
        s_head, s_tok = keys.stride(0), keys.stride(1)
        s_blk = block_size * s_tok
    if kmin.shape[-1] != d or kmin.dtype != keys.dtype or kmax.dtype != keys.dtype or kmin.stride(-1) != 1 or keys.stride(-1) != 1:
        raise ValueError("block_minmax: metadata must be [h, cap, d] in the keys' dtype, contiguous in d")
    call("lkv_block_minmax", ptr(keys), dtype_code(keys.dtype), h, n, block_size, d, s_head, s_blk, s_tok,
         ptr(kmin), ptr(kmax), kmin.stride(-3) if kmin.dim() >= 3 else kmin.shape[-2] * d, first_block, stream_handle(keys.device))


def pack_int8(pairs: torch.Tensor, records: torch.Tensor | None = None, kmin: torch.Tensor | None = None, kmax: torch.Tensor | None = None,
              first_block: int = 0, deq: torch.Tensor | None = None) -> torch.Tensor:
    """Records [n, h, W] for pairs [n, h, 2, bs, d]; optionally metadata and dequantised pairs.

    kmin/kmax, when given, are [h, cap, d] in the pairs' dtype (written at first_block + b).
    """
    require_cuda(pairs)
    n, h, two, bs, d = pairs.shape
    if two != 2:
        raise ValueError(f"expected a [..., 2, block_size, head_dim] KV pair, got {tuple(pairs.shape)}")
    pairs = pairs.contiguous()
    w = packed_pair_bytes(bs, d)
    if records is None:
        records = torch.empty((n, h, w), dtype=torch.uint8, device=pairs.device)
    m_head = 0 if kmin is None else kmin.stride(-3)
    call("lkv_pack_int8", ptr(pairs), dtype_code(pairs.dtype), n, h, bs, d, ptr(records), ptr(kmin), ptr(kmax), m_head, first_block,
         ptr(deq), stream_handle(pairs.device))
    return records


def unpack_int8(records: torch.Tensor, block_size: int, head_dim: int, dtype: torch.dtype) -> torch.Tensor:
    """[m, W] uint8 records -> [m, 2, bs, d] in `dtype`, bit-exact with the reference's unpack."""
    require_cuda(records)
    out = torch.empty((records.shape[0], 2, block_size, head_dim), dtype=dtype, device=records.device)
    if records.shape[0]:
        call("lkv_unpack_int8", ptr(records.contiguous()), records.shape[0], block_size, head_dim, ptr(out), dtype_code(dtype),
             stream_handle(records.device))
    return out


def fetch_pairs(src: torch.Tensor, src_rows: torch.Tensor, dst: torch.Tensor, dst_rows: torch.Tensor, block_size: int, head_dim: int) -> None:
    """dst row dst_rows[i] <- src row src_rows[i]; int8 records are dequantised into dst's dtype."""
    kind = L.LKV_COLD_INT8 if src.dtype == torch.uint8 else L.LKV_COLD_PAIRS
    n = src_rows.numel()
    if n == 0:
        return
    call("lkv_fetch_pairs", ptr(src), kind, ptr(src_rows), ptr(dst), ptr(dst_rows), n, block_size, head_dim, dtype_code(dst.dtype),
         stream_handle(dst.device))


def quest_topk(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, first_block: int, n_cand: int, k: int,
               bound_dtype: torch.dtype | None = None, out_blocks: torch.Tensor | None = None, want_bound: bool = False,
               bitmap: torch.Tensor | None = None, ws_slot: int = 1, by_block: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Top-k block ids [h, k] (int32) over candidates [first_block, first_block + n_cand) of
    metadata [h, cap, d]: descending bound with ties to the lower id, or ascending id when
    `by_block` (the same set, no sort); optionally the bounds [h, n_cand].

    Its workspace (slot 1 by default) keeps zeroed counters between calls, so it is never shared
    with the attention calls' workspace (slot 0)."""
    dev = require_cuda(query, kmin, kmax)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h = kmin.shape[-3]
    bound_dtype = bound_dtype or q.dtype
    if out_blocks is None:
        out_blocks = torch.empty((h, k), dtype=torch.int32, device=dev)
    if out_blocks.stride(-1) != 1 or out_blocks.shape[-1] < k:
        raise ValueError("quest_topk: out_blocks must be [h, >=k] int32 with unit column stride")
    bound = torch.empty((h, n_cand), dtype=torch.float32, device=dev) if want_bound else None
    nbytes = int(L.lib().lkv_quest_topk_workspace(h, n_cand))
    ws = workspace(dev, nbytes, ws_slot)
    words = 0 if bitmap is None else bitmap.shape[-1]
    call("lkv_quest_topk", ptr(q), dtype_code(q.dtype), hq, h, d, ptr(kmin), ptr(kmax), dtype_code(kmin.dtype), kmin.stride(-3),
         first_block, n_cand, k, dtype_code(bound_dtype), L.LKV_ORDER_BLOCK if by_block else L.LKV_ORDER_BOUND, ptr(out_blocks),
         out_blocks.stride(0), ptr(bound), ptr(bitmap), words, ptr(ws), ws.numel(),
         stream_handle(dev))
    return out_blocks, bound


def quest_topk_resident(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, first_block: int, n_cand: int, k: int,
                        out_blocks: torch.Tensor, block_slot: torch.Tensor, hot: torch.Tensor, bitmap: torch.Tensor,
                        bound_dtype: torch.dtype | None = None, ws_slot: int = 1) -> torch.Tensor:
    """The selection (block order) for an attention before the admit: out_blocks [h, k] the chosen
    ids, hot [h, >= k] (a view, unit column stride) each chosen block's current slot or -1, and the
    bitmap of the resident chosen blocks only (lkv_quest_topk_resident)."""
    dev = require_cuda(query, kmin, kmax, out_blocks, block_slot, hot, bitmap)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h = kmin.shape[-3]
    bound_dtype = bound_dtype or q.dtype
    if hot.stride(-1) != 1 or hot.shape[-1] < k or block_slot.stride(-1) != 1 or not block_slot.is_contiguous():
        raise ValueError("quest_topk_resident: hot must be [h, >=k] with unit column stride and block_slot contiguous [h, cap]")
    ws = workspace(dev, int(L.lib().lkv_quest_topk_workspace(h, n_cand)), ws_slot)
    call("lkv_quest_topk_resident", ptr(q), dtype_code(q.dtype), hq, h, d, ptr(kmin), ptr(kmax), dtype_code(kmin.dtype), kmin.stride(-3), first_block,
         n_cand, k, dtype_code(bound_dtype), ptr(out_blocks), out_blocks.stride(0), ptr(block_slot), block_slot.shape[-1], ptr(hot), hot.stride(0),
         ptr(bitmap), bitmap.shape[-1], ptr(ws), ws.numel(), stream_handle(dev))
    return out_blocks


def quest_bounds(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, first_block: int, n_cand: int, out: torch.Tensor,
                 bound_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The Quest bound of candidates [first_block, first_block + n_cand) into out [h, >= n_cand]
    (bf16 or float32; bf16 only with bf16 bounds), ranked as quest_topk ranks them; nothing else."""
    dev = require_cuda(query, kmin, kmax, out)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h = kmin.shape[-3]
    bound_dtype = bound_dtype or q.dtype
    if out.dim() != 2 or out.shape[0] != h or out.shape[1] < n_cand or out.stride(-1) != 1:
        raise ValueError(f"quest_bounds: out must be [{h}, >={n_cand}] with unit column stride, got {tuple(out.shape)}")
    call("lkv_quest_bounds", ptr(q), dtype_code(q.dtype), hq, h, d, ptr(kmin), ptr(kmax), dtype_code(kmin.dtype), kmin.stride(-3), first_block,
         n_cand, dtype_code(bound_dtype), ptr(out), dtype_code(out.dtype), out.stride(0), stream_handle(dev))
    return out


def topk_gathered(gathered: torch.Tensor, seg_n: list[int], k: int, rank: int, out_base: int, out: torch.Tensor,
                  bitmap: torch.Tensor | None = None, out_cols: int | None = None, block_slot: torch.Tensor | None = None,
                  hot: torch.Tensor | None = None) -> torch.Tensor:
    """Rank `rank`'s part of the global top-k over every rank's bounds gathered as [world, h, ld]
    (rank r holding seg_n[r] candidates after rank r-1's): out [h, >= out_cols] gets the chosen local
    ids (out_base + index in the rank), ascending, then -1; the bitmap those ids. With `block_slot`
    [h, cap] and `hot` [h, >= out_cols] (the resident split, lkv_topk_gathered_resident): hot gets
    each chosen block's current slot or -1, and the bitmap marks only the resident ones."""
    import ctypes

    dev = require_cuda(gathered, out)
    world, h, ld = gathered.shape
    if len(seg_n) != world or gathered.stride(-1) != 1 or not gathered.is_contiguous():
        raise ValueError("topk_gathered: gathered must be a contiguous [world, h, ld] with one count per rank")
    out_cols = out.shape[-1] if out_cols is None else out_cols
    counts = (ctypes.c_int32 * world)(*seg_n)
    words = 0 if bitmap is None else bitmap.shape[-1]
    if block_slot is None:
        call("lkv_topk_gathered", ptr(gathered), dtype_code(gathered.dtype), world, h, ld, ctypes.cast(counts, ctypes.c_void_p), k, rank, out_base,
             ptr(out), out.stride(0), out_cols, ptr(bitmap), words, stream_handle(dev))
    else:
        if hot is None or hot.stride(-1) != 1 or not block_slot.is_contiguous():
            raise ValueError("topk_gathered: the resident split needs hot [h, >=out_cols] (unit column stride) and a contiguous block_slot")
        call("lkv_topk_gathered_resident", ptr(gathered), dtype_code(gathered.dtype), world, h, ld, ctypes.cast(counts, ctypes.c_void_p), k, rank,
             out_base, ptr(out), out.stride(0), out_cols, ptr(bitmap), words, ptr(block_slot), block_slot.shape[-1], ptr(hot), hot.stride(0),
             stream_handle(dev))
    return out


def attention_workspace_bytes(h: int, hq: int, d: int, n_items: int) -> int:
    return int(L.lib().lkv_attention_workspace(h, hq, d, n_items))


def storage_rows(k_base: torch.Tensor, v_base: torch.Tensor, strides: tuple[int, int, int], h: int, block_size: int, d: int) -> int:
    """Storage rows addressable through (s_row, s_head, s_tok) for KV heads 0..h-1 inside both
    tensors' storage: the bound of the tensor-map loads (0 when not even one row fits)."""
    s_row, s_head, s_tok = strides
    reach = (h - 1) * s_head + (block_size - 1) * s_tok + d  # elements one row spans past its start
    rows = []
    for t in (k_base, v_base):
        avail = t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()
        rows.append(0 if avail < reach else (avail - reach) // s_row + 1)
    return max(0, min(rows))


def hot_attention(query: torch.Tensor, k_base: torch.Tensor, v_base: torch.Tensor, strides: tuple[int, int, int], blocks: torch.Tensor,
                  last_fill: int, scale: float, block_size: int, slot_of: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None, ws_slot: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of query [hq, d] over, per KV head j, the blocks listed in blocks[j] (int32 [h, n]).

    Block b of head j is storage row slot_of[j, b] (or b), its key (t, c) at
    k_base[row*s_row + j*s_head + t*s_tok + c]; the last listed block has `last_fill` live tokens.
    Returns float32 (out [hq, d], lse [hq]).
    """
    dev = require_cuda(query, k_base, v_base, blocks)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h, n = blocks.shape
    out = torch.empty((hq, d), dtype=torch.float32, device=dev) if out is None else out
    lse = torch.empty((hq,), dtype=torch.float32, device=dev) if lse is None else lse
    ws = workspace(dev, attention_workspace_bytes(h, hq, d, n), ws_slot)
    s_row, s_head, s_tok = strides
    n_rows = storage_rows(k_base, v_base, strides, h, block_size, d)
    call("lkv_hot_attention", ptr(q), hq, h, d, block_size, ptr(k_base), ptr(v_base), dtype_code(k_base.dtype), s_row, s_head, s_tok, n_rows,
         ptr(blocks), n, ptr(slot_of), 0 if slot_of is None else slot_of.stride(0), last_fill, scale, ptr(out), ptr(lse), ptr(ws), ws.numel(),
         stream_handle(dev))
    return out, lse


def cold_attention(query: torch.Tensor, cold: torch.Tensor, block_size: int, first_block: int, n_blocks: int, scale: float,
                   excluded: torch.Tensor | None = None, dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None, ws_slot: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Exact attention of query [hq, d] over blocks [first_block, first_block + n_blocks) of the
    cold store, minus the blocks set in excluded [h, words] (uint32 bitmap, viewed as int32).

    cold: int8 records [blocks, h, W] (uint8) or pairs [blocks, h, 2, bs, d]. Returns float32
    (out [hq, d], lse [hq]); a head with nothing left gets lse = -inf and out = 0.
    """
    dev = require_cuda(query, cold)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h = cold.shape[1]
    kind = L.LKV_COLD_INT8 if cold.dtype == torch.uint8 else L.LKV_COLD_PAIRS
    dt = q.dtype if dtype is None else dtype
    if kind == L.LKV_COLD_PAIRS and cold.dtype != dt:
        raise ValueError(f"cold pairs are {cold.dtype} but the query is {dt}")
    out = torch.empty((hq, d), dtype=torch.float32, device=dev) if out is None else out
    lse = torch.empty((hq,), dtype=torch.float32, device=dev) if lse is None else lse
    ws = workspace(dev, attention_workspace_bytes(h, hq, d, n_blocks), ws_slot)
    words = 0 if excluded is None else excluded.shape[-1]
    call("lkv_cold_attention", ptr(q), hq, h, d, block_size, ptr(cold), kind, dtype_code(dt), first_block, n_blocks, ptr(excluded), words,
         scale, ptr(out), ptr(lse), ptr(ws), ws.numel(), stream_handle(dev))
    return out, lse


def lse_merge(outs: torch.Tensor, lses: torch.Tensor, out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
              lse_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Merge partials outs [p, rows, d] / lses [p, rows] (float32) into (out [rows, d], lse [rows])."""
    dev = require_cuda(outs, lses)
    p, rows, d = outs.shape
    out = torch.empty((rows, d), dtype=out_dtype, device=dev) if out is None else out
    lse_out = torch.empty((rows,), dtype=torch.float32, device=dev) if lse_out is None else lse_out
    call("lkv_lse_merge", ptr(outs.contiguous()), ptr(lses.contiguous()), p, rows, d, ptr(out), dtype_code(out.dtype), ptr(lse_out),
         stream_handle(dev))
    return out, lse_out


def lse_merge_packed(parts: torch.Tensor, rows: int, d: int, out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                     lse_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Merge partials packed per part as out [rows, d] then lse [rows] (parts [p, rows * (d + 1)], float32)."""
    dev = require_cuda(parts)
    p = parts.shape[0]
    if parts.stride(-1) != 1 or parts.numel() != p * rows * (d + 1) or not parts.is_contiguous():
        raise ValueError("lse_merge_packed: parts must be contiguous [p, rows * (d + 1)] float32")
    out = torch.empty((rows, d), dtype=out_dtype, device=dev) if out is None else out
    lse_out = torch.empty((rows,), dtype=torch.float32, device=dev) if lse_out is None else lse_out
    call("lkv_lse_merge_packed", ptr(parts), p, rows, d, ptr(out), dtype_code(out.dtype), ptr(lse_out), stream_handle(dev))
    return out, lse_out


def bitmap_words(n_blocks: int) -> int:
    """uint32 words of a per-head block bitmap covering block ids [0, n_blocks)."""
    return max(1, math.ceil(n_blocks / 32))


def exact_attention(query: torch.Tensor, k_base: torch.Tensor, v_base: torch.Tensor, strides: tuple[int, int, int], blocks: torch.Tensor,
                    last_fill: int, cold: torch.Tensor, first_block: int, n_blocks: int, scale: float, block_size: int,
                    excluded: torch.Tensor | None = None, slot_of: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None, parts: tuple[torch.Tensor, torch.Tensor] | None = None,
                    ws_slot: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Hot pass, cold pass and their merge in one launch (plus the combine).

    The hot set is as in `hot_attention`, the cold set as in `cold_attention`; returns the merged
    (out [hq, d] in `out_dtype`, lse [hq] float32). `parts`, when given, receives the per-set float32
    partials (out [2, hq, d], lse [2, hq]), hot first.
    """
    dev = require_cuda(query, k_base, v_base, blocks, cold)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h, n = blocks.shape
    out_dtype = out_dtype or q.dtype
    out = torch.empty((hq, d), dtype=out_dtype, device=dev) if out is None else out
    lse = torch.empty((hq,), dtype=torch.float32, device=dev) if lse is None else lse
    ws = workspace(dev, int(L.lib().lkv_exact_attention_workspace(h, hq, d, n, n_blocks)), ws_slot)
    s_row, s_head, s_tok = strides
    hot = L.HotSet(ptr(k_base), ptr(v_base), dtype_code(k_base.dtype), s_row, s_head, s_tok, ptr(blocks), n, ptr(slot_of),
                   0 if slot_of is None else slot_of.stride(0), last_fill, storage_rows(k_base, v_base, strides, h, block_size, d))
    kind = L.LKV_COLD_INT8 if cold.dtype == torch.uint8 else L.LKV_COLD_PAIRS
    cs = L.ColdSet(ptr(cold), kind, first_block, n_blocks, ptr(excluded), 0 if excluded is None else excluded.shape[-1])
    po, pl = (None, None) if parts is None else parts
    call("lkv_exact_attention", ptr(q), hq, h, d, block_size, ctypes.byref(hot), ctypes.byref(cs), scale, ptr(out), dtype_code(out.dtype),
         ptr(lse), ptr(po), ptr(pl), ptr(ws), ws.numel(), stream_handle(dev))
    return out, lse


def device_status(clear: bool = True) -> int:
    """Status word of the kernels with bounded waits (0 = no wait ran out). Synchronises."""
    st = ctypes.c_int(0)
    call("lkv_device_status", ctypes.byref(st), int(clear))
    return st.value


_ATTACHED: set[int] = set()


def status_attach(device: torch.device | int | None = None) -> None:
    """Points the kernels on `device` at the host mirror of the status word (once per device)."""
    idx = torch.cuda.current_device() if device is None else (device if isinstance(device, int) else device.index)
    idx = torch.cuda.current_device() if idx is None else idx
    if idx in _ATTACHED:
        return
    with torch.cuda.device(idx):
        call("lkv_status_attach")
    _ATTACHED.add(idx)


def status_poll(clear: bool = True) -> int:
    """The host mirror of the status word, read without synchronising (0 when nothing was recorded,
    or when no device has been attached yet)."""
    if not _ATTACHED:
        return 0
    st = ctypes.c_int(0)
    call("lkv_status_poll", ctypes.byref(st), int(clear))
    return st.value


class DeviceWaitError(RuntimeError):
    """A kernel's bounded wait ran out (or a CTA's list overflowed): its output was poisoned."""


def raise_on_status(where: str) -> None:
    """Raises DeviceWaitError when the status mirror holds a code (clearing it)."""
    code = status_poll(clear=True)
    if code:
        what = {L.LKV_DEV_WAIT_TIMEOUT: "a bounded wait on the GPU ran out", L.LKV_DEV_LIST_OVERFLOW: "an attention CTA's item list overflowed"}
        raise DeviceWaitError(f"{where}: {what.get(code, f'device status {code}')} (an earlier step's output is not valid)")


def debug_set(key: int, value: int) -> None:
    """Test hooks of the bounded waits (lkv_debug_set)."""
    call("lkv_debug_set", key, value)


def tier_admit(chosen: torch.Tensor, block_slot: torch.Tensor, slot_block: torch.Tensor, last_used: torch.Tensor, evicted_at: torch.Tensor | None,
               step: int, store: torch.Tensor, pool: torch.Tensor, miss_blk: torch.Tensor, miss_slot: torch.Tensor, n_miss: torch.Tensor,
               slots_out: torch.Tensor | None = None, miss_total: torch.Tensor | None = None) -> None:
    """Device-side residency admit of `chosen` [h, k] plus the fetch of the misses (see lkv_tier_admit);
    `miss_total` (int64 scalar on the device, optional) accumulates the misses."""
    dev = require_cuda(chosen, block_slot, slot_block, last_used, store, pool)
    h, k = chosen.shape
    n_slots = slot_block.shape[1]
    bs, d = pool.shape[-2], pool.shape[-1]
    kind = L.LKV_COLD_INT8 if store.dtype == torch.uint8 else L.LKV_COLD_PAIRS
    call("lkv_tier_admit", ptr(chosen), h, k, chosen.stride(0), ptr(block_slot), block_slot.shape[1], ptr(slot_block), ptr(last_used), n_slots,
         ptr(evicted_at), step, ptr(store), kind, ptr(pool), bs, d, dtype_code(pool.dtype), ptr(miss_blk), ptr(miss_slot), ptr(n_miss),
         ptr(slots_out), 0 if slots_out is None else slots_out.stride(0), ptr(miss_total), stream_handle(dev))


def append_tokens(keys: torch.Tensor, values: torch.Tensor, slot: torch.Tensor, fill: int) -> None:
    """keys / values [h, T, d] (unit channel stride) into pool slot [h, 2, bs, d] at token positions
    fill .. fill + T - 1, in one launch (lkv_append_tokens)."""
    dev = require_cuda(keys, values, slot)
    h, t, d = keys.shape
    if values.shape != keys.shape or keys.dtype != slot.dtype or values.dtype != slot.dtype or keys.stride(-1) != 1 or values.stride(-1) != 1:
        raise ValueError("append_tokens needs keys and values [h, T, d] of the slot's dtype with unit channel stride")
    if not slot.is_contiguous() or slot.shape[0] != h or slot.shape[1] != 2 or slot.shape[-1] != d:
        raise ValueError(f"append_tokens needs a contiguous slot [{h}, 2, bs, {d}]")
    call("lkv_append_tokens", ptr(keys), keys.stride(0), keys.stride(1), ptr(values), values.stride(0), values.stride(1), h, t, d,
         dtype_code(slot.dtype), ptr(slot), slot.shape[2], fill, stream_handle(dev))


def mark_blocks(ids: torch.Tensor, bitmap: torch.Tensor) -> torch.Tensor:
    """Clear `bitmap` [h, words] and set the bit of every block id in `ids` [h, k] (int32; -1 is
    skipped), as the selection marks its own choice (lkv_mark_blocks). Returns `bitmap`."""
    dev = require_cuda(ids, bitmap)
    if ids.dtype != torch.int32 or bitmap.dtype != torch.int32 or ids.stride(-1) != 1 or not bitmap.is_contiguous():
        raise ValueError("mark_blocks needs int32 ids with unit column stride and a contiguous int32 bitmap")
    if ids.shape[0] != bitmap.shape[0]:
        raise ValueError(f"ids has {ids.shape[0]} heads, the bitmap {bitmap.shape[0]}")
    call("lkv_mark_blocks", ptr(ids), ids.shape[0], ids.shape[1], ids.stride(0), ptr(bitmap), bitmap.shape[1], stream_handle(dev))
    return bitmap


def quest_topk_admit(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, first_block: int, n_cand: int, k: int, chosen: torch.Tensor,
                     bitmap: torch.Tensor | None, block_slot: torch.Tensor, slot_block: torch.Tensor, last_used: torch.Tensor,
                     evicted_at: torch.Tensor | None, step: int, store: torch.Tensor, pool: torch.Tensor, miss_blk: torch.Tensor,
                     miss_slot: torch.Tensor, n_miss: torch.Tensor, slots_out: torch.Tensor | None = None,
                     bound_dtype: torch.dtype | None = None, ws_slot: int = 1, miss_total: torch.Tensor | None = None) -> torch.Tensor:
    """quest_topk in block order into `chosen` [h, k] (and the bitmap), then tier_admit of that
    selection, in one library call (lkv_quest_topk_admit). Returns `chosen`."""
    dev = require_cuda(query, kmin, kmax, chosen, block_slot, slot_block, last_used, store, pool)
    hq, d = query.shape[-3] if query.dim() == 4 else query.shape[0], query.shape[-1]
    q = query.reshape(hq, d).contiguous()
    h = kmin.shape[-3]
    if chosen.stride(-1) != 1 or chosen.shape[-1] < k:
        raise ValueError("quest_topk_admit: chosen must be [h, >=k] int32 with unit column stride")
    bound_dtype = bound_dtype or q.dtype
    ws = workspace(dev, int(L.lib().lkv_quest_topk_workspace(h, n_cand)), ws_slot)
    words = 0 if bitmap is None else bitmap.shape[-1]
    kind = L.LKV_COLD_INT8 if store.dtype == torch.uint8 else L.LKV_COLD_PAIRS
    call("lkv_quest_topk_admit", ptr(q), dtype_code(q.dtype), hq, h, d, ptr(kmin), ptr(kmax), dtype_code(kmin.dtype), kmin.stride(-3), first_block,
         n_cand, k, dtype_code(bound_dtype), ptr(chosen), chosen.stride(0), None, ptr(bitmap), words, ptr(ws), ws.numel(), ptr(block_slot),
         block_slot.shape[1], ptr(slot_block), ptr(last_used), slot_block.shape[1], ptr(evicted_at), step, ptr(store), kind, ptr(pool),
         pool.shape[-2], dtype_code(pool.dtype), ptr(miss_blk), ptr(miss_slot), ptr(n_miss), ptr(slots_out),
         0 if slots_out is None else slots_out.stride(0), ptr(miss_total), stream_handle(dev))
    return chosen


# -- the paged cache of a batch, the attention over a shared prefix, and draft verification --------------


_device_of = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream_of = L._RAW_STREAM if L._RAW_STREAM is not None else lambda index: torch.cuda.current_stream(index).cuda_stream
_ENTRY: dict[str, object] = {}  # entries that have been called
_F32, _BF16, _I8, _I32, _I64 = torch.float32, torch.bfloat16, torch.int8, torch.int32, torch.int64


def _run(name: str, args: bytes, index: int) -> None:
    """Entry `name` (an args struct and a stream) on the current stream of device `index`, which is made current."""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(L.lib(), name)
    if index == _device_of():
        rc = fn(args, _stream_of(index))  # type: ignore[operator]
    else:
        with torch.cuda.device(index):
            rc = fn(args, _stream_of(index))  # type: ignore[operator]
    if rc != 0:
        raise L.LkvError(f"{name} failed ({rc}): {L.last_error()}")


def _one_device(who: str, *tensors: torch.Tensor | None) -> int:
    """The index of the one CUDA device that all tensors are on."""
    index = -1
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if at < 0:
                require_cuda(t)
            if index < 0:
                index = at
            elif at != index:
                raise ValueError(f"{who}: tensors on cuda:{index} and cuda:{at}")
    return index


def _cache_geometry(who: str, pages: torch.Tensor, scales: torch.Tensor | None, table: torch.Tensor) -> tuple[int, int, int, int, int, int, int, int, int]:
    """(n_pages, h, bs, d, cache kind, scales' address) of pages [n_pages, h, 2, bs, d], and (batch, row stride,
    columns) of their table."""
    if pages.dim() != 5 or not pages.is_contiguous():
        raise ValueError(f"{who}: pages must be a contiguous [n_pages, h, 2, block_size, head_dim], got {tuple(pages.shape)}")
    n, h, two, bs, d = pages.shape
    if two != 2:
        raise ValueError(f"{who}: pages must be a contiguous [n_pages, h, 2, block_size, head_dim], got {tuple(pages.shape)}")
    if pages.dtype is _I8:
        if scales is None or scales.dtype is not _F32 or scales.shape != (n, h, 2, bs) or not scales.is_contiguous():
            raise ValueError(f"{who}: int8 pages need contiguous float32 scales [{n}, {h}, 2, {bs}]")
        kind, at = 1, scales.data_ptr()  # LKV_CACHE_INT8
    elif scales is not None:
        raise ValueError(f"{who}: scales belong to int8 pages, these are {pages.dtype}")
    else:
        kind, at = 0, 0  # LKV_CACHE_MODEL
    if table.dtype is not _I32 or table.dim() != 2:
        raise ValueError(f"{who}: the page table must be int32 [batch, columns] with unit column stride")
    (batch, cols), (ld, unit) = table.shape, table.stride()
    if unit != 1 and cols > 1:
        raise ValueError(f"{who}: the page table must be int32 [batch, columns] with unit column stride")
    return n, h, bs, d, kind, at, batch, ld, cols


def _per_sequence(who: str, name: str, t: torch.Tensor, batch: int) -> None:
    if t.dtype is not _I32 or t.dim() != 1 or t.numel() != batch or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous int32 [{batch}]")


def paged_write(keys: torch.Tensor, values: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                scales: torch.Tensor | None = None) -> None:
    """Tokens keys / values [batch, T, h, d] (any strides with contiguous channels) into positions
    starts[b] .. starts[b] + T - 1 of their sequences' pages, one launch (lkv_paged_write).

    pages [n_pages, h, 2, bs, d] hold the keys' dtype, or int8 codes with scales [n_pages, h, 2, bs]: one
    scale per token, head and key or value, the row's largest magnitude / 127. table [batch, columns]
    int32 lists each sequence's pages; a token whose page is missing (past the table, an id outside
    [0, n_pages)) is not written, so a batch may be padded. Two tokens must not share a row.
    """
    who = "paged_write"
    index = keys.get_device()
    if index < 0 or not (values.get_device() == pages.get_device() == table.get_device() == starts.get_device() == index) or (
            scales is not None and scales.get_device() != index):
        index = _one_device(who, keys, values, pages, table, starts, scales)
    dtype, shape = keys.dtype, keys.shape
    if keys.dim() != 4 or values.shape != shape or values.dtype is not dtype:
        raise ValueError(f"paged_write: keys and values must be alike, [batch, T, h, d]; got {tuple(shape)} and {tuple(values.shape)}")
    batch, t, h, d = shape
    n, ph, bs, pd, kind, at, rows, ld, cols = _cache_geometry(who, pages, scales, table)
    if ph != h or pd != d or (kind == 0 and pages.dtype is not dtype):
        raise ValueError(f"paged_write: {tuple(shape)} {dtype} tokens do not fit pages {tuple(pages.shape)} {pages.dtype}")
    (kb, kt, kh, kc), (vb, vt, vh, vc) = keys.stride(), values.stride()
    if rows != batch or kc != 1 or vc != 1:
        raise ValueError("paged_write: one table row per sequence, and contiguous channels")
    _per_sequence(who, "starts", starts, batch)
    _run("lkv_paged_write", L.PAGED_ARGS.pack(
        keys.data_ptr(), values.data_ptr(), kb, kt, kh, vb, vt, vh, 1 if dtype is _BF16 else dtype_code(dtype), batch, t, h, d, pages.data_ptr(), kind, at, n, bs,
        table.data_ptr(), ld, cols, starts.data_ptr(), 0, 0, 0), index)


def paged_read(pages: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, n_tokens: int, lens: torch.Tensor | None = None,
               scales: torch.Tensor | None = None, dtype: torch.dtype | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens starts[b] .. starts[b] + n_tokens - 1 of every sequence, read back as (keys, values)
    [batch, n_tokens, h, d], one launch (lkv_paged_read): code * scale rounded once to `dtype` (bfloat16
    by default; model-dtype pages are copied). Tokens at or past lens[b] (int32 [batch], optional) and
    tokens without a page are zeros.
    """
    who = "paged_read"
    index = pages.get_device()
    if index < 0 or not (table.get_device() == starts.get_device() == index) or (lens is not None and lens.get_device() != index) or (
            scales is not None and scales.get_device() != index):
        index = _one_device(who, pages, table, starts, lens, scales)
    n, h, bs, d, kind, at, batch, ld, cols = _cache_geometry(who, pages, scales, table)
    if kind == 0:
        if dtype is not None and dtype is not pages.dtype:
            raise ValueError(f"paged_read: {pages.dtype} pages are read back as {pages.dtype}, not {dtype}")
        dtype = pages.dtype
    elif dtype is None:
        dtype = _BF16
    code = 1 if dtype is _BF16 else dtype_code(dtype)
    if n_tokens < 0:
        raise ValueError(f"paged_read: {n_tokens} tokens")
    _per_sequence(who, "starts", starts, batch)
    if lens is not None:
        _per_sequence(who, "lens", lens, batch)
    if out is None:
        k = pages.new_empty((batch, n_tokens, h, d), dtype=dtype)
        v = torch.empty_like(k)
        out = k, v
    else:
        k, v = out
        for o in out:
            if o.shape != (batch, n_tokens, h, d) or o.dtype is not dtype or o.get_device() != index or not o.is_contiguous():
                raise ValueError(f"paged_read: out must be two contiguous {dtype} {(batch, n_tokens, h, d)} on cuda:{index}")
    _run("lkv_paged_read", L.PAGED_ARGS.pack(
        0, 0, 0, 0, 0, 0, 0, 0, code, batch, n_tokens, h, d, pages.data_ptr(), kind, at, n, bs, table.data_ptr(), ld, cols, starts.data_ptr(),
        0 if lens is None else lens.data_ptr(), k.data_ptr(), v.data_ptr()), index)
    return out


def paged_write_rotated(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, pages: torch.Tensor,
                        table: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, scales: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                        k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """New tokens from a layer's projections into the cache, one launch (lkv_paged_write_rotated): query [rows, hq, d]
    and keys [rows, h, d] are normalised per head (where q_weight / k_weight [d] are given: weight x / rms) and
    rotated to positions [rows] (int32), keys and values [rows, h, d] written into the pages as paged_write does.
    Returns the rotated query (in `out`, which may be `query` itself).

    Tokens are packed: sequence b's are rows offsets[b] .. offsets[b + 1] - 1 (offsets int32 [batch + 1]) and go to the
    last places of its lens[b] (int32 [batch]). Rows of no sequence are left alone (in a new `out`: not set), so a batch
    may be padded. Pair i of the len(frequencies) (float32, a multiple of 4, at most d / 2) turns by position x
    frequencies[i]: channels (i, i + len) or, interleaved, (2 i, 2 i + 1); the others do not turn. positions are the
    rotation's only, not the place in the pages.
    """
    who = "paged_write_rotated"
    index = keys.get_device()
    if index < 0 or not (query.get_device() == values.get_device() == positions.get_device() == frequencies.get_device() == pages.get_device() == table.get_device()
                         == lens.get_device() == offsets.get_device() == index):
        _one_device(who, query, keys, values, positions, frequencies, pages, table, lens, offsets)
    n, h, bs, d, kind, at, batch, ld, cols = _cache_geometry(who, pages, scales, table)
    dtype, shape, q_shape = keys.dtype, keys.shape, query.shape
    if len(q_shape) != 3 or len(shape) != 3 or shape[1:] != (h, d) or q_shape[::2] != shape[::2] or values.shape != shape or not (query.dtype is values.dtype is dtype) or (
            kind == 0 and pages.dtype is not dtype):
        raise ValueError(f"{who}: query [rows, hq, d], keys and values [rows, h, d] of one type must fit pages {tuple(pages.shape)} {pages.dtype}; got {query.dtype} "
                         f"{tuple(q_shape)}, {dtype} {tuple(shape)} and {values.dtype} {tuple(values.shape)}")
    rows, hq = shape[0], q_shape[1]
    (k_st, k_sh, kc), (v_st, v_sh, vc), (q_st, q_sh, qc) = keys.stride(), values.stride(), query.stride()
    if kc != 1 or vc != 1 or qc != 1:
        raise ValueError(f"{who}: channels must be contiguous")
    if positions.dtype is not _I32 or positions.shape != (rows,) or not positions.is_contiguous():
        raise ValueError(f"{who}: positions must be a contiguous int32 [{rows}]")
    pairs = frequencies.numel()
    if frequencies.dtype is not _F32 or frequencies.dim() != 1 or not frequencies.is_contiguous() or pairs & 3 or 2 * pairs > d:
        raise ValueError(f"{who}: frequencies must be a contiguous float32 [n], n a multiple of 4 and at most {d // 2}, got {frequencies.dtype} {tuple(frequencies.shape)}")
    weights = [0, 0]
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            if w.dtype is not dtype or w.shape != (d,) or not w.is_contiguous() or w.get_device() != index:
                raise ValueError(f"{who}: {'qk'[i]}_weight must be a contiguous {dtype} [{d}] on cuda:{index}, got {w.dtype} {tuple(w.shape)}")
            weights[i] = w.data_ptr()
    if not eps >= 0:
        raise ValueError(f"{who}: eps {eps}")
    _per_sequence(who, "lens", lens, batch)
    _per_sequence(who, "offsets", offsets, batch + 1)
    if out is None:
        out = query.new_empty(q_shape)
    elif out.shape != q_shape or out.dtype is not dtype or out.stride(2) != 1 or out.get_device() != index:
        raise ValueError(f"{who}: out must be {dtype} {tuple(q_shape)} with contiguous channels on cuda:{index}")
    o_st, o_sh, _ = out.stride()
    if scales is not None and scales.get_device() != index:
        _one_device(who, pages, scales)
    _run("lkv_paged_write_rotated", L.ROTATE_ARGS.pack(
        query.data_ptr(), keys.data_ptr(), values.data_ptr(), q_st, q_sh, k_st, k_sh, v_st, v_sh, out.data_ptr(), o_st, o_sh, 1 if dtype is _BF16 else dtype_code(dtype), rows, hq, h,
        d, positions.data_ptr(), frequencies.data_ptr(), pairs, interleaved, weights[0], weights[1], eps, pages.data_ptr(), kind, at, n, bs, table.data_ptr(), ld, cols,
        lens.data_ptr(), offsets.data_ptr(), batch), index)
    return out


def paged_evict(pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, sums: torch.Tensor, positions: torch.Tensor, keep: int,
                since: torch.Tensor | None = None, sinks: int = 0, scales: torch.Tensor | None = None,
                out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts each sequence's own tokens down to `keep` per KV head, one launch (lkv_paged_evict): the tokens at positions
    below `sinks` or from since[b] (int32 [batch]) on first, then those of the highest sums, ties to the lowest slot.

    lens [batch] counts the tokens in the pages' slots, sums [batch, h, cap] float32 are their weights (attention_sums) and
    positions [batch, h, cap] int32 what they were rotated to: heads keep different tokens. Kept tokens behind slot
    keep - 1 move into the slots of dropped ones, in place, with their scales, so slots are no longer in the order of
    the positions; attention does not need one, as long as new tokens follow in slots of their own. Returns (min(lens,
    keep), sums, positions): the last two new, or in `out`, which may be sums and positions themselves; 0 and -1 stand in
    slots without a token. Pages should reach to lens[b]: a token without a page is ranked like the others, and where either
    slot of a move has none, sum and position move without a row: the slot keeps the row it had, or the token is lost.
    """
    who = "paged_evict"
    index = pages.get_device()
    if index < 0 or not (table.get_device() == lens.get_device() == sums.get_device() == positions.get_device() == index) or (since is not None and since.get_device() != index) or (
            scales is not None and scales.get_device() != index):
        _one_device(who, pages, table, lens, sums, positions, since, scales)
    n, h, bs, d, kind, at, batch, ld, cols = _cache_geometry(who, pages, scales, table)
    _per_sequence(who, "lens", lens, batch)
    if since is not None:
        _per_sequence(who, "since", since, batch)
    shape = sums.shape
    if sums.dtype is not _F32 or len(shape) != 3 or shape[:2] != (batch, h) or not sums.is_contiguous():
        raise ValueError(f"{who}: sums must be a contiguous float32 [{batch}, {h}, slots], got {sums.dtype} {tuple(shape)}")
    if positions.dtype is not _I32 or positions.shape != shape or not positions.is_contiguous():
        raise ValueError(f"{who}: positions must be a contiguous int32 {tuple(shape)}, got {positions.dtype} {tuple(positions.shape)}")
    cap = shape[2]
    if not (1 <= keep < 2**31 and 0 <= sinks < 2**31):
        raise ValueError(f"{who}: a budget of {keep} tokens, the first {sinks} of them kept")
    code = 0 if kind == 1 else dtype_code(pages.dtype)
    if out is None:
        out = torch.empty_like(sums), torch.empty_like(positions)
    else:
        for o, like in zip(out, (sums, positions)):
            if o.dtype is not like.dtype or o.shape != shape or not o.is_contiguous() or o.get_device() != index:
                raise ValueError(f"{who}: out must be like sums and positions, {tuple(shape)} on cuda:{index}")
    left = torch.empty_like(lens)
    nbytes = batch * h * min(keep, cap - keep) * 8 if cap > keep else 0
    ws = lens.new_empty(nbytes // 4) if nbytes else None
    _run("lkv_paged_evict", L.EVICT_ARGS.pack(
        pages.data_ptr(), kind, code, at, n, h, bs, d, batch, table.data_ptr(), ld, cols, lens.data_ptr(), sums.data_ptr(), positions.data_ptr(), cap,
        out[0].data_ptr(), out[1].data_ptr(), left.data_ptr(), keep, sinks, 0 if since is None else since.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes), index)
    return left, out[0], out[1]


@functools.lru_cache(maxsize=4096)
def _prefix_workspace(batch: int, tokens: int, hq: int, h: int, d: int, prefix_len: int, kind: int, reach: int) -> int:
    return int(L.lib().lkv_prefix_attention_workspace(batch, tokens, hq, h, d, prefix_len, kind, reach))


def prefix_attention(query: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, prefix_table: torch.Tensor, prefix_len: int,
                     scale: float, scales: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of query [batch, T, hq, d] (bfloat16) for a batch that shares a prefix, whose pages are
    read once for all, up to 256 query rows per KV head (lkv_prefix_attention, two or three launches). Query t of sequence b attends the prefix_len
    tokens of the pages that prefix_table [columns] lists, and the first lens[b] - T + t + 1 of its own
    lens[b] tokens in the pages of table[b]: the step's T tokens (drafted ones included) are written
    before the call and are the last of lens[b].

    pages are bfloat16 or int8 with scales (paged_write). Returns (out [batch, T, hq, d] in `out_dtype`,
    bfloat16 by default, lse [batch, T, hq] float32); a row that attends nothing (no prefix, no own token,
    all pages missing) gets out = 0 and lse = -inf. lens and both tables are read on the device, so a
    captured graph follows them as they change; prefix_len and the shapes are fixed at capture.
    Scores, references and sums are float32. Weights enter the product with the values rounded: int8 pages 2^-11 of
    each (and 2^-31 of the row's largest weight times value); bfloat16 pages 2^-15 for a float32 output and up to 2^-8
    for a bfloat16 one, whose prefix of more than 16 rows per KV head is then a quarter faster.
    The partials' workspace comes from torch's allocator call by call, so calls on several streams and
    several captured graphs do not share it.
    """
    who = "prefix_attention"
    index = query.get_device()
    if index < 0 or not (pages.get_device() == table.get_device() == lens.get_device() == prefix_table.get_device() == index) or (
            scales is not None and scales.get_device() != index):
        index = _one_device(who, query, pages, table, lens, prefix_table, scales)
    if query.dim() != 4 or query.dtype is not _BF16:
        raise ValueError(f"prefix_attention: query must be bfloat16 [batch, T, hq, d], got {query.dtype} {tuple(query.shape)}")
    batch, t, hq, d = query.shape
    n, h, bs, pd, kind, at, rows, ld, cols = _cache_geometry(who, pages, scales, table)
    if pd != d or h < 1 or hq % h or rows != batch or (kind == 0 and pages.dtype is not _BF16):
        raise ValueError(f"prefix_attention: query {tuple(query.shape)} and table {tuple(table.shape)} do not fit {pages.dtype} pages {tuple(pages.shape)}")
    _per_sequence(who, "lens", lens, batch)
    pcols = prefix_table.numel()
    if prefix_table.dtype is not _I32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous() or not 0 <= prefix_len <= pcols * bs:
        raise ValueError(f"prefix_attention: prefix_table must be a contiguous int32 [columns] holding the {prefix_len} tokens of the prefix")
    sb, st, sh, sc = query.stride()
    if sc != 1 or (sb | st | sh) & 7 or query.data_ptr() & 15:
        query = query.clone(memory_format=torch.contiguous_format)
        sb, st, sh, _ = query.stride()
    if out is None:
        if out_dtype is None:
            out = torch.empty_like(query) if query.is_contiguous() else query.new_empty((batch, t, hq, d))
        else:
            out = query.new_empty((batch, t, hq, d), dtype=out_dtype)
    elif out.shape != query.shape or not out.is_contiguous() or (out_dtype is not None and out.dtype is not out_dtype) or out.get_device() != index:
        raise ValueError(f"prefix_attention: out must be a contiguous {tuple(query.shape)} on cuda:{index}")
    if lse is None:
        lse = query.new_empty((batch, t, hq), dtype=_F32)
    elif lse.shape != (batch, t, hq) or lse.dtype is not _F32 or not lse.is_contiguous() or lse.get_device() != index:
        raise ValueError(f"prefix_attention: lse must be a contiguous float32 {(batch, t, hq)} on cuda:{index}")
    code = 1 if out.dtype is _BF16 else dtype_code(out.dtype)
    nbytes = _prefix_workspace(batch, t, hq, h, d, prefix_len, kind, cols * bs)
    ws = query.new_empty((nbytes + 1) // 2) if nbytes else None
    _run("lkv_prefix_attention", L.PREFIX_ARGS.pack(
        query.data_ptr(), 1, sb, st, sh, pages.data_ptr(), kind, at, n, bs, batch, t, hq, h, d, table.data_ptr(), ld, cols, lens.data_ptr(),
        prefix_table.data_ptr(), pcols, prefix_len, scale, out.data_ptr(), code, lse.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes), index)
    return out, lse


@functools.lru_cache(maxsize=4096)
def _chunk_workspace(rows: int, batch: int, hq: int, h: int, d: int, prefix_len: int, reach: int) -> int:
    return int(L.lib().lkv_chunk_attention_workspace(rows, batch, hq, h, d, prefix_len, reach))


def chunk_attention(query: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, scale: float,
                    scales: torch.Tensor | None = None, prefix_table: torch.Tensor | None = None, prefix_len: int = 0, cap: float = 0.0,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of chunks of new tokens, of any length per sequence, over the paged cache (lkv_chunk_attention, two
    launches): query [rows, hq, d] bfloat16 is packed, sequence b's at rows offsets[b] .. offsets[b + 1] - 1 (int32
    [batch + 1]), the last of its lens[b] own tokens, which are in the pages already (paged_write_rotated). Each query
    attends the prefix_len tokens of the pages that prefix_table lists, and its sequence's own tokens up to itself; scores
    are scale q k or, with a cap, cap tanh(scale q k / cap).

    pages are bfloat16 or int8 with scales. Returns (out [rows, hq, d] bfloat16, lse [rows, hq] float32). A row that attends
    nothing gets out = 0 and lse = -inf; rows of no sequence are left alone (in new tensors: not set), so a batch may be
    padded, and sequences may have no new tokens. lens, offsets and the tables are read on the device, so a captured graph
    follows them as they change; the shapes and prefix_len are fixed at capture. Scores and sums are float32; weights are
    rounded where they multiply the values, of bfloat16 pages to bfloat16 (2^-8), of int8 pages to 2^-11 as in prefix_attention. The workspace comes from torch's allocator call by call.
    """
    who = "chunk_attention"
    index = query.get_device()
    if index < 0 or not (pages.get_device() == table.get_device() == lens.get_device() == offsets.get_device() == index):
        _one_device(who, query, pages, table, lens, offsets)
    n, h, bs, d, kind, at, batch, ld, cols = _cache_geometry(who, pages, scales, table)
    if query.dim() != 3 or query.dtype is not _BF16 or query.shape[2] != d or query.shape[1] < 1 or query.shape[1] % h or (kind == 0 and pages.dtype is not _BF16):
        raise ValueError(f"{who}: query must be bfloat16 [rows, heads, {d}], heads a multiple of {h}, over bfloat16 or int8 pages; got {query.dtype} "
                         f"{tuple(query.shape)}, {pages.dtype} pages {tuple(pages.shape)}")
    rows, hq, _ = query.shape
    _per_sequence(who, "lens", lens, batch)
    _per_sequence(who, "offsets", offsets, batch + 1)
    pcols = 0
    if prefix_table is not None:
        pcols = prefix_table.numel()
        if prefix_table.dtype is not _I32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous() or prefix_table.get_device() != index:
            raise ValueError(f"{who}: prefix_table must be a contiguous int32 [columns] on cuda:{index}")
    if not 0 <= prefix_len <= pcols * bs:
        raise ValueError(f"{who}: prefix_table of {pcols} pages of {bs} cannot hold {prefix_len} tokens")
    if not 0 <= cap < math.inf:
        raise ValueError(f"{who}: cap {cap}")
    st, sh, sc = query.stride()
    if sc != 1 or (st | sh) & 7 or query.data_ptr() & 15:
        query = query.clone(memory_format=torch.contiguous_format)
        st, sh, _ = query.stride()
    if out is None:
        out = query.new_empty((rows, hq, d))
    elif out.shape != (rows, hq, d) or out.dtype is not _BF16 or not out.is_contiguous() or out.get_device() != index:
        raise ValueError(f"{who}: out must be a contiguous bfloat16 {(rows, hq, d)} on cuda:{index}")
    if lse is None:
        lse = query.new_empty((rows, hq), dtype=_F32)
    elif lse.shape != (rows, hq) or lse.dtype is not _F32 or not lse.is_contiguous() or lse.get_device() != index:
        raise ValueError(f"{who}: lse must be a contiguous float32 {(rows, hq)} on cuda:{index}")
    if scales is not None and scales.get_device() != index:
        _one_device(who, query, scales)
    nbytes = _chunk_workspace(rows, batch, hq, h, d, prefix_len, cols * bs)
    ws = query.new_empty((nbytes + 1) // 2) if nbytes else None
    _run("lkv_chunk_attention", L.CHUNK_ARGS.pack(
        query.data_ptr(), st, sh, 1, rows, hq, h, d, pages.data_ptr(), kind, at, n, bs, table.data_ptr(), ld, cols, lens.data_ptr(), offsets.data_ptr(), batch,
        0 if prefix_table is None else prefix_table.data_ptr(), pcols, prefix_len, scale, cap, out.data_ptr(), lse.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes), index)
    return out, lse


@functools.lru_cache(maxsize=4096)
def _sums_workspace(batch: int, h: int, slots: int) -> int:
    return int(L.lib().lkv_attention_sums_workspace(batch, h, slots))


def attention_sums(query: torch.Tensor, lse: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, scale: float,
                   sums: torch.Tensor | None = None, last: int | None = None, cap: float = 0.0, scales: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The attention weight that every own token got from the queries of the chunks, added to `sums` (lkv_attention_sums, one
    or two launches): [batch, h, slots] float32, slots = columns * block size without sums or out. query, offsets, lens, scale and cap
    are those of chunk_attention, lse [rows, hq] what it (or prefix_attention) returned. With `last`, only the last so many
    query tokens of each chunk count. What paged_evict ranks tokens by.

    sums [batch, h, slots] are those of earlier steps (None: zeros) for the tokens in front of the chunk; the chunk's own
    start from 0, and slots without a token are 0. The result is new or in `out`, which may be sums itself. Sums are
    float32 in the order of the queries, the same every time.
    """
    who = "attention_sums"
    index = query.get_device()
    if index < 0 or not (lse.get_device() == pages.get_device() == table.get_device() == lens.get_device() == offsets.get_device() == index) or (
            scales is not None and scales.get_device() != index):
        _one_device(who, query, lse, pages, table, lens, offsets, scales)
    n, h, bs, d, kind, at, batch, ld, cols = _cache_geometry(who, pages, scales, table)
    if query.dim() != 3 or query.dtype is not _BF16 or query.shape[2] != d or query.shape[1] < 1 or query.shape[1] % h or (kind == 0 and pages.dtype is not _BF16):
        raise ValueError(f"{who}: query must be bfloat16 [rows, heads, {d}], heads a multiple of {h}, over bfloat16 or int8 pages; got {query.dtype} "
                         f"{tuple(query.shape)}, {pages.dtype} pages {tuple(pages.shape)}")
    rows, hq, _ = query.shape
    if lse.dtype is not _F32 or lse.shape != (rows, hq) or not lse.is_contiguous():
        raise ValueError(f"{who}: lse must be a contiguous float32 [{rows}, {hq}], got {lse.dtype} {tuple(lse.shape)}")
    _per_sequence(who, "lens", lens, batch)
    _per_sequence(who, "offsets", offsets, batch + 1)
    slots = cols * bs if sums is None and out is None else (out if sums is None else sums).shape[-1]
    for name, t in (("sums", sums), ("out", out)):
        if t is not None and (t.dtype is not _F32 or t.shape != (batch, h, slots) or not t.is_contiguous() or t.get_device() != index):
            raise ValueError(f"{who}: {name} must be a contiguous float32 [{batch}, {h}, {slots}] on cuda:{index}, got {t.dtype} {tuple(t.shape)}")
    if last is not None and last < 1:
        raise ValueError(f"{who}: the last {last} tokens of a chunk")
    if not 0 <= cap < math.inf:
        raise ValueError(f"{who}: cap {cap}")
    st, sh, sc = query.stride()
    if sc != 1 or (st | sh) & 7 or query.data_ptr() & 15:
        query = query.clone(memory_format=torch.contiguous_format)
        st, sh, _ = query.stride()
    if out is None:
        out = query.new_empty((batch, h, slots), dtype=_F32)
    nbytes = _sums_workspace(batch, h, slots)
    ws = query.new_empty((nbytes + 1) // 2) if nbytes else None
    _run("lkv_attention_sums", L.SUMS_ARGS.pack(
        query.data_ptr(), st, sh, 1, rows, hq, h, d, lse.data_ptr(), pages.data_ptr(), kind, at, n, bs, table.data_ptr(), ld, cols, lens.data_ptr(), offsets.data_ptr(), batch,
        2**31 - 1 if last is None else min(last, 2**31 - 1), 0 if sums is None else sums.data_ptr(), out.data_ptr(), slots, scale, cap,
        0 if ws is None else ws.data_ptr(), nbytes), index)
    return out


def verify_drafts(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, uniforms: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Which of k drafted tokens per sequence are kept, and the token that follows them (one launch,
    lkv_verify_drafts). target [batch, k + 1, vocab] and draft [batch, k, vocab] are float32
    probabilities (draft None: a draft that proposed its token with certainty), tokens [batch, k] int64,
    uniforms [batch, k + 1] float32 in [0, 1).

    Token i is kept while uniforms_i * draft_i(x_i) < target_i(x_i). After a rejection at n the next token
    is drawn from max(target_n - draft_n, 0), after k kept tokens from target_k, by inverting the
    cumulative sum at uniforms_k: kept tokens and drawn token are distributed as the target's own samples.
    A token outside [0, vocab) (say -1) ends its sequence's drafts, and the next one is drawn from the
    target there. Returns (kept [batch] int32, token [batch] int64); token is -1 where the weights are all
    zero or have no finite sum.
    """
    index = target.get_device()
    if index < 0 or not (tokens.get_device() == uniforms.get_device() == index) or (draft is not None and draft.get_device() != index):
        index = _one_device("verify_drafts", target, draft, tokens, uniforms)
    if target.dim() != 3 or tokens.dim() != 2:
        raise ValueError("verify_drafts: target must be [batch, k + 1, vocab] and tokens [batch, k]")
    batch, k = tokens.shape
    vocab = target.shape[2]
    if target.shape != (batch, k + 1, vocab) or uniforms.shape != (batch, k + 1) or (draft is not None and draft.shape != (batch, k, vocab)):
        raise ValueError(f"verify_drafts: {k} tokens drafted for {batch} sequences do not fit target {tuple(target.shape)}, uniforms "
                         f"{tuple(uniforms.shape)}, draft {None if draft is None else tuple(draft.shape)}")
    if target.dtype is not _F32 or uniforms.dtype is not _F32 or tokens.dtype is not _I64 or (draft is not None and draft.dtype is not _F32):
        raise ValueError("verify_drafts: probabilities and uniforms are float32, tokens int64")
    (pb, pt, pv), (tb, tk), (ub, uk) = target.stride(), tokens.stride(), uniforms.stride()
    qb, qt, qv = (0, 0, 1) if draft is None else draft.stride()
    if (vocab > 1 and (pv != 1 or qv != 1)) or (k > 1 and tk != 1) or (k > 0 and uk != 1):
        raise ValueError("verify_drafts: rows must be contiguous")
    token = tokens.new_empty(batch)
    kept = tokens.new_empty(batch, dtype=_I32)
    _run("lkv_verify_drafts", L.VERIFY_ARGS.pack(
        target.data_ptr(), pb, pt, 0 if draft is None else draft.data_ptr(), qb, qt, tokens.data_ptr(), tb, uniforms.data_ptr(), ub, batch, k, vocab,
        kept.data_ptr(), token.data_ptr()), index)
    return kept, token
