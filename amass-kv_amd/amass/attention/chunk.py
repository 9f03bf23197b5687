"""Attention of a chunk of new tokens over the paged cache (``amass_chunk_attention``).

What ``dense_paged_decode`` is for one token per request, for any number of them: prompts,
chunks of prompts that have tokens behind them already, drafted tokens and single tokens, mixed
in one batch.  Causal within the request (or not), with a sliding window on request, and with
the log-sum-exp of every row on request (to join the result with another part's).

The launches are fixed by the shapes of q, the block table and ``query_start``: lengths stay
on the device, nothing synchronises with the host, and a call can be captured in a HIP graph.
The scratch memory (the parts of rows whose keys several workgroups share) comes from torch's
allocator within the call, or from the caller.
"""
from __future__ import annotations

import torch

from .._hip import (ChunkArgs, cache_halves, call_on, check, device_index, load_library, packer,
                    vector)
from .rope import DTYPES

HEAD_DIMS = (64, 128)
MAX_INT = 2 ** 31 - 1
_pack_chunk = packer(ChunkArgs)
_SCRATCH = {}            # (GPU, requests, rows, kv heads, group, head dim) -> scratch bytes


def _chunk_args(q, kv_cache, block_table, seq_lens, query_start, out, scale, causal, window,
                lse):
    """(the argument struct's values up to the scratch, those behind it) of a checked call."""
    dt = q.dtype
    if not (dt in DTYPES and dt is kv_cache.dtype is out.dtype):
        raise ValueError("q, the cache and out must all be bf16 or all fp16")
    (nb, page, n_kv, d), k, v, cs = cache_halves(kv_cache)
    if v == 0:
        raise ValueError("the cache has no V half")
    shape = q.shape
    if len(shape) != 3 or shape[2] != d or out.shape != shape:
        raise ValueError(f"q and out must be (T, H, {d})")
    T, H, _ = shape
    if H == 0 or H % n_kv:
        raise ValueError(f"{H} query heads are not a multiple of {n_kv} kv heads")
    if d not in HEAD_DIMS:
        raise ValueError(f"head dim {d} (built for {HEAD_DIMS})")
    if page < 16 or page & (page - 1):
        raise ValueError(f"page {page} must be a power of two from 16 on")
    if window is not None and window < 1:
        raise ValueError("window must be positive (None: no window)")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 2e38:                 # (times log2 e it stays finite)
        raise ValueError(f"scale {scale} must be positive and finite")
    n_req = seq_lens.numel()
    vector(seq_lens, torch.int32, n_req, "seq_lens")
    vector(query_start, torch.int32, n_req + 1, "query_start")
    rows, width = block_table.shape
    bt_st, unit = block_table.stride()
    if block_table.dtype is not torch.int32 or (unit != 1 and width > 1) or rows < n_req or \
            width < 1:
        raise ValueError("block_table must be (R, max_pages) int32 with unit column stride")
    q_st, q_hs, q_unit = q.stride()
    o_st, o_hs, o_unit = out.stride()
    sb, st, sh, c_unit = cs
    if not q_unit == o_unit == c_unit == 1:
        raise ValueError("q / cache / out need unit stride on the head dim")
    if not (o_st or T == 1) or not (o_hs or H == 1):
        raise ValueError("rows or heads of out share memory")
    l_at = l_st = l_hs = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != (T, H):
            raise ValueError("lse must be (T, H) fp32")
        l_at = lse.data_ptr()
        l_st, l_hs = lse.stride()
        if not (l_st or T == 1) or not (l_hs or H == 1):
            raise ValueError("rows or heads of lse share memory")
    return ((q.data_ptr(), q_st, q_hs, k, v, sb, st, sh, block_table.data_ptr(), bt_st,
             seq_lens.data_ptr(), query_start.data_ptr(), out.data_ptr(), o_st, o_hs,
             l_at, l_st, l_hs),
            (scale, n_req, T, n_kv, H // n_kv, d, page, nb, width, 1 if causal else 0,
             min(window or 0, MAX_INT), DTYPES[dt]))


def _scratch_bytes(index, head, tail) -> int:
    key = (index, *tail[1:6])
    n = _SCRATCH.get(key)
    if n is None:
        with torch.cuda.device(index):
            n = load_library().amass_chunk_scratch_bytes(_pack_chunk(*head, 0, 0, *tail))
        if n < 0:
            check(n, "amass_chunk_scratch_bytes")
        if len(_SCRATCH) >= 4096:
            _SCRATCH.clear()
        _SCRATCH[key] = n
    return n


def chunk_scratch_bytes(q, kv_cache, block_table, seq_lens, query_start, out, *, scale=None,
                        causal: bool = True, window=None, lse=None) -> int:
    """Bytes of scratch that ``paged_chunk_attention`` takes for these shapes."""
    index = device_index(q, kv_cache, block_table, seq_lens, query_start, out, lse)
    return _scratch_bytes(index, *_chunk_args(q, kv_cache, block_table, seq_lens, query_start,
                                              out, scale, causal, window, lse))


def paged_chunk_attention(q, kv_cache, block_table, seq_lens, query_start, out, *, scale=None,
                          causal: bool = True, window: int | None = None, lse=None,
                          scratch=None) -> None:
    """Attend the rows of q (T, H, d) over their requests' keys and values, into out.

    Request r brings rows ``query_start[r] .. query_start[r + 1] - 1``, the last of its
    ``seq_lens[r]`` tokens, whose K and V the cache holds already (``rope_paged_write``).  The
    row at position p sees the request's positions ``j < seq_lens[r]``, with ``causal`` those
    ``j <= p``, with ``window`` those ``j > p - window``, and nothing in pages whose block is
    outside the cache or beyond the table's width.  Rows that see nothing get zeros (``lse``:
    -inf); rows of no request stay as they are.  ``scale`` defaults to ``d ** -0.5``; ``lse``
    (T, H) fp32 receives the rows' log-sum-exp of the scaled scores.  ``out`` may be q.

    bf16 or fp16, d 64 or 128, pages of 16 or a larger power of two, any number of query heads
    per kv head.  K and V need 16-byte aligned rows, as q and out do.

    ``scratch``: a uint8 tensor of ``chunk_scratch_bytes`` for programs that keep their own;
    calls that may run at the same time need one each."""
    index = device_index(q, kv_cache, block_table, seq_lens, query_start, out, lse, scratch)
    head, tail = _chunk_args(q, kv_cache, block_table, seq_lens, query_start, out, scale,
                             causal, window, lse)
    need = _scratch_bytes(index, head, tail)
    if scratch is None:
        scratch = q.new_empty(need // 2)
        size = need
    else:
        if scratch.dtype is not torch.uint8 or not scratch.is_contiguous():
            raise ValueError("scratch must be a contiguous uint8 tensor")
        size = scratch.numel()
        if size < need:
            raise ValueError(f"scratch of {size} bytes, {need} needed")
    call_on(index, "amass_chunk_attention",
            _pack_chunk(*head, scratch.data_ptr(), size, *tail))
