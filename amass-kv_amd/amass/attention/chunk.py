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

from .._hip import ChunkArgs, call_on, check, load_library, packer, same_device
from .decode import _split_kv
from .rope import DTYPES

HEAD_DIMS = (64, 128)
_pack_chunk = packer(ChunkArgs)


def _chunk_args(q, kv_cache, block_table, seq_lens, query_start, out, scale, causal, window,
                lse) -> ChunkArgs:
    same_device(q, kv_cache, block_table, seq_lens, query_start, out, lse)
    k, v = _split_kv(kv_cache)
    if v is None:
        raise ValueError("the cache has no V half")
    dt = q.dtype
    if dt not in DTYPES or k.dtype != dt or out.dtype != dt:
        raise ValueError("q, the cache and out must all be bf16 or all fp16")
    nb, page, n_kv, d = k.shape
    if q.dim() != 3 or q.shape[2] != d or out.shape != q.shape:
        raise ValueError(f"q and out must be (T, H, {d})")
    T, H = q.shape[:2]
    if H % n_kv or H == 0:
        raise ValueError(f"{H} query heads are not a multiple of {n_kv} kv heads")
    if d not in HEAD_DIMS:
        raise ValueError(f"head dim {d} (built for {HEAD_DIMS})")
    if page < 16 or page & (page - 1):
        raise ValueError(f"page {page} must be a power of two from 16 on")
    if window is not None and window < 1:
        raise ValueError("window must be positive (None: no window)")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 3e38:
        raise ValueError(f"scale {scale} must be positive and finite")
    n_req = seq_lens.shape[0]
    for t, name, n in ((seq_lens, "seq_lens", n_req), (query_start, "query_start", n_req + 1)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.shape[0] < n:
            raise ValueError(f"{name} must be a contiguous int32 vector of {n} entries")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or \
            block_table.stride(1) != 1 or block_table.shape[0] < n_req or \
            block_table.shape[1] < 1:
        raise ValueError("block_table must be (R, max_pages) int32 with unit column stride")
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
    if qs[2] != 1 or ks[3] != 1 or vs[3] != 1 or os_[2] != 1:
        raise ValueError("q / cache / out need unit stride on the head dim")
    ls = (0, 0)
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (T, H):
            raise ValueError("lse must be (T, H) fp32")
        ls = lse.stride()
    return _pack_chunk(                # in the struct's order
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0],
        vs[1], vs[2], block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(),
        query_start.data_ptr(), out.data_ptr(), os_[0], os_[1],
        0 if lse is None else lse.data_ptr(), ls[0], ls[1], 0, 0, scale, n_req, T, n_kv,
        H // n_kv, d, page, nb, block_table.shape[1], 1 if causal else 0, window or 0,
        DTYPES[dt])


def _scratch_bytes(a: ChunkArgs) -> int:
    n = load_library().amass_chunk_scratch_bytes(a)
    if n < 0:
        check(n, "amass_chunk_scratch_bytes")
    return n


def chunk_scratch_bytes(q, kv_cache, block_table, seq_lens, query_start, out, *, scale=None,
                        causal: bool = True, window=None, lse=None) -> int:
    """Bytes of scratch that ``paged_chunk_attention`` takes for these shapes."""
    return _scratch_bytes(_chunk_args(q, kv_cache, block_table, seq_lens, query_start, out,
                                      scale, causal, window, lse))


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
    (T, H) fp32 receives the rows' log-sum-exp of the scaled scores.

    bf16 or fp16, d 64 or 128, pages of 16 or a larger power of two, any number of query heads
    per kv head.  K and V need 16-byte aligned rows, as q and out do.

    ``scratch``: a uint8 tensor of ``chunk_scratch_bytes`` for programs that keep their own;
    calls that may run at the same time need one each."""
    a = _chunk_args(q, kv_cache, block_table, seq_lens, query_start, out, scale, causal, window,
                    lse)
    need = _scratch_bytes(a)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    else:
        same_device(q, scratch)
        if scratch.dtype != torch.uint8 or not scratch.is_contiguous():
            raise ValueError("scratch must be a contiguous uint8 tensor")
        if scratch.numel() < need:
            raise ValueError(f"scratch of {scratch.numel()} bytes, {need} needed")
    a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel()
    call_on(q.device, "amass_chunk_attention", a)
