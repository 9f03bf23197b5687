"""Block tables and slot maps of a step's new tokens, on the device (``amass_extend``).

A serving program keeps its free blocks in a list on the device: ``free[:top[0]]`` of an
int32 tensor ``free`` and the three-word ``top`` (free blocks, an arrival count that is zero
at rest, blocks short of the last call).  ``free_blocks`` makes both.

  extend_block_tables   every page that the step's tokens enter takes a block off the end of
                        the list; every token gets its position and its slot
  release_blocks        the blocks of finished requests go back

One launch each, fixed-shape, without allocation or host synchronisation, so both can be
captured in a HIP graph.  ``query_start`` (R + 1,) are the rows where the requests' tokens
start, ``seq_lens`` (R,) the requests' lengths with the new tokens, as the attention backend's
metadata has them.  A block belongs to one request.
"""
from __future__ import annotations

import torch

from .._hip import ExtendArgs, ReleaseArgs, call_on, packer, same_device

MAX_REQS = 4096      # requests of one call (the kernels rank them in LDS)
_pack_extend = packer(ExtendArgs)
_pack_release = packer(ReleaseArgs)


def free_blocks(num_blocks: int, device):
    """(free, top): a list of all blocks of a pool; block 0 is taken first."""
    free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
    return free, torch.tensor([num_blocks, 0, 0], dtype=torch.int32, device=device)


def _check_step(block_table, seq_lens, free, top, page, num_blocks):
    for t, name in ((seq_lens, "seq_lens"), (free, "free"), (top, "top")):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be (R, max_pages) int32 with unit column stride")
    n_req = seq_lens.shape[0]
    if block_table.shape[0] < n_req or block_table.shape[1] < 1:
        raise ValueError("block_table needs a row per request")
    if n_req > MAX_REQS:
        raise ValueError(f"{n_req} requests in one call (at most {MAX_REQS})")
    if top.shape[0] < 3:
        raise ValueError("top has three words (free_blocks)")
    if page < 1 or page & (page - 1):
        raise ValueError(f"page {page} is not a power of two")
    if num_blocks < 1:
        raise ValueError("num_blocks must be positive")
    return n_req


def extend_block_tables(block_table, seq_lens, query_start, free, top, slots, positions, *,
                        page: int, num_blocks: int, top_out=None) -> None:
    """Blocks for the pages that this step's tokens enter, slots and positions of its rows.

    Row ``t`` = ``query_start[r] + i`` of request r's ``n`` new tokens is at position
    ``seq_lens[r] - n + i``: ``positions[t]`` (int32), ``slots[t] = block * page + position %
    page`` (int64).  The k-th new page of the step, in (request, page) order, takes
    ``free[top[0] - 1 - k]`` and enters ``block_table``.  Rows of no request and rows before a
    request's position 0 get -1; a token at or past ``max_pages * page``, or in a page for
    which no block of ``[0, num_blocks)`` is there, gets slot -1.  ``slots`` gives the number of
    rows.

    ``top`` becomes the blocks left (``top[2]``: those that were short).  With ``top_out``,
    another such tensor, they go there and ``top`` stays, so that the step may be dropped."""
    same_device(block_table, seq_lens, query_start, free, top, slots, positions, top_out)
    n_req = _check_step(block_table, seq_lens, free, top, page, num_blocks)
    if query_start.dtype != torch.int32 or query_start.dim() != 1 or \
            not query_start.is_contiguous() or query_start.shape[0] < n_req + 1:
        raise ValueError("query_start must be a contiguous int32 vector of R + 1 rows")
    if slots.dtype != torch.int64 or positions.dtype != torch.int32 or slots.dim() != 1 or \
            positions.dim() != 1 or not (slots.is_contiguous() and positions.is_contiguous()) \
            or positions.shape[0] < slots.shape[0]:
        raise ValueError("slots (T,) int64 and positions (T,) int32 must be contiguous")
    if top_out is None:
        top_out = top
    elif top_out.dtype != torch.int32 or not top_out.is_contiguous() or top_out.numel() < 3:
        raise ValueError("top_out must be three contiguous int32 words")
    a = _pack_extend(                  # in the struct's order
        block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(),
        query_start.data_ptr(), free.data_ptr(), top.data_ptr(), top_out.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), n_req, slots.shape[0], block_table.shape[1],
        page, num_blocks, free.shape[0])
    call_on(block_table.device, "amass_extend", a)


def release_blocks(block_table, seq_lens, done, free, top, *, page: int,
                   num_blocks: int) -> None:
    """The blocks of the first ``ceil(seq_lens[r] / page)`` pages of every request with
    ``done[r]`` (bool) go behind the free list, in (request, page) order, and their table
    entries become -1.  Blocks past the list's length are dropped (``top[2]``)."""
    same_device(block_table, seq_lens, done, free, top)
    n_req = _check_step(block_table, seq_lens, free, top, page, num_blocks)
    if done.dtype not in (torch.bool, torch.uint8) or done.dim() != 1 or \
            not done.is_contiguous() or done.shape[0] < n_req:
        raise ValueError("done must be a contiguous bool vector, an entry per request")
    a = _pack_release(                 # in the struct's order
        block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(), done.data_ptr(),
        free.data_ptr(), top.data_ptr(), n_req, block_table.shape[1], page, num_blocks,
        free.shape[0])
    call_on(block_table.device, "amass_release", a)
