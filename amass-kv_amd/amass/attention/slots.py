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
metadata has them.  A block belongs to one request, and calls on one list run one after the
other (on one stream, or ordered by events).
"""
from __future__ import annotations

import torch

from .._hip import ExtendArgs, ReleaseArgs, call_on, device_index, packer, vector

MAX_REQS = 4096      # requests of one call (the kernels rank them in LDS)
_pack_extend = packer(ExtendArgs)
_pack_release = packer(ReleaseArgs)


def free_blocks(num_blocks: int, device):
    """(free, top): a list of all blocks of a pool; block 0 is taken first."""
    free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
    return free, torch.tensor([num_blocks, 0, 0], dtype=torch.int32, device=device)


def _table(block_table, n_req, page, num_blocks):
    """(row stride, width) of a checked block table."""
    rows, width = block_table.shape
    st, unit = block_table.stride()
    if block_table.dtype is not torch.int32 or (unit != 1 and width > 1):
        raise ValueError("block_table must be (R, max_pages) int32 with unit column stride")
    if st < width and rows > 1:
        raise ValueError("rows of block_table share memory")
    if rows < n_req or width < 1:
        raise ValueError("block_table needs a row per request")
    if n_req > MAX_REQS:
        raise ValueError(f"{n_req} requests in one call (at most {MAX_REQS})")
    if page < 1 or page & (page - 1):
        raise ValueError(f"page {page} is not a power of two")
    if num_blocks < 1:
        raise ValueError("num_blocks must be positive")
    return st, width


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
    index = device_index(block_table, seq_lens, query_start, free, top, slots, positions,
                         top_out)
    n_req, n_tokens, n_free = seq_lens.numel(), slots.numel(), free.numel()
    st, width = _table(block_table, n_req, page, num_blocks)
    vector(seq_lens, torch.int32, n_req, "seq_lens")
    vector(query_start, torch.int32, n_req + 1, "query_start")
    vector(free, torch.int32, n_free, "free")
    vector(top, torch.int32, 3, "top")
    vector(slots, torch.int64, n_tokens, "slots")
    vector(positions, torch.int32, n_tokens, "positions")
    if top_out is None:
        top_out = top
    else:
        vector(top_out, torch.int32, 3, "top_out")
    a = _pack_extend(                  # in the struct's order
        block_table.data_ptr(), st, seq_lens.data_ptr(), query_start.data_ptr(),
        free.data_ptr(), top.data_ptr(), top_out.data_ptr(), slots.data_ptr(),
        positions.data_ptr(), n_req, n_tokens, width, page, num_blocks, n_free)
    call_on(index, "amass_extend", a)


def release_blocks(block_table, seq_lens, done, free, top, *, page: int,
                   num_blocks: int) -> None:
    """The blocks of the first ``ceil(seq_lens[r] / page)`` pages of every request with
    ``done[r]`` (bool) go behind the free list, in (request, page) order, and their table
    entries become -1.  Blocks past the list's length are dropped (``top[2]``)."""
    index = device_index(block_table, seq_lens, done, free, top)
    n_req, n_free = seq_lens.numel(), free.numel()
    st, width = _table(block_table, n_req, page, num_blocks)
    vector(seq_lens, torch.int32, n_req, "seq_lens")
    vector(free, torch.int32, n_free, "free")
    vector(top, torch.int32, 3, "top")
    vector(done, torch.uint8 if done.dtype is torch.uint8 else torch.bool, n_req, "done")
    a = _pack_release(                 # in the struct's order
        block_table.data_ptr(), st, seq_lens.data_ptr(), done.data_ptr(), free.data_ptr(),
        top.data_ptr(), n_req, width, page, num_blocks, n_free)
    call_on(index, "amass_release", a)
