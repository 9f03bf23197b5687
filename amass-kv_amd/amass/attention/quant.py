"""A paged cache in 8 bits: its quantising write, its attention and the way back to 16 bits
(``amass_quant_write``, ``amass_quant_chunk_attention``, ``amass_quant_read``).

  codes    (NB, 2, page, n_kv, d) or (2, NB, ...) int8 or float8_e4m3fn
  scales   (NB, 2, n_kv) or (2, NB, n_kv) fp32, one for each block, half (K, V) and kv head

A number is ``code * scale``; where both first axes are 2, the first is the halves (as a 16-bit cache is
read).  Beside ``rope_paged_write`` and ``paged_chunk_attention`` it takes half the memory and half the
bytes of every decode step.  int8 resolves a block's numbers in 254 even
steps of its largest; e4m3 keeps 4 significant bits of each, for blocks of a few large numbers
among small ones.

A scale grows with its block: the write takes the largest magnitude of the tokens that enter the
block now and of those that are there, and where the scale grows it rounds the earlier tokens' codes
again.  The token in a block's first row starts the block anew.  An int8 number is off by at most half
a step of the last scale for its entry and for each growth after it.  So codes do not depend on how a
prompt was cut into chunks where no scale grows; where it grows g times they differ by (2 + g) / 2
steps at most (16 single tokens against one write: up to 2 steps among tokens of like size, several where
each is 1 percent larger than the one before).  An e4m3 number keeps its 4 bits through growths until
it is below 2^-6 of the scale.

Rows behind a run keep their codes, not their numbers: a run from the block's first row, or one that
makes the scale grow, leaves them under another scale.  So tokens enter a block in order; those that were
taken back are written again before anyone sees them.

All calls run on torch's current stream of the tensors' GPU, depend on shapes only, allocate
nothing but the attention's scratch, never synchronise and can be captured in a HIP graph.
"""
from __future__ import annotations

import torch

from .._hip import (QuantChunkArgs, QuantReadArgs, QuantWriteArgs, cache_halves, call_on, check,
                    device_index, load_library, packer, vector)
from .rope import DTYPES, LAYOUTS

HEAD_DIMS = (64, 128)
CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}      # AMASS_INT8, AMASS_E4M3
MIN_PAGE, MAX_PAGE = 16, 1024
MAX_INT = 2 ** 31 - 1
_pack_write = packer(QuantWriteArgs)
_pack_read = packer(QuantReadArgs)
_pack_chunk = packer(QuantChunkArgs)
_SCRATCH = {}            # (GPU, requests, rows, kv heads, group, head dim) -> scratch bytes


def quant_cache(num_blocks: int, page: int, n_kv: int, d: int, *, dtype=torch.int8,
                device=None):
    """(codes, scales) of a pool of ``num_blocks`` blocks, zeros with scales of one; ``dtype``
    torch.int8 or torch.float8_e4m3fn.

    The codes of a page of one head lie together (a view of (NB, 2, n_kv, page, d) memory).  The calls
    take any strides; over a contiguous (NB, 2, page, n_kv, d) the attention of 64 single tokens with
    8k keys (8 heads of 128, e4m3) takes 207 us where it takes 177 so."""
    _geometry(page, d, dtype)
    codes = torch.zeros(num_blocks, 2, n_kv, page, d, dtype=torch.int8, device=device)
    return (codes.transpose(2, 3).view(dtype),
            torch.ones(num_blocks, 2, n_kv, dtype=torch.float32, device=device))


def _geometry(page, d, dtype):
    if dtype not in CODES:
        raise ValueError(f"codes must be int8 or float8_e4m3fn, not {dtype}")
    if d not in HEAD_DIMS:
        raise ValueError(f"head dim {d} (built for {HEAD_DIMS})")
    if page < MIN_PAGE or page > MAX_PAGE or page & (page - 1):
        raise ValueError(f"page {page} must be a power of two from {MIN_PAGE} to {MAX_PAGE}")


def _halves(codes, scales, writes):
    """((blocks, page, n_kv, d), code type, (k, v, block, row, head strides of codes), (k, v, block,
    head strides of scales)) of a checked cache."""
    shape, st, dt = codes.shape, codes.stride(), codes.dtype
    if len(shape) != 5:
        raise ValueError("codes must be (NB, 2, page, n_kv, d) or (2, NB, page, n_kv, d)")
    n0, n1, page, n_kv, d = shape
    if scales.dtype is not torch.float32 or scales.shape != (n0, n1, n_kv):
        raise ValueError(f"scales must be ({n0}, {n1}, {n_kv}) fp32")
    if n0 == 2:
        nb = n1
        half, sb, row, head, unit = st
        s_half, s_sb, s_sh = scales.stride()
    elif n1 == 2:
        nb = n0
        sb, half, row, head, unit = st
        s_sb, s_half, s_sh = scales.stride()
    else:
        raise ValueError("codes must be (NB, 2, page, n_kv, d) or (2, NB, page, n_kv, d)")
    _geometry(page, d, dt)
    if unit != 1:
        raise ValueError("codes need unit stride on the head dim")
    if writes and (0 in (half, row, s_half) or (nb > 1 and 0 in (sb, s_sb)) or
                   (n_kv > 1 and 0 in (head, s_sh))):
        raise ValueError("rows of codes or scales share memory")
    at, s_at = codes.data_ptr(), scales.data_ptr()
    return ((nb, page, n_kv, d), CODES[dt], (at, at + half, sb, row, head),
            (s_at, s_at + 4 * s_half, s_sb, s_sh))


def quant_paged_write(k, v, codes, scales, slots, *, q=None, positions=None, table=None,
                      q_out=None, layout: str = "half") -> None:
    """Quantise k and v (T, n_kv, d), bf16 or fp16, into their slots of the cache.

    ``slots`` (T,) int64 from ``extend_block_tables``: the tokens of a block come as one run of
    rows with ascending slots, and a row whose slot is outside the cache is passed over.  Two
    runs of one call in one block leave a mixture there.  Numbers that are not finite make NaN of
    their block, half and head (until its first row is written again).

    With ``table`` (``rope_table``) and ``positions`` (T,) int32, k is turned by its position
    first (``layout`` as ``rope_paged_write`` has it, rot a multiple of 16), in float64, rounded
    to its type and then to a code; a row whose position is outside the table is passed over.
    With ``q`` (T, H, d) too, q is turned into ``q_out`` (``None``: in place), as
    ``rope_paged_write`` does.  k, v, q and codes need 16-byte aligned rows."""
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
        if (table is None) != (positions is None):
            raise ValueError("positions and table need each other")
    else:
        if table is None or positions is None:
            raise ValueError("q needs positions and table")
        if q_out is None:
            q_out = q
    index = device_index(k, v, codes, scales, slots, q, positions, table, q_out)
    dt = k.dtype
    if dt not in DTYPES or dt is not v.dtype or \
            (q is not None and not dt is q.dtype is q_out.dtype):
        raise ValueError("k, v, q and q_out must all be bf16 or all fp16")
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r}: 'half' or 'interleaved'")
    (nb, page, n_kv, d), kind, c, s = _halves(codes, scales, True)
    shape = k.shape
    T = shape[0]
    if shape != (T, n_kv, d) or v.shape != shape:
        raise ValueError(f"k and v must be (T, {n_kv}, {d})")
    vector(slots, torch.int64, T, "slots")
    k_st, k_hs, k_unit = k.stride()
    v_st, v_hs, v_unit = v.stride()
    q_at = q_st = q_hs = o_at = o_st = o_hs = H = 0
    q_unit = o_unit = 1
    if q is not None:
        shape = q.shape
        if len(shape) != 3 or shape[0] != T or shape[1] == 0 or shape[2] != d or \
                (q_out is not q and q_out.shape != shape):
            raise ValueError(f"q and q_out must be (T, H, {d})")
        H = shape[1]
        q_at = o_at = q.data_ptr()
        q_st, q_hs, q_unit = o_st, o_hs, o_unit = q.stride()
        if q_out is not q:
            o_at = q_out.data_ptr()
            o_st, o_hs, o_unit = q_out.stride()
        if (o_st == 0 and T > 1) or (o_hs == 0 and H > 1):
            raise ValueError("rows or heads of q_out share memory")
    if not k_unit == v_unit == q_unit == o_unit == 1:
        raise ValueError("k / v / q / q_out need unit stride on the head dim")
    tab_at = tab_st = pos_at = rot = max_pos = 0
    if table is not None:
        max_pos, rot = table.shape
        tab_st, unit = table.stride()
        if table.dtype is not torch.float32 or unit != 1 or rot % 16 or not 16 <= rot <= d:
            raise ValueError(f"table must be (max_pos, rot) fp32, rot a multiple of 16 up to {d}")
        vector(positions, torch.int32, T, "positions")
        tab_at, pos_at = table.data_ptr(), positions.data_ptr()
    if T == 0:
        return
    call_on(index, "amass_quant_write", _pack_write(       # in the struct's order
        k.data_ptr(), k_st, k_hs, v.data_ptr(), v_st, v_hs, q_at, q_st, q_hs, o_at, o_st, o_hs,
        *c, *s, tab_at, tab_st, pos_at, slots.data_ptr(), T, H, n_kv, d, rot, page, nb, max_pos,
        LAYOUTS[layout], DTYPES[dt], kind))


def quant_paged_read(codes, scales, src, kv_cache, dst) -> None:
    """Blocks ``src`` (n,) int32 of the 8-bit cache into blocks ``dst`` (n,) int32 of a bf16 or fp16
    one with the same pages and heads, (2, NB, page, n_kv, d) or (NB, 2, ...): what the decode path,
    the page summaries or ``paged_chunk_attention`` then read.  Pairs with a block outside its
    cache are passed over; a block appears once in ``dst``."""
    index = device_index(codes, scales, src, kv_cache, dst)
    if kv_cache.dtype not in DTYPES:
        raise ValueError("kv_cache must be bf16 or fp16")
    (nb, page, n_kv, d), kind, c, s = _halves(codes, scales, False)
    (nb_out, *shape), k, v, (o_sb, o_st, o_sh, unit) = cache_halves(kv_cache)
    if v == 0 or tuple(shape) != (page, n_kv, d):
        raise ValueError(f"kv_cache must have V and pages of ({page}, {n_kv}, {d})")
    if unit != 1 or not (o_sb or nb_out == 1) or not o_st or not (o_sh or n_kv == 1) or k == v:
        raise ValueError("kv_cache needs unit stride on the head dim and rows of their own")
    n = src.numel()
    if dst.numel() != n:
        raise ValueError(f"{n} blocks in src, {dst.numel()} in dst")
    vector(src, torch.int32, n, "src")
    vector(dst, torch.int32, n, "dst")
    if n == 0 or nb == 0 or nb_out == 0:
        return
    call_on(index, "amass_quant_read", _pack_read(         # in the struct's order
        *c, *s, k, v, o_sb, o_st, o_sh, src.data_ptr(), dst.data_ptr(), n, n_kv, d, page, nb,
        nb_out, DTYPES[kv_cache.dtype], kind))


def _chunk_args(q, codes, scales, block_table, seq_lens, query_start, out, scale, causal, window,
                lse):
    """(the argument struct's values up to the scratch, those behind it) of a checked call."""
    dt = q.dtype
    if dt not in DTYPES or dt is not out.dtype:
        raise ValueError("q and out must both be bf16 or both fp16")
    (nb, page, n_kv, d), kind, c, s = _halves(codes, scales, False)
    shape = q.shape
    if len(shape) != 3 or shape[2] != d or (out is not q and out.shape != shape):
        raise ValueError(f"q and out must be (T, H, {d})")
    T, H, _ = shape
    if H == 0 or H % n_kv:
        raise ValueError(f"{H} query heads are not a multiple of {n_kv} kv heads")
    if window is None:
        window = 0
    elif window < 1:
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
    if q_unit != 1 or o_unit != 1:
        raise ValueError("q / out need unit stride on the head dim")
    if (o_st == 0 and T > 1) or (o_hs == 0 and H > 1):
        raise ValueError("rows or heads of out share memory")
    l_at = l_st = l_hs = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != (T, H):
            raise ValueError("lse must be (T, H) fp32")
        l_at = lse.data_ptr()
        l_st, l_hs = lse.stride()
        if (l_st == 0 and T > 1) or (l_hs == 0 and H > 1):
            raise ValueError("rows or heads of lse share memory")
    return ((q.data_ptr(), q_st, q_hs, *c, *s, block_table.data_ptr(), bt_st, seq_lens.data_ptr(),
             query_start.data_ptr(), out.data_ptr(), o_st, o_hs, l_at, l_st, l_hs),
            (scale, n_req, T, n_kv, H // n_kv, d, page, nb, width, 1 if causal else 0,
             window if window < MAX_INT else MAX_INT, DTYPES[dt], kind))


def _scratch_bytes(index, head, tail) -> int:
    key = (index, *tail[1:6])
    n = _SCRATCH.get(key)
    if n is None:
        with torch.cuda.device(index):
            n = load_library().amass_quant_scratch_bytes(_pack_chunk(*head, 0, 0, *tail))
        if n < 0:
            check(n, "amass_quant_scratch_bytes")
        if len(_SCRATCH) >= 4096:
            _SCRATCH.clear()
        _SCRATCH[key] = n
    return n


def quant_scratch_bytes(q, codes, scales, block_table, seq_lens, query_start, out, *, scale=None,
                        causal: bool = True, window=None, lse=None) -> int:
    """Bytes of scratch that ``quant_chunk_attention`` takes for these shapes."""
    index = device_index(q, codes, scales, block_table, seq_lens, query_start, out, lse)
    return _scratch_bytes(index, *_chunk_args(q, codes, scales, block_table, seq_lens,
                                              query_start, out, scale, causal, window, lse))


def quant_chunk_attention(q, codes, scales, block_table, seq_lens, query_start, out, *,
                          scale=None, causal: bool = True, window: int | None = None, lse=None,
                          scratch=None) -> None:
    """``paged_chunk_attention`` over the 8-bit cache: the rows of q (T, H, d), bf16 or fp16,
    over their requests' keys and values, into out (which may be q).

    Requests, visible positions, ``causal``, ``window``, ``scale``, ``lse`` and ``scratch`` as
    there: row ``query_start[r] + i`` is one of the last tokens of request r's ``seq_lens[r]``,
    whose K and V the cache holds already (``quant_paged_write``).  Rows that see nothing get zeros
    (``lse``: -inf); rows of no request stay as they are.

    Scales are positive, V's count as at least 2^-64 and those of one request and kv head lie within
    2^80 of each other (pages of zeros aside, beside V of up to 2^40).  A scale that is not finite makes NaN of the rows that see its page, a NaN
    code of those that see its key."""
    index = device_index(q, codes, scales, block_table, seq_lens, query_start, out, lse, scratch)
    head, tail = _chunk_args(q, codes, scales, block_table, seq_lens, query_start, out, scale,
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
    call_on(index, "amass_quant_chunk_attention",
            _pack_chunk(*head, scratch.data_ptr(), size, *tail))
