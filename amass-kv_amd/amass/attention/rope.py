"""Rotary positions on q and k, with the K / V write to the paged cache (``amass_rope_write``).

  rope_table         (max_pos, rot) fp32 cosines and sines of every position, made once
  rope_paged_write   one layer's step: q turned, k turned and written, v written

The angle of pair i at position p is ``p * w_i``, ``w_i = base^(-2 i / rot)``, where ``rot`` is
the number of leading channels that turn (a head's others are copied).  Pairs are channels
``(i, i + rot / 2)`` (layout "half") or ``(2 i, 2 i + 1)`` ("interleaved").

Longer contexts than a model was trained on (``original_max`` positions) scale the angles:

  "linear"    p w_i / factor
  "ntk"       the base becomes base * factor^(rot / (rot - 2)): the slowest pair turns
              ``factor`` times slower, the fastest as before
  "by_parts"  pair i makes ``original_max w_i / 2 pi`` turns over the trained length: at
              ``fast`` turns (4) or more it stays, at ``slow`` (1) or fewer it is slowed by
              ``factor``, linear in the number of turns between them
  "yarn"      linear in the pair's index between the pairs of ``fast`` (32) and ``slow`` (1)
              turns, and cosines and sines times ``0.1 ln(factor) + 1``

Tables are computed in float64 and rounded once, so far positions keep the accuracy of near
ones.
"""
from __future__ import annotations

import math

import torch

from .._hip import RopeArgs, cache_halves, call_on, device_index, packer, vector

LAYOUTS = {"half": 0, "interleaved": 1}
DTYPES = {torch.bfloat16: 0, torch.float16: 1}      # AMASS_BF16, AMASS_FP16
_pack_rope = packer(RopeArgs)


def rope_frequencies(rot: int, *, base: float = 10000.0, scaling: str | None = None,
                     factor: float = 1.0, original_max: int | None = None,
                     fast: float | None = None, slow: float = 1.0):
    """(w (rot / 2,) float64, amplitude): the pairs' frequencies (module doc).  ``fast`` None: 4
    turns for "by_parts", 32 for "yarn"."""
    if rot < 2 or rot % 2:
        raise ValueError(f"rot {rot} must be even and positive")
    if not base > 1.0:
        raise ValueError(f"base {base} must exceed 1")
    if not factor >= 1.0:
        raise ValueError(f"factor {factor} must be at least 1")
    if scaling in ("by_parts", "yarn") and not (original_max and original_max > 0):
        raise ValueError(f"scaling {scaling!r} needs original_max")
    if fast is None:
        fast = 32.0 if scaling == "yarn" else 4.0
    if scaling in ("by_parts", "yarn") and not fast > slow > 0.0:
        raise ValueError("fast must exceed slow, and slow zero")
    if scaling == "ntk":
        if rot < 4:
            raise ValueError("scaling 'ntk' needs two pairs or more")
        base = base * factor ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64)
    w = base ** (-2.0 * i / rot)
    amplitude = 1.0
    if scaling is None or scaling == "ntk":
        pass
    elif scaling == "linear":
        w = w / factor
    elif scaling == "by_parts":
        turns = original_max * w / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        w = keep * w + (1.0 - keep) * w / factor
    elif scaling == "yarn":
        def pair(turns):                       # the pair that makes so many turns
            return rot * math.log(original_max / (2.0 * math.pi * turns)) / (2.0 * math.log(base))
        lo = max(math.floor(pair(fast)), 0)
        hi = min(math.ceil(pair(slow)), rot - 1)
        slowed = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        w = (1.0 - slowed) * w + slowed * w / factor
        amplitude = 0.1 * math.log(factor) + 1.0
    else:
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'ntk', 'by_parts' or 'yarn'")
    return w, amplitude


def rope_table(rot: int, max_pos: int, *, device=None, **scaling) -> torch.Tensor:
    """(max_pos, rot) fp32: cosines of every pair, then sines; ``scaling`` as
    ``rope_frequencies`` takes it."""
    if max_pos < 1:
        raise ValueError("max_pos must be positive")
    w, amplitude = rope_frequencies(rot, **scaling)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * w
    return (amplitude * torch.cat([angle.cos(), angle.sin()], 1)).to(torch.float32).to(device)


def rope_paged_write(q, k, v, positions, table, kv_cache, slots, q_out=None, *,
                     layout: str = "half") -> None:
    """Turn q (T, H, d) into ``q_out`` (``None``: in place) and k (T, n_kv, d) into its slots
    of the cache, and write v (T, n_kv, d; ``None`` for a cache without V) to them.

    ``positions`` (T,) int32, ``slots`` (T,) int64 (``extend_block_tables``), ``table`` from
    ``rope_table``, ``kv_cache`` one layer's (2, NB, page, n_kv, d), (NB, 2, ...) or, without V,
    (NB, 1, ...).  A row whose position is outside the table is passed over; one whose slot is
    outside the cache has its q turned and is not written.  A slot belongs to one row of a call.
    ``q_out`` is q or shares no memory with it.  bf16 or fp16."""
    q_out = q if q_out is None else q_out
    index = device_index(q, k, v, positions, table, kv_cache, slots, q_out)
    dt = q.dtype
    if not (dt in DTYPES and dt is k.dtype is kv_cache.dtype is q_out.dtype
            and (v is None or dt is v.dtype)):
        raise ValueError("q, k, v, q_out and the cache must all be bf16 or all fp16")
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r}: 'half' or 'interleaved'")
    (nb, page, n_kv, d), kc, vc, cs = cache_halves(kv_cache)
    if (v is None) != (vc == 0):
        raise ValueError("v comes with a cache that has V, and only with one")
    shape, k_shape = q.shape, k.shape
    if len(shape) != 3 or shape[2] != d or q_out.shape != shape or \
            k_shape != (shape[0], n_kv, d) or (v is not None and v.shape != k_shape):
        raise ValueError(f"q (T, H, {d}) and k, v (T, {n_kv}, {d}) expected, q_out like q")
    T, H, _ = shape
    max_pos, rot = table.shape
    tab_st, unit = table.stride()
    if table.dtype is not torch.float32 or unit != 1 or rot % 2 or not 2 <= rot <= d:
        raise ValueError(f"table must be (max_pos, rot) fp32 with an even rot of at most {d}")
    if d % 2 or page & (page - 1):
        raise ValueError(f"head dim {d} must be even and page {page} a power of two")
    vector(positions, torch.int32, T, "positions")
    vector(slots, torch.int64, T, "slots")
    if T == 0:
        return
    q_st, q_hs, q_unit = q.stride()
    k_st, k_hs, k_unit = k.stride()
    o_st, o_hs, o_unit = q_out.stride()
    sb, st, sh, c_unit = cs
    if not q_unit == k_unit == o_unit == c_unit == 1:
        raise ValueError("q / k / q_out / cache need unit stride on the head dim")
    if not (o_st or T == 1) or not (o_hs or H == 1):
        raise ValueError("rows or heads of q_out share memory")
    if not (sb or nb == 1) or not (st or page == 1) or not (sh or n_kv == 1):
        raise ValueError("rows of the cache share memory")
    v_at = v_st = v_hs = 0
    if v is not None:
        v_at = v.data_ptr()
        v_st, v_hs, v_unit = v.stride()
        if v_unit != 1:
            raise ValueError("v needs unit stride on the head dim")
    a = _pack_rope(                    # in the struct's order
        q.data_ptr(), q_st, q_hs, k.data_ptr(), k_st, k_hs, v_at, v_st, v_hs,
        q_out.data_ptr(), o_st, o_hs, kc, sb, st, sh, vc, sb, st, sh, table.data_ptr(), tab_st,
        positions.data_ptr(), slots.data_ptr(), T, H, n_kv, d, rot, page, nb, max_pos,
        LAYOUTS[layout], DTYPES[dt])
    call_on(index, "amass_rope_write", a)
