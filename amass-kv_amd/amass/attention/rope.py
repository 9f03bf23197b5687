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
              ``fast`` turns or more it stays, at ``slow`` or fewer it is slowed by ``factor``,
              linear in the number of turns between them
  "yarn"      the same ends, linear in the pair's index between the pairs of ``fast`` and
              ``slow`` turns, and cosines and sines times ``0.1 ln(factor) + 1``

Tables are computed in float64 and rounded once, so far positions keep the accuracy of near
ones.
"""
from __future__ import annotations

import math

import torch

from .._hip import RopeArgs, call_on, packer, same_device

LAYOUTS = {"half": 0, "interleaved": 1}
DTYPES = {torch.bfloat16: 0, torch.float16: 1}      # AMASS_BF16, AMASS_FP16
_pack_rope = packer(RopeArgs)
_NO_VIEW = (0, 0, 0)


def rope_frequencies(rot: int, *, base: float = 10000.0, scaling: str | None = None,
                     factor: float = 1.0, original_max: int | None = None, fast: float = 4.0,
                     slow: float = 1.0):
    """(w (rot / 2,) float64, amplitude): the pairs' frequencies (module doc)."""
    if rot < 2 or rot % 2:
        raise ValueError(f"rot {rot} must be even and positive")
    if not base > 1.0:
        raise ValueError(f"base {base} must exceed 1")
    if not factor >= 1.0:
        raise ValueError(f"factor {factor} must be at least 1")
    if scaling in ("by_parts", "yarn") and not (original_max and original_max > 0):
        raise ValueError(f"scaling {scaling!r} needs original_max")
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
    outside the cache has its q turned and is not written.  bf16 or fp16."""
    from .decode import _split_kv
    q_out = q if q_out is None else q_out
    same_device(q, k, v, positions, table, kv_cache, slots, q_out)
    kc, vc = _split_kv(kv_cache)
    dt = q.dtype
    if dt not in DTYPES or k.dtype != dt or kc.dtype != dt or q_out.dtype != dt or \
            (v is not None and v.dtype != dt):
        raise ValueError("q, k, v, q_out and the cache must all be bf16 or all fp16")
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r}: 'half' or 'interleaved'")
    if (v is None) != (vc is None):
        raise ValueError("v comes with a cache that has V, and only with one")
    nb, page, n_kv, d = kc.shape
    T, H = q.shape[:2]
    if q.shape != (T, H, d) or q_out.shape != q.shape or k.shape != (T, n_kv, d) or \
            (v is not None and v.shape != k.shape):
        raise ValueError(f"q (T, H, {d}) and k, v (T, {n_kv}, {d}) expected, q_out like q")
    max_pos, rot = table.shape
    if table.dtype != torch.float32 or table.stride(1) != 1 or rot % 2 or not 2 <= rot <= d:
        raise ValueError(f"table must be (max_pos, rot) fp32 with an even rot of at most {d}")
    if d % 2 or page & (page - 1):
        raise ValueError(f"head dim {d} must be even and page {page} a power of two")
    if positions.dtype != torch.int32 or slots.dtype != torch.int64 or \
            not (positions.is_contiguous() and slots.is_contiguous()) or \
            positions.dim() != 1 or slots.dim() != 1 or positions.shape[0] < T or \
            slots.shape[0] < T:
        raise ValueError("positions (T,) int32 and slots (T,) int64 must be contiguous")
    qs, ks, os_, cs = q.stride(), k.stride(), q_out.stride(), kc.stride()
    if qs[2] != 1 or ks[2] != 1 or os_[2] != 1 or cs[3] != 1:
        raise ValueError("q / k / q_out / cache need unit stride on the head dim")
    v_at = vc_at = 0
    vs = vcs = _NO_VIEW
    if v is not None:
        v_at, vs, vc_at, vcs = v.data_ptr(), v.stride(), vc.data_ptr(), vc.stride()
        if vs[2] != 1 or vcs[3] != 1:
            raise ValueError("v and its cache need unit stride on the head dim")
    a = _pack_rope(                    # in the struct's order
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v_at, vs[0], vs[1],
        q_out.data_ptr(), os_[0], os_[1], kc.data_ptr(), cs[0], cs[1], cs[2],
        vc_at, vcs[0], vcs[1], vcs[2], table.data_ptr(), table.stride(0),
        positions.data_ptr(), slots.data_ptr(), T, H, n_kv, d, rot, page, nb, max_pos,
        LAYOUTS[layout], DTYPES[dt])
    call_on(q.device, "amass_rope_write", a)
