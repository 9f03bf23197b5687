"""Chunk attention on the GPU at its edges: batches that are none, values that leave the ordinary."""
import math
import os
import re

import numpy as np
import pytest
import torch

from amass.attention import chunk_scratch_bytes, paged_chunk_attention
from helpers import announce
from test_gpu_chunk import DEV, Case, want_on_gpu

pytestmark = pytest.mark.gpu
INF = float("inf")


def test_starts_that_do_not_ascend_leave_other_memory_alone():
    """Requests whose rows together are several times the batch's, and a scratch that holds records of
    row tiles behind `out`: the rows there stay, and the scratch serves the next call."""
    announce("chunk attention: starts that do not ascend, a scratch of records")
    T, R = 1024, 5
    c = Case(new=[T], lens=[4000], n_kv=8)
    q, kv, table, _, _ = c.dev()
    wide = torch.full((2 * T, 32, 128), 7.0, dtype=c.dt, device=DEV)
    out = wide[:T]
    bad = dict(block_table=table.expand(R, -1).contiguous(),
               seq_lens=torch.full((R,), 4000, dtype=torch.int32, device=DEV),
               query_start=torch.tensor([0, T] * 3, dtype=torch.int32, device=DEV))
    need = chunk_scratch_bytes(q, kv, *bad.values(), out)
    # (request, row tile, parts, slot, first row, rows, tokens, 0) from byte 256 on, repeated
    record = torch.tensor([0, 0, 2, 0, T, T, 4000, 0], dtype=torch.int32)
    scratch = record.repeat(-(-need // 32) + 8).view(torch.uint8)[:need].to(DEV)
    paged_chunk_attention(q, kv, *bad.values(), out, scratch=scratch)
    torch.cuda.synchronize()
    assert (wide[T:] == 7.0).all()
    c = Case(new=[90, 3], lens=[3000, 900], n_kv=8)
    q, kv, table, lens, qs = c.dev()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    paged_chunk_attention(q, kv, table, lens, qs, out, lse=lse, scratch=scratch)
    c.check(out, lse)


@pytest.mark.parametrize("T,starts,rows", [(60, [0, 40, 20, 60], [*range(20), *range(40, 60)]),
                                           (12, [0, 9, 7, 12], [*range(7), *range(9, 12)])])
def test_rows_of_one_request_only_are_right_where_starts_do_not_ascend(T, starts, rows):
    announce(f"chunk attention: starts {starts}")
    c = Case(new=[T, 0, 0], lens=[150, 40, 230], n_kv=2)
    c.qs = torch.tensor(starts, dtype=torch.int32)
    c.check(*c.run(), rows=rows)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("new,lens,at", [([100], [230], 180), ([6], [300], 297), ([5], [6000], 5998),
                                         ([300], [2500], 2300), ([1], [40], 39)])
@pytest.mark.parametrize("value", [INF, -INF, float("nan")])
def test_v_that_is_not_finite_arrives_as_itself(new, lens, at, dtype, d, value):
    announce(f"chunk attention: {value} seen in a channel of V, {new} of {lens}, {dtype}")
    c = Case(new=new, lens=lens, n_kv=1, dtype=dtype, d=d)
    block, row = int(c.table[0, at // 16]), at % 16
    c.v[block, row, 0, 37] = value
    with np.errstate(invalid="ignore"):
        want = torch.tensor(c.want()[0][:, :, 37])
    out, _ = c.run()
    sees = at - (lens[0] - new[0])                  # the first row that does
    got = out[:, :, 37].double().cpu()
    assert torch.isfinite(got[:sees]).all()
    assert torch.equal(got[sees:].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0),
                       want[sees:].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0))


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("new,lens,first,second", [([90], [150], 70, 130), ([7], [2000], 1500, 1997),
                                                   ([300], [900], 650, 652)])
def test_opposite_infinities_in_v_make_nan(new, lens, first, second, dtype, d):
    """Rows that see one of them have it, rows that see both NaN; in other channels nothing."""
    announce(f"chunk attention: both infinities in V, {new} of {lens}, {dtype}")
    c = Case(new=new, lens=lens, n_kv=1, dtype=dtype, d=d)
    want = c.want()
    kept = {}
    for at, value in ((first, INF), (second, -INF)):
        b, i = int(c.table[0, at // 16]), at % 16
        kept[b, i] = c.v[b, i, 0, 5].clone()
        c.v[b, i, 0, 5] = value
    out, lse = c.run()
    start = lens[0] - new[0]
    one, both = max(first - start, 0), second - start
    x = out[:, :, 5].float()
    assert torch.isfinite(x[:one]).all() and (x[one:both] == INF).all()
    assert torch.isnan(x[both:]).all() and both < new[0]
    out[one:, :, 5] = torch.tensor(want[0][one:, :, 5], dtype=c.dt, device=DEV)
    for (b, i), v in kept.items():
        c.v[b, i, 0, 5] = v
    c.check(out, lse)


@pytest.mark.parametrize("dtype,q,k,scale", [
    ("fp16", 2.0 ** 15, 2.0 ** 15, None), ("fp16", -2.0 ** 15, 2.0 ** 14, None),
    ("fp16", 2.0 ** 11, 2.0 ** 11, 1.0), ("bf16", 2.0 ** 25, 2.0 ** 25, None),
    ("bf16", -2.0 ** 40, 2.0 ** 30, 0.3), ("bf16", 2.0 ** 60, 2.0 ** 58, 3.0),
    ("bf16", 2.0 ** 60, 2.0 ** 58, 1e30), ("bf16", -2.0 ** 60, 2.0 ** 58, 1e30),
    ("bf16", -2.0 ** 60, 2.0 ** 58, 0.1)])
@pytest.mark.parametrize("new,lens,d", [([1], [300], 128), ([5], [9000], 128), ([100], [300], 128),
                                        ([40], [6000], 64), ([2, 70], [40, 90], 64)])
def test_scores_far_from_zero(new, lens, d, dtype, q, k, scale):
    """Two keys have the largest score, every other one is thousands below: rows are the mean of the two
    keys' V.  Scores are exact in fp32 (d q k times 11/8 and 13/8, powers of two but for that), so
    are the two weights (1 each) and, but for 2^-24, their sum; the result is rounded once.  lse: at
    most eight roundings (constants, products, sums) of 2^-24 of its size.  A score that times the
    scale exceeds fp32 gives lse its infinity."""
    announce(f"chunk attention: scores around {d * q * k:g}, scale {scale}, {new} of {lens}")
    c = Case(new=new, lens=lens, dtype=dtype, d=d, n_kv=1, scale=scale)
    most, least = (1.625, 1.375) if q > 0 else (1.375, 1.625)
    c.q.fill_(q), c.k.fill_(least * k)
    want = torch.zeros(sum(new), 4, d, dtype=torch.float64)
    for r in range(len(new)):
        two = [(int(c.table[r, at // 16]), at % 16) for at in (3, lens[r] - new[r])]
        for b, i in two:
            c.k[b, i] = most * k
        want[int(c.qs[r]):int(c.qs[r + 1])] = sum(c.v[b, i].double() for b, i in two) / 2
    out, lse = c.run()
    u = torch.finfo(c.dt).eps / 2
    err = (out.double().cpu() - want).abs()
    size = 1.0 + 2.0 * want.abs()                   # (V is within a few of 1)
    assert (err <= u * want.abs() * 1.01 + 2.0 ** -22 * size).all(), err.max()
    top = most * d * q * k * c.scale
    if abs(top) * math.log2(math.e) < 3.4e38:
        assert ((lse.double() - (top + math.log(2.0))).abs() <= 2.0 ** -21 * abs(top) + 1e-6).all()
    else:
        assert (lse == math.copysign(INF, top)).all()


@pytest.mark.parametrize("n,to", [(1024, 256), (1500, 256), (700, 224)])
def test_short_row_tiles_stay_whole_beside_long_ones(n, to):
    """The rows of a prompt whose longest row tiles are cut in parts: those up to 4 tiles of 64 keys are
    as in a prompt that ends there, bit for bit."""
    announce(f"chunk attention: first {to} tokens of {n}")
    c = Case(new=[n], lens=[n], n_kv=1)
    out, lse = c.run()
    q, kv, table, lens, qs = c.dev()
    o, e = torch.full_like(q[:to], 7.0), torch.full_like(lse[:to], 7.0)
    paged_chunk_attention(q[:to], kv, table, torch.tensor([to], dtype=torch.int32, device=DEV),
                          torch.tensor([0, to], dtype=torch.int32, device=DEV), o, lse=e)
    assert torch.equal(lse[:to], e) and torch.equal(out[:to], o)


# batches whose keys no cache keeps: K and V of requests of one row tile are loaded past the caches
PAST = {
    "drafts": dict(new=[4, 1, 8, 3], lens=[9001, 12345, 8200, 9999]),
    "drafts fp16": dict(new=[3, 8, 5], lens=[17000, 10007, 9013], dtype="fp16"),
    "drafts d64": dict(new=[5, 2, 8, 7], lens=[20011, 17203, 19999, 15000], d=64),
    "drafts d64 fp16": dict(new=[4, 4, 8], lens=[30001, 25007, 20005], d=64, dtype="fp16", page=32),
    "chunks": dict(new=[10, 31, 9, 32], lens=[9003, 8230, 12001, 9100], pad=5),
    "chunks fp16": dict(new=[20, 9, 32], lens=[17005, 9012, 12300], dtype="fp16", halves_first=True),
    "chunks d64": dict(new=[10, 32, 17, 30], lens=[20001, 17217, 19000, 16003], d=64, page=64),
    "chunks d64 fp16": dict(new=[31, 9, 16], lens=[25011, 30030, 21001], d=64, dtype="fp16"),
    "seven heads": dict(new=[18, 5, 1, 16], lens=[17777, 15001, 9999, 23001], n_kv=4, G=7),
    "window": dict(new=[24, 5, 32], lens=[14001, 13007, 12345], window=11000),
    "beside a prompt": dict(new=[1500, 12, 3], lens=[3000, 9001, 8003]),
}


def loaded_past_the_caches(c):
    """Whether the requests of at most 128 rows are, by the kernel's rule: tiles of 64 keys of all row
    tiles (each counted as its request's longest) in bytes against the limit in the source."""
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "amass-kv_amd", "csrc", "chunk.hip")) as fh:
        limit = float(re.search(r"CK_ONCE = ([\d.e]+)f;", fh.read()).group(1))
    n_kv, d = c.k.shape[2:]
    G = c.q.shape[1] // n_kv
    keys = 0
    for n, length in zip((c.qs[1:] - c.qs[:-1]).tolist(), c.lens.tolist()):
        tiles = -(-n * G // 128)
        first = length - n + 128 * (tiles - 1) // G - (c.window or length) + 1    # its first key
        keys += tiles * (-(-length // 64) - max(first, 0) // 64)
    return keys * 64 * 4 * d * n_kv > limit


@pytest.mark.parametrize("name", PAST)
def test_keys_loaded_past_the_caches(name):
    announce(f"chunk attention: {name}, loaded past the caches")
    c = Case(**{**dict(n_kv=8, G=4), **PAST[name]})
    assert loaded_past_the_caches(c)
    c.want = lambda: want_on_gpu(c)
    c.check(*c.run())


@pytest.mark.parametrize("name", ["drafts d64 fp16", "chunks", "chunks d64"])
def test_v_that_is_not_finite_loaded_past_the_caches(name):
    """NaN in a channel of the last token of request 1, and everywhere behind the last tokens."""
    announce(f"chunk attention: {name}, loaded past the caches, V not finite")
    c = Case(**{**dict(n_kv=8, G=4), **PAST[name]})
    assert loaded_past_the_caches(c)
    want, finite = want_on_gpu(c), c.v.clone()
    for r, n in enumerate(c.lens.tolist()):
        last = c.table[r, (n - 1) // c.page]
        if n % c.page:
            c.k[last, n % c.page:] = float("nan")
            c.v[last, n % c.page:] = float("nan")
    n = int(c.lens[1])
    c.v[c.table[1, (n - 1) // c.page], (n - 1) % c.page, 2, 9] = float("nan")
    out, lse = c.run()
    t = int(c.qs[2]) - 1                            # the one row that sees it, by 4 heads
    assert torch.isnan(out[t, 8:12, 9].float()).all()
    out[t, 8:12, 9] = torch.tensor(want[0][t, 8:12, 9], dtype=c.dt, device=DEV)
    c.want, c.v = lambda: want, finite              # (the tolerance goes by V's largest)
    c.check(out, lse)


@pytest.mark.parametrize("new,lens", [([1], [300]), ([6], [5000]), ([100], [300]), ([300], [700])])
def test_largest_values_of_v_under_a_maximum_that_lags(new, lens):
    """A key whose weight is 2^7 times that of all keys before it, short of what moves the running
    maximum, has V of 2^123: its product with a weight above 1 would exceed fp32."""
    announce(f"chunk attention: V of 2^123, {new} of {lens}")
    c = Case(new=new, lens=lens, n_kv=1)
    c.q.zero_(), c.k.zero_(), c.v.zero_()
    c.q[:, :, 0] = 1.0
    block = int(c.table[0, 130 // 16])
    c.k[block, 130 % 16, 0, 0] = 7.0 * math.log(2.0) / c.scale
    c.v[block, 130 % 16, 0, 1::2] = 2.0 ** 123
    c.v[block, 130 % 16, 0, 4::8] = -1.5 * 2.0 ** 123
    c.check(*c.run())
