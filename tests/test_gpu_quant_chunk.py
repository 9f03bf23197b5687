"""Attention over the 8-bit cache on the GPU (amass_quant_chunk_attention) against the float64 oracle
of chunk attention on the numbers that the codes stand for.

Tolerance: that of test_gpu_chunk (weights and results rounded once to the element type, scores summed
in fp32), since codes are exact in the products.  Scales add to a score the roundings of log2 e scale sk, of
one fma and of the running maximum, each at most 2^-24 of 1.45 |score| + |log2 sv| (here at most 16): 8 more
terms of `reach`, and less than 2^-17 of `size`, which the 2^-16 there have room for (exponentials
and sums take 2^-17 at these lengths).  A weight below fp32's least normal number may be zero: lifted by 2^-8
at least, with V at most vmax, that is 2^-118 vmax for each key seen, which counts where the code of the key
that takes nearly all of the weight is 0 (a Gaussian V has no zeros, codes have): 2^-110 of it
in `size`, of which at least 2^-8 is allowed."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass._hip import AmassError
from amass.attention import quant_chunk_attention, quant_scratch_bytes
from helpers import announce
from test_gpu_chunk import CASES, ROUNDS, Case, want_on_gpu

pytestmark = pytest.mark.gpu
DEV = "cuda"
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class QuantCase(Case):
    """A Case whose K and V are random codes with random scales (no powers of two, a factor of 4 between the
    largest and the least)."""

    def __init__(self, new, lens, *, code="int8", seed=0, **kw):
        super().__init__(new, lens, seed=seed, **kw)
        g = torch.Generator().manual_seed(seed + 77)
        nb, page, n_kv, d = self.k.shape
        std = {"int8": 36.0, "e4m3": 128.0}[code]
        x = std * torch.randn(nb, 2, page, n_kv, d, generator=g)
        x = x.round().clamp(-127, 127) if code == "int8" else x.clamp(-448, 448)
        self.codes = x.to(CODES[code])
        self.scales = torch.exp2(2.0 * torch.rand(nb, 2, n_kv, generator=g) - 1.0) / std
        self.numbers()

    def numbers(self):
        x = self.codes.double() * self.scales.double()[:, :, None, :, None]
        self.k, self.v = x[:, 0], x[:, 1]

    def dev(self):
        codes, scales = self.codes.view(torch.int8).to(DEV), self.scales.to(DEV)
        if self.halves_first:
            codes, scales = codes.transpose(0, 1).contiguous(), scales.transpose(0, 1).contiguous()
        return (self.q.to(DEV), codes.view(self.codes.dtype), scales, self.table.to(DEV),
                self.lens.to(DEV), self.qs.to(DEV))

    def run(self, out=None, lse=None, **kw):
        args = self.dev()
        out = torch.full_like(args[0], 7.0) if out is None else out
        lse = torch.full(args[0].shape[:2], 7.0, device=DEV) if lse is None else lse
        quant_chunk_attention(*args, out, scale=self.scale, causal=self.causal,
                              window=self.window, lse=lse, **kw)
        torch.cuda.synchronize()
        return out, lse

    def check(self, out, lse, rows=None):
        want = self.want()
        least = 2.0 ** -110 * float(self.v.abs().max()) * want[2][:, None, None]
        if self.dt == torch.float16:
            least *= 2.0 ** 3                               # (2^-11 of it is allowed)
        more = (*want[:3], want[3] + least, want[4] * (1.0 + 8.0 / self.q.shape[2]))
        keep, self.want = self.want, lambda: more
        try:
            super().check(out, lse, rows)
        finally:
            self.want = keep

    def token(self, r, at):
        return int(self.table[r, at // self.page]), at % self.page


@pytest.mark.parametrize("name", [n for n in CASES if CASES[n].get("page", 16) <= 1024])
@pytest.mark.parametrize("code", CODES)
def test_matches_float64(name, code):
    announce(f"quant attention: {name}, {code}")
    c = QuantCase(code=code, **CASES[name])
    c.check(*c.run())


# batches of few rows only
FEW = {
    "one token": dict(new=[1], lens=[1]),
    "16 rows": dict(new=[4, 2, 4], lens=[1000, 40, 129]),
    "16 rows, one short": dict(new=[4, 1], lens=[333, 6000]),
    "17 rows": dict(new=[4, 1], lens=[333, 500], G=17),
    "one long row, split": dict(new=[1], lens=[9000], G=8),
    "split, 6 heads": dict(new=[3, 1], lens=[7000, 3000], n_kv=6, G=5),
    "past a period": dict(new=[2], lens=[20000], n_kv=2, G=1),
    "decode step": dict(new=[1] * 40, lens=[16 * i + 7 for i in range(40)], n_kv=8),
    "many requests": dict(new=[1 + i % 3 for i in range(150)], lens=[3 + 5 * i for i in range(150)], G=2),
    "thousands of requests": dict(new=[1] * 3400, lens=[1 + i % 29 for i in range(3400)], G=1),
    "empty requests": dict(new=[0, 3, 0, 4, 0], lens=[33, 9, 0, 77, 5], pad=6),
    "heads of 64": dict(new=[4, 1, 2], lens=[700, 64, 33], d=64, n_kv=4),
    "heads of 64, split": dict(new=[1], lens=[9000], d=64),
    "fp16": dict(new=[4, 1], lens=[700, 64], dtype="fp16"),
    "fp16 of 64": dict(new=[4, 1], lens=[700, 6400], dtype="fp16", d=64),
    "window": dict(new=[4, 2], lens=[400, 500], window=50),
    "window of one": dict(new=[4, 3], lens=[90, 70], window=1),
    "not causal": dict(new=[4, 2], lens=[100, 333], causal=False),
    "rows before position 0": dict(new=[4, 3], lens=[2, 3]),
    "pages of 64": dict(new=[4, 4], lens=[145, 700], page=64, n_kv=4),
    "pages of 1024, halves first": dict(new=[4, 4], lens=[145, 2700], page=1024, halves_first=True),
    "peaked": dict(new=[4, 3], lens=[200, 100], loud=12.0),
    "more than the chip takes": dict(new=[1] * 300, lens=[70 + i for i in range(300)], n_kv=8),
    "a few far longer": dict(new=[1] * 300, lens=[70 + 9000 * (i % 150 == 3) for i in range(300)], n_kv=8, G=2),
}


@pytest.mark.parametrize("name", FEW)
@pytest.mark.parametrize("code", CODES)
def test_few_rows(name, code):
    announce(f"quant attention: few rows, {name}, {code}")
    c = QuantCase(code=code, **FEW[name])
    c.check(*c.run())


def test_other_layouts():
    """A page of one head contiguous, and heads more than 2^30 bytes apart."""
    announce("quant attention: strides of heads")
    c = QuantCase(new=[4, 1, 2], lens=[700, 90, 33], n_kv=4)
    q, codes, scales, table, lens, qs = c.dev()
    major = codes.transpose(2, 3).contiguous().transpose(2, 3)
    nb = codes.shape[0]
    room = torch.empty(4, (1 << 30) + 16, dtype=torch.int8, device=DEV)
    far = room[:, :codes[:, :, :, 0].numel()].view(4, nb, 2, 16, 128).permute(1, 2, 3, 0, 4)
    far.copy_(codes)
    for cache in (major, far):
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
        quant_chunk_attention(q, cache, scales, table, lens, qs, out, lse=lse)
        c.check(out, lse)


@pytest.mark.parametrize("name", ROUNDS)
def test_more_tiles_than_the_chip_takes(name):
    announce(f"quant attention: {name}, more tiles than the chip takes at a time")
    c = QuantCase(code="e4m3" if len(name) % 2 else "int8", **{**dict(n_kv=8, G=4), **ROUNDS[name]})
    c.want = lambda: want_on_gpu(c)
    c.check(*c.run())


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("fp16", 128), ("fp16", 64)])
@pytest.mark.parametrize("code", CODES)
def test_every_code(code, dtype, d):
    """One visible key, whose V holds every code in some channel: the result is that number, rounded."""
    announce(f"quant attention: every code, {code} {dtype} {d}")
    n = 256 // d
    c = QuantCase(new=[1] * n, lens=[1] * n, code=code, dtype=dtype, d=d, n_kv=1, G=3)
    every = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.int8)
    every[every == -128] = 0
    if code == "e4m3":
        every[torch.isnan(every.view(torch.float8_e4m3fn).float())] = 0
    for i in range(n):
        c.codes.view(torch.int8)[int(c.table[i, 0]), 1, 0, 0] = every[i * d:(i + 1) * d]
    c.scales.fill_(0.25)
    c.numbers()
    out, _ = c.run()
    for i in range(n):
        want = c.v[int(c.table[i, 0]), 0, 0].to(c.dt).to(DEV)
        assert torch.equal(out[i], want.expand(3, d))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,lens", [([1, 20], [70, 50]), ([40], [150]), ([260], [333])])
def test_what_is_not_visible_is_not_used(new, lens, code):
    """NaN codes and scales behind a request's last token and in blocks of nobody, NaN scales of the
    blocks of the table behind it."""
    announce(f"quant attention: not finite behind the end, {new} of {lens}, {code}")
    c = QuantCase(new=new, lens=lens, code=code, n_kv=1)
    want = c.want()
    raw = c.codes.view(torch.int8)
    for r, n in enumerate(lens):
        raw[c.table[r, (n - 1) // 16], :, n % 16 or 16:] = 0x7F
    used = set(c.table[c.table >= 0].tolist())
    idle = [b for b in range(raw.shape[0]) if b not in used]
    raw[idle], c.scales[idle] = 0x7F, float("nan")
    c.table = torch.cat([c.table, torch.full((len(lens), 3), idle[0], dtype=torch.int32)], 1)
    out, lse = c.run()
    c.want = lambda: want
    c.check(out, lse)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("new,lens,at", [([100], [230], 180), ([6], [300], 297), ([3, 90], [80, 90], 40),
                                         ([5], [6000], 5998), ([270], [400], 250), ([1100], [1100], 700)])
@pytest.mark.parametrize("half", [0, 1])
def test_nan_codes_reach_only_rows_that_see_them(new, lens, at, dtype, d, half):
    announce(f"quant attention: a NaN code at {at} of {lens}, {dtype}, half {half}")
    c = QuantCase(new=new, lens=lens, dtype=dtype, d=d, n_kv=1, code="e4m3")
    r = len(new) - 1
    first = lens[r] - new[r]
    sees = [t for t in range(sum(new)) if t >= sum(new[:-1]) and first + t - sum(new[:-1]) >= at]
    rest = [t for t in range(sum(new)) if t not in sees]
    want = c.want()
    block, row = c.token(r, at)
    c.codes.view(torch.int8)[block, half, row, 0, 11] = -1 if half else 0x7F
    out, lse = c.run()
    assert sees and rest and torch.isnan(out[sees].float()).all()
    c.want = lambda: want
    c.check(out, lse, rows=rest)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,lens,page", [([100], [230], 10), ([6], [130], 8), ([270], [400], 16)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("half", [0, 1])
def test_scales_that_are_not_finite(new, lens, page, value, half, code):
    """They reach the rows that see a token of their page, and no others."""
    announce(f"quant attention: scale {value} of page {page} of {lens}, half {half}")
    c = QuantCase(new=new, lens=lens, n_kv=1, code=code)
    want = c.want()
    c.scales[int(c.table[0, page]), half, 0] = value
    out, lse = c.run()
    rest = [t for t in range(new[0]) if lens[0] - new[0] + t < 16 * page]
    sees = [t for t in range(new[0]) if t not in rest]
    assert sees and not torch.isfinite(out[sees].float()).all(2).any()
    c.want = lambda: want
    if rest:
        c.check(out, lse, rows=rest)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("half,head", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("what", ["code", "scale"])
def test_nan_of_one_head(what, half, head, dtype, d):
    """It reaches the rows of its head that see it: not the other head's, nor rows before."""
    announce(f"quant attention: a NaN {what} of head {head}, half {half}, {dtype}")
    for new, lens, at in (([4], [300], 298), ([4, 2], [80, 5000], 4999), ([3], [50], 48)):
        c = QuantCase(new=new, lens=lens, dtype=dtype, d=d, n_kv=2, G=2, code="e4m3")
        want = c.want()
        r = len(new) - 1
        block, row = c.token(r, at)
        if what == "code":
            c.codes.view(torch.int8)[block, half, row, head, 5] = 0x7F
        else:
            c.scales[block, half, head] = float("nan")
            at = at // 16 * 16
        out, lse = c.run()
        q0, q1 = int(c.qs[r]), int(c.qs[r + 1])
        sees = [q0 + i for i in range(q1 - q0) if lens[r] - new[r] + i >= at]
        heads = slice(2 * head, 2 * head + 2)
        assert sees and torch.isnan(out[sees][:, heads].float()).all()
        out[sees, heads] = torch.tensor(want[0][sees, heads], dtype=c.dt, device=DEV)
        lse[sees, heads] = torch.tensor(want[1][sees, heads], dtype=torch.float32, device=DEV)
        c.want = lambda: want
        c.check(out, lse)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("n_kv", [1, 2])
@pytest.mark.parametrize("new,lens", [([1, 3], [300, 200]), ([70], [300]), ([4], [5000]), ([280], [400])])
def test_pages_without_a_block_are_masked(new, lens, code, n_kv):
    announce(f"quant attention: blocks outside the pool, {new} of {lens}")
    c = QuantCase(new=new, lens=lens, n_kv=n_kv, spare=0, code=code)
    c.codes.view(torch.int8)[0] = 0x7F if code == "e4m3" else 99       # (block 0, read in their place)
    c.table[c.table == 0] = -1
    c.numbers()
    c.k, c.v = c.k.nan_to_num(), c.v.nan_to_num()
    nb = c.codes.shape[0]
    c.table[0, 1:8:2] = torch.tensor([-1, nb, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64).int()
    c.table[0, 10] = nb + 5
    c.check(*c.run())


def test_no_visible_page_at_all():
    announce("quant attention: every block outside the pool")
    for new, lens in (([2], [40]), ([50], [90]), ([260], [300])):
        c = QuantCase(new=new, lens=lens, n_kv=1)
        c.table.fill_(-1)
        out, lse = c.run()
        assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("new,lens", [([3, 1], [700, 90]), ([150], [400])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scales_far_apart(new, lens, dtype):
    """Pages of V of 2^-20 to 2^20 times the others (fp16: 2^-10 to 2^10), pages of zeros under the
    least scale."""
    announce(f"quant attention: scales far apart, {new} of {lens}, {dtype}")
    c = QuantCase(new=new, lens=lens, n_kv=2, dtype=dtype)
    far = 20 if dtype == "bf16" else 10
    g = torch.Generator().manual_seed(3)
    c.scales[:, 1] *= torch.exp2(torch.randint(-far, far + 1, c.scales[:, 1].shape, generator=g).float())
    c.scales[:, 1].clamp_(max=100.0)
    zero = [int(c.table[r, 2]) for r in range(len(new))]
    c.codes[zero, 1], c.scales[zero, 1] = 0, 2.0 ** -64
    c.numbers()
    c.check(*c.run())


@pytest.mark.parametrize("exponent", [-55, -30, 30, 100])
def test_scales_of_any_size(exponent):
    announce(f"quant attention: V scales about 2^{exponent}")
    c = QuantCase(new=[5, 40], lens=[300, 90], n_kv=1)
    c.scales[:, 1] *= 2.0 ** exponent
    c.numbers()
    c.check(*c.run())


@pytest.mark.parametrize("new,lens", [([2], [9000]), ([60], [9000])])
def test_keys_far_down_an_fp16_row_count_together(new, lens):
    """One key with V = 0, and thousands of weight e^-17.5, below half of fp16's least step."""
    announce(f"quant attention: faint keys, {new}")
    c = QuantCase(new=new, lens=lens, dtype="fp16", n_kv=1, G=2)
    c.q.zero_(), c.codes[:, 0].zero_(), c.codes[:, 1].abs_()
    c.q[:, :, 0] = 16.0
    c.codes[:, 0, ..., 0] = -99
    c.scales[:, 0] = 0.125                         # 16 * 12.375 / sqrt(128) = 17.5
    block, row = c.token(0, 5)
    c.codes[block, 0, row, :, 0] = 0
    c.codes[block, 1, row] = 0
    c.numbers()
    c.check(*c.run())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new,lens", [([4], [300]), ([150], [400])])
def test_scores_far_from_zero(new, lens, dtype):
    """Scores of millions, of both signs: the key of the largest takes all (its lead over the next exceeds
    the rounding of both)."""
    announce(f"quant attention: scores of millions, {new}, {dtype}")
    for sign in (1, -1):
        c = QuantCase(new=new, lens=lens, n_kv=1, G=2, dtype=dtype)
        c.q.zero_(), c.codes[:, 0].zero_()
        c.q[:, :, 0] = 2.0 ** 14
        pos = torch.arange(lens[0])
        block, row = c.table[0, pos // 16].long(), pos % 16
        c.codes[block, 0, row, 0, 0] = (sign * (120 - (pos * 7) % 11)).to(torch.int8)
        c.scales[:, 0] = 16.0
        c.scale = 0.25
        c.numbers()
        out, _ = c.run()
        want, _, _, size, _ = c.want()
        tol = 2.02 * torch.finfo(c.dt).eps * (size + np.abs(want)) + 2.0 ** -24
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


def test_table_narrower_than_the_request():
    announce("quant attention: requests longer than the table's row")
    c = QuantCase(new=[20, 3], lens=[100, 90], n_kv=1)
    c.table = c.table[:, :4].contiguous()
    c.check(*c.run())


@pytest.mark.parametrize("code", CODES)
def test_strided_tensors(code):
    """q and out as slices of wider buffers, codes and scales with gaps, a table with gaps, lse
    transposed."""
    announce(f"quant attention: strides, {code}")
    c = QuantCase(new=[30, 2], lens=[80, 60], n_kv=2, G=3, pad=4, code=code)
    q, codes, scales, table, lens, qs = c.dev()
    T, H, d = q.shape
    wide = torch.zeros(T, 2 * H + 1, 160, dtype=c.dt, device=DEV)
    qv = wide[:, 1:H + 1, :128]
    qv.copy_(q)
    res = torch.full((H, T + 1, 144), 7.0, dtype=c.dt, device=DEV)
    out = res.transpose(0, 1)[:T, :, 16:]
    lse_t = torch.full((H, T), 7.0, device=DEV)
    wt = torch.full((2, 9), -9, dtype=torch.int32, device=DEV)
    tv = wt[:, 3:3 + table.shape[1]]
    tv.copy_(table)
    nb, _, page, n_kv, _ = codes.shape
    room = torch.full((nb, 2, n_kv + 1, page + 1, 144), 0x7F, dtype=torch.int8, device=DEV)
    cv = room.transpose(2, 3)[:, :, :page, 1:, 16:]
    cv.copy_(codes.view(torch.int8))
    sroom = torch.full((n_kv, nb, 5), float("nan"), device=DEV)
    sv = sroom[:, :, 1:3].permute(1, 2, 0)
    sv.copy_(scales)
    quant_chunk_attention(qv, cv.view(codes.dtype), sv, tv, lens, qs, out, lse=lse_t.T)
    c.check(out, lse_t.T)
    assert (res[:, :, :16] == 7.0).all() and (res[:, T] == 7.0).all()


def test_far_offsets():
    """Blocks past 2^32 bytes of the cache."""
    announce("quant attention: blocks past 2^32 bytes")
    c = QuantCase(new=[40, 2], lens=[100, 50], n_kv=8, G=1, spare=0)
    q, codes, scales, table, lens, qs = c.dev()
    nb = (1 << 32) // (2 * 16 * 8 * 128) + 2000
    big = torch.empty(nb, 2, 16, 8, 128, dtype=torch.int8, device=DEV)
    big_s = torch.empty(nb, 2, 8, device=DEV)
    n = codes.shape[0]
    big[nb - n:], big_s[nb - n:] = codes, scales
    far = torch.where(table >= 0, table + (nb - n), table)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    quant_chunk_attention(q, big, big_s, far, lens, qs, out, lse=lse)
    c.check(out, lse)


@pytest.mark.parametrize("new,lens", [([4, 1], [3000, 70]), ([150, 3], [500, 90])])
def test_out_may_be_q(new, lens):
    announce(f"quant attention: in place, {new} of {lens}")
    c = QuantCase(new=new, lens=lens, n_kv=2)
    apart, alse = c.run()
    q, *rest = c.dev()
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    quant_chunk_attention(q, *rest, q, lse=lse)
    assert torch.equal(q, apart) and torch.equal(lse, alse)


def test_repeats_bit_for_bit():
    announce("quant attention: the same bits every time")
    c = QuantCase(new=[4, 60, 1], lens=[3000, 500, 2500], n_kv=2)
    first = c.run()
    for _ in range(3):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("code", CODES)
def test_captured_with_other_lengths(code):
    """One captured call, replayed with other lengths, tables, scales and row counts, between eager
    calls of the same shapes."""
    announce(f"quant attention: captured and replayed, {code}")
    shapes = [([5, 40, 1], [900, 70, 333]), ([1, 1, 1], [900, 2000, 17]), ([0, 46, 0], [5, 46, 9]),
              ([46, 0, 0], [2000, 1, 1])]
    T, width = 46, 125
    q = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    raw = torch.zeros(200, 2, 16, 2, 128, dtype=torch.int8, device=DEV)
    codes, scales = raw.view(CODES[code]), torch.ones(200, 2, 2, device=DEV)
    table = torch.zeros(3, width, dtype=torch.int32, device=DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    qs = torch.zeros(4, dtype=torch.int32, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(T, 8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        quant_chunk_attention(q, codes, scales, table, lens, qs, out, lse=lse)
    for i in range(8):
        new, ln = shapes[i % 4]
        c = QuantCase(new=new, lens=ln, seed=i, n_kv=2, G=4, code=code)
        cq, cc, cs, ct, cl, cqs = c.dev()
        q[:cq.shape[0]] = cq
        raw[:cc.shape[0]], scales[:cc.shape[0]] = cc.view(torch.int8), cs
        table[:, :ct.shape[1]] = ct
        lens.copy_(cl), qs.copy_(cqs)
        out.fill_(7.0), lse.fill_(7.0)
        graph.replay()
        n = cq.shape[0]
        assert (out[n:] == 7.0).all()
        c.check(out[:n], lse[:n])
        eager, eager_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        quant_chunk_attention(q, codes, scales, table, lens, qs, eager, lse=eager_lse)
        assert torch.equal(eager, out) and torch.equal(eager_lse, lse)


def test_two_streams_at_once():
    announce("quant attention: two streams")
    cases = [QuantCase(new=[4, 1], lens=[6000, 3000], n_kv=2, seed=s) for s in (1, 2)]
    dev = [c.dev() for c in cases]
    outs = [torch.full_like(d[0], 7.0) for d in dev]
    lses = [torch.full(d[0].shape[:2], 7.0, device=DEV) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for s, d, o, e in zip(streams, dev, outs, lses):
            with torch.cuda.stream(s):
                quant_chunk_attention(*d, o, lse=e)
    torch.cuda.synchronize()
    for c, o, e in zip(cases, outs, lses):
        c.check(o, e)


def test_scratch_of_the_caller():
    announce("quant attention: scratch")
    c = QuantCase(new=[3], lens=[4000], n_kv=1)
    args = c.dev()
    q = args[0]
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    need = quant_scratch_bytes(*args, out)
    scratch = torch.full((need + 512,), 0xAB, dtype=torch.uint8, device=DEV)
    quant_chunk_attention(*args, out, lse=lse, scratch=scratch)
    c.check(out, lse)
    assert (scratch[need:] == 0xAB).all()
    with pytest.raises(ValueError, match="needed"):
        quant_chunk_attention(*args, out, scratch=scratch[:need - 1])
    with pytest.raises(ValueError, match="uint8"):
        quant_chunk_attention(*args, out, scratch=scratch.view(torch.int8))


def test_wrapper_refuses():
    announce("quant attention: refusals")
    c = QuantCase(new=[3], lens=[40])
    q, codes, scales, table, lens, qs = c.dev()
    good = dict(q=q, codes=codes, scales=scales, block_table=table, seq_lens=lens, query_start=qs,
                out=torch.empty_like(q))
    odd = torch.zeros(3, 8, 136, dtype=c.dt, device=DEV)
    for over in (dict(q=q.float()), dict(q=q.half()), dict(out=torch.empty_like(q).half()),
                 dict(codes=codes[:, :1]), dict(codes=codes.view(torch.uint8)), dict(codes=codes.half()),
                 dict(scales=scales.double()), dict(scales=scales[:, :, :1]), dict(scales=scales[:-1]),
                 dict(q=q[:, :7], out=good["out"][:, :7]), dict(out=good["out"][:2]),
                 dict(seq_lens=lens.long()), dict(query_start=qs[:1]), dict(block_table=table.long()),
                 dict(window=0), dict(scale=0.0), dict(scale=float("nan")),
                 dict(lse=torch.zeros(3, 8, dtype=torch.float64, device=DEV)),
                 dict(lse=torch.zeros(3, 7, device=DEV)),
                 dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
                 dict(out=good["out"][:1].expand(3, 8, 128)),
                 dict(lse=torch.zeros(3, 1, device=DEV).expand(3, 8)),
                 dict(codes=codes[..., :8, :, :]), dict(codes=codes[..., :64].repeat(1, 1, 1, 1, 3))):
        with pytest.raises(ValueError):
            quant_chunk_attention(**{**good, **over})
    with pytest.raises(AmassError):          # rows that 16-byte loads do not fit
        quant_chunk_attention(**{**good, "q": odd[:, :, 4:132]})
    room = torch.zeros(*codes.shape[:-1], 136, dtype=torch.int8, device=DEV)
    with pytest.raises(AmassError):
        quant_chunk_attention(**{**good, "codes": room[..., :128]})
    quant_chunk_attention(q[:0], codes, scales, table, lens, qs, q[:0])       # nothing to do
    quant_chunk_attention(q, codes, scales, table[:0], lens[:0], qs[:1], good["out"])
