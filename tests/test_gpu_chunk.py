"""Chunk attention on the GPU (amass_chunk_attention) against the float64 oracle.

Tolerance, per element.  With u = eps / 2 of the element type: the weights are rounded once
(u of sum p |v| / l = `size`), so is the result (u of |out|).  Scores are sums of d products in
fp32 (off by at most d 2^-24 sum |q k| <= d 2^-24 `reach` once scaled), which moves a weight and its
sum by that much each; exponentials, sums and joins in fp32 add less than 2^-16 of `size` for
the lengths here (each at most 2^-24 per term).  fp16 adds its subnormal half steps: 2^-25 of
a weight (of weights that are 2^7 times the formula's, so of a sum that is at least 2^7) per
key seen, and of the result.  lse: the scores' and
the sums' error, and one rounding of its own size."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass.attention import chunk_scratch_bytes, paged_chunk_attention
from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


class Case:
    def __init__(self, new, lens, *, dtype="bf16", n_kv=2, G=4, d=128, page=16, pad=0, spare=3,
                 causal=True, window=None, scale=None, loud=1.0, halves_first=False, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.dt, self.page, self.causal, self.window = TYPES[dtype], page, causal, window
        self.scale = d ** -0.5 if scale is None else scale
        pages = [-(-max(a, 0) // page) for a in lens]
        nb = sum(pages) + spare
        perm = torch.randperm(nb, generator=g).int()
        self.table = torch.full((len(lens), max(pages + [1])), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(pages):
            self.table[r, :n] = perm[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.qs = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
        T, H = int(self.qs[-1]) + pad, n_kv * G
        self.q = (loud * torch.randn(T, H, d, generator=g)).to(self.dt)
        self.k = torch.randn(nb, page, n_kv, d, generator=g).to(self.dt)
        self.v = torch.randn(nb, page, n_kv, d, generator=g).to(self.dt)
        self.halves_first = halves_first

    def dev(self):
        kv = torch.stack([self.k, self.v], 0 if self.halves_first else 1).to(DEV)
        return self.q.to(DEV), kv, self.table.to(DEV), self.lens.to(DEV), self.qs.to(DEV)

    def run(self, out=None, lse=None, **kw):
        q, kv, table, lens, qs = self.dev()
        out = torch.full_like(q, 7.0) if out is None else out
        lse = torch.full(q.shape[:2], 7.0, device=DEV) if lse is None else lse
        paged_chunk_attention(q, kv, table, lens, qs, out, scale=self.scale, causal=self.causal,
                              window=self.window, lse=lse, **kw)
        torch.cuda.synchronize()
        return out, lse

    def want(self):
        return ochunk.attend(self.q.double().numpy(), self.k.double().numpy(),
                             self.v.double().numpy(), self.table.numpy(), self.lens.numpy(),
                             self.qs.numpy(), scale=self.scale, causal=self.causal,
                             window=self.window or 0, page=self.page)

    def check(self, out, lse, rows=None):
        """rows: the rows compared (all of the requests' by default)."""
        want, wlse, seen, size, reach = self.want()
        T = int(self.qs[-1])
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        assert (out[T:] == 7.0).all() and (lse[T:] == 7.0).all()       # rows of no request
        rows = np.arange(T) if rows is None else np.asarray(rows)
        d = self.q.shape[2]
        u = torch.finfo(self.dt).eps / 2
        moved = d * 2.0 ** -24 * reach
        tol = u * (1.01 * size + np.abs(want)) + (2.0 * moved[:, :, None] + 2.0 ** -16) * size
        if self.dt == torch.float16:
            vmax = float(self.v.abs().max())
            tol += 2.0 ** -25 + 2.0 ** -32 * seen[:, None, None] * vmax
        err = np.abs(out - want)
        bad = ~(err <= tol)
        assert not bad[rows].any(), (np.argwhere(bad[rows])[:4], err[rows].max())
        empty = np.isneginf(wlse)
        assert np.array_equal(np.isneginf(lse[rows]), empty[rows])
        fine = ~empty
        fine[T:] = False
        ltol = moved + 2.0 ** -16 + 2.0 ** -22 * np.abs(np.where(fine, wlse, 0.0))
        lerr = np.abs(np.where(fine, lse - np.where(fine, wlse, 0.0), 0.0))
        assert (lerr <= ltol)[rows].all(), lerr[rows].max()


CASES = {
    # the few-row layout: one wave's rows, waves over the keys
    "one token": dict(new=[1], lens=[1]),
    "one token, 4 keys": dict(new=[1], lens=[4], G=1, n_kv=1),
    "decode rows": dict(new=[1, 1, 1], lens=[17, 300, 64]),
    "drafts": dict(new=[5, 2, 8], lens=[1000, 40, 129]),
    "drafts fp16 d64": dict(new=[5, 2, 7], lens=[1000, 40, 129], dtype="fp16", d=64),
    "one long row, split": dict(new=[1], lens=[9000], n_kv=1, G=8),
    "two long drafts, split": dict(new=[3, 4], lens=[5001, 7777], n_kv=1, dtype="fp16"),
    # the shared-tile layout
    "prompt": dict(new=[200], lens=[200]),
    "prompt of 64": dict(new=[64], lens=[64], G=1),
    "prompt d64 fp16": dict(new=[333], lens=[333], d=64, dtype="fp16", n_kv=1),
    "prompt d64 bf16": dict(new=[130], lens=[190], d=64, G=2),
    "chunk behind a context": dict(new=[70], lens=[1500]),
    "chunk, keys split": dict(new=[40], lens=[6000], n_kv=1),
    "prompts of many lengths": dict(new=[1, 90, 33, 16, 65, 2], lens=[1, 90, 100, 600, 65, 31]),
    "mixed with decode rows": dict(new=[1, 1, 150, 1], lens=[400, 17, 200, 1025], G=7, n_kv=1),
    "empty requests": dict(new=[0, 9, 0, 40, 0], lens=[33, 9, 0, 77, 5], pad=6),
    "many requests": dict(new=[1 + i % 3 for i in range(150)], lens=[3 + 5 * i for i in range(150)],
                          n_kv=1, G=2),
    "thousands of requests": dict(new=[1] * 3400, lens=[1 + i % 29 for i in range(3400)], n_kv=1,
                                  G=1),
    "thousands of requests d64": dict(new=[1] * 1800, lens=[1 + i % 29 for i in range(1800)],
                                      n_kv=1, G=2, d=64),
    "pages of 256": dict(new=[5, 200], lens=[700, 300], page=256, n_kv=1),
    "pages of 4096": dict(new=[2, 70, 1], lens=[5000, 90, 4097], page=4096, n_kv=1, d=64, G=3),
    # prompts of many row tiles
    "long prompt": dict(new=[300], lens=[300]),
    "long prompt, one head": dict(new=[1030], lens=[1030], G=1, n_kv=1),
    "long prompt d64 fp16": dict(new=[270], lens=[420], d=64, dtype="fp16", n_kv=1),
    "long prompt d64 bf16": dict(new=[520], lens=[520], d=64, G=2, n_kv=1),
    "long prompt fp16": dict(new=[257], lens=[600], dtype="fp16", n_kv=1),
    "long, keys split": dict(new=[260], lens=[4000], n_kv=1),
    "long ragged": dict(new=[700, 1, 33, 300], lens=[700, 500, 90, 1000], G=5, n_kv=1, pad=9),
    "long window": dict(new=[600], lens=[900], window=130, G=2, n_kv=1),
    "long window of one": dict(new=[300], lens=[390], window=1, n_kv=1),
    "long, not causal": dict(new=[300], lens=[470], causal=False, n_kv=1),
    "long, rows before position 0": dict(new=[400], lens=[130], n_kv=1),
    "long, pages of 64": dict(new=[290], lens=[777], page=64, n_kv=1, halves_first=True),
    "long, forty heads": dict(new=[30], lens=[150], G=40, n_kv=1),
    "long, peaked": dict(new=[300], lens=[500], loud=12.0, n_kv=1),
    "long, peaked fp16": dict(new=[300], lens=[500], loud=12.0, n_kv=1, dtype="fp16"),
    "long, a window beyond everything": dict(new=[400], lens=[130], n_kv=1, window=2 ** 31 - 1),
    "a window past 32 bits": dict(new=[3, 40], lens=[50, 30], window=2 ** 40),
    "long, very peaked": dict(new=[300], lens=[400], loud=60.0, n_kv=1),
    # shapes
    "five heads per kv head": dict(new=[61, 3], lens=[90, 50], G=5, n_kv=3),
    "forty heads per kv head": dict(new=[7], lens=[150], G=40, n_kv=1),
    "pages of 32": dict(new=[45, 4], lens=[145, 70], page=32),
    "pages of 128": dict(new=[45, 4], lens=[145, 300], page=128, halves_first=True),
    # masks
    "not causal": dict(new=[70, 4], lens=[100, 333], causal=False),
    "window": dict(new=[150, 2], lens=[400, 500], window=50),
    "window of one": dict(new=[40, 3], lens=[90, 70], window=1),
    "window without causal": dict(new=[60], lens=[200], window=33, causal=False),
    "window wider than all": dict(new=[33], lens=[60], window=10 ** 6),
    "rows before position 0": dict(new=[50, 12], lens=[20, 3]),
    "rows before position 0, not causal": dict(new=[50, 12], lens=[20, 3], causal=False),
    "no tokens at all": dict(new=[5, 4], lens=[0, 4]),
    # scores
    "peaked": dict(new=[80, 3], lens=[200, 100], loud=12.0),
    "flat": dict(new=[40], lens=[100], scale=1e-6),
    "scale above one": dict(new=[40], lens=[100], scale=2.5, loud=0.3),
}


@pytest.mark.parametrize("name", CASES)
def test_matches_float64(name):
    announce(f"chunk attention: {name}")
    c = Case(**CASES[name])
    c.check(*c.run())


@pytest.mark.parametrize("new,lens", [([1, 20], [70, 50]), ([40], [150]), ([260], [333])])
def test_what_is_not_visible_is_not_used(new, lens):
    """Infinities and NaN behind a request's last token, in blocks of nobody and in K of masked
    positions."""
    announce(f"chunk attention: not finite behind the end, {new} of {lens}")
    c = Case(new=new, lens=lens, n_kv=1)
    want = c.want()
    for r, n in enumerate(lens):
        last = c.table[r, (n - 1) // 16]
        c.k[last, n % 16 or 16:] = float("nan")
        c.v[last, n % 16 or 16:] = float("nan")
    used = set(c.table[c.table >= 0].tolist())
    for b in range(c.k.shape[0]):
        if b not in used:
            c.k[b], c.v[b] = float("inf"), float("nan")
    out, lse = c.run()
    c.want = lambda: want
    c.check(out, lse)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("new,lens,at", [([100], [230], 180), ([6], [300], 297),
                                         ([3, 90], [80, 90], 40), ([5], [6000], 5998),
                                         ([270], [400], 250), ([1100], [1100], 700)])
def test_not_finite_tokens_reach_only_rows_that_see_them(new, lens, at, dtype, d):
    """A token of the last request has infinities in V and NaN in K: earlier rows are as if it
    were not there, the rows that see it are not finite."""
    announce(f"chunk attention: not finite at {at} of {lens}, {dtype}")
    c = Case(new=new, lens=lens, dtype=dtype, d=d, n_kv=1)
    r = len(new) - 1
    first = lens[r] - new[r]
    sees = [t for t in range(sum(new)) if t >= sum(new[:-1]) and first + t - sum(new[:-1]) >= at]
    rest = [t for t in range(sum(new)) if t not in sees]
    want = c.want()
    b = c.table[r, at // 16]
    c.v[b, at % 16] = float("inf")
    c.k[b, at % 16] = float("nan")
    out, lse = c.run()
    assert sees and rest and not torch.isfinite(out[sees].float()).any()
    c.want = lambda: want
    c.check(out, lse, rows=rest)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("new,lens,at", [([100], [230], 180), ([6], [300], 297), ([5], [6000], 5998),
                                         ([300], [2500], 2300), ([1], [40], 39)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_one_channel_of_v_that_is_not_finite(new, lens, at, dtype, d, value):
    """It reaches that channel of the rows that see its token, and nothing else."""
    announce(f"chunk attention: {value} in a channel, {new} of {lens}, {dtype}")
    c = Case(new=new, lens=lens, n_kv=1, dtype=dtype, d=d)
    block, row = int(c.table[0, at // 16]), at % 16
    keep = c.v[block, row, 0, 37].clone()
    c.v[block, row, 0, 37] = value
    out, lse = c.run()
    sees = at - (lens[0] - new[0])                  # the first row that does
    c.v[block, row, 0, 37] = keep
    assert not torch.isfinite(out[sees:, :, 37].float()).any()
    out[sees:, :, 37] = torch.tensor(c.want()[0][sees:, :, 37], dtype=c.dt, device=DEV)
    c.check(out, lse)


@pytest.mark.parametrize("new,lens", [([3, 1], [70, 400]), ([500], [3000])])
def test_a_cache_of_nans(new, lens):
    announce(f"chunk attention: V of NaN, {new} of {lens}")
    c = Case(new=new, lens=lens, n_kv=1)
    c.v.fill_(float("nan"))
    out, lse = c.run()
    assert torch.isnan(out.float()).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("new,lens", [([1, 3], [300, 200]), ([70], [300]), ([4], [5000]),
                                      ([280], [400])])
def test_pages_without_a_block_are_masked(new, lens):
    announce(f"chunk attention: blocks outside the pool, {new} of {lens}")
    c = Case(new=new, lens=lens, n_kv=1, spare=0)
    nb = c.k.shape[0]
    for r, bad in ((0, [-1, nb, 2 ** 31 - 1, -2 ** 31]),):
        c.table[r, 1:8:2] = torch.tensor(bad, dtype=torch.int64).int()
        c.table[r, 10] = nb + 5
    c.check(*c.run())


def test_no_visible_page_at_all():
    announce("chunk attention: every block outside the pool")
    for new, lens in (([2], [40]), ([50], [90]), ([260], [300])):
        c = Case(new=new, lens=lens, n_kv=1)
        c.table.fill_(-1)
        out, lse = c.run()
        assert (out == 0).all() and torch.isneginf(lse).all()


def test_scores_of_minus_infinity():
    """Rows whose every score is -inf count as empty; one finite score is enough otherwise."""
    announce("chunk attention: scores of -inf")
    c = Case(new=[3, 40], lens=[40, 64], n_kv=1, G=1)
    c.q.abs_()
    c.k[c.table[0, :3].long()] = float("-inf")
    c.k[c.table[1, 0], 1:] = float("-inf")
    with np.errstate(invalid="ignore"):
        want = c.want()
    want[3][:], want[4][:] = np.nan_to_num(want[3]), np.where(np.isfinite(want[4]), want[4], 0.0)
    out, lse = c.run()
    assert (out[:3] == 0).all() and torch.isneginf(lse[:3]).all()
    g = c.table[1, :4].long()
    assert torch.isfinite(lse[3:]).all() and torch.isfinite(out[3:].float()).all() and len(g)
    c.want = lambda: want
    # `reach` of a row with infinite keys says nothing: its finite keys' does
    kk, qq = c.k[g].reshape(-1, 128)[:64].double(), c.q[3:, 0].double()
    fine = torch.isfinite(kk).all(1)
    want[4][3:, 0] = c.scale * (qq @ kk[fine].abs().T).max(1).values.numpy()
    c.check(out, lse)


def test_table_narrower_than_the_request():
    announce("chunk attention: requests longer than the table's row")
    c = Case(new=[20, 3], lens=[100, 90], n_kv=1)
    c.table = c.table[:, :4].contiguous()
    c.check(*c.run())


def test_strided_tensors():
    """q and out as slices of wider buffers, a table with gaps, lse transposed."""
    announce("chunk attention: strides")
    c = Case(new=[30, 2], lens=[80, 60], n_kv=2, G=3, pad=4)
    q, kv, table, lens, qs = c.dev()
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
    paged_chunk_attention(qv, kv, tv, lens, qs, out, lse=lse_t.T)
    c.check(out, lse_t.T)
    assert (res[:, :, :16] == 7.0).all() and (res[:, T] == 7.0).all()


def test_far_offsets():
    """Blocks past 2^32 bytes and 2^31 elements of the cache."""
    announce("chunk attention: blocks past 2^32 bytes")
    c = Case(new=[40, 2], lens=[100, 50], n_kv=8, G=1, spare=0)
    q, kv, table, lens, qs = c.dev()
    nb = (1 << 32) // (2 * 16 * 8 * 128 * 2) + 2000
    big = torch.empty(nb, 2, 16, 8, 128, dtype=c.dt, device=DEV)
    n = kv.shape[0]
    big[nb - n:] = kv
    far = torch.where(table >= 0, table + (nb - n), table)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    paged_chunk_attention(q, big, far, lens, qs, out, lse=lse)
    c.check(out, lse)


def test_same_rows_in_any_batch_are_near():
    """A request's rows alone, and in a batch that splits and lays them out differently."""
    announce("chunk attention: alone and in a batch")
    new, lens = [4, 60, 1], [3000, 500, 2500]
    both = Case(new=new, lens=lens, n_kv=1, seed=5)
    out, lse = both.run()
    both.check(out, lse)
    q, kv, table, ln, qs = both.dev()
    for r in range(3):
        a, b = int(qs[r]), int(qs[r + 1])
        o = torch.empty_like(q[a:b])
        paged_chunk_attention(q[a:b], kv, table[r:r + 1], ln[r:r + 1],
                              torch.tensor([0, b - a], dtype=torch.int32, device=DEV), o)
        both_full = torch.full_like(q, 7.0)
        both_full[:] = out
        both_full[a:b] = o
        both.check(both_full, lse)


@pytest.mark.parametrize("new,lens", [([2], [9000]), ([60], [9000])])
def test_keys_far_down_an_fp16_row_count_together(new, lens):
    """One key with V = 0, and thousands of weight e^-17.5, below half of fp16's least step."""
    announce(f"chunk attention: faint keys, {new}")
    c = Case(new=new, lens=lens, dtype="fp16", n_kv=1, G=2)
    c.q.zero_(), c.k.zero_(), c.v.abs_()
    c.q[:, :, 0] = 16.0
    c.k[..., 0] = -12.375                           # 16 * 12.375 / sqrt(128) = 17.5
    first = int(c.table[0, 0])
    c.k[first, 5, :, 0] = 0.0
    c.v[first, 5] = 0.0
    c.check(*c.run())


@pytest.mark.parametrize("new,lens", [([4, 1], [3000, 70]), ([150, 3], [500, 90])])
def test_out_may_be_q(new, lens):
    announce(f"chunk attention: in place, {new} of {lens}")
    c = Case(new=new, lens=lens, n_kv=2)
    apart, alse = c.run()
    q, kv, table, ln, qs = c.dev()
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    paged_chunk_attention(q, kv, table, ln, qs, q, lse=lse)
    assert torch.equal(q, apart) and torch.equal(lse, alse)


def want_on_gpu(c):
    """Case.want for batches that fill the chip: the same formulas in float64 on the GPU."""
    q, k, v = (x.double().to(DEV) for x in (c.q, c.k, c.v))
    T, H, d = q.shape
    n_kv, G = k.shape[2], H // k.shape[2]
    out, size = torch.full_like(q, float("nan")), torch.zeros_like(q)
    lse, reach = (torch.zeros(T, H, dtype=torch.float64, device=DEV) for _ in range(2))
    seen = torch.zeros(T, dtype=torch.int64, device=DEV)
    lse[int(c.qs[-1]):] = float("nan")
    for r, L in enumerate(c.lens.tolist()):
        a, b = int(c.qs[r]), int(c.qs[r + 1])
        n, block = b - a, c.table[r, :-(-L // c.page)].long().to(DEV)
        p, j = torch.arange(L - n, L, device=DEV), torch.arange(L, device=DEV)
        see = (j <= p[:, None]) & (j > p[:, None] - (c.window or 2 ** 40))
        seen[a:b] = see.sum(1)
        see = see.repeat_interleave(G, 0)
        for h in range(n_kv):
            kk, vv = (x[block, :, h].reshape(-1, d)[:L] for x in (k, v))
            heads = slice(h * G, (h + 1) * G)
            qq = q[a:b, heads].reshape(-1, d)
            s = (c.scale * (qq @ kk.T.contiguous())).masked_fill(~see, -float("inf"))
            m = s.amax(1, keepdim=True)
            e = (s - m).exp()
            l = e.sum(1, keepdim=True)
            out[a:b, heads] = (e @ vv / l).view(n, G, d)
            size[a:b, heads] = (e @ vv.abs() / l).view(n, G, d)
            lse[a:b, heads] = (m + l.log()).view(n, G)
            t = c.scale * (qq.abs() @ kk.abs().T.contiguous())
            reach[a:b, heads] = t.masked_fill(~see, 0.0).amax(1).view(n, G)
    return tuple(x.cpu().numpy() for x in (out, lse, seen, size, reach))


ROUNDS = {        # 64 row tiles of 8 kv heads fill the chip once
    "66 tiles": dict(new=[2100], lens=[2400]),
    "the rest is a request's": dict(new=[100, 1900, 150], lens=[1500, 2000, 3000]),
    "the rest is of two requests": dict(new=[1950, 90, 130], lens=[1950, 2500, 1300], pad=3),
    "two rounds, 70 requests": dict(new=[40] * 70, lens=[100 + 37 * (i % 23) for i in range(70)]),
    "a row far longer than its share": dict(new=[4, 1900, 200], lens=[9000, 1900, 300]),
    "window": dict(new=[1500, 900], lens=[1500, 2900], window=700),
    "fp16": dict(new=[1950, 300], lens=[1950, 2000], dtype="fp16"),
}


@pytest.mark.parametrize("name", ["small"] + list(ROUNDS))
def test_more_tiles_than_the_chip_takes(name):
    announce(f"chunk attention: {name}, more tiles than the chip takes at a time")
    if name == "small":                             # the reference here against the oracle
        c = Case(new=[20, 3], lens=[70, 33], window=40)
        for x, y in zip(want_on_gpu(c), c.want()):
            assert np.allclose(x, y, rtol=1e-11, atol=1e-12)
        return
    c = Case(**{**dict(n_kv=8, G=4), **ROUNDS[name]})
    c.want = lambda: want_on_gpu(c)
    c.check(*c.run())


def test_repeats_bit_for_bit():
    announce("chunk attention: the same bits every time")
    c = Case(new=[4, 60, 1], lens=[3000, 500, 2500], n_kv=2)
    first = c.run()
    for _ in range(3):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_captured_with_other_lengths():
    """One captured call, replayed with other lengths, tables and row counts, between eager
    calls of the same shapes."""
    announce("chunk attention: captured and replayed")
    shapes = [([5, 40, 1], [900, 70, 333]), ([1, 1, 1], [900, 2000, 17]), ([0, 46, 0], [5, 46, 9]),
              ([46, 0, 0], [2000, 1, 1])]
    T, width = 46, 125
    kw = dict(n_kv=2, G=4)
    q = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    kv = torch.zeros(200, 2, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(3, width, dtype=torch.int32, device=DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    qs = torch.zeros(4, dtype=torch.int32, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(T, 8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_chunk_attention(q, kv, table, lens, qs, out, lse=lse)
    for i in range(8):
        new, ln = shapes[i % 4]
        c = Case(new=new, lens=ln, seed=i, **kw)
        cq, ckv, ct, cl, cs = c.dev()
        q[:cq.shape[0]] = cq
        kv[:ckv.shape[0]] = ckv
        table[:, :ct.shape[1]] = ct
        lens.copy_(cl), qs.copy_(cs)
        out.fill_(7.0), lse.fill_(7.0)
        graph.replay()
        n = cq.shape[0]
        assert (out[n:] == 7.0).all()
        c.check(out[:n], lse[:n])
        eager, eager_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        paged_chunk_attention(q, kv, table, lens, qs, eager, lse=eager_lse)
        assert torch.equal(eager, out) and torch.equal(eager_lse, lse)


def test_captured_prompts_and_padding():
    """One captured call of 2200 rows: more tiles than the chip takes, then mostly rows of nobody, and
    other requests."""
    announce("chunk attention: captured, from full to mostly padding")
    T, kw = 2200, dict(n_kv=8, G=4)
    steps = [([2100, 0, 0], [2400, 1, 1]), ([40, 30, 10], [900, 3000, 77]),
             ([1, 1900, 299], [2500, 1900, 800]), ([0, 0, 0], [5, 6, 7])]
    q = torch.zeros(T, 32, 128, dtype=torch.bfloat16, device=DEV)
    kv = torch.zeros(400, 2, 16, 8, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(3, 200, dtype=torch.int32, device=DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    qs = torch.zeros(4, dtype=torch.int32, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(T, 32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_chunk_attention(q, kv, table, lens, qs, out, lse=lse)
    for i in range(8):
        new, ln = steps[i % 4]
        c = Case(new=new, lens=ln, pad=T - sum(new), seed=i, **kw)
        cq, ckv, ct, cl, cs = c.dev()
        q.copy_(cq), lens.copy_(cl), qs.copy_(cs)
        kv[:ckv.shape[0]] = ckv
        table[:, :ct.shape[1]] = ct
        out.fill_(7.0), lse.fill_(7.0)
        graph.replay()
        eager, eager_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        paged_chunk_attention(q, kv, table, lens, qs, eager, lse=eager_lse)
        assert torch.equal(eager, out) and torch.equal(eager_lse, lse)
        if i < 4 and sum(new):
            live = [r for r in range(3) if new[r]]
            c.lens, c.table = c.lens[live], c.table[live]
            c.qs = torch.tensor(np.concatenate([[0], np.cumsum([new[r] for r in live])]),
                                dtype=torch.int32)
            c.want = lambda c=c: want_on_gpu(c)
            c.check(out, lse)


def test_two_streams_at_once():
    announce("chunk attention: two streams")
    cases = [Case(new=[4, 1], lens=[6000, 3000], n_kv=2, seed=s) for s in (1, 2)]
    dev = [c.dev() for c in cases]
    outs = [torch.full_like(d[0], 7.0) for d in dev]
    lses = [torch.full(d[0].shape[:2], 7.0, device=DEV) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for s, d, o, e in zip(streams, dev, outs, lses):
            with torch.cuda.stream(s):
                paged_chunk_attention(*d, o, lse=e)
    torch.cuda.synchronize()
    for c, o, e in zip(cases, outs, lses):
        c.check(o, e)


def test_scratch_of_the_caller():
    announce("chunk attention: scratch")
    c = Case(new=[3], lens=[4000], n_kv=1)
    q, kv, table, lens, qs = c.dev()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    need = chunk_scratch_bytes(q, kv, table, lens, qs, out)
    scratch = torch.full((need + 512,), 0xAB, dtype=torch.uint8, device=DEV)
    paged_chunk_attention(q, kv, table, lens, qs, out, lse=lse, scratch=scratch)
    c.check(out, lse)
    assert (scratch[need:] == 0xAB).all()
    with pytest.raises(ValueError, match="needed"):
        paged_chunk_attention(q, kv, table, lens, qs, out, scratch=scratch[:need - 1])
    with pytest.raises(ValueError, match="uint8"):
        paged_chunk_attention(q, kv, table, lens, qs, out, scratch=scratch.view(torch.int8))


def test_wrapper_refuses():
    announce("chunk attention: refusals")
    c = Case(new=[3], lens=[40])
    q, kv, table, lens, qs = c.dev()
    good = dict(q=q, kv_cache=kv, block_table=table, seq_lens=lens, query_start=qs,
                out=torch.empty_like(q))
    odd = torch.zeros(3, 8, 136, dtype=c.dt, device=DEV)
    for over in (dict(q=q.float()), dict(q=q.half()), dict(out=torch.empty_like(q).half()),
                 dict(kv_cache=kv[:, :1]), dict(q=q[:, :7], out=good["out"][:, :7]),
                 dict(out=good["out"][:2]), dict(seq_lens=lens.long()), dict(query_start=qs[:1]),
                 dict(block_table=table.long()), dict(window=0), dict(window=-3),
                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                 dict(lse=torch.zeros(3, 8, dtype=torch.float64, device=DEV)),
                 dict(lse=torch.zeros(3, 7, device=DEV)),
                 dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
                 dict(out=good["out"][:1].expand(3, 8, 128)),
                 dict(out=good["out"][:, :1].expand(3, 8, 128)),
                 dict(lse=torch.zeros(3, 1, device=DEV).expand(3, 8))):
        with pytest.raises(ValueError):
            paged_chunk_attention(**{**good, **over})
    from amass._hip import AmassError
    with pytest.raises(AmassError):          # rows that 16-byte loads do not fit
        paged_chunk_attention(**{**good, "q": odd[:, :, 4:132]})
    paged_chunk_attention(q[:0], kv, table, lens, qs, q[:0])       # nothing to do
    paged_chunk_attention(q, kv, table[:0], lens[:0], qs[:1], good["out"])
