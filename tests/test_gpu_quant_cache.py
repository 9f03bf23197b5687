"""The quantising write and the reading back on the GPU (amass_quant_write, amass_quant_read) against
the float64 oracle: codes and scales exactly, turned queries within the rounding of rope's test."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
import oracle.quant_cache as oq
from amass._hip import AmassError
from amass.attention import (quant_cache, quant_paged_read, quant_paged_write, rope_frequencies,
                             rope_paged_write, rope_table)
from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def num(codes):
    return codes.cpu().float().double().numpy()


def same(got, want):
    got, want = np.asarray(got), np.asarray(want)
    return np.array_equal(got, want, equal_nan=True)


class Step:
    """Tokens of some requests, at given first positions, in a pool of random contents."""

    def __init__(self, new, had, *, dtype="bf16", code="int8", n_kv=2, H=4, d=128, page=16, rot=0,
                 interleaved=False, pad=0, seed=0, loud=1.0):
        g = torch.Generator().manual_seed(seed)
        self.code, self.page, self.dt, self.rot = code, page, TYPES[dtype], rot
        self.interleaved = interleaved
        T = sum(new)
        pages = [-(-(h + n) // page) for h, n in zip(had, new)]
        nb = sum(pages) + 2
        perm = torch.randperm(nb, generator=g)
        at, slots, pos = 0, [], []
        for h, n, p in zip(had, new, pages):
            for i in range(h, h + n):
                slots.append(int(perm[at + i // page]) * page + i % page)
                pos.append(i)
            at += p
        self.T = T
        self.slots = torch.tensor(slots + [-1] * pad, dtype=torch.int64)
        self.pos = torch.tensor(pos + [0] * pad, dtype=torch.int32)
        self.q = torch.randn(T + pad, H, d, generator=g).to(self.dt)
        self.k, self.v = ((loud * torch.exp(torch.randn(T + pad, n_kv, 1, generator=g)) *
                           torch.randn(T + pad, n_kv, d, generator=g)).to(self.dt) for _ in range(2))
        x = (100.0 if code == "e4m3" else 40.0) * torch.randn(nb, 2, page, n_kv, d, generator=g)
        self.codes = (x.round().clamp(-127, 127) if code == "int8" else x.clamp(-448, 448)).to(CODES[code])
        # scales as writes leave them, some below what the new tokens need
        self.scales = torch.tensor([[[oq.step(float(m), code) for m in h] for h in b] for b in
                                    torch.exp(2.0 * torch.randn(nb, 2, n_kv, generator=g)).tolist()])
        self.table = rope_table(rot, max(pos + [0]) + 1, base=10000.0) if rot else None

    def dev(self):
        codes = self.codes.view(torch.int8).to(DEV).view(self.codes.dtype)
        return codes, self.scales.to(DEV)

    def run(self, codes, scales, q_out=None):
        kw = {}
        if self.rot:
            kw = dict(q=self.q.to(DEV), positions=self.pos.to(DEV), table=self.table.to(DEV), q_out=q_out,
                      layout="interleaved" if self.interleaved else "half")
        quant_paged_write(self.k.to(DEV), self.v.to(DEV), codes, scales, self.slots.to(DEV), **kw)
        torch.cuda.synchronize()

    def keys(self):
        """K as it enters the codes: turned in float64 by the table's angles, rounded twice."""
        if not self.rot:
            return self.k
        half = self.rot // 2
        ang = self.table[self.pos.long()].double().numpy()
        x = self.k.double().numpy().copy()
        i = np.arange(half)
        a, b = (2 * i, 2 * i + 1) if self.interleaved else (i, i + half)
        c, s = ang[:, None, :half], ang[:, None, half:]
        u, w = x[..., a], x[..., b]
        x[..., a], x[..., b] = u * c - w * s, w * c + u * s
        return torch.from_numpy(x).float().to(self.dt)

    def want(self):
        codes, scales = num(self.codes), self.scales.double().numpy()
        out = []
        for half, x in enumerate((self.keys(), self.v)):
            out.append(oq.write(codes[:, half], scales[:, half], x[:self.T].double().numpy(),
                                self.slots[:self.T].tolist(), self.page, self.code))
        return np.stack([o[0] for o in out], 1), np.stack([o[1] for o in out], 1)

    def check(self, codes, scales):
        wc, ws = self.want()
        assert same(scales.cpu().double().numpy(), ws)
        assert same(num(codes), wc)


STEPS = {
    "one token": dict(new=[1], had=[0]),
    "one token into a page": dict(new=[1], had=[7]),
    "last row of a page": dict(new=[1], had=[15]),
    "decode rows": dict(new=[1] * 9, had=[0, 1, 15, 16, 17, 31, 100, 64, 5]),
    "a whole page": dict(new=[16], had=[16]),
    "across pages": dict(new=[40], had=[9]),
    "prompts": dict(new=[33, 1, 70, 16], had=[0, 31, 5, 16], pad=3),
    "one kv head": dict(new=[20, 3], had=[3, 0], n_kv=1),
    "eleven kv heads": dict(new=[20, 3], had=[3, 0], n_kv=11),
    "d64": dict(new=[20, 3, 1], had=[3, 0, 40], d=64),
    "pages of 32": dict(new=[40, 3, 1], had=[3, 0, 40], page=32),
    "pages of 128, d64": dict(new=[200, 30, 1], had=[70, 0, 140], page=128, d=64),
    "pages of 1024": dict(new=[1500, 1], had=[100, 1023], page=1024, n_kv=1, d=64),
    "faint": dict(new=[20, 2], had=[0, 9], loud=2.0 ** -12),
    "loud": dict(new=[20, 2], had=[0, 9], loud=2.0 ** 6),
    "turned": dict(new=[20, 1, 3], had=[0, 99, 14], rot=128, pad=2),
    "turned in pairs": dict(new=[20, 1, 3], had=[0, 99, 14], rot=128, interleaved=True),
    "a quarter turned": dict(new=[20, 1, 3], had=[0, 99, 14], rot=32),
    "48 in pairs of 64": dict(new=[20, 1, 3], had=[0, 99, 14], rot=48, interleaved=True, d=64),
    "turned, pages of 64": dict(new=[150, 1], had=[30, 99], rot=64, page=64, d=64),
    "far positions": dict(new=[5, 1], had=[130000, 65536], rot=128),
    "hundreds of requests": dict(new=[1 + i % 3 for i in range(300)], had=[i % 37 for i in range(300)],
                                 n_kv=1, d=64),
}


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("dtype,code", [("bf16", "int8"), ("bf16", "e4m3"), ("fp16", "int8"),
                                        ("fp16", "e4m3")])
def test_write_is_the_formula(name, dtype, code):
    announce(f"quant write: {name}, {dtype} {code}")
    s = Step(dtype=dtype, code=code, **STEPS[name])
    codes, scales = s.dev()
    q = torch.full_like(s.q, 7.0).to(DEV)
    s.run(codes, scales, q)
    s.check(codes, scales)
    if s.rot:
        w, amp = rope_frequencies(s.rot, base=10000.0)
        want = ochunk.rotate(s.q.double().numpy(), s.pos.numpy(), w.numpy(), amp, s.interleaved)
        u = torch.finfo(s.dt).eps / 2
        x = s.q.double().numpy()
        # one rounding of the result, angles and products in fp32 (each within 2^-24 of |x| + |y|), and
        # the table's: cosines rounded to 2^-25
        tol = 1.01 * u * np.abs(want) + 2.0 ** -21 * np.abs(x).max() + 2.0 ** -25
        assert (np.abs(q.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("dtype,rot,interleaved", [("bf16", 128, False), ("bf16", 64, True), ("fp16", 128, True)])
def test_turned_keys_are_rounded_as_in_64_bits(dtype, rot, interleaved):
    """Millions of keys, of which some lie so near to a border of the 16-bit type that fp32 products round to
    the other side: all codes are those of the products in float64."""
    announce(f"quant write: keys at borders, {dtype}, {rot}")
    T, H = 4096, 8
    dt = TYPES[dtype]
    g = torch.Generator(DEV).manual_seed(9)
    k, v = (torch.randn(T, H, 128, generator=g, device=DEV).to(dt) for _ in range(2))
    k[:, 1] *= 2.0 ** -15                          # fp16: below its normal numbers
    pos = torch.randint(0, 60000, (T,), generator=g, device=DEV).int()
    table = rope_table(rot, 60000, base=500000.0, device=DEV)
    codes, scales = quant_cache(T // 16, 16, H, 128, device=DEV)
    quant_paged_write(k, v, codes, scales, torch.arange(T, device=DEV), positions=pos, table=table,
                      layout="interleaved" if interleaved else "half")
    c, s = table[pos.long()].double()[:, None].chunk(2, -1)
    x = k.double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else x[..., :rot].chunk(2, -1)
    u, w = a * c - b * s, b * c + a * s
    fast = a.float() * c.float() - b.float() * s.float()
    assert (u.float().to(dt) != fast.to(dt)).any()             # (fp32 alone would not do)
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    x = torch.cat([turned.float().to(dt).double(), x[..., rot:]], -1).view(T // 16, 16, H, 128)
    scale = scales[:, 0].double()[:, None, :, None]
    assert torch.equal(codes[:, 0].double(), (x / scale).round().clamp(-127, 127))


def test_a_page_token_by_token():
    """Sixteen steps of one token: every growth of a scale rounds the earlier codes again."""
    announce("quant write: a page token by token")
    for code in CODES:
        g = torch.Generator().manual_seed(5)
        k, v = (torch.exp(1.5 * torch.randn(16, 3, 1, generator=g)) * torch.randn(16, 3, 64, generator=g)
                for _ in range(2))
        k, v = k.bfloat16(), v.bfloat16()
        codes, scales = quant_cache(4, 16, 3, 64, dtype=CODES[code], device=DEV)
        wc = [np.zeros((4, 16, 3, 64)), np.zeros((4, 16, 3, 64))]
        ws = [np.ones((4, 3)), np.ones((4, 3))]
        grown = np.zeros(3)
        for i in range(16):
            slot = [2 * 16 + i]
            quant_paged_write(k[i:i + 1].to(DEV), v[i:i + 1].to(DEV), codes, scales,
                              torch.tensor(slot, device=DEV))
            for h, x in enumerate((k, v)):
                before = ws[h][2]
                wc[h], ws[h] = oq.write(wc[h], ws[h], x[i:i + 1].double().numpy(), slot, 16, code)
                grown += (ws[h][2] > before) * (h == 0)
            assert same(num(codes), np.stack(wc, 1)) and same(scales.cpu().double().numpy(), np.stack(ws, 1))
        # K: a rounding when the token enters and one with each growth, of half a step of at most the last
        # scale; e4m3: of 2^-4 of the number on entry, later none but below 2^-6 (steps of 2^-9)
        last = scales[2, 0].cpu().double().numpy()[None, :, None]
        got = num(codes)[2, 0] * last
        x, times = k.double().numpy(), (grown + 1)[None, :, None]
        tol = 0.5 * times * last if code == "int8" else 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * times * last
        assert (np.abs(got - x) <= tol).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_makes_nan_of_its_block_half_and_head(value, dtype, code):
    announce(f"quant write: {value}, {dtype} {code}")
    s = Step(new=[20, 1], had=[5, 9], dtype=dtype, code=code)
    s.k[3, 1, 77] = value
    s.v[20, 0, 0] = value
    codes, scales = s.dev()
    s.run(codes, scales)
    s.check(codes, scales)
    assert torch.isnan(scales).sum() == 2
    # it stays NaN for the next row, and ends with the block's first row
    b = int(s.slots[20]) // 16
    k = torch.ones(1, 2, 128, dtype=s.dt, device=DEV)
    for row, nan in ((10, True), (0, False)):
        quant_paged_write(k, k, codes, scales, torch.tensor([b * 16 + row], device=DEV))
        assert bool(torch.isnan(scales[b, 1, 0])) is nan
    assert num(codes[b, 1, 0, 0])[0] * float(scales[b, 1, 0]) == pytest.approx(1.0, rel=2 ** -7)


def test_extremes_of_the_types():
    """The largest and least numbers of each type, and blocks of zeros."""
    announce("quant write: extremes")
    for dtype, dt in TYPES.items():
        fi = torch.finfo(dt)
        tiny = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -24}[dtype]
        for code in CODES:
            for top in (fi.max, fi.max / 2, fi.tiny, tiny, 0.0, 1.0, 448.0, 127.0, 1.75, 1.7578125):
                s = Step(new=[16], had=[0], dtype=dtype, code=code, n_kv=1, d=64)
                s.k = (torch.linspace(-1, 1, 16 * 64, dtype=torch.float64) * top).view(16, 1, 64).to(dt)
                s.v = torch.zeros_like(s.k)
                s.v[0, 0, 0] = top
                codes, scales = s.dev()
                s.run(codes, scales)
                s.check(codes, scales)


def test_rows_that_are_passed_over():
    """Slots outside the cache and positions outside the table, in the middle of a run too."""
    announce("quant write: slots and positions outside")
    s = Step(new=[40], had=[0], rot=64, d=64)
    nb = s.codes.shape[0]
    first = int(s.slots[16])                       # (the second page keeps its run of rows 3 ..)
    for i, bad in ((16, -1), (17, nb * 16), (18, 2 ** 62)):
        s.slots[i] = bad
    s.pos[39], s.pos[38] = -1, 10 ** 6
    codes, scales = s.dev()
    q = torch.full_like(s.q, 7.0).to(DEV)
    s.run(codes, scales, q)
    assert (q[38:] == 7.0).all() and not (q[:38] == 7.0).all(2).any()
    s.slots[38:] = -1
    s.pos[38:] = 0
    s.check(codes, scales)
    assert first % 16 == 0


def test_halves_first_and_strides():
    announce("quant write: strides")
    for code in CODES:
        s = Step(new=[20, 1, 3], had=[3, 99, 14], code=code, rot=64, pad=2)
        codes, scales = s.dev()
        nb = codes.shape[0]
        room = torch.full((2, nb, 3, 17, 160), 99, dtype=torch.int8, device=DEV)
        cv = room.permute(0, 1, 3, 2, 4)[:, :, 1:, :2, 16:144]
        cv.copy_(codes.view(torch.int8).transpose(0, 1))
        sroom = torch.full((3, nb, 4), 5.0, device=DEV)
        sv = sroom[1:, :, ::2]
        sv.copy_(scales.transpose(0, 1))
        wide = torch.randn(s.q.shape[0], 4 + 2 + 2 + 1, 136, device=DEV).to(s.dt)
        q, k, v = (wide[:, a:b, 8:] for a, b in ((0, 4), (4, 6), (7, 9)))
        q.copy_(s.q), k.copy_(s.k), v.copy_(s.v)
        quant_paged_write(k, v, cv.view(CODES[code]), sv, s.slots.to(DEV), q=q, positions=s.pos.to(DEV),
                          table=s.table.to(DEV))
        s.check(cv.transpose(0, 1).contiguous().view(CODES[code]), sv.transpose(0, 1))
        assert (room[..., :16] == 99).all() and (room[..., 144:] == 99).all() and (room[:, :, 2] == 99).all()
        assert (room[:, :, :, 0] == 99).all() and (sroom[0] == 5.0).all() and (sroom[:, :, 1::2] == 5.0).all()


def test_queries_are_turned_as_rope_paged_write_turns_them():
    announce("quant write: queries beside rope_paged_write")
    for inter in (False, True):
        s = Step(new=[50, 1], had=[0, 999], rot=64, interleaved=inter)
        codes, scales = s.dev()
        mine = torch.zeros_like(s.q).to(DEV)
        s.run(codes, scales, mine)
        kv = torch.zeros(codes.shape[0], 2, 16, 2, 128, dtype=s.dt, device=DEV)
        ref = torch.zeros_like(mine)
        rope_paged_write(s.q.to(DEV), s.k.to(DEV), s.v.to(DEV), s.pos.to(DEV), s.table.to(DEV), kv,
                         s.slots.to(DEV), ref, layout="interleaved" if inter else "half")
        # both are within one rounding and the fp32 terms (test_write_is_the_formula) of the same formula;
        # which of two products is fused into the difference is not fixed, so they need not be equal
        u, x = torch.finfo(s.dt).eps / 2, float(s.q.abs().max())
        a, b = mine.double(), ref.double()
        assert ((a - b).abs() <= 2.02 * u * a.abs().maximum(b.abs()) + 2.0 ** -20 * x + 2.0 ** -24).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,n_kv,d", [(16, 2, 128), (16, 8, 64), (64, 3, 128), (1024, 1, 64), (32, 33, 64)])
def test_read_back(page, n_kv, d, dtype, code):
    announce(f"quant read: page {page}, {n_kv} heads of {d}, {dtype} {code}")
    s = Step(new=[1], had=[9 * page], dtype=dtype, code=code, n_kv=n_kv, d=d, page=page)
    codes, scales = s.dev()
    nb = codes.shape[0]
    want = (s.codes.float() * s.scales[:, :, None, :, None]).to(s.dt)     # (exact in fp32, rounded once)
    src = torch.tensor([3, 0, -1, nb, 7, 2 ** 31 - 1, 5], dtype=torch.int32, device=DEV)
    dst = torch.tensor([1, 4, 2, 0, -1, 5, 3], dtype=torch.int32, device=DEV)
    for first in (False, True):
        kv = torch.full((2, 6, page, n_kv, d) if first else (6, 2, page, n_kv, d), 7.0, dtype=s.dt, device=DEV)
        quant_paged_read(codes, scales, src, kv, dst)
        got = kv.transpose(0, 1) if first else kv
        ref = torch.full((6, 2, page, n_kv, d), 7.0, dtype=s.dt)
        for a, b in ((3, 1), (0, 4), (5, 3)):
            ref[b] = want[a]
        assert torch.equal(got.cpu(), ref)


def test_far_blocks():
    """Blocks past 2^32 bytes of the codes and of the 16-bit cache."""
    announce("quant write and read: blocks past 2^32 bytes")
    nb = (1 << 32) // (2 * 16 * 8 * 128) + 50
    codes = torch.zeros(nb, 2, 16, 8, 128, dtype=torch.int8, device=DEV)
    scales = torch.ones(nb, 2, 8, device=DEV)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 8, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    slots = torch.arange(3, device=DEV) + (nb - 3) * 16
    quant_paged_write(k, v, codes, scales, slots)
    small = torch.zeros(1, 2, 16, 8, 128, dtype=torch.int8, device=DEV), torch.ones(1, 2, 8, device=DEV)
    quant_paged_write(k, v, *small, torch.arange(3, device=DEV))
    assert torch.equal(codes[nb - 3], small[0][0]) and torch.equal(scales[nb - 3], small[1][0])
    assert not codes[:nb - 3].any() and not codes[nb - 2:].any()
    kv = torch.zeros(nb, 2, 16, 8, 128, dtype=torch.bfloat16, device=DEV)
    near = torch.zeros(1, 2, 16, 8, 128, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([nb - 3], dtype=torch.int32, device=DEV)
    quant_paged_read(codes, scales, at, kv, at + 1)
    quant_paged_read(*small, torch.zeros_like(at), near, torch.zeros_like(at))
    assert torch.equal(kv[nb - 2], near[0]) and not kv[nb - 3].any()


def test_captured_and_replayed():
    announce("quant write and read: captured")
    steps = [Step(new=n, had=h, rot=64, pad=40 - sum(n), seed=i, n_kv=2) for i, (n, h) in enumerate(
        [([40], [0]), ([1, 1, 1], [15, 16, 17]), ([20, 5], [3, 8]), ([0], [0])])]
    nb = 12
    codes, scales = quant_cache(nb, 16, 2, 128, device=DEV)
    q, k, v = (torch.zeros(40, h, 128, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    slots, pos = torch.full((40,), -1, device=DEV), torch.zeros(40, dtype=torch.int32, device=DEV)
    table = rope_table(64, 64, base=10000.0, device=DEV)
    src = torch.arange(nb, dtype=torch.int32, device=DEV)
    kv, qo = torch.zeros(nb, 2, 16, 2, 128, dtype=torch.bfloat16, device=DEV), torch.zeros_like(q)

    def call(codes, scales, kv, qo):
        quant_paged_write(k, v, codes, scales, slots, q=q, positions=pos, table=table, q_out=qo)
        quant_paged_read(codes, scales, src, kv, src)

    call(*(x.clone() for x in (codes, scales, kv, qo)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(codes, scales, kv, qo)
    for i in range(8):
        s = steps[i % 4]
        k.copy_(s.k), v.copy_(s.v), q.copy_(s.q), slots.copy_(s.slots), pos.copy_(s.pos)
        mine = [x.clone() for x in (codes, scales, kv, qo)]
        call(*mine)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(mine, (codes, scales, kv, qo)):
            assert torch.equal(a, b)


def test_wrappers_refuse():
    announce("quant write and read: refusals")
    s = Step(new=[3], had=[4], rot=64)
    codes, scales = s.dev()
    good = dict(k=s.k.to(DEV), v=s.v.to(DEV), codes=codes, scales=scales, slots=s.slots.to(DEV),
                q=s.q.to(DEV), positions=s.pos.to(DEV), table=s.table.to(DEV))
    k, q = good["k"], good["q"]
    for over in (dict(k=k.float()), dict(v=k.half()), dict(v=k[:2]), dict(slots=s.slots.int().to(DEV)),
                 dict(slots=good["slots"][:2]), dict(positions=None), dict(table=None),
                 dict(table=good["table"][:, :40]), dict(table=good["table"].double()),
                 dict(positions=good["positions"].long()), dict(q=q[:2]), dict(q=q[:, :0]),
                 dict(q=q.half()), dict(layout="other"), dict(codes=codes.view(torch.uint8)),
                 dict(codes=codes[:, :1]), dict(scales=scales[:, :, :1]), dict(scales=scales.half()),
                 dict(codes=codes[:1].expand(5, 2, 16, 2, 128)),
                 dict(scales=scales[..., :1].expand(*scales.shape)),
                 dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)),
                 dict(q_out=q[:1].expand(*q.shape)), dict(q=None, q_out=q)):
        with pytest.raises(ValueError):
            quant_paged_write(**{**good, **over})
    odd = torch.zeros(3, 2, 132, dtype=s.dt, device=DEV)[..., 4:]
    with pytest.raises(AmassError):
        quant_paged_write(**{**good, "k": odd})
    kv = torch.zeros(4, 2, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    for over in (dict(kv_cache=kv.float()), dict(kv_cache=kv[:, :1]), dict(kv_cache=kv[:, :, :8]),
                 dict(src=at.long()), dict(dst=at[:0]), dict(kv_cache=kv[:, :1].expand(4, 2, 16, 2, 128))):
        with pytest.raises(ValueError):
            quant_paged_read(**{**dict(codes=codes, scales=scales, src=at, kv_cache=kv, dst=at), **over})
    empty = k[:0]
    quant_paged_write(empty, empty, codes, scales, good["slots"][:0])         # nothing to do
    quant_paged_read(codes, scales, at[:0], kv, at[:0])
    for bad in (dict(dtype=torch.uint8), dict(page=8), dict(page=2048), dict(page=24), dict(d=96)):
        with pytest.raises(ValueError):
            quant_cache(**{**dict(num_blocks=2, page=16, n_kv=1, d=64), **bad})
