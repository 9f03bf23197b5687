"""Prompts, drafted tokens and decode steps over the 8-bit cache, as a serving program runs them: slots for
the step's tokens, the quantising rotary write, attention over the codes; then blocks read back to a 16-bit
cache, and this framework's decode and chunk attention over it."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass.attention import (dense_paged_decode, ensure_stage_b_buffers, extend_block_tables,
                             free_blocks, paged_chunk_attention, quant_cache, quant_chunk_attention,
                             quant_paged_read, quant_paged_write, release_blocks, rope_frequencies,
                             rope_table)
from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
N_KV, G = 2, 4
H = N_KV * G
U = 2.0 ** -8                                      # half a step of bf16
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Server:
    """R rows of requests over one layer's cache; the host keeps their turned keys and values in float64."""

    def __init__(self, R, nb, width, code, *, page=16, d=128, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.R, self.nb, self.page, self.d, self.code = R, nb, page, d, code
        self.codes, self.scales = quant_cache(nb, page, N_KV, d, dtype=CODES[code], device=DEV)
        # what an earlier program left in the memory
        self.codes.view(torch.int8).fill_(0x7F)
        self.scales.fill_(float("nan"))
        self.table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
        self.free, self.top = free_blocks(nb, DEV)
        self.angles = rope_table(d, 2048, device=DEV)
        self.w = rope_frequencies(d)[0].numpy()
        self.lens = np.zeros(R, np.int64)
        self.held = [np.zeros((0, 2, N_KV, d)) for _ in range(R)]
        self.steps = 0

    def write(self, new, pad=0):
        """Slots and the quantising write of a step; (q turned, lens, query_start)."""
        T, d = int(sum(new)) + pad, self.d
        self.lens += np.asarray(new)
        self.steps += 1
        qkv = torch.randn(T, H + 2 * N_KV, d, generator=self.gen)
        qkv[:, H:] *= torch.exp(torch.randn(T, 2 * N_KV, 1, generator=self.gen))
        qkv = qkv.to(torch.bfloat16)
        q, k, v = qkv.to(DEV).split([H, N_KV, N_KV], 1)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        qs = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)
        slots = torch.empty(T, dtype=torch.int64, device=DEV)
        pos = torch.empty(T, dtype=torch.int32, device=DEV)
        extend_block_tables(self.table, lens, qs, self.free, self.top, slots, pos, page=self.page,
                            num_blocks=self.nb)
        out_q = torch.zeros(T, H, d, dtype=torch.bfloat16, device=DEV)
        quant_paged_write(k, v, self.codes, self.scales, slots, q=q, positions=pos,
                          table=self.angles, q_out=out_q)
        at = 0
        for r, n in enumerate(new):
            rows = qkv[at:at + n].double().numpy()
            p = np.arange(self.lens[r] - n, self.lens[r])
            turned = ochunk.rotate(rows[:, H:H + N_KV], p, self.w, 1.0, False)
            self.held[r] = np.concatenate([self.held[r], np.stack([turned, rows[:, H + N_KV:]], 1)])
            at += n
        return out_q, lens, qs

    def numbers(self):
        """What the cache holds, float64 (NB, 2, page, n_kv, d), and its scales."""
        scales = self.scales.double().cpu().numpy()
        codes = self.codes.cpu().float().double().numpy()
        return np.nan_to_num(codes * scales[:, :, None, :, None]), scales

    def check_cache(self):
        """Every token's K and V, off by bf16's rounding of K, a rounding to a code on entry, and one with
        each growth of its scale: a write call makes one at most, of half a step of at most the last
        scale (e4m3: on entry 2^-4 of the number, later below 2^-6 of a scale only)."""
        x, scales = self.numbers()
        for r, want in enumerate(self.held):
            n = len(want)
            if not n:
                continue
            at = np.arange(n)
            block = self.table[r].cpu().numpy()[at // self.page]
            got, s = x[block, :, at % self.page], scales[block][..., None]
            assert np.isfinite(s).all()
            tol = U * np.abs(want)
            tol += 0.5 * self.steps * s if self.code == "int8" else \
                2.0 ** -4 * (1 + U) * np.abs(want) + 2.0 ** -10 * self.steps * s
            assert (np.abs(got - want) <= tol).all(), r

    def attend(self, q, lens, qs, **kw):
        out = torch.zeros_like(q)
        quant_chunk_attention(q, self.codes, self.scales, self.table, lens, qs, out, **kw)
        return out

    def check_attention(self, q, lens, qs, out):
        """Against the oracle on the numbers that the cache holds and the turned q: weights and results rounded
        once (U of size and of the value), scores summed in fp32 (d + 8 terms of `reach`), and 2^-16 of
        size for exponentials and sums."""
        x, _ = self.numbers()
        want, _, _, size, reach = ochunk.attend(
            q.double().cpu().numpy(), x[:, 0], x[:, 1], self.table.cpu().numpy(), lens.tolist(), qs.tolist(),
            scale=self.d ** -0.5, causal=True, window=0, page=self.page)
        n = int(qs[-1])
        moved = (self.d + 8) * 2.0 ** -24 * reach[:n, :, None]
        tol = U * (1.01 * size[:n] + np.abs(want[:n])) + (2.0 * moved + 2.0 ** -16) * size[:n]
        assert (np.abs(out[:n].double().cpu().numpy() - want[:n]) <= tol).all()
        assert (out[n:] == 0).all()
        return want[:n], size[:n], reach[:n]


@pytest.mark.parametrize("code,page,d", [("int8", 16, 128), ("e4m3", 16, 128), ("int8", 64, 64),
                                         ("e4m3", 32, 64)])
def test_prompts_drafts_and_decode_steps(code, page, d):
    announce(f"a server's steps over the 8-bit cache: {code}, pages of {page}, heads of {d}")
    s = Server(R=4, nb=96 * 16 // page + 8, width=640 // page, code=code, page=page, d=d)
    steps = [([70, 0, 33, 5], 3), ([1, 90, 1, 1], 0), ([5, 40, 1, 3], 7), ([1, 1, 1, 1], 0)]
    for new, pad in steps:
        q, lens, qs = s.write(new, pad)
        s.check_cache()
        out = s.attend(q, lens, qs)
        want, size, reach = s.check_attention(q, lens, qs, out)
    # the pages of all requests to a 16-bit cache, under other blocks: rounding its numbers to bf16 moves a
    # score by U reach at most, so a weight and its sum by e^(U reach) each, and V by U
    pages = [-(-int(n) // page) for n in s.lens]
    src = torch.cat([s.table[r, :n] for r, n in enumerate(pages)])
    dst = torch.arange(len(src), dtype=torch.int32, device=DEV).flip(0)
    kv = torch.full((len(src), 2, page, N_KV, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    quant_paged_read(s.codes, s.scales, src, kv, dst.contiguous())
    table = torch.full_like(s.table, -1)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = dst[at:at + n]
        at += n
    other = torch.zeros_like(q)
    paged_chunk_attention(q, kv, table, lens, qs, other)
    tol = (np.exp(2.02 * U * reach)[:, :, None] - 1.0 + 4.0 * U) * size + 2.0 * U * np.abs(want)
    assert (np.abs(other.double().cpu().numpy() - want) <= tol).all()
    if page == 16 and d == 128:
        st = type("S", (), dict(max_reqs=4, n_kv=N_KV, G=G, D=d))()
        ensure_stage_b_buffers(st, DEV)
        dec = torch.zeros_like(q)
        dense_paged_decode(q, kv, table, lens, st, dec, scale=d ** -0.5)
        assert (np.abs(dec.double().cpu().numpy() - want) <= tol).all()
    # a finished request's blocks serve the next one, whose scales start anew
    before = set(s.table[1, :pages[1]].tolist())
    done = torch.tensor([False, True, False, False], device=DEV)
    release_blocks(s.table, lens, done, s.free, s.top, page=page, num_blocks=s.nb)
    s.lens[1], s.held[1] = 0, s.held[1][:0]
    q, lens, qs = s.write([1, 60, 1, 1])
    assert set(s.table[1, :-(-60 // page)].tolist()) <= before
    s.check_cache()
    s.check_attention(q, lens, qs, s.attend(q, lens, qs))


def test_drafts_that_are_taken_back():
    """Tokens rejected and written again in the middle of a page: what stays is within the steps that the
    scales so far have."""
    announce("drafts taken back over the 8-bit cache")
    s = Server(R=2, nb=16, width=8, code="int8", seed=3)
    s.write([13, 30])
    for keep in (2, 0, 3, 1):
        s.write([5, 5])                            # five drafted tokens, of which `keep` stay
        s.lens -= 5 - keep
        s.held = [h[:n] for h, n in zip(s.held, s.lens)]
        # (blocks of pages that hold no token any more go back by hand)
        for r, n in enumerate(s.lens):
            last = -(-int(n) // 16)
            gone = s.table[r, last:][s.table[r, last:] >= 0]
            t = int(s.top[0])
            s.free[t:t + len(gone)] = gone.flip(0)
            s.top[0] += len(gone)
            s.table[r, last:] = -1
    q, lens, qs = s.write([1, 1])
    s.check_cache()
    s.check_attention(q, lens, qs, s.attend(q, lens, qs))


@pytest.mark.parametrize("code", CODES)
def test_captured_decode_step(code):
    """A whole step in one graph (slots, quantising write, attention, reading back), replayed over page
    borders, every replay against the eager calls."""
    announce(f"a server's decode step over the 8-bit cache: captured, 20 replays, {code}")
    R, nb = 3, 32
    s = Server(R=R, nb=nb, width=16, code=code, seed=4)
    q, lens, qs = s.write([14, 30, 1])
    qkv = torch.zeros(R, H + 2 * N_KV, 128, dtype=torch.bfloat16, device=DEV)
    qs = torch.arange(R + 1, dtype=torch.int32, device=DEV)
    slots = torch.zeros(R, dtype=torch.int64, device=DEV)
    pos = torch.zeros(R, dtype=torch.int32, device=DEV)
    ids = torch.arange(nb, dtype=torch.int32, device=DEV)
    qo, out = (torch.zeros(R, H, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kv = torch.zeros(nb, 2, 16, N_KV, 128, dtype=torch.bfloat16, device=DEV)

    def step(table, lens, top, codes, scales, qo, out, kv):
        q, k, v = qkv.split([H, N_KV, N_KV], 1)
        lens += 1
        extend_block_tables(table, lens, qs, s.free, top, slots, pos, page=16, num_blocks=nb)
        quant_paged_write(k, v, codes, scales, slots, q=q, positions=pos, table=s.angles, q_out=qo)
        quant_chunk_attention(qo, codes, scales, table, lens, qs, out)
        quant_paged_read(codes, scales, ids, kv, ids)

    mine = (s.table, lens, s.top, s.codes, s.scales, qo, out, kv)
    other = [x.clone() for x in mine]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*mine)
    for i in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=s.gen))
        graph.replay()
        step(*other)
        torch.cuda.synchronize()
        for a, b in zip(mine, other):
            raw = torch.int8 if a.element_size() == 1 else torch.int16 if a.element_size() == 2 else torch.int32
            assert torch.equal(a.view(raw), b.view(raw)), i
        assert torch.isfinite(out.float()).all(), i
    assert lens.tolist() == [34, 50, 21]


def test_on_another_stream():
    """The whole sequence on a stream of its own, while another one runs another server."""
    announce("two servers over 8-bit caches on two streams")
    servers = [Server(R=3, nb=64, width=24, code=c, seed=i) for i, c in enumerate(CODES)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in servers]
    last = [None, None]
    for new in ([50, 3, 17], [1, 40, 1], [4, 1, 2]):
        for i, (s, stream) in enumerate(zip(servers, streams)):
            with torch.cuda.stream(stream):
                q, lens, qs = s.write(new)
                last[i] = (q, lens, qs, s.attend(q, lens, qs))
    torch.cuda.synchronize()
    for s, x in zip(servers, last):
        s.check_cache()
        s.check_attention(*x)
