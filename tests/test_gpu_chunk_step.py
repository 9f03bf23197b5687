"""Prompts, drafted tokens and decode steps through the operators together, as a serving program
runs them: slots for the step's tokens, rotary positions and the cache write, chunk attention;
then this framework's decode over the cache that they filled."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
import oracle.decode as odec
import oracle.select as osel
from amass.attention import (ResidentVSource, dense_paged_decode, ensure_stage_b_buffers,
                             extend_block_tables, free_blocks, paged_chunk_attention,
                             release_blocks, rope_frequencies, rope_paged_write, rope_table)
from amass.selection import QuadState, derive_page_params
from amass.selection.quad_build import quad_build_bulk, quad_build_delta
from amass.selection.quad_score import select_then_attend
from helpers import announce, npf, npi

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE, N_KV, G, D = 16, 2, 4, 128
H = N_KV * G


class Server:
    """R rows of requests over one layer's cache; the host keeps every request's turned keys,
    values and queries in float64."""

    def __init__(self, R, nb, width, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.R, self.nb = R, nb
        self.kv = torch.full((nb, 2, PAGE, N_KV, D), float("nan"), dtype=torch.bfloat16, device=DEV)
        self.table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
        self.free, self.top = free_blocks(nb, DEV)
        self.angles = rope_table(D, 2048, device=DEV)
        self.w = rope_frequencies(D)[0].numpy()
        self.lens = np.zeros(R, np.int64)
        self.keys = [np.zeros((0, N_KV, D)) for _ in range(R)]
        self.values = [np.zeros((0, N_KV, D)) for _ in range(R)]

    def write(self, new, pad=0):
        """Slots, rotary positions and the cache write of a step; (q turned, lens, query_start)."""
        T = int(sum(new)) + pad
        self.lens += np.asarray(new)
        qkv = torch.randn(T, H + 2 * N_KV, D, generator=self.gen).to(torch.bfloat16)
        dev = qkv.to(DEV)
        q, k, v = dev.split([H, N_KV, N_KV], 1)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        qs = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)
        slots = torch.empty(T, dtype=torch.int64, device=DEV)
        pos = torch.empty(T, dtype=torch.int32, device=DEV)
        extend_block_tables(self.table, lens, qs, self.free, self.top, slots, pos, page=PAGE,
                            num_blocks=self.nb)
        out_q = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
        rope_paged_write(q, k, v, pos, self.angles, self.kv, slots, out_q)
        at = 0
        for r, n in enumerate(new):
            p = np.arange(self.lens[r] - n, self.lens[r])
            rows = qkv[at:at + n].double().numpy()
            turned = ochunk.rotate(rows[:, H:H + N_KV], p, self.w, 1.0, False)
            self.keys[r] = np.concatenate([self.keys[r], turned])
            self.values[r] = np.concatenate([self.values[r], rows[:, H + N_KV:]])
            at += n
        self.q64 = qkv.double().numpy()[:, :H]
        return out_q, lens, qs

    def attention(self, new):
        """The step's attention in float64 from the host's own keys and values."""
        out, at = [], 0
        for r, n in enumerate(new):
            if not n:
                continue
            length = int(self.lens[r])
            q = ochunk.rotate(self.q64[at:at + n], np.arange(length - n, length), self.w, 1.0, False)
            o, *_ = ochunk.attend(q, self.keys[r][None], self.values[r][None],
                                  np.zeros((1, 1), np.int64), [length], [0, n], scale=D ** -0.5,
                                  causal=True, window=0, page=length)
            out.append(o)
            at += n
        return np.concatenate(out)


def _near(got, want):
    """q and k were each rounded to bf16 (2^-8 of a channel): a score of N(0, 1) channels is off
    by 2^-8 sum |q k| d^-1/2 twice, at most 2^-7 d^1/2 2.5 = 0.22 for |q k| means up to 2.5 -- in
    the worst case of one sign; weights move by e^(2 * 0.22) - 1 = 0.56 at the very most, and V
    and out by a rounding.  The errors' signs are random, so the mean over an output must be
    far below that: d^1/2 times smaller (0.05), with the roundings 0.06."""
    got = got.double().cpu().numpy()
    scale = np.abs(want).mean()
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= 0.56 * np.abs(want).max() + 2.0 ** -7
    assert np.abs(got - want).mean() <= 0.06 * scale


def test_prompts_drafts_and_decode_steps():
    announce("a server's steps: prompts, chunks, drafts, decode, release")
    s = Server(R=4, nb=96, width=40)
    steps = [([70, 0, 33, 5], 3), ([1, 90, 1, 1], 0), ([5, 40, 1, 3], 7), ([1, 1, 1, 1], 0)]
    for new, pad in steps:
        q, lens, qs = s.write(new, pad)
        out = torch.zeros_like(q)
        paged_chunk_attention(q, s.kv, s.table, lens, qs, out)
        _near(out[:sum(new)], s.attention(new))
        assert (out[sum(new):] == 0).all()
        used = int(sum(-(-s.lens // PAGE)))
        assert s.top.tolist() == [s.nb - used, 0, 0]
    # the last step had one token per request: the decode over the same cache agrees
    st = type("S", (), dict(max_reqs=4, n_kv=N_KV, G=G, D=D))()
    ensure_stage_b_buffers(st, DEV)
    dec = torch.zeros_like(q)
    dense_paged_decode(q, s.kv, s.table, lens, st, dec, scale=D ** -0.5)
    a, b = out.float(), dec.float()
    # both round their weights and results once: 2 (u + u) of values up to the rows' largest
    assert ((a - b).abs() <= 4 * 2.0 ** -8 * a.abs().amax(-1, keepdim=True) + 2.0 ** -8).all()
    # a finished request's blocks serve the next one
    before = set(s.table[1, :-(-int(s.lens[1]) // PAGE)].tolist())
    done = torch.tensor([False, True, False, False], device=DEV)
    release_blocks(s.table, lens, done, s.free, s.top, page=PAGE, num_blocks=s.nb)
    s.lens[1], s.keys[1], s.values[1] = 0, s.keys[1][:0], s.values[1][:0]
    new = [1, 60, 1, 1]
    q, lens, qs = s.write(new)
    assert set(s.table[1, :4].tolist()) <= before
    out = torch.zeros_like(q)
    paged_chunk_attention(q, s.kv, s.table, lens, qs, out)
    _near(out, s.attention(new))


def test_captured_decode_step():
    """A whole step in one graph (slots, rotary write, attention), replayed over page borders,
    every replay against the eager calls."""
    announce("a server's decode step: captured, 20 replays")
    R, nb = 3, 32
    s = Server(R=R, nb=nb, width=16, seed=4)
    q, lens, qs = s.write([14, 30, 1])
    qkv = torch.zeros(R, H + 2 * N_KV, D, dtype=torch.bfloat16, device=DEV)
    qs = torch.arange(R + 1, dtype=torch.int32, device=DEV)
    slots = torch.zeros(R, dtype=torch.int64, device=DEV)
    pos = torch.zeros(R, dtype=torch.int32, device=DEV)
    qo, out = (torch.zeros(R, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def step(table, lens, top, kv, qo, out):
        q, k, v = qkv.split([H, N_KV, N_KV], 1)
        lens += 1
        extend_block_tables(table, lens, qs, s.free, top, slots, pos, page=PAGE, num_blocks=nb)
        rope_paged_write(q, k, v, pos, s.angles, kv, slots, qo)
        paged_chunk_attention(qo, kv, table, lens, qs, out)

    other = [x.clone() for x in (s.table, lens, s.top, s.kv, qo, out)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s.table, lens, s.top, s.kv, qo, out)
    for i in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=s.gen))
        graph.replay()
        step(*other)
        assert torch.equal(lens, other[1]) and torch.equal(s.table, other[0]), i
        assert torch.equal(out, other[5]) and torch.isfinite(out.float()).all(), i
    assert lens.tolist() == [34, 50, 21] and s.top.tolist() == other[2].tolist()


@pytest.mark.parametrize("budget", [0.15, 1.0])
def test_sparse_decode_over_the_cache_that_they_filled(budget):
    """Prompts through the operators, summaries of the pages that they filled, then decode steps:
    slots, rotary write, summaries of new pages, score, selection and sparse decode.  The pages
    kept are those of the scores; the output is the attention over them, and over all pages
    (budget 1) the chunk attention's of the same step.  Both kernels round their weights and results
    once: 2 (u + u) of values up to the rows' largest."""
    announce(f"sparse decode over the cache that the operators filled, budget {budget}")
    R, nb, width = 3, 128, 48
    s = Server(R=R, nb=nb, width=width, seed=7)
    new = [600, 200, 333]
    q, lens, qs = s.write(new, 5)
    out = torch.zeros_like(q)
    paged_chunk_attention(q, s.kv, s.table, lens, qs, out)
    _near(out[:sum(new)], s.attention(new))
    st = QuadState(DEV, num_layers=1, num_blocks=nb, n_kv=N_KV, G=G, head_dim=D, page=PAGE,
                   max_reqs=R, max_pages=width, rank=8, budget=budget, combine="nrm")
    ensure_stage_b_buffers(st, DEV)
    full = sum(int(n) // PAGE for n in new)
    assert quad_build_bulk(st, [s.kv[:, 0]], s.table, lens, R) == full
    built = 0
    for step in range(20):                          # every request fills a page or two
        q, lens, qs = s.write([1] * R)
        built += quad_build_delta(st, [s.kv[:, 0]], s.table, lens, R)
        derive_page_params(st, lens, R)
        got = torch.full_like(q, float("nan"))
        select_then_attend(st, 0, q, s.kv, s.table, lens, R, D ** -0.5, got, ResidentVSource(s.kv))
        if step % 6 and step < 19:
            continue
        tab, cnt, _ = osel.select(npf(st.score), npi(st.n_pages), npi(st.n_sel_hi), npi(st.b_fix),
                                  sink=1, max_pages=width, mode=0, coverage=1.0, tie_mode=0,
                                  score_kind=1)
        assert np.array_equal(npi(st.page_table), tab) and np.array_equal(npi(st.page_cnt), cnt)
        pages = -(-s.lens // PAGE)
        assert (cnt == pages[:, None]).all() if budget == 1.0 else (cnt < pages[:, None]).all()
        # (rows behind the last token hold NaN, and the oracle multiplies them by zero)
        k, v = (np.nan_to_num(npf(s.kv[:, j])) for j in (0, 1))
        want = odec.attend(npf(q), k, v, npi(s.table), npi(lens), tab, cnt, scale=D ** -0.5, G=G)
        tol = 4 * 2.0 ** -8 * np.abs(want).max(-1, keepdims=True) + 2.0 ** -8
        assert (np.abs(npf(got) - want) <= tol).all(), step
        if budget == 1.0:
            out = torch.zeros_like(q)
            paged_chunk_attention(q, s.kv, s.table, lens, qs, out)
            assert (np.abs(npf(got) - npf(out)) <= tol).all(), step
    assert built == sum(int(n) // PAGE for n in s.lens) - full
