"""Block tables and slot maps on the GPU (amass_extend, amass_release) against the oracle's plain
loops: whole numbers, so every comparison is exact."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass.attention import extend_block_tables, free_blocks, release_blocks
from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


class Step:
    """A step's inputs on both sides; the table's old pages hold blocks of a permutation."""

    def __init__(self, new, lens, *, page=16, width=None, spare=5, pad=0, short=0, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.new, self.lens = page, list(new), list(lens)
        had = [max(-(-max(a - n, 0) // page), 0) for a, n in zip(lens, new)]
        need = [-(-max(a, 0) // page) for a in lens]
        width = max(need + [1]) if width is None else width
        want = sum(max(b - a, 0) for a, b in zip(had, need))
        self.nb = sum(had) + want + spare + 1
        perm = rng.permutation(self.nb)
        self.table = np.full((len(lens), width), -7, np.int32)
        at = 0
        for r, n in enumerate(had):
            self.table[r, :n] = perm[at:at + n][:width]
            at += n
        free = perm[at:]
        self.top = max(want + spare - short, 0) if short else len(free)
        self.free = free.astype(np.int32)
        self.qs = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.qs[-1]) + pad

    def run(self, top_out=None):
        d = dict(table=_i32(self.table), free=_i32(self.free), top=_i32([self.top, 0, 0]),
                 slots=torch.full((self.T,), 99, dtype=torch.int64, device=DEV),
                 positions=torch.full((self.T,), 99, dtype=torch.int32, device=DEV))
        extend_block_tables(d["table"], _i32(self.lens), _i32(self.qs), d["free"], d["top"],
                            d["slots"], d["positions"], page=self.page, num_blocks=self.nb,
                            top_out=top_out)
        torch.cuda.synchronize()
        return d

    def want(self):
        return ochunk.extend(self.table, self.lens, self.qs, self.free, self.top, self.T,
                             self.page, self.nb)

    def check(self):
        d = self.run()
        table, slots, positions, left, short = self.want()
        assert np.array_equal(d["table"].cpu().numpy(), table)
        assert np.array_equal(d["slots"].cpu().numpy(), slots)
        assert np.array_equal(d["positions"].cpu().numpy(), positions)
        assert d["top"].tolist() == [left, 0, short]
        assert np.array_equal(d["free"].cpu().numpy(), self.free)
        return d


STEPS = {
    "one token": dict(new=[1], lens=[1]),
    "one token, page starts": dict(new=[1] * 4, lens=[17, 16, 33, 18]),
    "decode step": dict(new=[1] * 67, lens=[int(x) for x in
                                            np.random.default_rng(5).integers(1, 900, 67)]),
    "prompts": dict(new=[40, 1, 333, 16], lens=[40, 50, 333, 32], pad=9),
    "empty requests": dict(new=[0, 5, 0, 0, 7, 0], lens=[30, 5, 0, 16, 100, 8], pad=2),
    "drafts in pages of 64": dict(new=[5, 3, 9], lens=[66, 63, 200], page=64),
    "pages of one token": dict(new=[3, 2], lens=[3, 9], page=1),
    "several workgroups": dict(new=[1500, 2, 2000, 1, 900], lens=[1500, 300, 2100, 64, 5000],
                               pad=300),
    "more requests than threads": dict(new=[1] * 700, lens=list(range(1, 701)), pad=5),
    "the most requests": dict(new=[1] * 4096, lens=[16 * (i % 3) + 1 for i in range(4096)]),
    "list runs dry": dict(new=[100, 30, 50], lens=[100, 60, 50], spare=0, short=4),
    "empty list": dict(new=[17, 1], lens=[17, 40], spare=0, short=10 ** 6),
    "chunk longer than its request": dict(new=[20, 4], lens=[13, 4]),
    "table too narrow": dict(new=[100, 3], lens=[100, 20], width=4),
    "only padding": dict(new=[0, 0], lens=[5, 0], pad=40),
}


@pytest.mark.parametrize("name", STEPS)
def test_extend_matches_the_oracle(name):
    announce(f"extend: {name}")
    Step(**STEPS[name]).check()


def test_bad_blocks_count_as_none():
    announce("extend: blocks outside the pool")
    s = Step(new=[4, 33], lens=[20, 33])    # (the first request's tokens start a page)
    s.free[s.top - 2] = -5                  # the second new page's block
    d = s.check()
    assert (d["slots"][:4] >= 0).all() and (d["slots"][4:20] == -1).all()
    assert (d["slots"][20:] >= 0).all() and d["table"][1, 0] == -1
    s = Step(new=[3, 2], lens=[20, 2])
    s.table[0, 1] = s.nb + 3                # the page the first request's tokens lie in
    d = s.check()
    assert (d["slots"][:3] == -1).all() and (d["slots"][3:] >= 0).all()


@pytest.mark.parametrize("T", [50, 5000])
def test_top_out_leaves_the_list_as_it_was(T):
    announce(f"extend: top_out, {T} tokens")
    s = Step(new=[T], lens=[T])
    out = torch.full((3,), 7, dtype=torch.int32, device=DEV)
    d = s.run(top_out=out)
    _, _, _, left, short = s.want()
    assert d["top"].tolist() == [s.top, 0, 0] and out.tolist() == [left, 7, short]


def test_table_rows_and_columns_beyond_the_step_stay():
    announce("extend: strided table")
    wide = torch.full((6, 9), -3, dtype=torch.int32, device=DEV)
    table = wide[1:4, 2:7]
    free, top = free_blocks(20, DEV)
    slots = torch.empty(40, dtype=torch.int64, device=DEV)
    pos = torch.empty(40, dtype=torch.int32, device=DEV)
    extend_block_tables(table, _i32([33, 2]), _i32([0, 33, 35]), free, top, slots, pos, page=16,
                        num_blocks=20)
    want = np.full((6, 9), -3)
    want[1, 2:5] = [0, 1, 2]
    want[2, 2] = 3
    assert np.array_equal(wide.cpu().numpy(), want)
    assert top.tolist() == [16, 0, 0]
    assert slots[35:].tolist() == [-1] * 5 and slots[33:35].tolist() == [48, 49]


@pytest.mark.parametrize("R,page,seed", [(1, 16, 0), (5, 16, 1), (3000, 16, 2), (40, 64, 3)])
def test_release_matches_the_oracle(R, page, seed):
    announce(f"release: {R} requests, pages of {page}")
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 40 * page // max(1, R // 200), R)
    done = rng.random(R) < 0.6
    width = max(-(-int(lens.max()) // page) - 1, 1)          # (some rows are longer than it)
    nb = R * width + 10
    table = rng.permutation(nb)[:R * width].reshape(R, width).astype(np.int32)
    table[rng.random(table.shape) < 0.05] = -1
    free = np.full(nb - R, 3, np.int32)
    dt, df, dtop = _i32(table), _i32(free), _i32([4, 0, 0])
    release_blocks(dt, _i32(lens), torch.tensor(done, device=DEV), df, dtop, page=page,
                   num_blocks=nb)
    wt, wf, left, dropped = ochunk.release(table, lens, done, free, 4, page, nb)
    assert np.array_equal(dt.cpu().numpy(), wt) and np.array_equal(df.cpu().numpy(), wf)
    assert dtop.tolist() == [left, 0, dropped]


def test_release_drops_what_does_not_fit():
    announce("release: full list")
    table = np.arange(12, dtype=np.int32).reshape(2, 6)
    dt, df, dtop = _i32(table), _i32(np.full(8, 77)), _i32([5, 0, 0])
    release_blocks(dt, _i32([96, 50]), torch.tensor([True, True], device=DEV), df, dtop, page=16,
                   num_blocks=12)
    assert df.tolist() == [77] * 5 + [0, 1, 2] and dtop.tolist() == [8, 0, 7]


def test_blocks_circulate_through_a_captured_step():
    """Decode steps of a replayed graph, with requests that end and start between them: every
    block is in one place, and the tables are the oracle's."""
    announce("extend + release: captured, 40 steps")
    R, page, nb, width = 6, 16, 64, 8
    rng = np.random.default_rng(3)
    table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    lens, qs = _i32([0] * R), _i32(range(R + 1))
    done = torch.zeros(R, dtype=torch.bool, device=DEV)
    free, top = free_blocks(nb, DEV)
    slots = torch.empty(R + 2, dtype=torch.int64, device=DEV)
    pos = torch.empty(R + 2, dtype=torch.int32, device=DEV)

    def step():
        release_blocks(table, lens, done, free, top, page=page, num_blocks=nb)
        lens.copy_(torch.where(done, 1, lens + 1))
        extend_block_tables(table, lens, qs, free, top, slots, pos, page=page, num_blocks=nb)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    w_table, w_free, w_left = np.full((R, width), -1, np.int32), np.arange(nb)[::-1].copy(), nb
    w_lens = np.ones(R, np.int64)
    w_table, _, _, w_left, _ = ochunk.extend(w_table, w_lens, range(R + 1), w_free, w_left, R + 2,
                                             page, nb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(40):
        flags = (rng.random(R) < 0.15) | (w_lens >= page * width)
        done.copy_(torch.tensor(flags))
        graph.replay()
        w_table, w_free, w_left, _ = ochunk.release(w_table, w_lens, flags, w_free, w_left, page, nb)
        w_lens = np.where(flags, 1, w_lens + 1)
        w_table, w_slots, w_pos, w_left, short = ochunk.extend(
            w_table, w_lens, range(R + 1), w_free, w_left, R + 2, page, nb)
        assert np.array_equal(table.cpu().numpy(), w_table), i
        assert np.array_equal(slots.cpu().numpy(), w_slots), i
        assert np.array_equal(pos.cpu().numpy(), w_pos), i
        assert top.tolist() == [w_left, 0, short], i
        held = w_table[w_table >= 0].tolist() + free[:w_left].tolist()
        assert sorted(held) == list(range(nb)), i


def test_wrapper_refuses():
    announce("extend, release: refusals")
    table, lens, qs = _i32([[0, 0]]), _i32([3]), _i32([0, 3])
    free, top = free_blocks(4, DEV)
    slots = torch.empty(3, dtype=torch.int64, device=DEV)
    pos = torch.empty(3, dtype=torch.int32, device=DEV)
    good = dict(block_table=table, seq_lens=lens, query_start=qs, free=free, top=top, slots=slots,
                positions=pos)
    for over, kw in ((dict(block_table=table.long()), {}), (dict(seq_lens=lens.long()), {}),
                     (dict(query_start=qs[:1]), {}), (dict(slots=slots.int()), {}),
                     (dict(positions=pos[:2]), {}), (dict(top=top[:2]), {}),
                     (dict(slots=slots[::2]), {}), ({}, dict(page=12)), ({}, dict(num_blocks=0)),
                     (dict(seq_lens=_i32([1, 2])), {}), ({}, dict(top_out=top[:2]))):
        with pytest.raises(ValueError):
            extend_block_tables(**{**good, **over}, **{**dict(page=16, num_blocks=4), **kw})
    with pytest.raises(ValueError, match="share memory"):
        extend_block_tables(table.expand(2, 2), _i32([1, 1]), _i32([0, 1, 2]), free, top, slots, pos,
                            page=16, num_blocks=4)
    with pytest.raises(ValueError, match="at most 4096"):
        n = 4097
        extend_block_tables(torch.zeros(n, 2, dtype=torch.int32, device=DEV), _i32([1] * n),
                            _i32(range(n + 1)), free, top, slots, pos, page=16, num_blocks=4)
    with pytest.raises(ValueError):
        release_blocks(table, lens, lens, free, top, page=16, num_blocks=4)
    # nothing to do is no error
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    extend_block_tables(table[:0], none, qs[:1], free, top, slots[:0], pos[:0], page=16,
                        num_blocks=4)
    release_blocks(table[:0], none, none.bool(), free, top, page=16, num_blocks=4)
    assert top.tolist() == [4, 0, 0]
