"""The 8-bit cache where it could go wrong.  Attention: scores beside which log2 of V's scale is lost, caches that
are read past the GPU's own, starts that do not ascend, captured prompts that become padding.  The write: batches
of many tokens, whose runs start and end anywhere in the windows that are looked through."""
import numpy as np
import pytest
import torch

from amass.attention import quant_chunk_attention, quant_scratch_bytes
from helpers import announce
from test_gpu_chunk import want_on_gpu
from test_gpu_quant_cache import Step
from test_gpu_quant_chunk import CODES, DEV, QuantCase

pytestmark = pytest.mark.gpu


def far_case(new, lens, e, sign, **kw):
    """Scores of sign * {1, 2, 4} 2^e to the rounding of log2 e (2^(e-2) between unlike ones at least, so the
    largest alone count), each on pages of two K scales; the products of equal scores are equal in fp32,
    whose scales differ by a power of two."""
    c = QuantCase(new=new, lens=lens, n_kv=1, G=2, **kw)
    c.q.zero_(), c.codes[:, 0].zero_()
    c.q[:, :, 0] = 2.0 ** 10
    c.scale = 0.25
    for r, n in enumerate(lens):
        pos = torch.arange(n)
        block, row = c.table[r, pos // 16].long(), pos % 16
        level = torch.tensor([8, 16, 32])[pos * 7 % 3]
        half = 1 + pos // 16 % 2
        c.codes[block, 0, row, 0, 0] = (sign * level // half).to(c.codes.dtype)
        c.scales[block, 0, 0] = half * 2.0 ** (e - 11)
    c.numbers()
    return c


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("e", [13, 20, 26, 31, 60])
@pytest.mark.parametrize("new,lens", [([4], [300]), ([1, 2], [40, 700]), ([150], [400]), ([1], [9000]),
                                      ([40], [9000])])
def test_scores_far_from_zero(new, lens, e, code, dtype, d):
    """Only the keys of the largest score count, as much as their V's scales say: each weight is rounded once
    and its log2 sv to 2^-19 (under 32, in a few steps), sums to 2^-16; the result once.  A lse keeps the
    roundings of log2 e, the scaled score, the sum of both parts, ln 2 and their product: 5 of 2^-24."""
    for sign in (1, -1):
        announce(f"quant attention: scores {sign} 2^{e}, {new} of {lens}, {code}, {dtype} {d}")
        c = far_case(new, lens, e, sign, code=code, dtype=dtype, d=d)
        out, lse = c.run()
        want, wlse, _, size, _ = c.want()
        tol = torch.finfo(c.dt).eps / 2 * (1.01 * size + np.abs(want)) + 2.0 ** -14 * size + 2.0 ** -24
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:4], err.max())
        assert (np.abs(lse.double().cpu().numpy() - wlse) <= 5 * 2.0 ** -24 * np.abs(wlse) + 2.0 ** -14).all()


@pytest.mark.parametrize("new,lens", [([4], [300]), ([150], [400])])
def test_scores_far_from_zero_beside_v_scales_far_apart(new, lens):
    """As above where the equal scores' pages have V scales of 2^-40 to 2^40."""
    announce(f"quant attention: scores of 2^31, scales of V far apart, {new}")
    c = far_case(new, lens, 31, 1)
    g = torch.Generator().manual_seed(5)
    c.scales[:, 1] *= torch.exp2(torch.randint(-40, 41, c.scales[:, 1].shape, generator=g).float())
    c.numbers()
    out, _ = c.run()
    want, _, _, size, _ = c.want()
    tol = torch.finfo(c.dt).eps / 2 * (1.01 * size + np.abs(want)) + 2.0 ** -14 * size
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,dtype,d", [([1] * 45, "bf16", 128), ([2] * 45, "fp16", 128), ([1] * 90, "bf16", 64)])
def test_more_codes_than_the_caches_hold(new, code, dtype, d):
    """Few rows over more than 128 MB of codes, as a batch of long requests has (here they share blocks, each
    in an order of its own)."""
    announce(f"quant attention: {len(new)} long requests, {code}, {dtype} {d}")
    c = QuantCase(new=new, lens=[4100], n_kv=8, G=2, code=code, dtype=dtype, d=d)
    g = torch.Generator().manual_seed(9)
    c.table = torch.stack([c.table[0][torch.randperm(c.table.shape[1], generator=g)] for _ in new])
    c.lens = torch.tensor([3999 + 7 * i % 101 for i in range(len(new))], dtype=torch.int32)
    assert int(c.lens.sum()) * 8 * d > 128e6
    c.want = lambda: want_on_gpu(c)
    c.check(*c.run())


def test_starts_that_do_not_ascend_leave_other_memory_alone():
    """Requests whose rows together are several times the batch's, and a scratch that holds records of
    row tiles behind `out`: the rows there stay, and the scratch serves the next call."""
    announce("quant attention: starts that do not ascend, a scratch of records")
    T, R = 1024, 5
    c = QuantCase(new=[T], lens=[4000], n_kv=8)
    q, codes, scales, table, _, _ = c.dev()
    wide = torch.full((2 * T, *q.shape[1:]), 7.0, dtype=c.dt, device=DEV)
    out = wide[:T]
    bad = (table.expand(R, -1).contiguous(), torch.full((R,), 4000, dtype=torch.int32, device=DEV),
           torch.tensor([0, T] * 3, dtype=torch.int32, device=DEV))
    need = quant_scratch_bytes(q, codes, scales, *bad, out)
    # (request, row tile, parts, slot, first row, rows, tokens, 0) from byte 256 on, repeated
    record = torch.tensor([0, 0, 2, 0, T, T, 4000, 0], dtype=torch.int32)
    scratch = record.repeat(-(-need // 32) + 8).view(torch.uint8)[:need].to(DEV)
    quant_chunk_attention(q, codes, scales, *bad, out, scratch=scratch)
    torch.cuda.synchronize()
    assert (wide[T:] == 7.0).all()
    c = QuantCase(new=[90, 3], lens=[3000, 900], n_kv=8)
    c.check(*c.run(scratch=scratch))


@pytest.mark.parametrize("T,starts,rows", [(60, [0, 40, 20, 60], [*range(20), *range(40, 60)]),
                                           (12, [0, 9, 7, 12], [*range(7), *range(9, 12)])])
def test_rows_of_one_request_only_are_right_where_starts_do_not_ascend(T, starts, rows):
    announce(f"quant attention: starts {starts}")
    c = QuantCase(new=[T, 0, 0], lens=[150, 40, 230], n_kv=2)
    c.qs = torch.tensor(starts, dtype=torch.int32)
    c.check(*c.run(), rows=rows)


@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "fp16")])
def test_captured_prompts_become_padding_and_back(code, dtype):
    """One graph over 2200 rows: prompts, then a few rows of other requests, then prompts again; the eager
    call between the replays has a scratch of its own."""
    announce(f"quant attention: captured prompts and padding, {code}, {dtype}")
    c = QuantCase(new=[1300, 900], lens=[1500, 2400], n_kv=2, G=2, code=code, dtype=dtype)
    q, codes, scales, table, lens, qs = c.dev()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    call = (q, codes, scales, table, lens, qs, out)
    scratch = torch.empty(quant_scratch_bytes(*call, lse=lse), dtype=torch.uint8, device=DEV)
    quant_chunk_attention(*call, lse=lse, scratch=scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        quant_chunk_attention(*call, lse=lse, scratch=scratch)
    for step, (new, at) in enumerate([([1300, 900], [1500, 2400]), ([3, 1], [1400, 2000]), ([0, 0], [1500, 2400]),
                                      ([1, 200], [17, 2400]), ([1300, 900], [1500, 2400])]):
        announce(f"replay {step}: {new} of {at}")
        c.lens = torch.tensor(at, dtype=torch.int32)
        c.qs = torch.tensor([0, new[0], sum(new)], dtype=torch.int32)
        lens.copy_(c.lens), qs.copy_(c.qs)
        out.fill_(7.0), lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager, elsewhere = c.run()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)) and torch.equal(lse, elsewhere)
        c.want = lambda: want_on_gpu(c)
        if sum(new):
            c.check(out, lse)
        else:
            assert (out == 7.0).all() and (lse == 7.0).all()


LARGE = {         # more than 256 tokens are looked through by fours, more than 1024 by sixteens
    "260 single tokens": dict(new=[1] * 260, had=[i % 50 for i in range(260)], n_kv=1),
    "1100 single tokens": dict(new=[1] * 1100, had=[i * 7 % 40 for i in range(1100)], n_kv=1, d=64),
    "runs of 1 to 21": dict(new=[1 + i * 5 % 21 for i in range(130)], had=[i * 11 % 37 for i in range(130)], n_kv=3),
    "a prompt among drafts": dict(new=[3, 5, 1000, 2, 4, 90], had=[9, 14, 5, 15, 31, 0], rot=128),
    "pages of 64, in pairs": dict(new=[61, 700, 1, 400], had=[3, 60, 63, 0], page=64, rot=64, interleaved=True, d=64),
    "a run of a whole large page": dict(new=[7, 2100], had=[1, 1000], page=1024, n_kv=1, d=64, rot=32),
}


@pytest.mark.parametrize("dtype,code", [("bf16", "int8"), ("fp16", "e4m3")])
@pytest.mark.parametrize("holes", [False, True])
@pytest.mark.parametrize("name", LARGE)
def test_writes_of_many_tokens(name, holes, dtype, code):
    """The formula, exactly.  Holes: blocks that stay as they were, of padding in the middle of the batch."""
    announce(f"quant write: {name}, {'holes, ' * holes}{dtype} {code}")
    s = Step(dtype=dtype, code=code, **LARGE[name])
    if holes:
        s.slots[s.slots // s.page % 3 == 1] = -1
    codes, scales = s.dev()
    s.run(codes, scales, torch.full_like(s.q, 7.0).to(DEV))
    s.check(codes, scales)
