"""NaN codes of an 8-bit cache that the write appends to: rounding a block's earlier rows again keeps them."""
import numpy as np
import pytest
import torch

from amass.attention import quant_chunk_attention, quant_paged_write
from helpers import announce
from test_gpu_quant_cache import Step, num, same

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [dict(new=[1], had=[9]), dict(new=[5, 1], had=[7, 60], d=64),
                                   dict(new=[20, 3], had=[17, 30], page=32), dict(new=[70], had=[130], page=256),
                                   dict(new=[1] * 300, had=[1 + i % 15 for i in range(300)], n_kv=1)])
def test_nan_codes_stay_where_a_scale_grows(shape, dtype):
    """Both NaN codes in every channel place of a word, in rows before the run, at it and behind it."""
    announce(f"quant write: NaN codes in earlier rows, {shape}, {dtype}")
    s = Step(dtype=dtype, code="e4m3", **shape)
    raw = s.codes.view(torch.int8)
    nb, _, page, n_kv, d = raw.shape
    c = torch.arange(d)
    for row in range(page):
        raw[:, :, row, :, c % 13 == row % 13] = 0x7F
        raw[:, :, row, :, c % 29 == row % 29] = -1
    before = s.codes.clone()
    s.scales *= 2.0 ** -12                                  # (every run makes its block's scale grow)
    codes, scales = s.dev()
    s.run(codes, scales)
    s.check(codes, scales)
    got, was = codes.cpu().view(torch.uint8), before.view(torch.uint8)
    nan = torch.isnan(before.float())
    slots = s.slots[:s.T]
    written = torch.zeros(nb, page, dtype=torch.bool)
    written[slots // page, slots % page] = True
    old = nan & ~written[:, None, :, None, None]
    assert old.any() and torch.equal(got[old], was[old])    # (the code itself, its sign too)


def test_a_nan_key_stays_one_through_decode_steps():
    """A cache with a NaN in V, a token after it that is far larger: the rows that see the NaN are NaN, in its
    head alone."""
    announce("quant write: a NaN in V before a decode step")
    n_kv, d = 2, 128
    g = torch.Generator().manual_seed(3)
    codes = (64.0 * torch.randn(3, 2, 16, n_kv, d, generator=g)).to(torch.float8_e4m3fn)
    codes.view(torch.int8)[1, 1, 4, 0, 77] = 0x7F
    codes = codes.view(torch.int8).to(DEV).view(torch.float8_e4m3fn)
    scales = torch.full((3, 2, n_kv), 2.0 ** -8, device=DEV)
    k, v = ((100.0 * torch.randn(1, n_kv, d, generator=g)).bfloat16().to(DEV) for _ in range(2))
    quant_paged_write(k, v, codes, scales, torch.tensor([16 + 9], device=DEV))
    assert (scales[1] > 2.0 ** -8).all() and torch.isnan(codes[1, 1, 4, 0, 77].float())
    q = torch.randn(1, 4, d, generator=g).bfloat16().to(DEV)
    out = torch.empty_like(q)
    i32 = dict(dtype=torch.int32, device=DEV)
    quant_chunk_attention(q, codes, scales, torch.ones(1, 1, **i32), torch.tensor([10], **i32),
                          torch.tensor([0, 1], **i32), out)
    assert torch.isnan(out[0, :2].float()).all() and torch.isfinite(out[0, 2:].float()).all()


def test_numbers_are_rounded_again_as_before():
    """The formula, exactly, for codes of every value."""
    announce("quant write: every code rounded again")
    for code in ("int8", "e4m3"):
        s = Step(new=[1, 2], had=[15, 14], code=code)
        every = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.int8)
        every = every[every != -128] if code == "int8" else every
        s.codes.view(torch.int8).copy_(every[torch.arange(s.codes.numel()) % len(every)].view(s.codes.shape))
        s.scales *= 2.0 ** -2
        codes, scales = s.dev()
        s.run(codes, scales)
        s.check(codes, scales)
        assert np.isnan(num(codes)).any() == (code == "e4m3") and same(num(s.codes).shape, num(codes).shape)
