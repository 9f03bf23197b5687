"""Attention over the 8-bit cache in fp16 where V's scales lie far apart: a weight with V's scale has fewer
bits the further its page is below the largest."""
import pytest
import torch

from helpers import announce
from test_gpu_quant_chunk import QuantCase

pytestmark = pytest.mark.gpu


def apart_case(new, lens, bits, code, first, n_kv=1, **kw):
    """Every fifth page has V scales of 2^bits times the others' and codes of zero in all channels but every
    eighth, where they are small enough for the result to stay in fp16.  first: whether such a page comes first."""
    c = QuantCase(new=new, lens=lens, n_kv=n_kv, G=2, code=code, dtype="fp16", **kw)
    for r, n in enumerate(lens):
        blocks = c.table[r, :-(-n // c.page)].long()
        loud = blocks[0 if first else min(3, len(blocks) - 1)::5]
        c.scales[loud, 1] *= 2.0 ** bits
        c.codes.view(torch.int8)[loud, 1] = 0
        if bits <= 14:                                     # (numbers below 2^13)
            c.codes[loud, 1, :, :, ::8] = torch.tensor(7.0).to(c.codes.dtype)
    c.numbers()
    return c


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("bits", [5, 9, 14, 21, 28, 40, 74])
@pytest.mark.parametrize("new,lens,d", [([4, 1], [300, 70], 128), ([2], [2000], 64), ([150], [400], 128),
                                        ([130, 3], [200, 900], 64), ([1], [9000], 128), ([60], [9000], 64)])
def test_fp16_weights_of_pages_far_below_the_largest(new, lens, d, bits, code):
    """The channels where the large pages hold zeros come from the other pages alone, to the tolerance of
    any other channel (of the weighted mean of |v| there)."""
    for first in (False, True):
        announce(f"quant attention: fp16, V scales 2^{bits} apart, {new} of {lens}, {code}, {d}, "
                 f"{'large page first' if first else 'large pages behind'}")
        c = apart_case(new, lens, bits, code, first, d=d)
        small = float(c.v[:, :, :, 1].abs().max())         # (a channel without large numbers)
        out, lse = c.run()
        keep = c.v
        want = c.want()
        c.want = lambda: want
        if bits > 14:
            c.v = keep[..., 1:2]                            # the tolerance's largest V: that of what is compared
        assert float(c.v.abs().max()) >= small
        c.check(out, lse)


@pytest.mark.parametrize("new,lens", [([4], [300]), ([200], [333])])
def test_fp16_scales_from_2_to_the_minus_30_to_the_10(new, lens):
    """Random scales; the numbers of the least pages are below fp16's least."""
    announce(f"quant attention: fp16, V scales of 2^-30 to 2^10, {new} of {lens}")
    c = QuantCase(new=new, lens=lens, n_kv=2, dtype="fp16")
    g = torch.Generator().manual_seed(8)
    c.scales[:, 1] *= torch.exp2(torch.randint(-30, 11, c.scales[:, 1].shape, generator=g).float())
    c.numbers()
    c.check(*c.run())


@pytest.mark.parametrize("window,causal", [(40, True), (None, False)])
def test_fp16_pages_far_apart_under_masks(window, causal):
    """Pages that some rows see and others do not, pages without a block, pages of the table behind the end."""
    announce(f"quant attention: fp16, V scales far apart, window {window}, causal {causal}")
    for new, lens in (([3, 2], [333, 90]), ([140], [300])):
        c = apart_case(new, lens, 30, "int8", False, window=window, causal=causal, spare=2)
        c.table[0, 4] = -1
        want = c.want()
        c.want = lambda: want
        c.v = c.v[..., 1:2]
        c.check(*c.run())
