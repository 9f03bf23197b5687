"""Attention over the 8-bit cache where V holds the largest numbers of bf16: scales up to those that the write
makes of them (2^121 int8, 2^119 e4m3), and larger ones of caches quantised elsewhere."""
import numpy as np
import pytest
import torch

from helpers import announce
from test_gpu_quant_chunk import QuantCase
from test_gpu_quant_edges import far_case

pytestmark = pytest.mark.gpu


def largest_case(new, lens, e, code, most, **kw):
    """Rows whose first new token's key takes all of the weight (a lead of 141, beside which the rest is below
    2^-190 of it), from a page of V scale 2^e whose codes are -most .. most, zeros among them."""
    c = QuantCase(new=new, lens=lens, n_kv=1, G=2, code=code, **kw)
    c.q.zero_(), c.codes.view(torch.int8)[:, 0].zero_()
    c.q[:, :, 0] = 16.0
    c.scales[:, 0] = 1.0
    c.scales[:, 1] *= 2.0 ** (e - 40)
    d = c.q.shape[2]
    for r, (n, length) in enumerate(zip(new, lens)):
        if n:
            block, row = c.token(r, length - n)
            c.codes[block, 0, row, 0, 0] = torch.tensor(100.0 * (d / 128) ** 0.5).round().to(c.codes.dtype)
            levels = torch.linspace(-most, most, 9).round()
            c.codes[block, 1] = levels[torch.arange(16 * d) % 9].view(16, 1, d).to(c.codes.dtype)
            c.scales[block, 1] = 2.0 ** e
    c.numbers()
    return c


# (e, code, largest code): 127 2^121 is just below bf16's largest
LEVELS = [(119, "int8", 127), (120, "int8", 127), (121, "int8", 127), (125, "int8", 7), (127, "int8", 1),
          (119, "e4m3", 448), (122, "e4m3", 60), (127, "e4m3", 1)]


@pytest.mark.parametrize("e,code,most", LEVELS)
@pytest.mark.parametrize("new,lens,d", [([1, 1, 3], [1, 40, 300], 128), ([1, 4], [17, 90], 64), ([150], [150], 128),
                                        ([130, 1], [400, 30], 64), ([1], [9000], 128), ([60], [9000], 64),
                                        ([0, 40], [5, 6000], 128)])
def test_a_page_of_the_largest_numbers(new, lens, d, e, code, most):
    """One key's row of V, each number of it to the rounding of the result; zeros stay zeros."""
    announce(f"quant attention: V scales of 2^{e}, codes to {most}, {new} of {lens}, {code}, {d}")
    c = largest_case(new, lens, e, code, most, d=d)
    out, lse = c.run()
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    c.check(out, lse)


@pytest.mark.parametrize("code,exponent", [("int8", 121), ("e4m3", 119)])
@pytest.mark.parametrize("new,lens", [([5], [300]), ([200], [200]), ([2], [7000])])
def test_pages_of_the_largest_numbers(new, lens, code, exponent):
    """Every page under the largest scale of the write; single tokens see one of them, others a mean of many."""
    announce(f"quant attention: all V scales 2^{exponent}, {new} of {lens}, {code}")
    c = QuantCase(new=new, lens=lens, n_kv=1, code=code)
    c.scales[:, 1] = 2.0 ** exponent
    c.numbers()
    out, lse = c.run()
    assert torch.isfinite(out.float()).all()
    c.check(out, lse)


@pytest.mark.parametrize("e", [13, 20, 31, 60])
@pytest.mark.parametrize("new,lens", [([4], [300]), ([150], [400]), ([1], [9000]), ([40], [9000])])
def test_scores_far_from_zero_beside_the_largest_v_scales(new, lens, e):
    """Equal scores of 2^e, on pages of V scales from 2^56 to 2^116: the pages of the largest take all, and as much
    each as its scale says.  Tolerances of test_scores_far_from_zero."""
    announce(f"quant attention: scores of 2^{e}, V scales to 2^116, {new} of {lens}")
    for sign in (1, -1):
        c = far_case(new, lens, e, sign)
        g = torch.Generator().manual_seed(5)
        c.scales[:, 1] *= torch.exp2(torch.randint(62, 121, c.scales[:, 1].shape, generator=g).float())
        c.numbers()
        out, lse = c.run()
        want, wlse, _, size, _ = c.want()
        tol = torch.finfo(c.dt).eps / 2 * (1.01 * size + np.abs(want)) + 2.0 ** -14 * size
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:4], (err / tol).max())
        assert (np.abs(lse.double().cpu().numpy() - wlse) <= 5 * 2.0 ** -24 * np.abs(wlse) + 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new,lens,d", [([4, 1], [300, 90], 128), ([150], [400], 64), ([2], [9000], 128)])
def test_pages_of_zeros_count_in_full(new, lens, d, dtype):
    """Every other page of V is zeros under the least scale, beside numbers of 2^40 (fp16: 2^12): its keys' weights
    are in every row's sum."""
    announce(f"quant attention: pages of zeros beside large numbers, {new} of {lens}, {d}, {dtype}")
    c = QuantCase(new=new, lens=lens, n_kv=2, d=d, dtype=dtype)
    c.scales[:, 1] *= 2.0 ** (38 if dtype == "bf16" else 10)
    for r, n in enumerate(lens):
        zero = c.table[r, :-(-n // 16)][r % 2::2].long()
        c.codes[zero, 1], c.scales[zero, 1] = 0, 2.0 ** -64
    c.numbers()
    c.check(*c.run())
