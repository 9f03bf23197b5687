"""What a page of the 8-bit cache holds after its scale has grown (on the oracle, which the kernels match code for
code): how far it is from the tokens, and how far its codes from those of one write."""
import numpy as np
import pytest

import oracle.quant_cache as oq

ROWS = {
    "N(0, 1)": lambda g, i: g.normal(size=64),
    "0.8 percent a token": lambda g, i: np.clip(g.normal(size=64), -2.5, 2.5) / 2.5 * 1.008 ** i,
    "2 percent a token": lambda g, i: np.clip(g.normal(size=64), -2.5, 2.5) / 2.5 * 1.02 ** i,
    "twice a token": lambda g, i: g.normal(size=64) * 2.0 ** i,
}


def token_by_token(x, page, code):
    """(codes, scale, growths) of one page that took its rows one at a time."""
    c, s, grown = np.zeros((1, page, 1, x.shape[1])), np.ones((1, 1)), 0
    for i in range(page):
        before = s[0, 0]
        c, s = oq.write(c, s, x[i:i + 1, None], [i], page, code)
        grown += i > 0 and s[0, 0] > before
    return c[0, :, 0], s[0, 0], grown


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("name", ROWS)
def test_int8_token_by_token_is_half_a_step_for_the_entry_and_each_growth(name, page):
    g = np.random.default_rng(4)
    x = np.stack([ROWS[name](g, i) for i in range(page)])
    c, s, grown = token_by_token(x, page, "int8")
    whole, ws = oq.write(np.zeros((1, page, 1, 64)), np.ones((1, 1)), x[:, None], range(page), page, "int8")
    assert s == ws[0, 0]                                   # (the largest number's, however it came)
    assert (np.abs(c * s - x) <= 0.5 * s * (1 + grown) * (1 + 1e-9)).all()
    apart = np.abs(c - whole[0, :, 0]).max()
    assert apart <= 0.5 * (2 + grown)
    if name == "0.8 percent a token":                      # more than one step: growths add up
        assert apart > 2


def test_e4m3_is_rounded_again_without_loss_above_its_least_normal_number():
    g = np.random.default_rng(4)
    x = np.stack([ROWS["twice a token"](g, i) for i in range(6)])
    c, s, grown = token_by_token(np.concatenate([x, np.zeros((10, 64))]), 16, "e4m3")
    assert grown >= 4
    big = np.abs(x) >= 2.0 ** -6 * s
    assert big.sum() > 100 and (np.abs(c[:6] * s - x)[big] <= 2.0 ** -4 * np.abs(x)[big]).all()
    # below 2^-6 of the last scale: half a step of 2^-9 of the scale for the entry and each growth
    assert (np.abs(c[:6] * s - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * s * (1 + grown)).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_rows_behind_a_run_keep_codes_and_not_numbers(code):
    """A second write of a page's first rows starts the page anew; one that makes the scale grow rounds
    only the rows before it again."""
    g = np.random.default_rng(4)
    x = g.normal(size=(16, 1, 8))
    x[9] *= 50.0
    c, s = oq.write(np.zeros((1, 16, 1, 8)), np.ones((1, 1)), x, range(16), 16, code)
    again, s2 = oq.write(c, s, x[:4], range(4), 16, code)
    assert s2[0, 0] < s[0, 0] and np.array_equal(again[0, 4:], c[0, 4:])
    grown, s3 = oq.write(c, s, 1000.0 * x[4:6], [4, 5], 16, code)
    assert s3[0, 0] > s[0, 0] and np.array_equal(grown[0, 6:], c[0, 6:]) and not np.array_equal(grown[0, :4], c[0, :4])
    same, s4 = oq.write(c, s, x[4:6], [4, 5], 16, code)
    assert s4[0, 0] == s[0, 0] and np.array_equal(same, c)     # (from a later row: the same codes again)
