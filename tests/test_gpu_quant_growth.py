"""A page whose scale grows a little with every token, and the order of halves in a pool of two blocks."""
import numpy as np
import pytest
import torch

import oracle.quant_cache as oq
from amass.attention import quant_cache, quant_paged_read, quant_paged_write
from helpers import announce
from test_gpu_quant_cache import CODES, num, same

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("by", [1.008, 1.02, 1.3])
def test_slow_growth_token_by_token(by, code):
    """Every step's codes and scales are the oracle's."""
    announce(f"quant write: a page that grows by {by} a token, {code}")
    g = torch.Generator().manual_seed(6)
    k, v = ((torch.randn(16, 2, 64, generator=g).clamp(-2.5, 2.5) * by ** torch.arange(16.0)[:, None, None]).bfloat16()
            for _ in range(2))
    codes, scales = quant_cache(3, 16, 2, 64, dtype=CODES[code], device=DEV)
    wc = [np.zeros((3, 16, 2, 64)), np.zeros((3, 16, 2, 64))]
    ws = [np.ones((3, 2)), np.ones((3, 2))]
    for i in range(16):
        slot = [16 + i]
        quant_paged_write(k[i:i + 1].to(DEV), v[i:i + 1].to(DEV), codes, scales, torch.tensor(slot, device=DEV))
        for h, x in enumerate((k, v)):
            wc[h], ws[h] = oq.write(wc[h], ws[h], x[i:i + 1].double().numpy(), slot, 16, code)
        assert same(num(codes), np.stack(wc, 1)) and same(scales.cpu().double().numpy(), np.stack(ws, 1))


def test_a_pool_of_two_blocks_has_its_halves_first():
    """(2, 2, ...) may be read both ways: all calls take the first axis as K and V, as they do 16-bit caches."""
    announce("quant cache: two blocks")
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(20, 2, 64, generator=g).bfloat16() for _ in range(2))
    codes, scales = quant_cache(2, 16, 2, 64, device=DEV)
    quant_paged_write(k.to(DEV), v.to(DEV), codes, scales, torch.arange(20, device=DEV))
    for half, x in enumerate((k, v)):
        wc, ws = oq.write(np.zeros((2, 16, 2, 64)), np.ones((2, 2)), x.double().numpy(), range(20), 16, "int8")
        assert same(num(codes[half]), wc) and same(scales[half].cpu().double().numpy(), ws)
    kv = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    which = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    quant_paged_read(codes, scales, which, kv, which)
    want = (codes.float() * scales[:, :, None, :, None]).bfloat16()
    assert torch.equal(kv, want)
