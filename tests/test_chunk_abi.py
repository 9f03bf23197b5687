"""include/amass_chunk.h against its bindings, the entry points' refusals (checked on the host
before any launch, so no GPU is touched) and the wrappers' argument checks on the CPU."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass import _hip
from amass.attention import (extend_block_tables, free_blocks, paged_chunk_attention,
                             release_blocks, rope_frequencies, rope_paged_write, rope_table)

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "include", "amass_chunk.h")
KIND = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "float": ctypes.c_float}


def _text():
    with open(HEADER) as fh:
        return re.sub(r"/\*.*?\*/", "", fh.read(), flags=re.S)


def test_structs_and_symbols_mirror_the_header():
    lib = _hip.load_library()
    txt = _text()
    structs = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", txt, flags=re.S):
        fields = []
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            typ, names = re.match(r"((?:const\s+)?\w+\s*\**)\s*(.*)", decl).groups()
            for nm in names.split(","):
                ptr = "*" in typ or "*" in nm
                kind = typ.replace("const", "").strip(" *")
                fields.append((nm.strip(" *"), ctypes.c_void_p if ptr else KIND[kind]))
        structs[name] = fields
    assert set(structs) == set(_hip.CHUNK_STRUCTS)
    for name, (idx, st) in _hip.CHUNK_STRUCTS.items():
        assert list(st._fields_) == structs[name], name
        assert ctypes.sizeof(st) == lib.amass_chunk_struct_size(idx), name
    names = re.findall(r"^\s*(?:int|int64_t|size_t)\s+(amass_\w+)\s*\(", txt, flags=re.M)
    assert len(names) == 7
    for n in names:
        assert hasattr(lib, n), n
    assert lib.amass_chunk_struct_size(4) == 0
    version = int(re.search(r"AMASS_CHUNK_ABI_VERSION (\d+)", txt).group(1))
    assert lib.amass_chunk_abi_version() == _hip.CHUNK_ABI_VERSION == version


def _chunk(**over):
    a = _hip.ChunkArgs()
    base = dict(q=0x1000, q_st=512, q_hs=128, k=0x1000, v=0x1000,
                kv_sb=32768, kv_st=1024, kv_sh=128, block_table=0x1000, bt_st=4, seq_lens=0x1000,
                query_start=0x1000, out=0x1000, o_st=512, o_hs=128, scale=0.1, n_req=1,
                n_tokens=3, n_kv=8, G=4, d=128, page=16, nb=4, max_pages=4, causal=1)
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(q=None), -1), (dict(v=None), -1), (dict(query_start=None), -1), (dict(d=96), -3),
    (dict(dtype=2), -3), (dict(page=8), -2), (dict(page=24), -2), (dict(scale=0.0), -2),
    (dict(scale=-1.0), -2), (dict(scale=math.nan), -2), (dict(scale=math.inf), -2),
    (dict(window=-1), -2), (dict(G=0), -2), (dict(n_kv=0), -2), (dict(nb=0), -2),
    (dict(q=0x1008), -2), (dict(kv_st=1028), -2), (dict(o_hs=124), -2), (dict(kv_st=1 << 30), -2),
    (dict(kv_st=-1024), -2), (dict(kv_sb=1 << 30), -2), (dict(kv_sb=-32768), -2),
    (dict(n_tokens=1 << 29), -2), (dict(max_pages=0), -2)])
def test_chunk_attention_refuses(over, status):
    lib = _hip.load_library()
    a = _chunk(**over)
    assert lib.amass_chunk_scratch_bytes(ctypes.byref(a)) == status
    a.scratch, a.scratch_bytes = 0x1000, 1 << 40
    assert lib.amass_chunk_attention(ctypes.byref(a), None) == status


def test_chunk_attention_refuses_a_small_or_missing_scratch():
    lib = _hip.load_library()
    a = _chunk()
    need = lib.amass_chunk_scratch_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.amass_chunk_attention(ctypes.byref(a), None) == -1
    a.scratch, a.scratch_bytes = 0x1000, need - 1
    assert lib.amass_chunk_attention(ctypes.byref(a), None) == -6
    a.scratch, a.scratch_bytes = 0x1010, need
    assert lib.amass_chunk_attention(ctypes.byref(a), None) == -6
    assert lib.amass_chunk_attention(None, None) == -1
    for empty in (dict(n_tokens=0), dict(n_req=0)):
        a = _chunk(**empty)
        assert lib.amass_chunk_scratch_bytes(ctypes.byref(a)) == 0
        assert lib.amass_chunk_attention(ctypes.byref(a), None) == 0


def test_chunk_attention_refuses_more_workgroups_than_a_launch_has():
    lib = _hip.load_library()
    a = _chunk(n_tokens=1 << 20, n_kv=4096)
    a.scratch, a.scratch_bytes = 0x1000, lib.amass_chunk_scratch_bytes(ctypes.byref(a))
    assert a.scratch_bytes > 0
    assert lib.amass_chunk_attention(ctypes.byref(a), None) == -2


def _fill(st, **over):
    a = st()
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_extend_release_and_rope_refuse():
    lib = _hip.load_library()
    P = 0x1000
    ext = dict(block_table=P, bt_st=4, seq_lens=P, query_start=P, free_list=P, top=P, top_out=P,
               slots=P, positions=P, n_req=2, n_tokens=5, max_pages=4, page=16, nb=8, capacity=8)
    for over, status in ((dict(top=None), -1), (dict(slots=None), -1), (dict(page=12), -2),
                         (dict(page=0), -2), (dict(nb=0), -2), (dict(n_tokens=-1), -2),
                         (dict(max_pages=0), -2), (dict(n_req=4097), -6)):
        a = _fill(_hip.ExtendArgs, **{**ext, **over})
        assert lib.amass_extend(ctypes.byref(a), None) == status, over
    rel = dict(block_table=P, bt_st=4, seq_lens=P, done=P, free_list=P, top=P, n_req=2,
               max_pages=4, page=16, nb=8, capacity=8)
    for over, status in ((dict(done=None), -1), (dict(page=3), -2), (dict(n_req=5000), -6)):
        a = _fill(_hip.ReleaseArgs, **{**rel, **over})
        assert lib.amass_release(ctypes.byref(a), None) == status, over
    rope = dict(q=P, q_st=4096, q_hs=128, k=P, k_st=1024, k_hs=128, q_out=P, qo_st=4096,
                qo_hs=128, k_cache=P, kc_sb=16384, kc_st=1024, kc_sh=128, table=P, tab_st=128,
                positions=P, slots=P, n_tokens=3, n_heads=32, n_kv=8, d=128, rot=128, page=16,
                nb=4, max_pos=9)
    for over, status in ((dict(q=None), -1), (dict(v=P), -1), (dict(rot=130), -2),
                         (dict(rot=3), -2), (dict(d=127), -2), (dict(page=10), -2),
                         (dict(dtype=5), -3), (dict(max_pos=0), -2), (dict(nb=0), -2),
                         (dict(n_tokens=1 << 30), -2)):       # more threads than a launch has
        a = _fill(_hip.RopeArgs, **{**rope, **over})
        assert lib.amass_rope_write(ctypes.byref(a), None) == status, over
    a = _fill(_hip.RopeArgs, **{**rope, "n_tokens": 0})
    assert lib.amass_rope_write(ctypes.byref(a), None) == 0


def test_wrappers_reject_cpu_tensors():
    i32 = dict(dtype=torch.int32)
    bt, sl, qs = torch.zeros(1, 4, **i32), torch.ones(1, **i32), torch.tensor([0, 1], **i32)
    kv = torch.zeros(4, 2, 16, 1, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    slots, pos = torch.zeros(1, dtype=torch.int64), torch.zeros(1, **i32)
    free, top = free_blocks(4, "cpu")
    for call in (lambda: paged_chunk_attention(q, kv, bt, sl, qs, q.clone()),
                 lambda: extend_block_tables(bt, sl, qs, free, top, slots, pos, page=16,
                                             num_blocks=4),
                 lambda: release_blocks(bt, sl, torch.ones(1, dtype=torch.bool), free, top,
                                        page=16, num_blocks=4),
                 lambda: rope_paged_write(q, q[:, :1], q[:, :1], pos, rope_table(64, 8), kv,
                                          slots)):
        with pytest.raises(_hip.AmassError, match="CPU tensor"):
            call()


def test_free_blocks():
    free, top = free_blocks(5, "cpu")
    assert free.tolist() == [4, 3, 2, 1, 0] and top.tolist() == [5, 0, 0]


# ---------------------------------------------------------------- rotary tables (host maths)
def test_rope_table_is_rounded_once_at_far_positions():
    table = rope_table(64, 200001, base=500000.0)
    w = 500000.0 ** (-np.arange(0, 64, 2) / 64)
    for p in (0, 1, 77777, 200000):
        want = np.concatenate([np.cos(p * w), np.sin(p * w)])
        # one rounding to fp32, and the float64 angle's own: p w 2^-52 radians
        assert np.abs(table[p].double().numpy() - want).max() <= 2.0 ** -24 + p * 2.0 ** -50


def test_rope_scalings():
    plain, one = rope_frequencies(128, base=10000.0)
    assert one == 1.0 and plain[0] == 1.0
    assert torch.allclose(plain, torch.tensor([10000.0 ** (-i / 64) for i in range(64)],
                                              dtype=torch.float64), rtol=1e-14)
    lin, _ = rope_frequencies(128, base=10000.0, scaling="linear", factor=4.0)
    assert torch.equal(lin, plain / 4.0)
    ntk, _ = rope_frequencies(128, base=10000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4.0, rel_tol=1e-12)
    parts, amp = rope_frequencies(128, base=500000.0, scaling="by_parts", factor=8.0,
                                  original_max=8192)
    base, _ = rope_frequencies(128, base=500000.0)
    turns = 8192 * base / (2 * math.pi)
    assert amp == 1.0
    assert torch.equal(parts[turns >= 4.0], base[turns >= 4.0])
    assert torch.allclose(parts[turns <= 1.0], base[turns <= 1.0] / 8.0, rtol=1e-14)
    mid = (turns > 1.0) & (turns < 4.0)
    assert mid.any() and ((parts < base) & (parts > base / 8.0))[mid].all()
    yarn, amp = rope_frequencies(128, base=10000.0, scaling="yarn", factor=16.0,
                                 original_max=4096, fast=32.0, slow=1.0)
    assert math.isclose(amp, 0.1 * math.log(16.0) + 1.0)
    assert yarn[0] == 1.0 and math.isclose(yarn[-1], plain[-1] / 16.0, rel_tol=1e-12)
    assert (yarn[1:] < yarn[:-1]).all()
    table = rope_table(128, 3, base=10000.0, scaling="yarn", factor=16.0, original_max=4096,
                       fast=32.0, slow=1.0)
    assert torch.equal(table[0, :64], torch.full((64,), amp, dtype=torch.float64).float())


@pytest.mark.parametrize("L,base", [(4096, 10000.0), (8192, 500000.0)])
def test_rope_scalings_by_their_defaults(L, base):
    """Without `fast` and `slow`: by parts between 4 turns and 1, yarn between 32 and 1."""
    rot, factor = 128, 8.0
    pairs = range(rot // 2)
    w = [base ** (-2 * i / rot) for i in pairs]
    turns = [L * x / (2 * math.pi) for x in w]
    keep = [min(max((t - 1) / 3, 0.0), 1.0) for t in turns]
    got, _ = rope_frequencies(rot, base=base, scaling="by_parts", factor=factor, original_max=L)
    assert np.allclose(got.numpy(), [x * (k + (1 - k) / factor) for x, k in zip(w, keep)], rtol=1e-11,
                       atol=0.0)
    # the last pair of at least 32 turns stays, the first of at most one is slowed whole
    first = max(i for i in pairs if turns[i] >= 32)
    last = min(i for i in pairs if turns[i] <= 1)
    slowed = [min(max((i - first) / (last - first), 0.0), 1.0) for i in pairs]
    got, _ = rope_frequencies(rot, base=base, scaling="yarn", factor=factor, original_max=L)
    assert np.allclose(got.numpy(), [x * (1 - s + s / factor) for x, s in zip(w, slowed)], rtol=1e-11,
                       atol=0.0)
    assert torch.equal(rope_table(rot, 9, base=base, scaling="yarn", factor=factor, original_max=L),
                       rope_table(rot, 9, base=base, scaling="yarn", factor=factor, original_max=L,
                                  fast=32.0, slow=1.0))


@pytest.mark.parametrize("bad", [dict(rot=7), dict(rot=0), dict(base=1.0), dict(factor=0.5),
                                 dict(scaling="by_parts", factor=2.0), dict(scaling="other"),
                                 dict(scaling="yarn", factor=2.0),
                                 dict(scaling="yarn", original_max=64, fast=1.0, slow=2.0),
                                 dict(scaling="ntk", rot=2)])
def test_rope_frequencies_refuses(bad):
    with pytest.raises(ValueError):
        rope_frequencies(**{"rot": 64, **bad})


# ---------------------------------------------------------------- the oracle itself
def test_oracle_attention_is_a_softmax():
    """Against torch's softmax of a dense causal mask, one contiguous request."""
    g = torch.Generator().manual_seed(1)
    n, H, d = 7, 4, 8
    q, k, v = (torch.randn(n, h, d, generator=g, dtype=torch.float64) for h in (H, 2, 2))
    out, lse, seen, _, _ = ochunk.attend(q.numpy(), k.numpy()[None], v.numpy()[None],
                                         np.zeros((1, 1), np.int32), [n], [0, n], scale=0.3,
                                         causal=True, window=0, page=n)
    s = 0.3 * torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1))
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
    want = torch.einsum("hij,jhd->ihd", s.softmax(-1), v.repeat_interleave(2, 1))
    assert np.allclose(out, want.numpy(), atol=1e-13)
    assert np.allclose(lse, s.logsumexp(-1).T.numpy(), atol=1e-13)
    assert seen.tolist() == list(range(1, n + 1))


def test_oracle_tables_hand_out_each_block_once():
    table, slots, pos, left, short = ochunk.extend(
        np.full((3, 4), -1), [20, 3, 33], [0, 20, 20, 21], np.arange(6), 6, 23, 16, 6)
    # request 0: two new pages; request 1 brings nothing; request 2's token starts page 2
    assert table.tolist() == [[5, 4, -1, -1], [-1] * 4, [-1, -1, 3, -1]]
    assert left == 3 and short == 0
    assert slots.tolist() == [80 + i for i in range(16)] + [64 + i for i in range(4)] + [48, -1, -1]
    assert pos[20] == 32 and pos[21] == -1
