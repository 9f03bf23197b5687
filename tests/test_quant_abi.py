"""include/amass_quant.h against its bindings, the entry points' refusals (checked on the host before any
launch, so no GPU is touched), the wrappers' argument checks on the CPU, and the oracle itself."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

import oracle.quant_cache as oq
from amass import _hip
from amass.attention import (quant_cache, quant_chunk_attention, quant_paged_read, quant_paged_write)

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "include", "amass_quant.h")
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
    assert set(structs) == set(_hip.QUANT_STRUCTS)
    for name, (idx, st) in _hip.QUANT_STRUCTS.items():
        assert list(st._fields_) == structs[name], name
        assert ctypes.sizeof(st) == lib.amass_quant_struct_size(idx), name
    names = re.findall(r"^\s*(?:int|int64_t|size_t)\s+(amass_\w+)\s*\(", txt, flags=re.M)
    assert len(names) == 6
    for n in names:
        assert hasattr(lib, n), n
    assert lib.amass_quant_struct_size(3) == 0
    version = int(re.search(r"AMASS_QUANT_ABI_VERSION (\d+)", txt).group(1))
    assert lib.amass_quant_abi_version() == _hip.QUANT_ABI_VERSION == version


def _fill(st, base, over):
    a = st()
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return a


P = 0x1000
CHUNK = dict(q=P, q_st=512, q_hs=128, k_codes=P, v_codes=P, c_sb=32768, c_st=1024, c_sh=128, k_scale=P,
             v_scale=P, s_sb=16, s_sh=1, block_table=P, bt_st=4, seq_lens=P, query_start=P, out=P, o_st=512,
             o_hs=128, scale=0.1, n_req=1, n_tokens=3, n_kv=8, G=4, d=128, page=16, nb=4, max_pages=4,
             causal=1)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), -1), (dict(v_codes=None), -1), (dict(k_scale=None), -1), (dict(query_start=None), -1),
    (dict(d=96), -3), (dict(dtype=2), -3), (dict(code=2), -3), (dict(code=-1), -3), (dict(page=8), -2),
    (dict(page=2048), -2), (dict(page=24), -2), (dict(scale=0.0), -2), (dict(scale=math.nan), -2),
    (dict(scale=math.inf), -2), (dict(window=-1), -2), (dict(G=0), -2), (dict(n_kv=0), -2), (dict(nb=0), -2),
    (dict(q=0x1008), -2), (dict(c_st=1032), -2), (dict(k_codes=0x1008), -2), (dict(o_hs=124), -2),
    (dict(c_st=1 << 28), -2), (dict(c_st=-1024), -2), (dict(c_sb=1 << 31), -2), (dict(c_sb=-32768), -2),
    (dict(n_tokens=1 << 29), -2), (dict(max_pages=0), -2)])
def test_attention_refuses(over, status):
    lib = _hip.load_library()
    a = _fill(_hip.QuantChunkArgs, CHUNK, over)
    assert lib.amass_quant_scratch_bytes(ctypes.byref(a)) == status
    a.scratch, a.scratch_bytes = 0x1000, 1 << 40
    assert lib.amass_quant_chunk_attention(ctypes.byref(a), None) == status


def test_attention_refuses_a_small_or_missing_scratch():
    lib = _hip.load_library()
    a = _fill(_hip.QuantChunkArgs, CHUNK, {})
    need = lib.amass_quant_scratch_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.amass_quant_chunk_attention(ctypes.byref(a), None) == -1
    for at, size in ((0x1000, need - 1), (0x1010, need)):
        a.scratch, a.scratch_bytes = at, size
        assert lib.amass_quant_chunk_attention(ctypes.byref(a), None) == -6
    assert lib.amass_quant_chunk_attention(None, None) == -1
    for empty in (dict(n_tokens=0), dict(n_req=0)):
        a = _fill(_hip.QuantChunkArgs, CHUNK, empty)
        assert lib.amass_quant_scratch_bytes(ctypes.byref(a)) == 0
        assert lib.amass_quant_chunk_attention(ctypes.byref(a), None) == 0
    a = _fill(_hip.QuantChunkArgs, CHUNK, dict(n_tokens=1 << 20, n_kv=4096))     # more workgroups than fit
    a.scratch, a.scratch_bytes = 0x1000, lib.amass_quant_scratch_bytes(ctypes.byref(a))
    assert a.scratch_bytes > 0
    assert lib.amass_quant_chunk_attention(ctypes.byref(a), None) == -2


WRITE = dict(k=P, k_st=1024, k_hs=128, v=P, v_st=1024, v_hs=128, q=P, q_st=4096, q_hs=128, q_out=P,
             qo_st=4096, qo_hs=128, k_codes=P, v_codes=P, c_sb=32768, c_st=1024, c_sh=128, k_scale=P,
             v_scale=P, s_sb=16, s_sh=1, table=P, tab_st=128, positions=P, slots=P, n_tokens=3, n_heads=32,
             n_kv=8, d=128, rot=128, page=16, nb=4, max_pos=9)
READ = dict(k_codes=P, v_codes=P, c_sb=32768, c_st=1024, c_sh=128, k_scale=P, v_scale=P, s_sb=16, s_sh=1,
            k_cache=P, v_cache=P, o_sb=32768, o_st=1024, o_sh=128, src=P, dst=P, n=3, n_kv=8, d=128,
            page=16, nb=4, nb_out=4)


@pytest.mark.parametrize("over,status", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1), (dict(k_scale=None), -1),
    (dict(q_out=None), -1), (dict(positions=None), -1), (dict(table=None), -1), (dict(rot=24), -2),
    (dict(rot=144), -2), (dict(rot=0), -2), (dict(max_pos=0), -2), (dict(d=96), -3), (dict(dtype=3), -3),
    (dict(code=2), -3), (dict(page=8), -2), (dict(page=2048), -2), (dict(page=48), -2), (dict(nb=0), -2),
    (dict(n_kv=0), -2), (dict(n_heads=0), -2), (dict(k=0x1008), -2), (dict(k_st=1020), -2),
    (dict(c_sh=136), -2), (dict(tab_st=130), -2), (dict(q_hs=132), -2), (dict(n_tokens=-1), -2),
    (dict(n_tokens=1 << 30), -2)])
def test_write_refuses(over, status):
    a = _fill(_hip.QuantWriteArgs, WRITE, over)
    assert _hip.load_library().amass_quant_write(ctypes.byref(a), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(k_codes=None), -1), (dict(v_cache=None), -1), (dict(src=None), -1), (dict(dst=None), -1),
    (dict(d=80), -3), (dict(dtype=2), -3), (dict(code=7), -3), (dict(page=8), -2), (dict(nb=0), -2),
    (dict(nb_out=0), -2), (dict(n=-1), -2), (dict(k_cache=0x1008), -2), (dict(o_st=1028), -2),
    (dict(c_st=1032), -2), (dict(n=1 << 30), -2)])
def test_read_refuses(over, status):
    a = _fill(_hip.QuantReadArgs, READ, over)
    assert _hip.load_library().amass_quant_read(ctypes.byref(a), None) == status


def test_nothing_to_do():
    lib = _hip.load_library()
    assert lib.amass_quant_write(ctypes.byref(_fill(_hip.QuantWriteArgs, WRITE, dict(n_tokens=0))), None) == 0
    assert lib.amass_quant_read(ctypes.byref(_fill(_hip.QuantReadArgs, READ, dict(n=0))), None) == 0
    assert lib.amass_quant_write(None, None) == lib.amass_quant_read(None, None) == -1


def test_wrappers_reject_cpu_tensors():
    i32 = dict(dtype=torch.int32)
    bt, sl, qs = torch.zeros(1, 4, **i32), torch.ones(1, **i32), torch.tensor([0, 1], **i32)
    codes, scales = quant_cache(4, 16, 1, 64)
    assert codes.shape == (4, 2, 16, 1, 64) and scales.shape == (4, 2, 1) and (scales == 1).all()
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: quant_chunk_attention(q, codes, scales, bt, sl, qs, q.clone()),
                 lambda: quant_paged_write(q[:, :1], q[:, :1], codes, scales,
                                           torch.zeros(1, dtype=torch.int64)),
                 lambda: quant_paged_read(codes, scales, sl, torch.zeros(4, 2, 16, 1, 64).half(), sl)):
        with pytest.raises(_hip.AmassError, match="CPU tensor"):
            call()


# ---------------------------------------------------------------- the oracle itself
def test_oracle_codes_are_the_nearest():
    g = np.random.default_rng(0)
    y = np.concatenate([g.normal(size=4000) * 150.0, g.normal(size=4000) * 2.0 ** -8, [0.5, 1.5, 2.5, -0.5]])
    c = oq.to_code(y, "int8")
    assert (np.abs(c - np.clip(y, -127, 127)) <= 0.5).all() and c[-4:].tolist() == [0.0, 2.0, 2.0, 0.0]
    every = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).double()
    every = np.unique(every[torch.isfinite(every)].numpy())
    near = every[np.abs(np.clip(y, -448, 448)[:, None] - every).argmin(1)]
    c = oq.to_code(y, "e4m3")
    assert (np.abs(c - y) <= np.abs(near - y)).all() and np.isin(c, every).all()


def test_oracle_steps_are_the_smallest():
    g = np.random.default_rng(1)
    for m in [1.0, 127.0, 448.0, 1.75, 2.0 ** -20, *np.exp(g.normal(size=200) * 10.0)]:
        m = float(torch.tensor(m).bfloat16())
        s = oq.step(m, "int8")
        assert s * 127.0 >= m and float(torch.tensor(s).bfloat16()) == s
        less = float(np.nextafter(np.float32(s), np.float32(0)))
        less = float((torch.tensor(less).view(torch.int32) & -0x10000).view(torch.float32))
        assert less * 127.0 < m
        s = oq.step(m, "e4m3")
        assert 448.0 * s >= m > 224.0 * s and math.frexp(s)[0] == 0.5
    assert oq.step(0.0, "int8") == oq.step(0.0, "e4m3") == 2.0 ** -64


def test_oracle_write_starts_a_block_anew_and_grows_it():
    codes, scales = np.full((2, 16, 1, 2), 5.0), np.full((2, 1), 0.5)
    x = np.array([[[127.0, 1.0]], [[254.0, -3.0]]])
    c, s = oq.write(codes, scales, x[:1], [16], 16, "int8")
    assert s[1, 0] == 1.0 and c[1, 0, 0].tolist() == [127.0, 1.0] and c[1, 1, 0, 0] == 5.0
    c, s = oq.write(c, s, x[1:], [17], 16, "int8")
    assert s[1, 0] == 2.0 and c[1, :2, 0].tolist() == [[64.0, 0.0], [127.0, -2.0]]
    assert (c[0] == 5.0).all() and s[0, 0] == 0.5
