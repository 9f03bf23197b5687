"""Rotary positions and the paged write on the GPU (amass_rope_write) against float64.

Tolerance.  A turned channel is x c - y s in fp32: the table's c and s are off by 2^-25 (one
rounding of a value below 1; amplitude up to 1.4 doubles it), the two products and the sum by
2^-24 of |x| + |y| each, so 2^-22 (|x| + |y|) covers them; the result is rounded once, half a
step of the type (eps / 2 of the value, 2^-25 below fp16's normal range)."""
import numpy as np
import pytest
import torch

import oracle.chunk as ochunk
from amass.attention import rope_frequencies, rope_paged_write, rope_table
from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _pairs_size(x, rot, interleaved):
    """|x| + |y| of each channel's pair; 0 for the channels that do not turn."""
    a = np.abs(x)
    size = np.zeros_like(a)
    i = np.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    size[..., p] = size[..., q] = a[..., p] + a[..., q]
    return size


def _check(got, x, positions, w, amp, rot, interleaved, dt):
    x = x.double().cpu().numpy()
    want = ochunk.rotate(x, positions, w, amp, interleaved)
    tol = (torch.finfo(dt).eps / 2 * 1.01) * np.abs(want) + \
        2.0 ** -22 * _pairs_size(x, rot, interleaved) + 2.0 ** -25
    bad = ~(np.abs(got.double().cpu().numpy() - want) <= tol)
    assert not bad.any(), np.argwhere(bad)[:4]
    copied = got[..., rot:].cpu()
    assert torch.equal(copied, torch.from_numpy(x[..., rot:]).to(dt))


SHAPES = [
    # dtype, T, H, n_kv, d, rot, layout, page, cache with the two halves first
    ("bf16", 1, 4, 1, 128, 128, "half", 16, False),
    ("bf16", 33, 32, 8, 128, 128, "half", 16, True),
    ("fp16", 17, 7, 7, 64, 64, "half", 32, False),
    ("bf16", 9, 6, 2, 128, 64, "interleaved", 16, False),
    ("fp16", 130, 3, 3, 64, 16, "interleaved", 64, False),
    ("bf16", 5, 2, 1, 128, 32, "half", 16, False),
    # shapes that 16-byte accesses do not fit
    ("bf16", 6, 3, 1, 128, 72, "half", 16, False),
    ("fp16", 6, 5, 5, 40, 40, "half", 1, False),
    ("bf16", 4, 2, 2, 66, 6, "interleaved", 16, False),
    ("fp16", 3, 1, 1, 2, 2, "half", 2, False),
]


@pytest.mark.parametrize("dtype,T,H,n_kv,d,rot,layout,page,halves_first", SHAPES)
def test_rope_write_matches_float64(dtype, T, H, n_kv, d, rot, layout, page, halves_first):
    announce(f"rope {dtype} T={T} H={H} n_kv={n_kv} d={d} rot={rot} {layout} page={page}")
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(T + rot)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dt) for h in (H, n_kv, n_kv))
    nb = -(-T // page) + 3
    max_pos = 100000
    scaling = dict(base=500000.0)
    positions = torch.randint(0, max_pos, (T,), generator=g)
    positions[0], positions[-1] = 0, max_pos - 1
    slots = torch.randperm(nb * page, generator=g)[:T]
    shape = (2, nb, page, n_kv, d) if halves_first else (nb, 2, page, n_kv, d)
    kv = torch.full(shape, 5.0, dtype=dt, device=DEV)
    out = torch.full((T, H, d), 9.0, dtype=dt, device=DEV)
    rope_paged_write(q.to(DEV), k.to(DEV), v.to(DEV), positions.int().to(DEV),
                     rope_table(rot, max_pos, device=DEV, **scaling), kv, slots.to(DEV), out,
                     layout=layout)
    w, amp = rope_frequencies(rot, **scaling)
    pairs = layout == "interleaved"
    _check(out, q, positions.numpy(), w.numpy(), amp, rot, pairs, dt)
    kc, vc = (kv[0], kv[1]) if halves_first else (kv[:, 0], kv[:, 1])
    flat_k, flat_v = (x.reshape(nb * page, n_kv, d).cpu() for x in (kc, vc))
    _check(flat_k[slots], k, positions.numpy(), w.numpy(), amp, rot, pairs, dt)
    assert torch.equal(flat_v[slots], v)
    rest = torch.ones(nb * page, dtype=torch.bool)
    rest[slots] = False
    assert (flat_k[rest] == 5.0).all() and (flat_v[rest] == 5.0).all()


def test_in_place_views_and_scaled_table():
    """q in place, q / k / v slices of one projection, a scaled table with an amplitude."""
    announce("rope: in place on a projection's slices, yarn table")
    T, H, n_kv, d, rot = 21, 4, 2, 128, 128
    dt = torch.bfloat16
    kw = dict(base=10000.0, scaling="yarn", factor=8.0, original_max=4096, fast=32.0, slow=1.0)
    qkv = torch.randn(T, H + 2 * n_kv, d, generator=torch.Generator().manual_seed(2)).to(dt)
    dev = qkv.to(DEV)
    q, k, v = dev.split([H, n_kv, n_kv], 1)
    kv = torch.zeros(2, 2, 16, n_kv, d, dtype=dt, device=DEV)
    pos = torch.arange(30000, 30000 + T)
    rope_paged_write(q, k, v, pos.int().to(DEV), rope_table(rot, 32768, device=DEV, **kw), kv,
                     torch.arange(T, device=DEV))
    w, amp = rope_frequencies(rot, **kw)
    assert amp > 1.2
    _check(dev[:, :H], qkv[:, :H], pos.numpy(), w.numpy(), amp, rot, False, dt)
    assert torch.equal(dev[:, H:].cpu(), qkv[:, H:])
    flat = kv[0].reshape(32, n_kv, d)[:T]        # (2, ...) is the two halves
    _check(flat, qkv[:, H:H + n_kv], pos.numpy(), w.numpy(), amp, rot, False, dt)


def test_padded_rows_and_rows_without_a_slot():
    announce("rope: positions and slots outside their ranges")
    T, d = 8, 64
    dt = torch.float16
    q = torch.randn(T, 2, d, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
    k, v = q[:, :1].contiguous(), q[:, 1:].contiguous()
    kv = torch.full((2, 2, 16, 1, d), 3.0, dtype=dt, device=DEV)
    out = torch.full_like(q, 9.0)
    pos = torch.tensor([-1, 0, 99, 100, 2 ** 31 - 1, 5, 6, -2 ** 31], dtype=torch.int32)
    slots = torch.tensor([1, -1, 7, 2, 3, 32, 2 ** 40, 4])
    rope_paged_write(q, k, v, pos.to(DEV), rope_table(d, 100, device=DEV), kv, slots.to(DEV), out)
    w, _ = rope_frequencies(d)
    live = [1, 2, 5, 6]
    _check(out[live], q[live], pos.numpy()[live], w.numpy(), 1.0, d, False, dt)
    assert (out[[0, 3, 4, 7]] == 9.0).all()
    flat_k, flat_v = (kv[j].reshape(32, 1, d) for j in (0, 1))
    _check(flat_k[7:8], k[2:3], pos.numpy()[2:3], w.numpy(), 1.0, d, False, dt)
    assert torch.equal(flat_v[7], v[2])
    rest = [i for i in range(32) if i != 7]
    assert (flat_k[rest] == 3.0).all() and (flat_v[rest] == 3.0).all()


def test_cache_without_v_and_far_offsets():
    """A K-only cache whose last blocks lie past 2^32 bytes."""
    announce("rope: K-only cache, blocks past 2^32 bytes")
    n_kv, d, dt = 8, 128, torch.bfloat16
    nb = (1 << 32) // (16 * n_kv * d * 2) + 64
    kv = torch.empty(nb, 1, 16, n_kv, d, dtype=dt, device=DEV)
    k = torch.randn(3, n_kv, d, generator=torch.Generator().manual_seed(1)).to(dt).to(DEV)
    q = k[:, :1].contiguous()
    slots = torch.tensor([5, (nb - 1) * 16 + 15, (nb - 40) * 16 + 2], device=DEV)
    kv.view(-1, n_kv, d)[slots] = 0
    pos = torch.zeros(3, dtype=torch.int32, device=DEV)
    rope_paged_write(q, k, None, pos, rope_table(d, 4, device=DEV), kv, slots)
    assert torch.equal(kv.view(-1, n_kv, d)[slots], k)       # (position 0 turns by nothing)


def test_captured_on_another_stream():
    announce("rope: captured and replayed with other positions and slots")
    T, H, n_kv, d, dt = 12, 4, 2, 128, torch.bfloat16
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.zeros(T, h, d, dtype=dt, device=DEV) for h in (H, n_kv, n_kv))
    kv = torch.zeros(3, 2, 16, n_kv, d, dtype=dt, device=DEV)
    pos = torch.zeros(T, dtype=torch.int32, device=DEV)
    slots = torch.zeros(T, dtype=torch.int64, device=DEV)
    out = torch.zeros(T, H, d, dtype=dt, device=DEV)
    table = rope_table(d, 1000, device=DEV)
    w, _ = rope_frequencies(d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope_paged_write(q, k, v, pos, table, kv, slots, out)
    for i in range(4):
        x = torch.randn(T, H, d, generator=g).to(dt)
        p, s = torch.randint(0, 1000, (T,), generator=g), torch.randperm(48, generator=g)[:T]
        q.copy_(x), k.copy_(x[:, :n_kv]), v.copy_(x[:, n_kv:]), pos.copy_(p), slots.copy_(s)
        graph.replay()
        _check(out, x, p.numpy(), w.numpy(), 1.0, d, False, dt)
        eager = torch.zeros_like(kv)
        rope_paged_write(q, k, v, pos, table, eager, slots, out)
        flat = lambda c: c.transpose(1, 2).reshape(48, 2, n_kv, d)[s]  # noqa: E731
        assert torch.equal(flat(kv), flat(eager))


def test_wrapper_refuses():
    announce("rope: refusals")
    dt = torch.bfloat16
    q = torch.zeros(4, 2, 64, dtype=dt, device=DEV)
    k, v = q[:, :1].contiguous(), q[:, :1].contiguous()
    kv = torch.zeros(3, 2, 16, 1, 64, dtype=dt, device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    slots = torch.zeros(4, dtype=torch.int64, device=DEV)
    table = rope_table(64, 8, device=DEV)
    good = dict(q=q, k=k, v=v, positions=pos, table=table, kv_cache=kv, slots=slots)
    wide = torch.zeros(4, 2, 128, dtype=dt, device=DEV)[:, :, ::2]
    for over in (dict(q=q.float()), dict(k=k.half()), dict(v=None), dict(v=v[:3]),
                 dict(k=k[:, :, :32]), dict(positions=pos.long()), dict(positions=pos[:3]),
                 dict(slots=slots.int()), dict(table=table.double()),
                 dict(table=rope_table(66, 8, device=DEV)), dict(q=wide), dict(layout="other"),
                 dict(q_out=torch.zeros(4, 3, 64, dtype=dt, device=DEV)),
                 dict(kv_cache=kv[:, :1]), dict(q_out=q[:1].expand(4, 2, 64)),
                 dict(q_out=q[:, :1].expand(4, 2, 64)), dict(kv_cache=kv[:1].expand(3, 2, 16, 1, 64)),
                 dict(kv_cache=kv[:, :, :1].expand(3, 2, 16, 1, 64))):
        with pytest.raises(ValueError):
            rope_paged_write(**{**good, **over})
    rope_paged_write(q[:0], k[:0], v[:0], pos[:0], table, kv, slots[:0])      # nothing to do
