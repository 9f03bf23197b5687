"""The operators of a paged cache held in 8 bits, as a serving program runs them.

A case is a dict of plain values; ``op`` names the operator:

  write   a step's keys (turned by their positions with the queries, where ``rot`` is not zero)
          and values quantised as they enter the cache (``quant_paged_write``)
  read    blocks of the cache read back into a 16-bit one (``quant_paged_read``)
  attend  attention of a step's new tokens over the cache (``quant_chunk_attention``)

The cache holds int8 or e4m3 codes with an fp32 scale for each block, half (K, V) and kv head.
``B`` requests bring ``n_lo`` .. ``n_hi`` new tokens each (the last one ``tail`` if that is not
zero: a prompt's chunk beside decode rows) and hold ``c_lo`` .. ``c_hi`` tokens already; a read
moves ``blocks`` blocks.  Sizes are those of the repository's benchmark configurations (8 kv
heads, 4 query heads each, 128 channels, pages of 16, 4K to 64K tokens) and generic ragged and odd
ones around them.  Queries, keys and values are N(0, 1), louder in some blocks and heads than
in others; a twentieth of the blocks hold keys pulled towards their kv head's mean query.  Block
tables are random permutations of one pool.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "amass-kv_amd"))

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "e4m3": 448.0}           # the largest code
LEAST_SCALE = 2.0 ** -64
MOST_SCALE = {"int8": 2.0 ** 121, "e4m3": 2.0 ** 119}
BASE = 500000.0                    # of the rotary frequencies
SPARE = 8                          # blocks of the pool beyond those in use
PIECE = 1 << 28                    # scores that the plain attention holds at a time

COMMON = dict(B=1, n_lo=1, n_hi=1, tail=0, c_lo=0, c_hi=0, pad=0, page=16, n_kv=8, G=4, d=128,
              dtype="bf16", code="int8", rot=128, interleaved=False, blocks=0, causal=True, window=0,
              lse=False)


def _case(name, op, **over):
    return dict(dict(COMMON, op=op, **over), name=name)


def listed():
    return [
        # a decode step of 16 users
        _case("write_16x1", "write", B=16, c_lo=1000, c_hi=60000),
        # one prompt of 8K tokens
        _case("write_1x8k", "write", n_lo=8192, n_hi=8192),
        # half of each head turned in pairs, fp16, chunks of three prompts that start inside a page
        _case("write_part_pairs", "write", B=3, n_lo=411, n_hi=771, c_hi=9000, dtype="fp16",
              code="e4m3", rot=64, interleaved=True, page=32, pad=5),
        # the pages of a short request, to the 16-bit cache that the page summaries are made from
        _case("read_37", "read", blocks=37, page=16),
        # a context of 64K tokens, fp16, heads of 64
        _case("read_64k", "read", blocks=4096, code="e4m3", dtype="fp16", n_kv=16, d=64),
        # one user's five drafted tokens to verify at 4K: latency and launches count
        _case("attend_1x5_4k", "attend", n_lo=5, n_hi=5, c_lo=4096, c_hi=4096),
        # a decode step of 64 users at 8K: the cache's bytes
        _case("attend_64x1_8k", "attend", B=64, c_lo=8000, c_hi=8191, code="e4m3"),
        # eight users' four drafted tokens at 8K to 24K
        _case("attend_8x4_24k", "attend", B=8, n_lo=4, n_hi=4, c_lo=8000, c_hi=24000, lse=True),
        # 23 decode rows beside a chunk of a thousand tokens, seven query heads per kv head
        _case("attend_mixed", "attend", B=24, c_lo=300, c_hi=9000, tail=1000, n_kv=4, G=7,
              code="e4m3"),
        # a whole prompt of 8K tokens
        _case("attend_1x8k", "attend", n_lo=8192, n_hi=8192),
        # the chunk of 2K tokens of a prompt that has 62K behind it
        _case("attend_2k_at_62k", "attend", n_lo=2048, n_hi=2048, c_lo=63488, c_hi=63488,
              code="e4m3", lse=True),
        # ragged chunks with a sliding window, heads of 64 channels in fp16, pages of 64
        _case("attend_window", "attend", B=5, n_lo=33, n_hi=1500, c_hi=12000, d=64, G=8, n_kv=2,
              dtype="fp16", window=1025, page=64, pad=13),
    ]


def _spread(rng, lo, hi):
    """A size of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend"])
    d = rng.choice([64, 128, 128])
    n_kv = rng.choice([1, 2, 3, 4, 8, 8])
    shape = dict(page=rng.choice([16, 16, 32, 64, 128]), n_kv=n_kv, d=d,
                 G=min(rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), 32 // n_kv), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 code=rng.choice(["int8", "e4m3"]))
    if op == "read":
        return dict(COMMON, op=op, blocks=_spread(rng, 1, 65536 // shape["page"]), **shape)
    if op == "write":
        B = _spread(rng, 1, 256)
        hi = _spread(rng, 1, max(1, 8192 // B))
        return dict(COMMON, op=op, B=B, n_lo=max(1, hi // rng.choice([1, 3])), n_hi=hi,
                    c_hi=_spread(rng, 1, 60000), rot=rng.choice([0, d, d, d // 2, d // 4]),
                    interleaved=rng.random() < 0.4, pad=rng.choice([0, 0, 5]), **shape)
    kind = rng.choice(["draft", "mixed", "prompt", "chunk"])
    shape.update(lse=rng.random() < 0.4, causal=rng.random() < 0.9, pad=rng.choice([0, 0, 9]))
    if kind == "draft":
        B, n = _spread(rng, 1, 32), rng.randint(1, 9)
        c = _spread(rng, 500, 24000)
        return dict(COMMON, op=op, B=B, n_lo=1, n_hi=n, c_lo=c // 3, c_hi=c, **shape)
    shape["window"] = rng.choice([0, 0, _spread(rng, 1, 5000)]) if shape["causal"] else 0
    if kind == "mixed":
        return dict(COMMON, op=op, B=_spread(rng, 2, 32), c_hi=_spread(rng, 100, 12000),
                    tail=_spread(rng, 17, 2000), **shape)
    if kind == "prompt":
        B = _spread(rng, 1, 12)
        n = _spread(rng, 17, 8192 // B)
        return dict(COMMON, op=op, B=B, n_lo=max(1, n // 5), n_hi=n, **shape)
    n = _spread(rng, 17, 2048)
    return dict(COMMON, op=op, n_lo=n, n_hi=n, c_hi=_spread(rng, 500, 60000), **shape)


# ------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """(new tokens, all tokens) of each request: the case's own lengths, the largest of them
    those it names, in an order that the seed gives."""
    B = case["B"]
    rng = random.Random(repr([case[x] for x in ("B", "n_lo", "n_hi", "c_lo", "c_hi", "tail")]))
    new = [rng.randint(case["n_lo"], case["n_hi"]) for _ in range(B)]
    had = [rng.randint(case["c_lo"], case["c_hi"]) for _ in range(B)]
    new[-1], had[0] = case["n_hi"], case["c_hi"]
    if case["tail"]:
        new[-1], had[-1] = case["tail"], had[-1] // 4
    order = random.Random(seed).sample(range(B), B)
    return [new[r] for r in order], [new[r] + had[r] for r in order]


def _tables(pages, spare, gen):
    """(block tables padded with 0, number of blocks): every request's pages are blocks of one
    random permutation."""
    total = sum(pages)
    perm = torch.randperm(total + spare, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(len(pages), max(pages), dtype=torch.int32, device=DEV)
    live = torch.arange(table.shape[1], device=DEV) < torch.tensor(pages, device=DEV)[:, None]
    table[live] = perm[:total]
    return table, total + spare


def _scale_of(most, code):
    """The scale of numbers of at most ``most``: for int8 a 127th of it, rounded up to 8
    significant bits, for e4m3 the least power of two by which it fits."""
    if code == "int8":
        bits = (most / MOST[code]).view(torch.int32)
        scale = ((bits + 0xFFFF) & -0x10000).view(torch.float32)
    else:
        part, power = torch.frexp(most)                # most = part 2^power, part in [0.5, 1)
        power = power - torch.where(part <= 0.875, 9, 8)           # 448 = 0.875 2^9
        power = torch.where(most > 0, power, -64).clamp(-64, 119).int()
        scale = ((power + 127) << 23).view(torch.float32)
    return scale.clamp(LEAST_SCALE, MOST_SCALE[code])


def _round(x, scale, code):
    """Codes of fp32 numbers (whole blocks of them are rounded half to even)."""
    y = (x / scale).clamp(-MOST[code], MOST[code])
    return (torch.round(y) if code == "int8" else y).to(CODES[code])


def _cache(case, nb, gen, mean=None):
    """(codes, scales) of a pool of nb blocks, quantised block by block."""
    page, n_kv, d = case["page"], case["n_kv"], case["d"]
    codes = torch.empty(nb, 2, page, n_kv, d, dtype=CODES[case["code"]], device=DEV)
    scales = torch.empty(nb, 2, n_kv, device=DEV)
    loud = torch.exp(0.5 * torch.randn(nb, 2, 1, n_kv, 1, generator=gen, device=DEV))
    heavy = torch.rand(nb, generator=gen, device=DEV) < 0.05
    step = max(1, (1 << 27) // (2 * page * n_kv * d))
    for i in range(0, nb, step):
        x = torch.randn(*codes[i:i + step].shape, generator=gen, device=DEV)
        if mean is None:
            x *= loud[i:i + step]
        else:                          # (louder keys would make every row see one key alone)
            x[:, 1] *= loud[i:i + step, 1]
            x[:, 0] += heavy[i:i + step, None, None, None] * mean
        x = x.to(TYPES[case["dtype"]]).float()
        s = _scale_of(x.abs().amax((2, 4)), case["code"])
        scales[i:i + step] = s
        codes[i:i + step] = _round(x, s[:, :, None, :, None], case["code"])
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    page, n_kv, d, dt = case["page"], case["n_kv"], case["d"], TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    if case["op"] == "read":
        n = case["blocks"]
        s = dict(case=case)
        s["codes"], s["scales"] = _cache(case, n + SPARE, gen)
        perm = lambda: torch.randperm(n + SPARE, generator=gen, device=DEV)[:n].int()  # noqa: E731
        s["src"], s["dst"] = perm(), perm()
        s["kv"] = torch.zeros(n + SPARE, 2, page, n_kv, d, dtype=dt, device=DEV)
        return s
    new, lens = _lengths(case, seed)
    B, T, H = case["B"], sum(new), n_kv * case["G"]
    n_tokens = T + case["pad"]
    # (a write's pool holds the pages that the step enters and no others)
    before = [(a - n) // page if case["op"] == "write" else 0 for a, n in zip(lens, new)]
    pages = [-(-a // page) - b for a, b in zip(lens, before)]
    table, nb = _tables(pages, SPARE, gen)
    s = dict(case=case, T=T, n_tokens=n_tokens, table=table,
             seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             query_start=torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32),
             out=torch.zeros(n_tokens, H, d, dtype=dt, device=DEV))
    if case["op"] == "write":
        s["codes"], s["scales"] = _cache(case, nb, gen)
        # q, k and v are views of one projection's output, as a model has them
        qkv = randn(n_tokens, H + 2 * n_kv, d)
        qkv[:, H:] *= torch.exp(0.3 * randn(n_tokens, 2 * n_kv, 1))
        s["q"], s["k"], s["v"] = qkv.to(dt).split([H, n_kv, n_kv], 1)
        req = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
        start = s["seq_lens"] - s["query_start"][1:]      # position of a token - its row
        pos = torch.arange(T, device=DEV) + start[req]
        page_in = pos // page - torch.tensor(before, device=DEV)[req]
        slot = table[req, page_in].long() * page + pos % page
        tail = torch.full((case["pad"],), -1, device=DEV)
        s["positions"], s["slots"] = torch.cat([pos, tail]).int(), torch.cat([slot, tail])
        if case["rot"]:
            freq = BASE ** (-torch.arange(0, case["rot"], 2, device=DEV).double() / case["rot"])
            angle = torch.arange(max(lens), device=DEV).double()[:, None] * freq
            s["angles"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    mean = randn(n_kv, d)
    s["q"] = (randn(n_tokens, n_kv, case["G"], d) + 0.5 * mean[:, None]).view(-1, H, d).to(dt)
    s["codes"], s["scales"] = _cache(case, nb, gen, mean)
    s["lse"] = torch.zeros(n_tokens, H, device=DEV) if case["lse"] else None
    # what the plain form does at once: (requests, their new tokens from, to)
    most = max(1, PIECE // (max(lens) * H))
    if max(new) <= 16:
        step = max(1, most // max(new))
        s["pieces"] = [(r, min(B, r + step), 0, max(new)) for r in range(0, B, step)]
    else:
        s["pieces"] = [(r, r + 1, i, min(n, i + most)) for r, n in enumerate(new)
                       for i in range(0, n, most)]
    s["pages"] = pages
    return s


# -------------------------------------------------------------------------- the plain forms
def _turned(x, cos, sin, rot, interleaved):
    """x with its first ``rot`` channels turned, in the type of cos and sin."""
    x = x.to(cos.dtype)
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _write(s):
    case, T, code, dt = s["case"], s["T"], s["case"]["code"], s["k"].dtype
    page, n_kv, d = case["page"], case["n_kv"], case["d"]
    codes, scales, out = s["codes"], s["scales"], s["out"]
    nb = len(codes)
    block, at = s["slots"][:T] // page, s["slots"][:T] % page
    k, v = s["k"][:T], s["v"][:T]
    if case["rot"]:
        cos, sin = s["angles"][s["positions"][:T].long()].chunk(2, -1)
        out[:T] = _turned(s["q"][:T], cos, sin, case["rot"], case["interleaved"]).to(dt)
        # (the keys' rounding decides their codes: in 64 bits, as it is defined)
        k = _turned(k, cos.double(), sin.double(), case["rot"], case["interleaved"]).float().to(dt)
    x = torch.stack([k, v], 1).float()                             # (T, 2, n_kv, d)
    # the blocks that the step enters: their first new row, and the largest number in each
    first = torch.full((nb,), page, device=DEV).scatter_reduce_(0, block, at, "amin")
    most = torch.zeros(nb, 2, n_kv, device=DEV).scatter_reduce_(
        0, block[:, None, None].expand(T, 2, n_kv), x.abs().amax(-1), "amax")
    entered = first < page
    keep = (first > 0)[:, None, None] & entered[:, None, None]
    new = torch.where(entered[:, None, None],
                      torch.maximum(_scale_of(most, code), torch.where(keep, scales, 0.0)), scales)
    # rows before the step's, where the scale grew
    ids = (first > 0).logical_and(entered).nonzero()[:, 0]
    held = codes[ids].float() * scales[ids][:, :, None, :, None]
    again = _round(held, new[ids][:, :, None, :, None], code)
    old = torch.arange(page, device=DEV)[:, None, None] < first[ids][:, None, None, None, None]
    grown = (new > scales)[ids][:, :, None, :, None]
    codes.view(torch.int8)[ids] = torch.where(old & grown, again.view(torch.int8),
                                              codes[ids].view(torch.int8))
    codes.view(torch.int8).transpose(1, 2)[block, at] = \
        _round(x, new[block][..., None], code).view(torch.int8)
    scales.copy_(new)
    return (out, codes, scales) if case["rot"] else (codes, scales)


def _read(s):
    src = s["src"].long()
    x = s["codes"].view(torch.int8)[src].view(s["codes"].dtype).float()
    s["kv"][s["dst"].long()] = (x * s["scales"][src][:, :, None, :, None]).to(s["kv"].dtype)
    return s["kv"]


def _attend(s):
    case, page, d = s["case"], s["case"]["page"], s["case"]["d"]
    G, n_kv, window = case["G"], case["n_kv"], case["window"]
    out, lse, qs = s["out"], s["lse"], s["query_start"]
    for r0, r1, i0, i1 in s["pieces"]:
        R, n, MP = r1 - r0, i1 - i0, max(s["pages"][r0:r1])
        row = qs[r0:r1, None] + torch.arange(i0, i1, device=DEV)
        live = row < qs[r0 + 1:r1 + 1, None]
        row_in = row.clamp(max=s["n_tokens"] - 1)
        ids = s["table"][r0:r1, :MP].long()
        kv = s["codes"].view(torch.int8)[ids].view(s["codes"].dtype).float()
        kv = kv * s["scales"][ids][:, :, :, None, :, None]         # (R, MP, 2, page, n_kv, d)
        k, v = (kv[:, :, j].reshape(R, MP * page, n_kv, d).transpose(1, 2) for j in (0, 1))
        q = s["q"][row_in].view(R, n, n_kv, G, d).permute(0, 2, 1, 3, 4)
        sc = q.reshape(R, n_kv, n * G, d).float() @ k.transpose(2, 3) * d ** -0.5
        key = torch.arange(MP * page, device=DEV)
        sl = s["seq_lens"][r0:r1, None, None]
        pos = row[:, :, None] - qs[r0 + 1:r1 + 1, None, None] + sl
        see = (key < sl) & (pos >= 0)
        if case["causal"]:
            see = see & (key <= pos)
        if window:
            see = see & (key > pos - window)
        see = see[:, None, :, None, :].expand(R, n_kv, n, G, MP * page).reshape(sc.shape)
        sc = sc.masked_fill(~see, -math.inf)
        m = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - m.clamp(min=torch.finfo(torch.float32).min))
        l = p.sum(-1, keepdim=True)
        o = (p @ v / l.clamp(min=torch.finfo(torch.float32).tiny)).view(R, n_kv, n, G, d)
        o = o.permute(0, 2, 1, 3, 4).reshape(R, n, n_kv * G, d).to(out.dtype)
        out[row[live].long()] = o[live]
        if lse is not None:
            x = (m + l.log()).view(R, n_kv, n, G).permute(0, 2, 1, 3).reshape(R, n, n_kv * G)
            lse[row[live].long()] = x[live]
    return out if lse is None else (out, lse)


# ----------------------------------------------------------------------------------- a pass
def run(s):
    case = s["case"]
    if own:
        from amass.attention import quant_chunk_attention, quant_paged_read, quant_paged_write
        if case["op"] == "write":
            if not case["rot"]:
                quant_paged_write(s["k"], s["v"], s["codes"], s["scales"], s["slots"])
                return s["codes"], s["scales"]
            quant_paged_write(s["k"], s["v"], s["codes"], s["scales"], s["slots"], q=s["q"],
                              positions=s["positions"], table=s["angles"], q_out=s["out"],
                              layout="interleaved" if case["interleaved"] else "half")
            return s["out"], s["codes"], s["scales"]
        if case["op"] == "read":
            quant_paged_read(s["codes"], s["scales"], s["src"], s["kv"], s["dst"])
            return s["kv"]
        quant_chunk_attention(s["q"], s["codes"], s["scales"], s["table"], s["seq_lens"],
                              s["query_start"], s["out"], scale=case["d"] ** -0.5,
                              causal=case["causal"], window=case["window"] or None, lse=s["lse"])
        return s["out"] if s["lse"] is None else (s["out"], s["lse"])
    return {"write": _write, "read": _read, "attend": _attend}[case["op"]](s)


def _pairs(n, length, causal, window):
    """Visible (new token, key) pairs of a request."""
    if not causal:
        return n * length
    first = length - n + 1                     # keys that the first new token sees
    if not window:
        return n * (first + length) // 2
    full = max(0, min(n, length - max(first, window) + 1))       # tokens with a whole window
    rest = n - full
    return full * window + rest * (2 * first + rest - 1) // 2


def work(case):
    d, n_kv, H, page = case["d"], case["n_kv"], case["n_kv"] * case["G"], case["page"]
    if case["op"] == "read":
        n = case["blocks"] * 2 * n_kv
        return {"bytes": n * (3 * page * d + 4) + 8 * case["blocks"], "flops": n * page * d}
    new, lens = _lengths(case, 0)
    T = sum(new)
    if case["op"] == "write":
        entered = sum(-(-a // page) - (a - n) // page for a, n in zip(lens, new))
        rot = case["rot"]
        turned = T * (4 * H * d + 4 * rot + 4) if rot else 0
        return {"bytes": turned + T * (6 * n_kv * d + 8) + 8 * entered * n_kv,
                "flops": 3 * T * (H + n_kv) * rot + 4 * T * n_kv * d}
    pairs = sum(_pairs(n, a, case["causal"], case["window"]) for n, a in zip(new, lens))
    seen = sum(min(a, case["window"] + n - 1) if case["window"] else a for n, a in zip(new, lens))
    return {"bytes": 4 * T * H * d + 2 * seen * n_kv * d + 8 * (seen // page) * n_kv +
            (4 * T * H if case["lse"] else 0),
            "flops": 4 * pairs * H * d}


# ------------------------------------------------------------- the definitions, in 64 bits
def _binade(x):
    """The powers of two at or below float64 numbers from 2^-200 on, as integers."""
    return torch.frexp(x.clamp(min=2.0 ** -200))[1].double() - 1


def _exact_codes(x, code):
    """Round half to even of float64 numbers to whole ones or to e4m3's (4 significant bits,
    steps of 2^-9 below 2^-6)."""
    if code == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(_binade(x.abs()).clamp(min=-6) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_scale(most, code):
    if code == "int8":
        grid = torch.exp2(_binade(most / 127) - 7)                 # 8 significant bits
        s = torch.ceil(most / 127 / grid) * grid
    else:
        s = torch.exp2(_binade(most / 448))
        s = torch.where(448 * s < most, 2 * s, s)
    return s.clamp(LEAST_SCALE, MOST_SCALE[code])


def exact(case, seed):
    """Outputs from the operators' definitions, request by request."""
    s = prepare(case, seed)
    page, code = case["page"], case["code"]
    if case["op"] == "read":
        kv = s["kv"].double()
        for i, j in zip(s["src"].tolist(), s["dst"].tolist()):
            kv[j] = s["codes"][i].double() * s["scales"][i].double()[:, None, :, None]
        return kv
    n_tokens = s["n_tokens"]
    qs, lens = s["query_start"].tolist(), s["seq_lens"].tolist()
    if case["op"] == "write":
        rot, T, dt = case["rot"], s["T"], s["k"].dtype
        out, k, v = s["out"].double(), s["k"][:T].double(), s["v"][:T].double()
        if rot:
            i = torch.arange(rot // 2, device=DEV)
            first = 2 * i if case["interleaved"] else i
            second = first + (1 if case["interleaved"] else rot // 2)
            w = torch.exp(-2.0 * i.double() / rot * math.log(BASE))
            angle = s["positions"][:T].double()[:, None, None] * w

            def turned(x, turn):
                y = x.clone()
                z = torch.complex(y[..., first], y[..., second]) * turn
                y[..., first], y[..., second] = z.real, z.imag
                return y

            out[:T] = turned(s["q"][:T].double(), torch.polar(torch.ones_like(angle), angle))
            held = s["angles"][s["positions"][:T].long()].double()[:, None]
            # (keys enter as the operator defines them: by the table's angles, rounded)
            k = turned(k, torch.complex(*held.chunk(2, -1))).float().to(dt).double()
        codes, scales = s["codes"].double(), s["scales"].double()
        slots = s["slots"][:T].tolist()
        t = 0
        while t < T:
            b, a = divmod(slots[t], page)
            n = 1
            while a + n < page and t + n < T and slots[t + n] == slots[t] + n:
                n += 1
            for half, x in enumerate((k, v)):
                part = x[t:t + n]                                   # (n, n_kv, d)
                step = _exact_scale(part.abs().amax((0, 2)), code)
                old = scales[b, half]
                now = torch.maximum(step, old) if a else step
                if a:
                    moved = _exact_codes(codes[b, half, :a] * old[:, None] / now[:, None], code)
                    codes[b, half, :a] = torch.where((now > old)[:, None], moved, codes[b, half, :a])
                codes[b, half, a:a + n] = _exact_codes(part / now[:, None], code)
                scales[b, half] = now
            t += n
        codes = codes.to(torch.int8) if code == "int8" else codes
        return (out, codes, scales) if rot else (codes, scales)
    G, d = case["G"], case["d"]
    out = torch.zeros(n_tokens, case["n_kv"] * G, d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device=DEV)
    for r, length in enumerate(lens):
        blocks = s["table"][r, :-(-length // page)].long()
        for h in range(case["n_kv"]):
            k, v = ((s["codes"].view(torch.int8)[blocks, j, :, h].view(s["codes"].dtype).double() *
                     s["scales"][blocks, j, h].double()[:, None, None]).view(-1, d)[:length]
                    for j in (0, 1))
            for a in range(qs[r], qs[r + 1], 512):
                b = min(qs[r + 1], a + 512)
                at = torch.arange(a, b, device=DEV) - qs[r + 1] + length
                hi = at if case["causal"] else torch.full_like(at, length - 1)
                lo = at - case["window"] + 1 if case["window"] else torch.zeros_like(at)
                key = torch.arange(length, device=DEV)
                hide = (key > hi[:, None]) | (key < lo[:, None])
                q = s["q"][a:b, h * G:(h + 1) * G].double().transpose(0, 1)
                score = (q.reshape(-1, d) @ k.T).view(G, b - a, length) / math.sqrt(d)
                score = score.masked_fill(hide, -math.inf)
                z = torch.logsumexp(score, -1)
                out[a:b, h * G:(h + 1) * G] = ((score - z[..., None]).exp() @ v).transpose(0, 1)
                lse[a:b, h * G:(h + 1) * G] = z.T
    return (out, lse) if case["lse"] else out
