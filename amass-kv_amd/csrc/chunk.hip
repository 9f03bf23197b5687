// Attention of a chunk of new tokens over the paged cache for gfx950 (amass_chunk_attention).
//
// Mathematics.  The rows of (request, kv head) are its n new tokens times the G query heads
// of the group (row rho: token rho / G, head rho % G), so a K / V tile serves all of them.
// A workgroup of four waves takes CK_BM rows (a row tile) and walks keys 64 at a time with
// the running maximum m, sum l and unnormalised output O of a softmax:
//   S^T[key][row] = K Q^T     v_mfma 32x32x16, A = K rows (LDS), B = Q^T (registers)
//   p = 2^(c s - c m), c = scale log2 e        one fma and one exp2 per score, rounded to the
//                                              element type for the second product, summed as fp32
//   O^T[d][row] += V^T P^T    A = V^T (LDS, transposing 64-bit reads), B = P^T
// In S^T a lane holds one row's scores (column = lane % 32), so the row maximum is a chain of
// v_max in the lane and one exchange with lane ^ 32, the rescale one factor per lane, and the
// accumulator registers of S^T, packed to 16 bits, already are the B operand of the second
// product: the contraction order over keys is free, and V^T is read in the order they have.
//
// K and V go from HBM to LDS with 16-byte direct loads (no registers), each lane's source
// chosen so that the LDS image is swizzled: 16-byte chunk c of row t is at chunk
// c ^ swz(t), which spreads both the K reads (16 rows, one chunk) and the transposing V reads
// (4 rows, 2 chunks) over the banks.
//
// Two layouts, chosen per row tile (d = 128, bf16, 8 kv heads of 4 query heads unless stated):
//   many (more than 32 rows): wave w owns rows 32 w .. 32 w + 31; the workgroup shares each
//     64-key tile, double-buffered (2 x 32 KB at d = 128), one barrier per tile.  The matrix cores
//     bound it: a prompt of 8192 tokens 536 us with both launches, 1.03 PFLOP/s (60 % of the matrix
//     cores' cycles, 5.8 vector instructions beside every product), 2048 tokens behind 63488
//     2007 us, 1.08 PFLOP/s (66 %), on a card whose product of 8192^3 reaches 1.24 to 1.39; 506 and
//     1853 on the fastest met.  A wave of 64 rows (O and Q in the accumulator half of the registers)
//     took 549 and 2005 us on one where this took 509 to 546 and 1869 to 2016.
//   few (32 rows or less: single tokens, drafts, a chunk's remainder): the rows fit one wave,
//     so the waves take 32 keys each in turn, each with a K and a V buffer of its own and no
//     barrier, and merge their (m, l, O) through LDS at the end.  Memory bounds it: 8 requests of 4
//     drafted tokens with 8k to 24k keys 104 us, 5.6 TB/s; 64 single tokens with 8k keys 335 us,
//     6.4 TB/s.  The many-row layout, three of four waves idle, takes 116 for the drafts.
// Splitting.  A row tile of many keys is cut into S parts when the batch has fewer tiles
// than the chip has room for (plan below, on the device: the launch needs no lengths on the
// host and can be captured); parts leave (m, l, O) in scratch and a second launch joins them.
// 5 drafted tokens behind 4096: 9.8 us of 17 parts and 4.0 us of joining (medians; least 8.7 and 3.2).
#include <atomic>
#include <type_traits>

#include "../../include/amass_chunk.h"
#include "common.h"

namespace amass {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr int CK_WAVES = 4;
// workgroups per CU (waves per SIMD): 256 registers a lane at d = 128, 170 at d = 64
constexpr int ck_wgs(int d) { return d == 128 ? 2 : 3; }
constexpr int CK_BM = 32 * CK_WAVES;       // rows of a row tile
constexpr int CK_FEW = 32;                 // rows up to which the waves share the rows
constexpr int CK_KEYS = 64;                // keys of a tile
// a row tile is cut in one part per this many tiles of keys at most: joining costs what two do (5
// tokens behind 4096: 13.1 us at 4, 14.7 at 2, 13.7 at 8)
constexpr int CK_MIN_SPLIT = 4;
// cut tiles for parts of at most 2 / 3 of the longest (at most half: 1000 tokens behind 1600 with 7
// heads per kv head 49.8 -> 59.8 us, ragged chunks under a sliding window 33.4 -> 32.0)
constexpr int CK_WORTH = 3;
// Keys that one row tile alone reads are loaded past the caches where the batch's row tiles read
// more bytes of K and V than this, half of the memory-side cache: 4 drafted tokens of 8 requests,
// 580 MB, 118 -> 103 us; 8 tokens with 8 heads per kv head, 164 MB, 43.7 -> 40.4; but 41 MB that the
// last call left there 24.1 -> 29.1 (1 kv head) and 21.8 -> 22.1 (8).
constexpr float CK_ONCE = 128e6f;
constexpr float CK_LAZY = 8.f;             // a maximum may lag by this power of two
// maxima (times c) beyond this take the products with care: there a weight may be off by 2^(1/16);
// from 16 times as much on it may exceed fp16, from 2^11 times fp32
constexpr float CK_FAR = 0x1p20f;
// Weights are 2^CK_LIFT times those of the formula (sums too, so the result is the same): fp16
// has no bits below 2^-24, and thousands of keys that far down a row count together.  2^15, the
// largest with the lag, is below fp16's largest.  bf16 has the exponents of fp32, and so has V: no
// weight exceeds 1, or a product with V near the largest value would exceed fp32.
template <int DT>
constexpr float CK_LIFT = DT == AMASS_FP16 ? 7.f : -CK_LAZY;

// ------------------------------------------------------------------ the 16-bit types
template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (DT == AMASS_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {       // to nearest even
    if constexpr (DT == AMASS_BF16) return pack_bf16x2(lo, hi);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
}
// bits 15 / 31 set where a half of x is an infinity or a NaN
template <int DT>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) {
    return DT == AMASS_BF16 ? (x & 0x7F807F80u) + 0x00800080u : (x & 0x7C007C00u) + 0x04000400u;
}
// bits 15 / 31 set where a half of x is a NaN
template <int DT>
__device__ __forceinline__ uint32_t nan2(uint32_t x) {
    return (x & 0x7FFF7FFFu) + (DT == AMASS_BF16 ? 0x007F007Fu : 0x03FF03FFu);
}

// ------------------------------------------------------------------ LDS
// XOR of a row's 16-byte chunks: the 16 rows of a K read land in 16 places of the 256 bytes
// that the banks serve, and the 4 rows (of 64 bytes) of half a wave's transposing V read in
// different quarters of them.
template <int D>
__device__ __forceinline__ int swz(int row) {
    return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3)
                    : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// (the compiler warns of m0, a reserved register, among the clobbers: the loads take their LDS address
// there, and it has to know)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes per lane from base + off (off per lane) to LDS at `to` + 16 lane (`to` uniform).
// No register waits for it: the caller waits with dma_wait before anyone reads the place.
__device__ __forceinline__ void dma16(uint32_t to, const char* base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(to), "v"(off), "s"(base)
                 : "memory", "m0");
}
// N of them, load n from base + off[n] + 1024 n to `to` + 1024 n + 16 lane: the instruction's
// offset counts on both sides, so `to` is set once.  ONCE: what nobody reads again soon (it need
// not stay in a cache).
#define CK_LOAD(n, at, hint) "\n\tglobal_load_lds_dwordx4 %" #n ", %1 offset:" #at hint
#define CK_LOADS2(hint) "s_mov_b32 m0, %0\n\ts_nop 0" CK_LOAD(2, 0, hint) CK_LOAD(3, 1024, hint)
#define CK_LOADS4(hint) CK_LOADS2(hint) CK_LOAD(4, 2048, hint) CK_LOAD(5, 0xc00, hint)
template <bool ONCE, int N>
__device__ __forceinline__ void dma16_n(uint32_t to, const char* base, const uint32_t (&off)[N]) {
    if constexpr (N == 4 && ONCE)
        asm volatile(CK_LOADS4(" nt")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[1]), "v"(off[N - 2]), "v"(off[N - 1])
                     : "memory", "m0");
    else if constexpr (N == 4)
        asm volatile(CK_LOADS4("")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[1]), "v"(off[N - 2]), "v"(off[N - 1])
                     : "memory", "m0");
    else if constexpr (ONCE)
        asm volatile(CK_LOADS2(" nt")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[1])
                     : "memory", "m0");
    else
        asm volatile(CK_LOADS2("") : : "s"(to), "s"(base), "v"(off[0]), "v"(off[1]) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void dma_wait() {        // all but the last N loads have arrived
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}
// four 16-bit values down a column of a 4-row block (lane i of 16: row i / 4, chunk half i % 4;
// returns column i)
__device__ __forceinline__ u32x2_t lds_tr4(uint32_t addr) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4_t*)(uintptr_t)addr));
}

// ------------------------------------------------------------------ ranges and plan
struct ChunkPlan {
    int sh;              // log2 page
    int cap;             // positions that a block-table row covers
    int target;          // workgroups per kv head that fill the chip
    int slots;           // scratch slots per kv head
    int slot_rows;       // rows of a slot
    int tiles_max;       // row tiles of the batch at most
    int items;           // items of the batch at most
    uint32_t g_mul;      // x / G = x g_mul >> (30 + g_sh) for x < 2^30
    int g_sh;
};

struct Span {            // keys [64 lo, 64 lo + 64 n) hold the visible ones below hi
    int lo, n, hi;
};

struct Req {
    int q0, n, len;      // first row, new tokens, tokens
};

__device__ __forceinline__ int div_g(const ChunkPlan& pl, int x) {
    return (int)(((uint64_t)(uint32_t)x * pl.g_mul) >> (30 + pl.g_sh));
}
__device__ __forceinline__ Req load_req(const amass_chunk_args& a, int r) {
    Req q;
    q.q0 = min(max(a.query_start[r], 0), a.n_tokens);
    q.n = max(min(max(a.query_start[r + 1], 0), a.n_tokens) - q.q0, 0);
    q.len = max(a.seq_lens[r], 0);
    return q;
}
__device__ __forceinline__ int row_tiles(const amass_chunk_args& a, const Req& q) {
    return (int)((uint32_t)(q.n * a.G + CK_BM - 1) / CK_BM);
}

// visible keys [lo, hi) of the token at position p
__device__ __forceinline__ int key_hi(const amass_chunk_args& a, const ChunkPlan& pl, int len, int p) {
    const int l = min(len, pl.cap);
    return p < 0 ? 0 : a.causal ? min(l, p + 1) : l;
}
__device__ __forceinline__ int key_lo(const amass_chunk_args& a, int p) {
    return a.window > 0 && p >= a.window ? p - a.window + 1 : 0;
}
__device__ __forceinline__ Span tile_span(const amass_chunk_args& a, const ChunkPlan& pl,
                                          const Req& q, int tile) {
    const int r0 = tile * CK_BM, r1 = min(q.n * a.G, r0 + CK_BM) - 1;
    const int p0 = q.len - q.n + div_g(pl, r0), p1 = q.len - q.n + div_g(pl, r1);
    Span s;
    s.hi = key_hi(a, pl, q.len, p1);
    s.lo = key_lo(a, p0) / CK_KEYS;
    s.n = max(0, (s.hi + CK_KEYS - 1) / CK_KEYS - s.lo);
    return s;
}
// the most tiles of keys that a row tile of the request has (the last one's, or under a
// window that of the last whole one)
__device__ __forceinline__ int req_work(const amass_chunk_args& a, const ChunkPlan& pl,
                                        const Req& q, int tiles) {
    int w = 0;
    if (tiles > 0) w = tile_span(a, pl, q, tiles - 1).n;
    if (tiles > 1 && a.window > 0) w = max(w, tile_span(a, pl, q, tiles - 2).n);
    return w;
}

// The batch's row tiles per kv head, `target` of which the chip takes at a time, are dispatched in
// the requests' order, a request's last (causal: longest) first.  Whole rounds of `target` tiles
// are left whole; the `rest` behind them (all of them where they are fewer than a round) is cut
// so that it fills the chip once: S_r = ceil(w_r / len) parts of a request's tiles, w_r the
// longest's tiles of keys, for the smallest len >= max(CK_MIN_SPLIT, sum_r rest_r w_r / target)
// with at most `target` parts; a shorter tile of the request has no more of them than one per
// CK_MIN_SPLIT tiles of keys that it begins.  Where some
// tile is much longer than a workgroup's share of all the work, that share is `len`, and there are
// no whole rounds.  (2100 tokens behind 60k, 66 tiles for 64: 3037 us uncut, 1951 with the rest cut.)
// Items, slots and records are bounded by the row tiles that ascending starts can make (chunk_plan
// below).  Starts that do not ascend may make more, whose items no workgroup would take and
// whose records nobody would write: such a batch is passed over whole (`fits`).
// Every wave computes it from the lengths, 64 requests at a time, one per lane; of more than 64
// requests the workgroup holds what that takes in LDS (256 single tokens with 500 keys each: 111 us
// with a round of memory per pass and 64 requests, 105 so).
struct Held {            // in LDS
    Req q;
    int tiles, work;     // row tiles, and the most tiles of keys that one has
};
struct LaneReq {
    Req q;
    int tiles, rest;     // row tiles; those behind the whole rounds (the first `rest` of them)
    float cost;          // the longest's tiles of keys
};
__device__ __forceinline__ Held held_req(const amass_chunk_args& a, const ChunkPlan& pl, int r) {
    Held h = {{0, 0, 0}, 0, 0};
    if (r < a.n_req) h.q = load_req(a, r);
    h.tiles = row_tiles(a, h.q);
    h.work = req_work(a, pl, h.q, h.tiles);
    return h;
}

struct Parts {
    const Held* held;    // the first n_held requests'
    int n_held;
    bool fits;           // no more row tiles than ascending starts make
    int whole;           // tiles of the whole rounds
    float inv;           // 1 / len, a little less, so that no rounding makes a part more
    float keys;          // tiles of keys of all row tiles
    LaneReq x0;          // of the first 64 requests
};
// (before: tiles of the requests before the 64)
__device__ __forceinline__ LaneReq lane_req(const amass_chunk_args& a, const ChunkPlan& pl,
                                            const Parts& p, int r, int before) {
    Held h;
    if (r < p.n_held) h = p.held[r];
    else h = held_req(a, pl, r);
    LaneReq x = {h.q, h.tiles, h.tiles, 0.f};
    if (p.whole > 0) {
        x.rest = min(max(before + wave_incl_scan(h.tiles) - p.whole, 0), h.tiles);
        if (x.rest < h.tiles) h.work = x.rest > 0 ? req_work(a, pl, h.q, x.rest) : 0;
    }
    x.cost = (float)h.work;
    return x;
}
__device__ __forceinline__ int parts_of(const LaneReq& x, float inv) {
    return max(1, (int)ceilf(x.cost * inv));
}
template <class F>
__device__ __forceinline__ void every_req(const amass_chunk_args& a, const ChunkPlan& pl,
                                          const Parts& p, F f) {
    f(p.x0);
    if (a.n_req <= WAVE) return;
    int before = wave_sum_uniform(p.x0.tiles);
    for (int base = WAVE; base < a.n_req; base += WAVE) {
        const LaneReq x = lane_req(a, pl, p, base + (threadIdx.x & 63), before);
        before += wave_sum_uniform(x.tiles);
        f(x);
    }
}
__device__ __forceinline__ int count_items(const amass_chunk_args& a, const ChunkPlan& pl,
                                           const Parts& p, float inv) {
    int tot = 0;
    every_req(a, pl, p, [&](const LaneReq& x) { tot += wave_sum_uniform(x.rest * parts_of(x, inv)); });
    return tot;
}
__device__ __forceinline__ Parts plan_parts(const amass_chunk_args& a, const ChunkPlan& pl,
                                            const Held* held, int n_held) {
    constexpr float LESS = 1.f - 0x1p-20f;
    const int lane = threadIdx.x & 63;
    Parts p = {held, n_held, true, 0, 0.f, 0.f, {{0, 0, 0}, 0, 0, 0.f}};
    p.x0 = lane_req(a, pl, p, lane, 0);
    int tiles;
    float work, longest, share;
    const auto add_up = [&] {
        work = 0.f;
        tiles = 0;
        longest = 0.f;
        every_req(a, pl, p, [&](const LaneReq& x) {
            work += (float)x.rest * x.cost;
            tiles = min(tiles + wave_sum_uniform(x.rest), 1 << 30);
            longest = fmaxf(longest, wave_maxf_uniform(x.cost));
        });
        work = wave_sumf_uniform(work);
        share = fmaxf((float)CK_MIN_SPLIT, work / ((float)pl.target * LESS));
    };
    // joining costs what two or three tiles do: cut only for a part well below the longest tile
    const auto pays = [&](float len) { return CK_WORTH * len <= longest * (CK_WORTH - 1); };
    add_up();
    p.keys = work;
    p.fits = tiles <= pl.tiles_max;
    if (!p.fits) return p;
    if (tiles >= pl.target) {
        if (pays(share)) {
            p.inv = LESS / share;
            return p;
        }
        p.whole = tiles - tiles % pl.target;
        p.x0 = lane_req(a, pl, p, lane, 0);
        add_up();
    }
    float len = share;
    if (len < longest && count_items(a, pl, p, LESS / len) > pl.target) {
        // parts <= cost / len + 1 each: at this length the items are few enough
        float few = fminf(longest, share * (float)pl.target / (float)(pl.target - tiles) + 1.f);
        while (few - len > len * (1.f / 32)) {
            const float mid = 0.5f * (len + few);
            if (count_items(a, pl, p, LESS / mid) <= pl.target) few = mid;
            else len = mid;
        }
        len = few;
    }
    p.inv = pays(len) ? LESS / len : LESS / fmaxf(longest, 1.f);      // (else no tile is cut)
    return p;
}

struct Item {
    int r, tile, part, parts;
    int slot;            // of this part, where parts > 1
    int cut;             // index of the row tile among those cut
    Req q;
};

// Item y of the batch; false past the end.
__device__ __forceinline__ bool find_item(const amass_chunk_args& a, const ChunkPlan& pl,
                                          const Parts& p, int y, Item& it) {
    int base = 0, before = 0, slots = 0, cuts = 0;       // those of earlier requests
    bool found = false;
    every_req(a, pl, p, [&](const LaneReq& x) {
        const int S = parts_of(x, p.inv), full = x.tiles - x.rest;
        const int n = full + x.rest * S, ns = S > 1 ? x.rest * S : 0, nc = S > 1 ? x.rest : 0;
        const int incl = wave_incl_scan(n), incl_s = wave_incl_scan(ns), incl_c = wave_incl_scan(nc);
        const int all = __builtin_amdgcn_readlane(incl, WAVE - 1);
        if (!found && y < before + all) {
            found = true;
            const int src = __ffsll((long long)__ballot(before + incl > y)) - 1;
            const int at = y - before - __builtin_amdgcn_readlane(incl - n, src);
            const int f = __builtin_amdgcn_readlane(full, src), b = at - f;
            const int s = b < 0 ? 1 : __builtin_amdgcn_readlane(S, src), t = b / s;
            it.r = base + src;
            it.parts = s;
            it.tile = b < 0 ? __builtin_amdgcn_readlane(x.tiles, src) - 1 - at
                            : __builtin_amdgcn_readlane(x.rest, src) - 1 - t;
            it.part = b < 0 ? 0 : b - t * s;
            it.slot = slots + __builtin_amdgcn_readlane(incl_s - ns, src) + b;
            it.cut = cuts + __builtin_amdgcn_readlane(incl_c - nc, src) + t;
            it.q.q0 = __builtin_amdgcn_readlane(x.q.q0, src);
            it.q.n = __builtin_amdgcn_readlane(x.q.n, src);
            it.q.len = __builtin_amdgcn_readlane(x.q.len, src);
        }
        base += WAVE;
        before += all;
        slots += __builtin_amdgcn_readlane(incl_s, WAVE - 1);
        cuts += __builtin_amdgcn_readlane(incl_c, WAVE - 1);
    });
    return found;
}
__device__ __forceinline__ int count_cut(const amass_chunk_args& a, const ChunkPlan& pl,
                                         const Parts& p) {
    int tot = 0;
    every_req(a, pl, p, [&](const LaneReq& x) {
        tot += wave_sum_uniform(parts_of(x, p.inv) > 1 ? x.rest : 0);
    });
    return tot;
}

// tiles of keys per part of a row tile of n, of whose request's longest there are `parts`
__device__ __forceinline__ int part_len(int n, int parts) {
    parts = max(1, min(parts, (n + CK_MIN_SPLIT - 1) / CK_MIN_SPLIT));
    return max(1, (n + parts - 1) / parts);
}

// ------------------------------------------------------------------ scratch
// The number of cut row tiles, a record of each, then the slots of their parts, by kv head.  A
// slot: per group of 32 rows D / 32 tiles of 16 x 64 floats, then the rows' m and l.
struct CutTile {
    int r, tile, parts, slot;
    Req q;
    int pad;
};
constexpr int CK_HEAD = 256;
constexpr int CK_STATS = 64;             // floats: m (32), l (32)

__device__ __forceinline__ CutTile* cut_tile(const amass_chunk_args& a, int i) {
    return reinterpret_cast<CutTile*>((char*)a.scratch + CK_HEAD) + i;
}
template <int D>
__device__ __forceinline__ float* slot_group(const amass_chunk_args& a, const ChunkPlan& pl, int kh,
                                             int slot, int group) {
    const int64_t at = ((int64_t)kh * pl.slots + slot) * (pl.slot_rows / 32) + group;
    return reinterpret_cast<float*>(cut_tile(a, pl.slots)) + at * (32 * D + CK_STATS);
}

// ------------------------------------------------------------------ one wave's state
template <int D>
struct RowState {
    f32x16_t o[D / 32];      // O^T: d = 32 x + 8 (i / 4) + 4 (lane / 32) + i % 4, row lane % 32
    float m, l;              // maximum (raw score); this lane's half of the sum
};

template <int D>
__device__ __forceinline__ void reset(RowState<D>& st) {
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[x][i] = 0.f;
    st.m = -__FLT_MAX__;
    st.l = 0.f;
}

// This lane's LDS reads, as byte offsets within a K or V image.  The swizzle only turns bits of
// the 16-byte chunk, and so does going to another chunk of the same row, so one offset each
// and an XOR reach all of them.
template <int D>
struct LdsLane {
    uint32_t k, v;
    __device__ __forceinline__ LdsLane(int lane) {
        const int row = lane & 31, h = lane >> 5, i16 = lane & 15, sub = (lane >> 4) & 1;
        k = row * (2 * D) + ((h ^ swz<D>(row)) << 4);
        const int t = 4 * h + (i16 >> 2), c = 2 * sub + ((i16 >> 1) & 1);
        v = t * (2 * D) + ((c ^ swz<D>(t)) << 4) + (i16 & 1) * 8;
    }
    // channels 16 i + 8 h .. of key row % 32 + 32 x
    __device__ __forceinline__ u32x4_t k_frag(uint32_t ks, int i, int x) const {
        return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)(
            ((ks + k) ^ (uint32_t)(i << 5)) + x * (64 * D));
    }
    // d tile x of the 16 keys from 16 y: four keys from 4 h, four from 8 + 4 h (whose rows
    // turn the chunk's second bit)
    __device__ __forceinline__ u32x4_t v_frag(uint32_t vs, int x, int y) const {
        const uint32_t at = (vs + v) ^ (uint32_t)(x << 6);
        const u32x2_t a = lds_tr4(at + y * (32 * D));
        const u32x2_t b = lds_tr4((at ^ 32u) + y * (32 * D) + 16 * D);
        return (u32x4_t){a[0], a[1], b[0], b[1]};
    }
};

// S^T of 32 NK keys
template <int DT, int D, int NK>
__device__ __forceinline__ void scores(uint32_t ks, const LdsLane<D>& ll,
                                       const u32x4_t (&q)[D / 16], f32x16_t (&s)[NK]) {
#pragma unroll
    for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int x = 0; x < NK; ++x)
            s[x] = mfma32<DT>(ll.k_frag(ks, i, x), q[i], s[x]);
}

// -inf for the keys (relative to the tile) outside [lo, hi) of this lane's row, and those of
// 16-key groups without a block
template <int NK>
__device__ __forceinline__ void mask_scores(f32x16_t (&s)[NK], int lo, int hi, uint32_t groups,
                                            int lane) {
    const int h4 = 4 * (lane >> 5);
    lo -= h4;
    hi -= h4;
#pragma unroll
    for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = 32 * x + 8 * (i >> 2) + (i & 3);
            const bool see = key >= lo && key < hi && (groups >> (2 * x + (i >> 3)) & 1);
            s[x][i] = see ? s[x][i] : -INFINITY;
        }
}

// The running maximum after these scores, and the rescale of what was summed.  The maximum
// may lag the true one by 2^CK_LAZY, which the weights (of any size) and fp32 sums hold exactly
// as well, so most tiles skip the rescale.
__device__ __forceinline__ float row_max(const f32x16_t& s) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    return mx;
}
// O times al, passed over where every lane's is 1.  Written out with its own skip, on registers
// of its own choice: as a branch of the program the products would be new values, and the compiler moves
// all of O (64 registers) twice a tile to join them.  The waits cover a matrix product's result
// before, and its operand after.
#define CK_MUL1(r) "v_mul_f32 v" #r ", %[al], v" #r "\n\t"
#define CK_MUL16(a, b, c, d, e, f, g, h, i, j, k, l, m, n, o, p)                               \
    CK_MUL1(a) CK_MUL1(b) CK_MUL1(c) CK_MUL1(d) CK_MUL1(e) CK_MUL1(f) CK_MUL1(g) CK_MUL1(h)     \
    CK_MUL1(i) CK_MUL1(j) CK_MUL1(k) CK_MUL1(l) CK_MUL1(m) CK_MUL1(n) CK_MUL1(o) CK_MUL1(p)
#define CK_MUL_0 CK_MUL16(128, 129, 130, 131, 132, 133, 134, 135, 136, 137, 138, 139, 140, 141, 142, 143)
#define CK_MUL_1 CK_MUL16(144, 145, 146, 147, 148, 149, 150, 151, 152, 153, 154, 155, 156, 157, 158, 159)
#define CK_MUL_2 CK_MUL16(160, 161, 162, 163, 164, 165, 166, 167, 168, 169, 170, 171, 172, 173, 174, 175)
#define CK_MUL_3 CK_MUL16(176, 177, 178, 179, 180, 181, 182, 183, 184, 185, 186, 187, 188, 189, 190, 191)
#define CK_SKIP "v_cmp_neq_f32 vcc, 1.0, %[al]\n\ts_cbranch_vccz 1f\n\ts_nop 15\n\ts_nop 15\n\t"
template <int D>
__device__ __forceinline__ void scale_o(RowState<D>& st, float al) {
    if constexpr (D == 128)
        asm volatile(CK_SKIP CK_MUL_0 CK_MUL_1 CK_MUL_2 CK_MUL_3 "s_nop 7\n1:"
                     : "+{v[128:143]}"(st.o[0]), "+{v[144:159]}"(st.o[1]),
                       "+{v[160:175]}"(st.o[D / 32 - 2]), "+{v[176:191]}"(st.o[D / 32 - 1])
                     : [al] "v"(al)
                     : "vcc");
    else
        asm volatile(CK_SKIP CK_MUL_0 CK_MUL_1 "s_nop 7\n1:"
                     : "+{v[128:143]}"(st.o[0]), "+{v[144:159]}"(st.o[1])
                     : [al] "v"(al)
                     : "vcc");
}
// the maximum and the sum for a higher maximum; the factor for O
template <int D>
__device__ __forceinline__ float raise(float mx, float c, RowState<D>& st) {
    const float m = fmaxf(st.m, mx);
    const float al = __builtin_amdgcn_exp2f((st.m - m) * c);
    st.m = m;
    st.l *= al;
    return al;
}
template <int D>
__device__ __forceinline__ bool lags(float mx, float c, const RowState<D>& st) {
    return __any((mx - st.m) * c > CK_LAZY);
}
template <int D, int NK>
__device__ __forceinline__ void maximum(const f32x16_t (&s)[NK], float c, RowState<D>& st) {
    float mx = row_max(s[0]);
    if constexpr (NK == 2) mx = fmaxf(mx, row_max(s[1]));
    mx = xor32_maxf(mx);
    float al = 1.f;
    const bool lag = lags(mx, c, st);
    if (lag) al = raise(mx, c, st);
    scale_o(st, al);
}

// Weights p = 2^(c s - c m) and O^T += V^T P^T, 32 keys at a time: the exponentials of the
// second 32 run under the products of the first.  Scores (2 x, 8 y ..) packed are the B operand of
// 16-key step 2 x + y.
template <int DT, int D, int NK>
__device__ __forceinline__ void weigh(uint32_t vs, const LdsLane<D>& ll, const f32x16_t (&s)[NK],
                                      float c, RowState<D>& st) {
    const float mc = fmaxf(st.m * c, -__FLT_MAX__) - CK_LIFT<DT>;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NK; ++x) {
        u32x4_t p[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], c, -mc));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i + 1], c, -mc));
            sum[i & 2] += e0;
            sum[(i & 2) + 1] += e1;
            p[i >> 3][(i >> 1) & 3] = pack2<DT>(e0, e1);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int z = 0; z < D / 32; ++z)
                st.o[z] = mfma32<DT>(ll.v_frag(vs, z, 2 * x + y), p[y], st.o[z]);
    }
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A tile of 64 keys, in a fixed order (each step ends in a scheduling
// barrier): the matrix products follow each other with four fragments in flight, and the
// vector work runs under them:
//   scores of keys 0..31 | scores of 32..63, weights of 0..31 | maximum |
//   products with V of 0..31, weights of 32..63 | products with V of 32..63
// The first weights are made with the maximum so far and made again in the rare tile whose
// scores exceed it by more than it may lag.  MASKS: the lane's row sees the keys [lo, hi) of the
// tile; without, all.
template <int DT, int D, bool MASKS>
__device__ __forceinline__ void ordered_tile(uint32_t ks, uint32_t vs, const LdsLane<D>& ll,
                                             const u32x4_t (&q)[D / 16], float c, RowState<D>& st,
                                             int lo, int hi, int lane) {
    lo -= 4 * (lane >> 5);
    hi -= 4 * (lane >> 5);
    const uint32_t seen = (uint32_t)max(hi - lo, 0);
    const auto masked = [&](float v, int x, int i) {
        const int key = 32 * x + 8 * (i >> 2) + (i & 3);
        return !MASKS || (uint32_t)(key - lo) < seen ? v : -INFINITY;
    };
    constexpr int N = D / 16, Z = D / 32;      // products of 32 keys with K or V; d tiles
    u32x4_t f[4], p[4];
    f32x16_t s[2], zero;
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0.f;
    const auto k_frag = [&](int n) { return ll.k_frag(ks, n % N, n / N); };
    const auto step = [] { __builtin_amdgcn_sched_barrier(0); };
    float mc = fmaxf(st.m * c, -__FLT_MAX__) - CK_LIFT<DT>, sum[4] = {0.f, 0.f, 0.f, 0.f};
    const auto weight = [&](int x, int i, bool fresh = true) {    // weights 2 i and 2 i + 1 of half x
        if (x == 0 && fresh) {                 // (half 1 is masked before the maximum)
            s[0][2 * i] = masked(s[0][2 * i], 0, 2 * i);
            s[0][2 * i + 1] = masked(s[0][2 * i + 1], 0, 2 * i + 1);
        }
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][2 * i], c, -mc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][2 * i + 1], c, -mc));
        sum[2 * (i & 1)] += e0;
        sum[2 * (i & 1) + 1] += e1;
        uint32_t w = pack2<DT>(e0, e1);
        asm volatile("" : "+v"(w));            // (made here, not behind the branch below)
        p[2 * x + (i >> 2)][i & 3] = w;
    };
#pragma unroll
    for (int n = 0; n < 4; ++n) f[n] = k_frag(n);
    step();
    __builtin_amdgcn_s_setprio(1);             // (products before the other wave's vector work)
#pragma unroll
    for (int n = 0; n < N; ++n) {
        s[0] = mfma32<DT>(f[n & 3], q[n], n ? s[0] : zero);
        f[n & 3] = k_frag(n + 4);
        step();
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        s[1] = mfma32<DT>(f[n & 3], q[n], n ? s[1] : zero);
        if (n + 4 < N) f[n & 3] = k_frag(N + n + 4);
        else f[n & 3] = ll.v_frag(vs, (n + 4 - N) % Z, (n + 4 - N) / Z);
#pragma unroll
        for (int i = 8 * n / N; i < 8 * (n + 1) / N; ++i) weight(0, i);
        step();
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (MASKS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[1][i] = masked(s[1][i], 1, i);
    }
    const float mx = xor32_maxf(fmaxf(row_max(s[0]), row_max(s[1])));
    const bool lag = lags(mx, c, st);
    float al = 1.f;
    if (lag) {
        al = raise(mx, c, st);
        mc = fmaxf(st.m * c, -__FLT_MAX__) - CK_LIFT<DT>;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) weight(0, i, false);
    }
    scale_o(st, al);
    __builtin_amdgcn_s_setprio(1);
    step();
    // V fragment n: 16-key step n / Z, d tile n % Z
#pragma unroll
    for (int n = 0; n < 2 * N; ++n) {
        st.o[n % Z] = mfma32<DT>(f[n & 3], p[n / Z], st.o[n % Z]);
        if (n + 4 < 2 * N) f[n & 3] = ll.v_frag(vs, (n + 4) % Z, (n + 4) / Z);
        if (n < N) {
#pragma unroll
            for (int i = 8 * n / N; i < 8 * (n + 1) / N; ++i) weight(1, i);
        }
        step();
    }
    __builtin_amdgcn_s_setprio(0);
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// whether a row that is there needs the products with care below.  Either O is not finite: V of keys
// that the row sees is not, or of keys that it does not see (zero times that is NaN, and stays).
// Asked once per row tile, 64 products a lane; asking V of every tile with masks takes 160
// instructions and 32 LDS reads each time.  Or the maximum is far from zero: the weights' exponents
// are c s less c m rounded, which is off by 2^-24 of it, and then a weight of one turns to 0 or infinity.
template <int D>
__device__ __forceinline__ bool needs_care(const RowState<D>& st, float c, bool live) {
    float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i & 3] = __builtin_fmaf(st.o[x][i], 0.f, z[i & 3]);
    const bool far = st.m > -__FLT_MAX__ && fabsf(st.m) * c > CK_FAR;
    return __any(live && (far || !((z[0] + z[1]) + (z[2] + z[3]) == 0.f)));
}

// `weigh` with exponents from s - m, exact where s is near m, and for V that is not finite
// everywhere, where the weight zero of a key that a row does not see would make NaN.  The products
// take zeros in place of what is not finite; then products of the largest bf16 values (where a row
// sees a key that is not finite in the channel; zeros elsewhere) make an infinity of V's sign of
// that row's channel, and one of the opposite sign too, NaN with the first, where V is NaN.  Rare,
// and written for few registers.
template <int DT, int D, int NK>
__device__ __forceinline__ void weigh_careful(uint32_t vs, const LdsLane<D>& ll,
                                              const f32x16_t (&s)[NK], float c, RowState<D>& st) {
    constexpr uint32_t MOST = 0x7F7Fu;
    const auto step = [] { __builtin_amdgcn_sched_barrier(0); };
    const auto halves = [](uint32_t tops) { return ((tops >> 15) & 0x00010001u) * 0xFFFFu; };
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < 2 * NK; ++y) {
        u32x4_t p, see;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float s0 = s[y >> 1][8 * (y & 1) + i], s1 = s[y >> 1][8 * (y & 1) + i + 1];
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0 - st.m, c, CK_LIFT<DT>));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s1 - st.m, c, CK_LIFT<DT>));
            sum += e0 + e1;
            p[i >> 1] = pack2<DT>(e0, e1);
            see[i >> 1] = (s0 != -INFINITY ? MOST : 0u) | (s1 != -INFINITY ? MOST << 16 : 0u);
            step();
        }
#pragma unroll
        for (int z = 0; z < D / 32; ++z) {
            u32x4_t v = ll.v_frag(vs, z, y), most, other;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t bad = halves(nonfinite2<DT>(v[j])), nan = halves(nan2<DT>(v[j]));
                most[j] = bad & (MOST << 16 | MOST | (v[j] & 0x80008000u));
                other[j] = nan & (most[j] ^ 0x80008000u);
                v[j] &= ~bad;
            }
            st.o[z] = mfma32<DT>(v, p, st.o[z]);
            st.o[z] = mfma32<AMASS_BF16>(most, see, st.o[z]);
            st.o[z] = mfma32<AMASS_BF16>(other, see, st.o[z]);
            step();
        }
    }
    st.l += sum;
}

// ------------------------------------------------------------------ staging
// One request's pages of one kv head.  Everything but the lane offsets is uniform.
template <int D>
struct Pages {
    static constexpr int ROWS = 512 / D;           // rows of one 1-KB load
    static constexpr int LOADS = 16 / ROWS;        // loads of 16 rows
    static constexpr int BACK = 1024 * (LOADS - 1);
    const __attribute__((address_space(4))) int32_t* table;   // the request's row
    const char* k;                                 // of the kv head, BACK before it
    int64_t to_v;                                  // from a K row to its V row
    uint32_t sb, st;                               // bytes of a block, a row
    int sh, nb, last;                              // last: a position that has a table entry
    uint32_t lane_off[LOADS];                      // this lane's source in a 16-row group, less the
                                                   // load's own 1024 n, from BACK before it
    int lane;

    __device__ __forceinline__ Pages(const amass_chunk_args& a, const ChunkPlan& pl, int r, int kh,
                                     int hi, int lane_)
        : table((const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.block_table +
                                                                              r * a.bt_st)),
          k((const char*)a.k + kh * a.kv_sh * 2 - BACK), to_v((const char*)a.v - (const char*)a.k),
          sb((uint32_t)a.kv_sb * 2), st((uint32_t)a.kv_st * 2), sh(pl.sh), nb(a.nb),
          last(max(hi - 1, 0)), lane(lane_) {
        const int chunk = lane & (D / 8 - 1), lr = lane / (D / 8);
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int row = ROWS * n + lr;
            lane_off[n] = (uint32_t)row * st + ((uint32_t)(chunk ^ swz<D>(row)) << 4) + BACK - 1024 * n;
        }
    }
    // table entry of position t (of `last` behind it) and whether the pool has that block
    __device__ __forceinline__ int entry(int t) const { return table[min(t, last) >> sh]; }
    __device__ __forceinline__ bool has(int id) const { return (uint32_t)id < (uint32_t)nb; }
    __device__ __forceinline__ const char* row(int id, int t) const {
        return k + (uint64_t)(uint32_t)id * sb + (uint32_t)(t & ((1 << sh) - 1)) * st;
    }
    // 16 rows to LDS
    template <bool ONCE = false>
    __device__ __forceinline__ void load(uint32_t to, const char* src) const {
        dma16_n<ONCE>(to, src, lane_off);
    }
    __device__ __forceinline__ void load(uint32_t to, const char* src, bool once) const {
        if (once) load<true>(to, src);
        else load(to, src);
    }
    // the first `rows` of 16 rows, zero behind them (the weight of a masked key is zero, and
    // zero times what lies behind a request's last token could be NaN)
    __device__ __forceinline__ void load_part(char* dst, uint32_t to, const char* src,
                                              int rows) const {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            if (ROWS * n + lane / (D / 8) < rows) dma16(to + 1024 * n, src + 1024 * n, lane_off[n]);
            else *reinterpret_cast<u32x4_t*>(dst + 1024 * n + 16 * lane) = (u32x4_t){0u, 0u, 0u, 0u};
        }
    }
};

// ------------------------------------------------------------------ results
// Rows of a wave, normalised: 16 bytes per store after an exchange between the half waves
// (lane l: d 32 x + 16 u .. + 7, lane l + 32: the next 8).
template <int DT, int D>
__device__ __forceinline__ void store_row(uint16_t* out, int x, const float (&o)[16], int lane) {
    // (out: the row, null for none; x: the d tile)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        uint32_t e[2], f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const auto s = __builtin_amdgcn_permlane32_swap(
                pack2<DT>(o[8 * u + 2 * j], o[8 * u + 2 * j + 1]),
                pack2<DT>(o[8 * u + 4 + 2 * j], o[8 * u + 4 + 2 * j + 1]), false, false);
            e[j] = s[0];
            f[j] = s[1];
        }
        if (out)
            *reinterpret_cast<u32x4_t*>(out + 32 * x + 16 * u + 8 * (lane >> 5)) =
                (u32x4_t){e[0], e[1], f[0], f[1]};
    }
}

template <int D>
__device__ __forceinline__ void save_tile(float* g, int x, const float (&o)[16], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(g + (x * 4 + i) * 4 * WAVE + 4 * lane) =
            make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
}

template <int D>
__device__ __forceinline__ void save_stats(float* g, float m, float l, int lane) {
    g[32 * D + lane] = lane < 32 ? m : l;        // (both halves of the wave hold the rows)
}

struct RowOut {
    uint16_t* out;       // the row, null for none
    float* lse;
};

__device__ __forceinline__ RowOut row_out(const amass_chunk_args& a, const ChunkPlan& pl,
                                          const Req& q, int kh, int row) {
    RowOut w = {nullptr, nullptr};
    if (row < q.n * a.G) {
        const int i = div_g(pl, row);
        const int64_t t = q.q0 + i;
        const int64_t h = kh * a.G + (row - i * a.G);
        w.out = (uint16_t*)a.out + t * a.o_st + h * a.o_hs;
        if (a.lse) w.lse = a.lse + t * a.l_st + h * a.l_hs;
    }
    return w;
}

template <int DT>
__device__ __forceinline__ void store_lse(const RowOut& w, float m, float l, float c, int lane) {
    if (w.lse && lane < 32) {
        *w.lse = l == 0.f ? -INFINITY : (m * c - CK_LIFT<DT> + __log2f(l)) * 0.693147180559945309f;
    }
}

template <int D>
struct __align__(1024) ChunkLds {
    char kv[2 * 2 * CK_KEYS * 2 * D];              // staging, then the waves' O
    float m[CK_WAVES][WAVE], l[CK_WAVES][WAVE];
    int gaps[CK_WAVES];                            // a page without a block
    int bad[CK_WAVES];                             // rows that need care
};

// ------------------------------------------------------------------ kernel
// grid: kv head fastest (workgroups of one kv head share an XCD's L2 where n_kv is a multiple
// of 8), then the items.
template <int DT, int D>
__global__ __launch_bounds__(CK_WAVES * WAVE)
__attribute__((amdgpu_waves_per_eu(ck_wgs(D), ck_wgs(D)))) void
chunk_kernel(const amass_chunk_args a, const ChunkPlan pl) {
    __shared__ ChunkLds<D> lds;
    constexpr int KB = CK_KEYS * 2 * D;            // bytes of a K (or V) tile
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kh = blockIdx.x % a.n_kv;
    Item it;
    float keys;
    {
        Held* held = reinterpret_cast<Held*>(lds.kv);
        const int n_held = a.n_req > WAVE ? min(a.n_req, (int)(sizeof(lds.kv) / sizeof(Held))) : 0;
        for (int r = threadIdx.x; r < n_held; r += CK_WAVES * WAVE) held[r] = held_req(a, pl, r);
        if (n_held > 0) __syncthreads();
        const Parts p = plan_parts(a, pl, held, n_held);
        if (blockIdx.x == 0 && w == 0) {
            const int cuts = p.fits ? count_cut(a, pl, p) : 0;
            if (lane == 0) *(int*)a.scratch = cuts;
        }
        keys = p.keys;
        if (!p.fits || !find_item(a, pl, p, blockIdx.x / a.n_kv, it)) return;
        if (n_held > 0) __syncthreads();           // (before the keys take its place)
    }
    const Span sp = tile_span(a, pl, it.q, it.tile);
    const int per = part_len(sp.n, it.parts);
    const int j0 = min(sp.n, it.part * per), j1 = min(sp.n, j0 + per);   // tiles of this part
    if (it.part > 0 && j0 >= j1) return;
    const bool whole = per >= sp.n;                // no other part has keys
    if (it.parts > 1 && it.part == 0 && kh == 0 && threadIdx.x == 0)
        *cut_tile(a, it.cut) = {it.r, it.tile, (sp.n + per - 1) / per, it.slot, it.q, 0};
    const int rows = min(CK_BM, it.q.n * a.G - it.tile * CK_BM);
    const bool few = rows <= CK_FEW;
    const bool once = it.q.n * a.G <= CK_BM &&
                      __builtin_amdgcn_readfirstlane(keys * (float)(2 * KB) * (float)a.n_kv > CK_ONCE);
    const int group = few ? 0 : w;                 // 32-row group of this wave
    const int row = it.tile * CK_BM + 32 * group + (lane & 31);
    const int last = it.tile * CK_BM + min(rows, 32 * group + 32) - 1;    // of the wave
    const int start = it.q.len - it.q.n;
    const float c = a.scale * 1.44269504088896341f;
    const Pages<D> pg(a, pl, it.r, kh, sp.hi, lane);
    const int len = min(it.q.len, pl.cap);
    // this lane's visible keys; the wave's rows see at least [lo_hi, hi_lo), at most [lo_lo, hi_hi)
    const bool live = row < it.q.n * a.G;
    const int tok = div_g(pl, row);
    const int pos = start + tok;
    const int hi = live ? key_hi(a, pl, it.q.len, pos) : 0, lo = live ? key_lo(a, pos) : 0;
    const int first = it.tile * CK_BM + 32 * group;
    const bool idle = first > last;
    const int p_first = start + div_g(pl, first), p_last = start + div_g(pl, last);
    const int hi_lo = key_hi(a, pl, it.q.len, p_first), hi_hi = key_hi(a, pl, it.q.len, p_last);
    const int lo_lo = key_lo(a, p_first), lo_hi = key_lo(a, p_last);

    u32x4_t q[D / 16];
    {
        const uint16_t* src = (const uint16_t*)a.q + (int64_t)(it.q.q0 + tok) * a.q_st +
                              (int64_t)(kh * a.G + (row - tok * a.G)) * a.q_hs + 8 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            q[i] = live ? *reinterpret_cast<const u32x4_t*>(src + 16 * i) : (u32x4_t){0u, 0u, 0u, 0u};
    }
    // (here, not in the loop over the keys, where a wait would also wait for the next tile's loads)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(q[i]));
    const LdsLane<D> ll(lane);
    RowState<D> st;
    reset(st);

    if (!few) {
        // ---- many rows: the workgroup shares the tiles -------------------------------------
        // Wave w requests the 16 keys 64 j + 16 w .. of tile j, one tile ahead; their table entry
        // is looked up another tile ahead, so that no request waits for it.
        const uint32_t base = lds_addr(lds.kv);
        int t_next = CK_KEYS * (sp.lo + j0) + 16 * w, id = pg.entry(t_next);
        const auto request = [&](int buf) {
            const uint32_t kd = base + 2 * KB * buf + 16 * w * 2 * D, vd = kd + KB;
            const char* src = pg.row(id, t_next);
            if (t_next + 16 <= len && pg.has(id)) {
                if (once) {
                    pg.template load<true>(kd, src);
                    pg.template load<true>(vd, src + pg.to_v);
                } else {
                    pg.load(kd, src);
                    pg.load(vd, src + pg.to_v);
                }
            } else {
                const int rows = pg.has(id) ? min(len - t_next, 16) : 0;
                if (rows > 0) pg.load(kd, src);
                pg.load_part(lds.kv + (vd - base), vd, src + pg.to_v, rows);
            }
            t_next += CK_KEYS;
            id = pg.entry(t_next);
        };
        // whether every page that a row of the workgroup sees in this part has a block
        {
            bool has = true;
            const int from = max(CK_KEYS * (sp.lo + j0), key_lo(a, start + div_g(pl, it.tile * CK_BM)));
            const int to = (min(CK_KEYS * (sp.lo + j1), sp.hi) - 1) >> pg.sh;    // the last page
            for (int p = (from >> pg.sh) + threadIdx.x; p <= to; p += CK_WAVES * WAVE)
                has &= pg.has(a.block_table[it.r * a.bt_st + p]);
            const bool all = __all(has);
            if (lane == 0) lds.gaps[w] = !all;
        }
        const auto turn = [&](int j) {
            dma_wait<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (j + 1 < j1) request((j + 1 - j0) & 1);
        };
        const auto seen = [&](int j) {             // by some row of the wave
            const int t0 = CK_KEYS * (sp.lo + j);
            return !idle && t0 < hi_hi && t0 + CK_KEYS > lo_lo;
        };
        const auto tile = [&](int j, auto masks) {
            const uint32_t ks = base + 2 * KB * ((j - j0) & 1);
            const int t0 = CK_KEYS * (sp.lo + j);
            ordered_tile<DT, D, masks>(ks, ks + KB, ll, q, c, st, lo - t0, hi - t0, lane);
        };
        bool again = false;
        if (j0 < j1) {
            request(0);
            turn(j0);
            again = __builtin_amdgcn_readfirstlane(lds.gaps[0] | lds.gaps[1] | lds.gaps[2] |
                                                   lds.gaps[3]) != 0;
        }
        if (!again) {
            // tiles [f0, f1) hold only keys that all of the wave's rows see
            const int f1 = idle ? j1 : min(j1, hi_lo / CK_KEYS - sp.lo);
            const int f0 = idle ? j1 : min(f1, max(j0, (lo_hi + CK_KEYS - 1) / CK_KEYS - sp.lo));
            int j = j0;
            while (j < f0) {
                if (seen(j)) tile(j, std::true_type());
                if (++j < j1) turn(j);
            }
            while (j < f1) {
                tile(j, std::false_type());
                if (++j < j1) turn(j);
            }
            while (j < j1) {
                if (seen(j)) tile(j, std::true_type());
                if (++j < j1) turn(j);
            }
            const bool bad = needs_care(st, c, live);
            if (lane == 0) lds.bad[w] = bad;
            __syncthreads();
            again = __builtin_amdgcn_readfirstlane(lds.bad[0] | lds.bad[1] | lds.bad[2] |
                                                   lds.bad[3]) != 0;
        }
        // Pages without a block, something that is not finite or far from zero: (all over again) with
        // care
        if (again) {
            reset(st);
            t_next = CK_KEYS * (sp.lo + j0) + 16 * w;
            id = pg.entry(t_next);
            request(0);
            for (int j = j0; j < j1; ++j) {
                turn(j);
                if (!seen(j)) continue;
                const uint32_t ks = base + 2 * KB * ((j - j0) & 1);
                const int t0 = CK_KEYS * (sp.lo + j);
                uint32_t groups = 0;
#pragma unroll
                for (int g = 0; g < 4; ++g) groups |= (pg.has(pg.entry(t0 + 16 * g)) ? 1u : 0u) << g;
                f32x16_t s[2];
                scores<DT, D, 2>(ks, ll, q, s);
                mask_scores<2>(s, lo - t0, hi - t0, groups, lane);
                maximum<D, 2>(s, c, st);
                weigh_careful<DT, D, 2>(ks + KB, ll, s, c, st);
            }
        }
    } else {
        // ---- few rows: each wave its own 32 keys, w + 4, w + 8, ... ------------------------
        constexpr int HB = KB / 2;                 // 32 keys
        char* own = lds.kv + 2 * HB * w;           // K, then V
        const uint32_t base = lds_addr(own);
        constexpr int LOADS = 2 * Pages<D>::LOADS;
        const int b0 = 2 * (sp.lo + j0) + w, b1 = 2 * (sp.lo + j1);
        int id[2];
        const auto find = [&](int b) {
#pragma unroll
            for (int g = 0; g < 2; ++g) id[g] = pg.entry(32 * b + 16 * g);
        };
        // both return whether the usual number of loads is in flight
        const auto issue_k = [&](int b) -> bool {
#pragma unroll
            for (int g = 0; g < 2; ++g)
                if (pg.has(id[g])) pg.load(base + g * (HB / 2), pg.row(id[g], 32 * b + 16 * g), once);
            return pg.has(id[0]) && pg.has(id[1]);
        };
        const auto issue_v = [&](int b) -> bool {
            if (pg.has(id[0]) && pg.has(id[1]) && 32 * b + 32 <= len) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
                    pg.load(base + HB + g * (HB / 2), pg.row(id[g], 32 * b + 16 * g) + pg.to_v, once);
                return true;
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int t = 32 * b + 16 * g;
                pg.load_part(own + HB + g * (HB / 2), base + HB + g * (HB / 2),
                             pg.row(id[g], t) + pg.to_v, pg.has(id[g]) ? len - t : 0);
            }
            return false;
        };
        bool kfull = false, vfull = false;
        if (b0 < b1) {
            find(b0);
            issue_k(b0);
            vfull = issue_v(b0);
        }
        for (int b = b0; b < b1; b += CK_WAVES) {
            const int t0 = 32 * b;
            const uint32_t groups = (pg.has(id[0]) ? 1u : 0u) | (pg.has(id[1]) ? 2u : 0u);
            const bool more = b + CK_WAVES < b1;
            f32x16_t s[1];
            if (vfull) dma_wait<LOADS>();
            else dma_wait<0>();
            scores<DT, D, 1>(base, ll, q, s);
            dma_wait<63>();                        // (the K reads have returned)
            if (more) {
                find(b + CK_WAVES);
                kfull = issue_k(b + CK_WAVES);
            }
            const bool masked = t0 < lo_hi || t0 + 32 > hi_lo || groups != 3u;
            if (masked) mask_scores<1>(s, lo - t0, hi - t0, groups, lane);
            maximum<D, 1>(s, c, st);
            if (more && kfull) dma_wait<LOADS>();
            else dma_wait<0>();
            const uint32_t vs = base + HB;
            weigh<DT, D, 1>(vs, ll, s, c, st);
            dma_wait<63>();
            if (more) vfull = issue_v(b + CK_WAVES);
        }
        if (needs_care(st, c, live)) {             // (as above, this wave alone)
            reset(st);
            for (int b = b0; b < b1; b += CK_WAVES) {
                const int t0 = 32 * b;
                find(b);
                issue_k(b);
                issue_v(b);
                dma_wait<0>();
                const uint32_t groups = (pg.has(id[0]) ? 1u : 0u) | (pg.has(id[1]) ? 2u : 0u);
                f32x16_t s[1];
                scores<DT, D, 1>(base, ll, q, s);
                mask_scores<1>(s, lo - t0, hi - t0, groups, lane);
                maximum<D, 1>(s, c, st);
                weigh_careful<DT, D, 1>(base + HB, ll, s, c, st);
                dma_wait<0>();                     // (the reads have returned)
            }
        }
        // the waves' (m, l, O) through LDS: wave w takes d tile w of all of them
        dma_wait<0>();
        __syncthreads();
        lds.m[w][lane] = st.m;
        lds.l[w][lane] = st.l + xor32_f(st.l);
        float* of = reinterpret_cast<float*>(lds.kv) + w * (32 * D);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
            float o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = st.o[x][i];
            save_tile<D>(of, x, o, lane);
        }
        __syncthreads();
        float m = -__FLT_MAX__, l = 0.f, wt[CK_WAVES];
#pragma unroll
        for (int v = 0; v < CK_WAVES; ++v) m = fmaxf(m, lds.m[v][lane]);
#pragma unroll
        for (int v = 0; v < CK_WAVES; ++v) {
            // (a wave without a finite score has l = 0 and O = 0)
            wt[v] = __builtin_amdgcn_exp2f((lds.m[v][lane] - m) * c);
            l += lds.l[v][lane] * wt[v];
        }
        if (w >= D / 32) return;
        float o[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int v = 0; v < CK_WAVES; ++v) {
                const float4 y = *reinterpret_cast<const float4*>(
                    reinterpret_cast<float*>(lds.kv) + v * (32 * D) + (w * 4 + i) * 4 * WAVE + 4 * lane);
                z.x += y.x * wt[v];
                z.y += y.y * wt[v];
                z.z += y.z * wt[v];
                z.w += y.w * wt[v];
            }
            o[4 * i] = z.x;
            o[4 * i + 1] = z.y;
            o[4 * i + 2] = z.z;
            o[4 * i + 3] = z.w;
        }
        if (whole) {
            const RowOut ro = row_out(a, pl, it.q, kh, row);
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= inv;
            store_row<DT, D>(ro.out, w, o, lane);
            if (w == 0) store_lse<DT>(ro, m, l, c, lane);
        } else {
            float* g = slot_group<D>(a, pl, kh, it.slot, 0);
            save_tile<D>(g, w, o, lane);
            if (w == 0) save_stats<D>(g, m, l, lane);
        }
        return;
    }
    if (idle) return;
    const float l = st.l + xor32_f(st.l);
    const RowOut ro = row_out(a, pl, it.q, kh, row);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float* g = whole ? nullptr : slot_group<D>(a, pl, kh, it.slot, group);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = st.o[x][i] * (whole ? inv : 1.f);
        if (whole) store_row<DT, D>(ro.out, x, o, lane);
        else save_tile<D>(g, x, o, lane);
    }
    if (whole) store_lse<DT>(ro, st.m, l, c, lane);
    else save_stats<D>(g, st.m, l, lane);
}

// Joins the parts of cut row tiles, a d tile per workgroup (grid: cut tile x kv head, 32-row group, d
// tile).  Bound by the latency of its loads: record, statistics and O, 4.0 us at 17 parts of one
// tile, 6.6 us at 310 tiles of two parts (20 MB; medians).  A wave issues the loads of
// CM_BATCH parts before it uses any.  Up to that many parts it joins a group alone, and one
// workgroup takes all groups of the tile (a workgroup of waves with a part each, joining in LDS,
// took 8.7 us there); beyond, wave w takes parts w, w + 4, ... of one group and the waves join
// through LDS.  Batches without cut tiles leave a launch that reads the count, 4.8 us.
constexpr int CM_WAVES = 4;
constexpr int CM_BATCH = 4;

template <int DT, int D>
__global__ __launch_bounds__(CM_WAVES * WAVE) void chunk_merge_kernel(const amass_chunk_args a,
                                                                      const ChunkPlan pl) {
    __shared__ float ms[CM_WAVES][32], ls[CM_WAVES][32], os[CM_WAVES][16][WAVE];
    const int lane = threadIdx.x & 63, rl = lane & 31;
    const int x = blockIdx.z;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kh = blockIdx.x % a.n_kv, i = blockIdx.x / a.n_kv;
    const int cuts = *(const int*)a.scratch;
    const CutTile ct = *cut_tile(a, i);            // (inside the scratch; read before it is known)
    if (i >= cuts || ct.parts < 2) return;
    const int rows = min(CK_BM, ct.q.n * a.G - ct.tile * CK_BM);
    const float c = a.scale * 1.44269504088896341f;
    const int64_t step = (int64_t)(pl.slot_rows / 32) * (32 * D + CK_STATS);
    const bool alone = ct.parts <= CM_BATCH;
    const int group = alone ? w : blockIdx.y, w0 = alone ? 0 : w, waves = alone ? 1 : CM_WAVES;
    if (32 * group >= rows || (alone && blockIdx.y > 0)) return;
    const float* g0 = slot_group<D>(a, pl, kh, ct.slot, group);
    float m = -__FLT_MAX__, l = 0.f, o[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = 0.f;
    for (int s0 = w0; s0 < ct.parts; s0 += waves * CM_BATCH) {
        float pm[CM_BATCH], ps[CM_BATCH];
        float4 y[CM_BATCH][4];
#pragma unroll
        for (int u = 0; u < CM_BATCH; ++u) {
            const int s = s0 + u * waves;
            pm[u] = -__FLT_MAX__;
            ps[u] = 0.f;
            if (s < ct.parts) {                // (scalar)
                const float* g = g0 + s * step;
                pm[u] = g[32 * D + rl];
                ps[u] = g[32 * D + 32 + rl];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    y[u][j] = *reinterpret_cast<const float4*>(g + (x * 4 + j) * 4 * WAVE + 4 * lane);
            }
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < CM_BATCH; ++u) mx = fmaxf(mx, pm[u]);
        const float al = __builtin_amdgcn_exp2f((m - mx) * c);
        m = mx;
        l *= al;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] *= al;
#pragma unroll
        for (int u = 0; u < CM_BATCH; ++u)
            if (s0 + u * waves < ct.parts) {
                const float wt = __builtin_amdgcn_exp2f((pm[u] - m) * c);
                l += ps[u] * wt;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[4 * j] += y[u][j].x * wt;
                    o[4 * j + 1] += y[u][j].y * wt;
                    o[4 * j + 2] += y[u][j].z * wt;
                    o[4 * j + 3] += y[u][j].w * wt;
                }
            }
    }
    if (!alone) {
        if (lane < 32) {
            ms[w][lane] = m;
            ls[w][lane] = l;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) os[w][j][lane] = o[j];
        __syncthreads();
        if (w > 0) return;
        m = -__FLT_MAX__;
        l = 0.f;
#pragma unroll
        for (int v = 0; v < CM_WAVES; ++v) m = fmaxf(m, ms[v][rl]);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = 0.f;
#pragma unroll
        for (int v = 0; v < CM_WAVES; ++v) {
            const float wt = __builtin_amdgcn_exp2f((ms[v][rl] - m) * c);
            l += ls[v][rl] * wt;
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] += os[v][j][lane] * wt;
        }
    }
    const RowOut ro = row_out(a, pl, ct.q, kh, ct.tile * CK_BM + 32 * group + rl);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] *= inv;
    store_row<DT, D>(ro.out, x, o, lane);
    if (x == 0) store_lse<DT>(ro, m, l, c, lane);
}

// ------------------------------------------------------------------ host
// compute units of the current device, asked for once per device
static int chunk_cus() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
        return 256;
    if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

static bool chunk_empty(const amass_chunk_args& a) { return a.n_tokens == 0 || a.n_req == 0; }

static int chunk_check(const amass_chunk_args& a) {
    if (chunk_empty(a)) return AMASS_OK;
    if (!a.q || !a.k || !a.v || !a.block_table || !a.seq_lens || !a.query_start || !a.out)
        return AMASS_ERR_NULL;
    if (a.dtype != AMASS_BF16 && a.dtype != AMASS_FP16) return AMASS_ERR_UNSUPPORTED;
    if (a.d != 64 && a.d != 128) return AMASS_ERR_UNSUPPORTED;
    if (a.page < 16 || a.page > (1 << 20) || (a.page & (a.page - 1))) return AMASS_ERR_GEOMETRY;
    if (a.n_req < 0 || a.n_tokens < 0 || a.n_kv < 1 || a.G < 1 || a.nb < 1 || a.max_pages < 1 ||
        a.window < 0 || !(a.scale > 0.f) || a.scale > 2e38f)
        return AMASS_ERR_GEOMETRY;
    if (a.n_kv > 4096 || a.G > 4096 || (int64_t)a.n_tokens * a.G > (1 << 30)) return AMASS_ERR_GEOMETRY;
    const auto off = [](const void* p) { return ((uintptr_t)p & 15) != 0; };
    if (off(a.q) || off(a.k) || off(a.v) || off(a.out) ||
        ((a.q_st | a.q_hs | a.kv_sb | a.kv_st | a.kv_sh | a.o_st | a.o_hs) & 7))
        return AMASS_ERR_GEOMETRY;
    // the kernel has 32 bits for a row's offset (bytes) within its block
    if (a.kv_sb < 0 || a.kv_sb >= (1 << 30) || a.kv_st < 0 || a.kv_st * a.page >= (1 << 30))
        return AMASS_ERR_GEOMETRY;
    return AMASS_OK;
}

static ChunkPlan chunk_plan(const amass_chunk_args& a) {
    ChunkPlan p;
    p.sh = 0;
    while ((1 << p.sh) < a.page) ++p.sh;
    const int64_t cap = (int64_t)a.max_pages << p.sh;
    p.cap = cap > 0x7FFF0000 ? 0x7FFF0000 : (int)cap;    // (positions a tile ahead fit an int)
    p.target = ck_wgs(a.d) * chunk_cus() / a.n_kv;
    if (p.target < 1) p.target = 1;
    const int64_t rows = (int64_t)a.n_tokens * a.G;
    p.tiles_max = (int)(rows / CK_BM) + (a.n_req < a.n_tokens ? a.n_req : a.n_tokens);
    // the rest's parts are at most `target`; without whole rounds those of cut tiles are at most twice
    // sum_r tiles_r w_r / len <= target
    p.slots = p.tiles_max < p.target ? p.target : 2 * p.target;
    p.items = p.tiles_max < p.target ? p.target : p.tiles_max + p.target;
    p.slot_rows = rows <= CK_FEW ? CK_FEW : CK_BM;
    p.g_sh = 0;
    while ((1 << p.g_sh) < a.G) ++p.g_sh;
    p.g_mul = (uint32_t)((((uint64_t)1 << (30 + p.g_sh)) + a.G - 1) / a.G);
    return p;
}

static int64_t chunk_scratch(const amass_chunk_args& a, const ChunkPlan& p) {
    return CK_HEAD + (int64_t)p.slots * sizeof(CutTile) +
           (int64_t)a.n_kv * p.slots * (p.slot_rows / 32) * (32 * a.d + CK_STATS) * sizeof(float);
}

template <int DT, int D>
static int launch_chunk(const amass_chunk_args& a, const ChunkPlan& p, hipStream_t s) {
    const int64_t items = (int64_t)p.items * a.n_kv;
    if (items * CK_WAVES * WAVE > 0xFFFFFFFFll) return AMASS_ERR_GEOMETRY;    // (threads of a launch)
    hipLaunchKernelGGL((chunk_kernel<DT, D>), dim3((unsigned)items), dim3(CK_WAVES * WAVE), 0, s, a, p);
    const int rc = check_launch();
    if (rc) return rc;
    // a cut tile has two slots at least
    const int cuts = p.tiles_max < (p.slots + 1) / 2 ? p.tiles_max : (p.slots + 1) / 2;
    hipLaunchKernelGGL((chunk_merge_kernel<DT, D>), dim3(cuts * a.n_kv, p.slot_rows / 32, D / 32),
                       dim3(CM_WAVES * WAVE), 0, s, a, p);
    return check_launch();
}

}  // namespace amass

using namespace amass;

extern "C" int64_t amass_chunk_scratch_bytes(const amass_chunk_args* a) {
    if (!a) return AMASS_ERR_NULL;
    const int rc = chunk_check(*a);
    return rc || chunk_empty(*a) ? rc : chunk_scratch(*a, chunk_plan(*a));
}

extern "C" int amass_chunk_attention(const amass_chunk_args* ain, void* stream) {
    if (!ain) return AMASS_ERR_NULL;
    const amass_chunk_args& a = *ain;
    const int rc = chunk_check(a);
    if (rc) return rc;
    if (chunk_empty(a)) return AMASS_OK;
    if (!a.scratch) return AMASS_ERR_NULL;
    const ChunkPlan p = chunk_plan(a);
    if (((uintptr_t)a.scratch & 255) || a.scratch_bytes < chunk_scratch(a, p)) return AMASS_ERR_CAPACITY;
    hipStream_t s = (hipStream_t)stream;
    if (a.dtype == AMASS_BF16)
        return a.d == 128 ? launch_chunk<0, 128>(a, p, s) : launch_chunk<0, 64>(a, p, s);
    return a.d == 128 ? launch_chunk<1, 128>(a, p, s) : launch_chunk<1, 64>(a, p, s);
}

extern "C" int amass_chunk_abi_version(void) { return AMASS_CHUNK_ABI_VERSION; }

extern "C" size_t amass_chunk_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(amass_extend_args);
        case 1: return sizeof(amass_release_args);
        case 2: return sizeof(amass_rope_args);
        case 3: return sizeof(amass_chunk_args);
        default: return 0;
    }
}
