// What the kernels of attention over a paged cache share (chunk.hip, quant_chunk.hip): the plan
// that cuts a batch's row tiles into parts, a wave's softmax state, the LDS image of a tile of keys
// in 16 bits, and how results leave (rows, parts, the join of parts).  chunk.hip's comment has the
// mathematics and the layouts.
#pragma once

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
constexpr float CK_LAZY = 8.f;             // a maximum may lag by this power of two
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
#define CK_LOADS1(hint) "s_mov_b32 m0, %0\n\ts_nop 0" CK_LOAD(2, 0, hint)
#define CK_LOADS2(hint) CK_LOADS1(hint) CK_LOAD(3, 1024, hint)
#define CK_LOADS4(hint) CK_LOADS2(hint) CK_LOAD(4, 2048, hint) CK_LOAD(5, 0xc00, hint)
template <bool ONCE, int N>
__device__ __forceinline__ void dma16_n(uint32_t to, const char* base, const uint32_t (&off)[N]) {
    if constexpr (N == 4 && ONCE)
        asm volatile(CK_LOADS4(" nt")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[N / 2 - 1]), "v"(off[N - 2]), "v"(off[N - 1])
                     : "memory", "m0");
    else if constexpr (N == 4)
        asm volatile(CK_LOADS4("")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[N / 2 - 1]), "v"(off[N - 2]), "v"(off[N - 1])
                     : "memory", "m0");
    else if constexpr (N == 1 && ONCE)
        asm volatile(CK_LOADS1(" nt") : : "s"(to), "s"(base), "v"(off[0]) : "memory", "m0");
    else if constexpr (N == 1)
        asm volatile(CK_LOADS1("") : : "s"(to), "s"(base), "v"(off[0]) : "memory", "m0");
    else if constexpr (ONCE)
        asm volatile(CK_LOADS2(" nt")
                     :
                     : "s"(to), "s"(base), "v"(off[0]), "v"(off[N - 1])
                     : "memory", "m0");
    else
        asm volatile(CK_LOADS2("") : : "s"(to), "s"(base), "v"(off[0]), "v"(off[N - 1]) : "memory", "m0");
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

// What O is multiplied by at the end, sums being 2^UP times those of the weights: ROW_UP, then row_scale.  In one, a
// row of bf16 whose weight lies on a page of V scale s would take 2^8 s, beyond fp32 from s = 2^120 on (such a
// page's numbers are in the type); of two, the second is 2^124 at most for any s.
template <int UP>
constexpr float ROW_UP = (float)(1 << (UP - UP / 4));
template <int UP>
__device__ __forceinline__ float row_scale(float l) {
    return l == 0.f ? 0.f : (float)(1 << (UP / 4)) / l;
}

template <int DT, int UP>
__device__ __forceinline__ void store_lse(const RowOut& w, float m, float l, float c, int lane) {
    if (w.lse && lane < 32) {
        *w.lse = l == 0.f ? -INFINITY
                          : (m * c - (CK_LIFT<DT> + UP) + __log2f(l)) * 0.693147180559945309f;
    }
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

// c: powers of two that a maximum counts by; the sums are 2^UP times those of the weights.
template <int DT, int D, int UP>
__device__ __forceinline__ void merge_parts(const amass_chunk_args& a, const ChunkPlan& pl,
                                            const float c) {
    __shared__ float ms[CM_WAVES][32], ls[CM_WAVES][32], os[CM_WAVES][16][WAVE];
    const int lane = threadIdx.x & 63, rl = lane & 31;
    const int x = blockIdx.z;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kh = blockIdx.x % a.n_kv, i = blockIdx.x / a.n_kv;
    const int cuts = *(const int*)a.scratch;
    const CutTile ct = *cut_tile(a, i);            // (inside the scratch; read before it is known)
    if (i >= cuts || ct.parts < 2) return;
    const int rows = min(CK_BM, ct.q.n * a.G - ct.tile * CK_BM);
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
    const float inv = row_scale<UP>(l);
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = o[j] * ROW_UP<UP> * inv;
    store_row<DT, D>(ro.out, x, o, lane);
    if (x == 0) store_lse<DT, UP>(ro, m, l, c, lane);
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

}  // namespace amass
