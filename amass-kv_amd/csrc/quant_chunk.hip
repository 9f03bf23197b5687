// Attention of a chunk of new tokens over a paged cache in 8 bits for gfx950
// (amass_quant_chunk_attention).
//
// Mathematics.  That of chunk.hip with k_j = c_j sk and v_j = c'_j sv, where sk and sv belong to a page (16
// keys or a multiple).  Codes are exact in 16 bits, so the matrix products take them as they are,
// and the scales enter where a lane holds one row's scores of 16 keys of one page:
//   x_j = (scale log2 e sk) (q . c_j) + log2 sv       one fma, as without scales
//   w_j = 2^(x_j - M), M the running maximum of x     the weight with V's scale, rounded once
//   O  += w_j c'_j,  l += (sum of the 16 w_j) / sv    V's scale leaves the sum again, per 16 keys
//   out = O / l,  lse = ln 2 (M + log2 l)
// So a page costs a few instructions per 16 keys and nothing per key.
//
// Layouts, parts and results are those of chunk.hip (chunk_core.h).  Codes are widened to 16 bits on the way:
//   many rows (more than 32): each wave brings 16 keys of a 64-key tile into registers two tiles ahead and writes
//     them to LDS widened, one tile ahead, under the products with the tile before; an int8 takes 1.5 instructions
//     (bf16; fp16 1.25), an e4m3 half a one, once for the four waves.  Vector work bounds it: a prompt of 8192 tokens
//     (8 kv heads of 4 query heads, d 128, bf16) takes 576 us with int8, 10 vector instructions beside every product
//     and 43 % of the matrix cores' cycles, 539 with e4m3, where chunk.hip over the same numbers in 16 bits takes
//     507 and 490; 2048 tokens behind 63488 2034 us with e4m3 (1820), 1.06 PFLOP/s.  Cards differ: 576 to 601,
//     2022 to 2106.  d 64: the prompt 359 and 342 us (312 and 304).
//   few rows: each wave brings its own 32 keys to LDS as they are, one step ahead, reads K by rows and V by columns
//     of 8-bit elements, and widens them in registers.  Memory bounds it: 64 single tokens with 8k keys 196 to 207 us, 5.1
//     to 5.4 TB/s (16 bits: 341), 177 where the codes of a page of one head lie together (quant_cache), 6.0 TB/s; 8
//     requests of 4 drafted tokens with 8k to 24k keys 68 us, in a graph over two caches in turn 73 (110) and 64.  Tried
//     there where 64 single tokens took 196, to no gain: two heads a wave (256 neighbouring bytes a key, 196, and it
//     needs more parts), all heads of a token in one workgroup (196), more in flight (206), loads that other caches
//     keep (225).
#include "chunk_core.h"
#include "quant_codes.h"

namespace amass {

// Sums are 2^QC_UP times those of the weights: with bf16's lift, 1 / sv of the largest scale would
// leave fp32's normal numbers.
constexpr int QC_UP = 16;

// As CK_ONCE of chunk.hip: more bytes of codes than this are loaded past the caches, where one row tile
// alone reads them.
constexpr float QC_ONCE = 128e6f;

// Maxima beyond this take their request again with care: log2 sv less the maximum, rounded, moves the weights of
// one page against another's by 2^-12 there, and from 2^27 on makes weights of any size.
constexpr float QC_FAR = 0x1p12f;

// fp16: V scales that are more powers of two than this from their first page's take their request with care, too.  A
// weight with V's scale of 2^-21 of the largest has no bits to lose, so what counts in channels where a large page
// holds zeros would.  As the rule leaves pages (12 powers of two apart), weights of a row's largest to 2^-9 of it keep
// all bits everywhere.  Pages below 2^-35 do not count: their numbers are beneath half of fp16's least.  (With care a
// prompt of 8192 tokens takes 1660 us for 630, 64 single tokens with 8k keys 414 for 198; the look at the scales 0.7 %.)
constexpr float QC_APART = 6.f;
constexpr float QC_NOUGHT = -35.f;

struct Scales {
    const float *k, *v;
    int64_t sb, sh;
};

// The pages of a wave's next 64 groups of 16 keys, one a lane, PER of them a step (a tile of 64
// keys, or a wave's 32): looked up once in 64 / PER steps, a period ahead, so that no step waits for
// a table entry or a scale.
template <int DT, int PER>
struct Lookup {
    static constexpr int STEPS = WAVE / PER;
    static constexpr uint32_t NO_REF = 0xFFFFFFFFu, APART = 0xFFFFFFFEu;      // (as numbers, NaN)
    const int32_t* table;          // the request's row
    const float *ks, *vs;          // of the kv head
    int64_t sb;
    int sh, nb, last;              // last: the last position that counts
    int t, jump;                   // this lane's first position; positions of a period
    float c;
    int id, next_id;               // -1: no block
    float sk, off, inv;            // scale log2 e sk, log2 sv, 2^QC_UP / sv
    float next_k, next_v;
    unsigned long long has;
    uint32_t ref = NO_REF;         // fp16: log2 sv of the first page that counts (NO_REF: none so far), APART once
                                   // a page is far from it

    __device__ __forceinline__ int find(int at) const {
        const int e = table[max(min(at, last), 0) >> sh];
        return at <= last && (uint32_t)e < (uint32_t)nb ? e : -1;
    }
    __device__ __forceinline__ void fetch(int e, float& k, float& v) const {
        k = v = 1.f;
        if (e >= 0) {
            k = ks[e * sb];
            v = vs[e * sb];
        }
    }
    __device__ __forceinline__ void take(int e, float k, float v) {
        id = e;
        has = __ballot(e >= 0);
        sk = k < INFINITY ? k * c : __builtin_nanf("");
        if (v < LEAST_SCALE) v = LEAST_SCALE;
        off = e < 0 ? -INFINITY : __log2f(v);      // (a page without a block: weights of zero)
        inv = (float)(1 << QC_UP) / v;
        if constexpr (DT == AMASS_FP16) {
            const unsigned long long counts = __ballot(off > QC_NOUGHT);
            if (counts && ref == NO_REF)
                ref = __builtin_amdgcn_readlane(__float_as_uint(off), __ffsll((long long)counts) - 1);
            if (__any(off > QC_NOUGHT && fabsf(off - __uint_as_float(ref)) > QC_APART)) ref = APART;
        }
    }
    // first: this lane's first position
    __device__ __forceinline__ void start(int first, int period) {
        t = first;
        jump = period;
        ref = NO_REF;
        float k, v;
        const int e = find(t);
        fetch(e, k, v);
        take(e, k, v);
        next_id = find(t + jump);
    }
    // before step s of a period
    __device__ __forceinline__ void ahead(int s) {
        if (s == STEPS / 2) fetch(next_id, next_k, next_v);
    }
    __device__ __forceinline__ bool apart() const { return DT == AMASS_FP16 && ref == APART; }
    // behind its last step
    __device__ __forceinline__ void turn() {
        take(next_id, next_k, next_v);
        t += jump;
        next_id = find(t + jump);
    }
    // block of group g of step s (of the next period from STEPS on), negative for none
    __device__ __forceinline__ int block(int s, int g) const {
        return s < STEPS ? __builtin_amdgcn_readlane(id, PER * s + g)
                         : __builtin_amdgcn_readlane(next_id, PER * (s - STEPS) + g);
    }
    __device__ __forceinline__ uint32_t groups(int s) const {
        return (uint32_t)(has >> (PER * s)) & ((1u << PER) - 1);
    }
};

// ------------------------------------------------------------------ staging
// 16 rows of codes of a page, 16 channels of a row in each of a lane's LOADS registers of 16 bytes.  8 neighbouring
// lanes, whose 16-byte chunks a cycle of an LDS write takes, hold 4 of each of two rows whose swizzles differ in the
// lowest bit, so that they fill the banks once (with 8 lanes a row every write took two cycles for one, a quarter
// of LDS' time).
template <int D>
struct Codes {
    static constexpr int LPR = D / 16, RPL = WAVE / LPR, LOADS = 16 / RPL;
    uint32_t off, st;              // of the lane's first 16 bytes in a page; bytes between rows
    uint32_t lds;                  // its first chunk in the image
    int row;

    __device__ __forceinline__ Codes(uint32_t st_, int lane) : st(st_) {
        const int c = (lane & 3) + (D == 128 ? (lane >> 1) & 4 : 0);
        row = D == 128 ? (lane >> 4) + (lane & 4) : ((lane >> 3) & 3) + (lane & 4) + 8 * (lane >> 5);
        off = (uint32_t)row * st + 16 * c;
        lds = row * (2 * D) + (((2 * c) ^ swz<D>(row)) << 4);
    }
    __device__ __forceinline__ void load(u32x4_t* z, const uint8_t* page) const {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) z[n] = *reinterpret_cast<const u32x4_t*>(page + off + n * RPL * st);
    }
    // 8 codes of register n (the half h of it), widened, to the image of its 16 rows at `to` (row + 8 turns
    // the chunk's second bit)
    template <int DT, int CT>
    __device__ __forceinline__ void put(uint32_t to, int n, int h, const u32x4_t& z) const {
        u32x4_t a;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t lo, hi, x = z[2 * h + j];
            asm("" : "+v"(x));                     // (widened here, not byte by byte where it was loaded)
            widen4<DT, CT>(x, lo, hi);
            a[2 * j] = lo;
            a[2 * j + 1] = hi;
        }
        const uint32_t at = ((to + lds) ^ (uint32_t)(32 * n + 16 * h)) + n * RPL * (2 * D);
        *(__attribute__((address_space(3))) u32x4_t*)(uintptr_t)at = a;
    }
    // V's register n without the rows from `rows` on (what lies behind the last token may be a NaN, and the
    // weight zero times that is one)
    __device__ __forceinline__ void clip(u32x4_t& z, int n, int rows) const {
        if (row + n * RPL >= rows) z = (u32x4_t){0u, 0u, 0u, 0u};
    }
    // a key whose V holds a NaN: its K becomes NaN instead, so that the rows that see it, and no others,
    // become NaN
    __device__ __forceinline__ void poison(u32x4_t& k, u32x4_t& v) const {
        int bad = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= (int)nan_codes(v[j]);
        bad |= dpp_i<DPP_XOR2>(bad);
        bad |= dpp_i<DPP_XOR1>(bad);
        if constexpr (LPR == 8) bad |= __shfl_xor(bad, 8);
        if (bad) {
            k = (u32x4_t){0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};
            v = (u32x4_t){0u, 0u, 0u, 0u};
        }
    }
};

// ------------------------------------------------------------------ a tile
template <int N>
struct Factors {                   // of N groups of 16 keys
    float sk[N], off[N], inv[N];
    template <int DT, int PER>
    __device__ __forceinline__ Factors(const Lookup<DT, PER>& lk, int s) {
#pragma unroll
        for (int g = 0; g < N; ++g) {
            sk[g] = readlane_f(lk.sk, PER * s + g);
            off[g] = readlane_f(lk.off, PER * s + g);
            inv[g] = readlane_f(lk.inv, PER * s + g);
        }
    }
};

// nothing moves across (the order is the program's, and few values wait in registers)
__device__ __forceinline__ void step() { __builtin_amdgcn_sched_barrier(0); }

// The largest of 8 scores, by three a instruction.  (A NaN stays one: a maximum that drops it asks for
// another instruction a score, which tells signalling ones apart.  Its row is not finite then, and is
// done again with care.)
__device__ __forceinline__ float group_max(const f32x16_t& s, int half) {
    const auto max3 = [](float a, float b, float c) {
        return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
    };
    const int i = 8 * half;
    return max3(max3(max3(s[i], s[i + 1], s[i + 2]), s[i + 3], s[i + 4]), max3(s[i + 5], s[i + 6], s[i + 7]),
                -INFINITY);
}
// the running maximum and sum for a higher maximum; the factor for O
template <int D>
__device__ __forceinline__ float lift_max(float mx, RowState<D>& st) {
    const float m = fmaxf(st.m, mx);
    const float al = __builtin_amdgcn_exp2f(st.m - m);
    st.m = m;
    st.l *= al;
    return al;
}

// -inf for the keys (relative to the tile) outside [lo, hi) of this lane's row, and those of groups of 16
// whose bit is not set
template <int NK>
__device__ __forceinline__ void mask_scores(f32x16_t (&s)[NK], int lo, int hi, uint32_t groups, int lane) {
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

// The weights of 32 NK keys, packed for the second product, and what they add to the maximum and the
// sum.
template <int DT, int D, int NK>
__device__ __forceinline__ void weigh_tile(const f32x16_t (&s)[NK], const Factors<2 * NK>& f,
                                           RowState<D>& st, u32x4_t (&p)[2 * NK]) {
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 2 * NK; ++g)
        mx = fmaxf(mx, __builtin_fmaf(group_max(s[g >> 1], g & 1), f.sk[g], f.off[g]));
    mx = xor32_maxf(mx);
    float al = 1.f;
    const bool lag = __any(mx - st.m > CK_LAZY);
    if (lag) al = lift_max(mx, st);
    scale_o(st, al);
    const float base = CK_LIFT<DT> - st.m;
#pragma unroll
    for (int g = 0; g < 2 * NK; ++g) {
        const float off = f.off[g] + base;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + i], f.sk[g], off));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + i + 1], f.sk[g], off));
            sum += e0 + e1;
            p[g][i >> 1] = pack2<DT>(e0, e1);
        }
        step();
        st.l = __builtin_fmaf(sum, f.inv[g], st.l);
    }
}

// The same with care: for factors that are not finite, which must not reach what a row does not see, for scores
// far from zero, beside which log2 sv is lost, and for V scales far apart in fp16.  The weights count from the largest
// key's product (st.m, rounded as every product is, so that differences are exact where they matter) and its log2 sv
// (mo), kept apart.  Codes are exact in bf16, too, which has fp32's exponents: weights of fp16 rows are two numbers of
// it each (16 bits together) and V's codes are widened to it.
constexpr int CAREFUL_DT = AMASS_BF16;
template <int DT>
constexpr int LIMBS = DT == AMASS_FP16 ? 2 : 1;
template <int N, int L>
struct Weights {
    u32x4_t p[L][N];
};
template <int DT, int D, int NK>
__device__ __forceinline__ void weigh_careful(const f32x16_t (&s)[NK], const Factors<2 * NK>& f,
                                              RowState<D>& st, float& mo, Weights<2 * NK, LIMBS<DT>>& wt) {
#pragma clang fp contract(off)
    float m = st.m, o = mo;
    const auto larger = [&](float pm, float po) {      // (both half waves find the same one)
        const float d = (pm - m) + (po - o);
        const bool is = pm != -INFINITY && (d > 0.f || (d == 0.f && pm > m));
        m = is ? pm : m;
        o = is ? po : o;
    };
#pragma unroll
    for (int g = 0; g < 2 * NK; ++g) larger(group_max(s[g >> 1], g & 1) * f.sk[g], f.off[g]);
    larger(__shfl_xor(m, 32), __shfl_xor(o, 32));
    const float al = __builtin_amdgcn_exp2f((st.m - m) + (mo - o));
    st.m = m;
    mo = o;
    st.l *= al;
    scale_o(st, al);
#pragma unroll
    for (int g = 0; g < 2 * NK; ++g) {
        const float off = (f.off[g] - mo) + CK_LIFT<DT>;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float e[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float sc = s[g >> 1][8 * (g & 1) + i + j];
                const float x = (sc * f.sk[g] - m) + off;
                e[j] = __builtin_amdgcn_exp2f(sc == -INFINITY ? -INFINITY : x);
                sum += e[j];
            }
#pragma unroll
            for (int k = 0; k < LIMBS<DT>; ++k) {
                const uint32_t w = pack2<CAREFUL_DT>(e[0], e[1]);
                wt.p[k][g][i >> 1] = w;
                e[0] -= __uint_as_float(w << 16);
                e[1] -= __uint_as_float(w & 0xFFFF0000u);
            }
        }
        step();
        if (sum != 0.f) st.l += sum * f.inv[g];
    }
}
// One number to count from again: the two together near zero, else the product, with the sums taken times sv.  Those
// are 2^-QC_DOWN times that, for any sv's sake, and the number is larger by it: the same for every wave, so that what
// is lost of it beside a product beyond 2^24 is lost of all alike.
constexpr float QC_DOWN = 32.f;
template <int D>
__device__ __forceinline__ void careful_end(RowState<D>& st, float mo) {
    const bool far = fabsf(st.m) > QC_FAR;
    const float by = __builtin_amdgcn_exp2f(far ? mo - QC_DOWN : 0.f);
    st.m += far ? QC_DOWN : mo;
    st.l *= by;
    scale_o(st, by);
}

template <int D, int NK, int L>
__device__ __forceinline__ void add_values(uint32_t vs, const LdsLane<D>& ll, const Weights<2 * NK, L>& wt,
                                           RowState<D>& st) {
#pragma unroll
    for (int y = 0; y < 2 * NK; ++y)
#pragma unroll
        for (int z = 0; z < D / 32; ++z) {
            const u32x4_t v = ll.v_frag(vs, z, y);
#pragma unroll
            for (int k = 0; k < L; ++k) st.o[z] = mfma32<CAREFUL_DT>(v, wt.p[k][y], st.o[z]);
            if (z & 1) step();
        }
}

// A tile of 64 keys of the many-row layout, in a fixed order (each step ends in a scheduling barrier):
// the matrix products follow each other with four fragments in flight, and the vector work runs under them:
//   scores of keys 0..31, the next tile's K into LDS | scores of 32..63, weights of 0..31 | maximum |
//   products with V of 0..31, weights of 32..63 | products with V of 32..63, the next tile's V into LDS
// The first weights are made with the maximum so far and made again in the rare tile whose scores exceed
// it by more than it may lag.  MASKS: the lane's row sees the keys [lo, hi) of the tile; without, all.
// bring_k, bring_v: put 8 codes a lane (the argument: which) of the next tile.
template <int DT, int D, bool MASKS, class BringK, class BringV>
__device__ __forceinline__ void ordered_tile(uint32_t ks, uint32_t vs, const LdsLane<D>& ll,
                                             const u32x4_t (&q)[D / 16], const Factors<4>& fa,
                                             RowState<D>& st, int lo, int hi, int lane, BringK bring_k,
                                             BringV bring_v) {
    lo -= 4 * (lane >> 5);
    hi -= 4 * (lane >> 5);
    const uint32_t seen = (uint32_t)max(hi - lo, 0);
    const auto masked = [&](float v, int x, int i) {
        const int key = 32 * x + 8 * (i >> 2) + (i & 3);
        return !MASKS || (uint32_t)(key - lo) < seen ? v : -INFINITY;
    };
    constexpr int N = D / 16, Z = D / 32;      // products of 32 keys with K or V; d tiles
    constexpr int EVERY = N / (2 * Codes<D>::LOADS);
    u32x4_t f[4], p[4];
    f32x16_t s[2], zero;
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0.f;
    const auto k_frag = [&](int n) { return ll.k_frag(ks, n % N, n / N); };
    float off[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
    const auto offsets = [&] {
#pragma unroll
        for (int g = 0; g < 4; ++g) off[g] = fa.off[g] + (CK_LIFT<DT> - st.m);
    };
    offsets();
    const auto weight = [&](int x, int i, bool fresh = true) {    // weights 2 i and 2 i + 1 of half x
        const int g = 2 * x + (i >> 2);
        if (x == 0 && fresh) {                 // (half 1 is masked before the maximum)
            s[0][2 * i] = masked(s[0][2 * i], 0, 2 * i);
            s[0][2 * i + 1] = masked(s[0][2 * i + 1], 0, 2 * i + 1);
        }
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][2 * i], fa.sk[g], off[g]));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][2 * i + 1], fa.sk[g], off[g]));
        sum[g] += e0 + e1;
        uint32_t w = pack2<DT>(e0, e1);
        asm volatile("" : "+v"(w), "+v"(sum[g]));     // (made here, not behind the branch below)
        p[g][i & 3] = w;
    };
#pragma unroll
    for (int n = 0; n < 4; ++n) f[n] = k_frag(n);
    step();
    __builtin_amdgcn_s_setprio(1);             // (products before the other wave's vector work)
#pragma unroll
    for (int n = 0; n < N; ++n) {
        s[0] = mfma32<DT>(f[n & 3], q[n], n ? s[0] : zero);
        f[n & 3] = k_frag(n + 4);
        if (n % EVERY == EVERY - 1) bring_k(n / EVERY);
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
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g)
        mx = fmaxf(mx, __builtin_fmaf(group_max(s[g >> 1], g & 1), fa.sk[g], fa.off[g]));
    mx = xor32_maxf(mx);
    const bool lag = __any(mx - st.m > CK_LAZY);
    float al = 1.f;
    if (lag) {
        al = lift_max(mx, st);
        offsets();
        sum[0] = sum[1] = 0.f;
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
        } else if (n % EVERY == EVERY - 1) {
            bring_v((n - N) / EVERY);
        }
        step();
    }
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int g = 0; g < 4; ++g) st.l = __builtin_fmaf(sum[g], fa.inv[g], st.l);
}

// ------------------------------------------------------------------ few rows: codes in LDS
// Rows of D bytes, 16-byte chunk c of row t at c ^ turn(t): the 16 rows of a K read (one chunk) and the 8 rows of a
// transposing V read (two chunks) fill the banks once.
template <int D>
struct RawRows {
    static constexpr int ROWS = 1024 / D;          // of one 1-KB load
    static constexpr int LOADS = 16 / ROWS;        // of 16 rows
    static constexpr int BACK = 1024 * (LOADS - 1);
    uint32_t off[LOADS];                           // this lane's source in 16 rows, less the load's own 1024 n,
                                                   // from BACK before it
    uint32_t k, v;                                 // its reads, within 32 rows
    int lane;

    static __device__ __forceinline__ int turn(int row) {
        return D == 128 ? ((row >> 2) & 1) | (row & 2) | ((row >> 1) & 4) : (row >> 2) & 3;
    }
    __device__ __forceinline__ RawRows(uint32_t st, int lane_) : lane(lane_) {
        const int chunk = lane & (D / 16 - 1), lr = lane / (D / 16);
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int row = ROWS * n + lr;
            off[n] = (uint32_t)row * st + ((uint32_t)(chunk ^ turn(row)) << 4) + BACK - 1024 * n;
        }
        const int row = lane & 31, h = lane >> 5, i16 = lane & 15, sub = (lane >> 4) & 1;
        k = row * D + ((h ^ turn(row)) << 4);
        const int t = ((i16 >> 1) & 3) + 8 * (i16 >> 3) + 4 * h;
        v = t * D + ((sub ^ turn(t)) << 4) + (i16 & 1) * 8;
    }
    // 16 rows to LDS
    template <bool ONCE>
    __device__ __forceinline__ void load(uint32_t to, const uint8_t* src) const {
        dma16_n<ONCE>(to, (const char*)src - BACK, off);
    }
    // the first `rows` of them, zero behind
    __device__ __forceinline__ void load_part(char* dst, uint32_t to, const uint8_t* src, int rows) const {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            if (ROWS * n + lane / (D / 16) < rows)
                dma16(to + 1024 * n, (const char*)src - BACK + 1024 * n, off[n]);
            else *reinterpret_cast<u32x4_t*>(dst + 1024 * n + 16 * lane) = (u32x4_t){0u, 0u, 0u, 0u};
        }
    }
    // channels 32 n + 16 h .. of key row % 32
    __device__ __forceinline__ u32x4_t row_codes(uint32_t at, int n) const {
        return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)((at + k) ^ (uint32_t)(n << 5));
    }
    // channel 32 x + lane % 32 of the keys 16 y + 4 h + 0..3 and + 8..11
    __device__ __forceinline__ u32x2_t column_codes(uint32_t at, int x, int y) const {
        typedef int i32x2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2_t*)(uintptr_t)(((at + v) ^ (uint32_t)(x << 5)) + y * (16 * D))));
    }
};

// S^T of 32 keys (ks, and their V at vs).  CARE: a key whose V holds a NaN scores NaN.
template <int DT, int CT, int D, bool CARE>
__device__ __forceinline__ void few_scores(uint32_t ks, uint32_t vs, const RawRows<D>& raw,
                                           const u32x4_t (&q)[D / 16], f32x16_t& s) {
    uint32_t bad = 0;
    if constexpr (CARE && CT == AMASS_E4M3) {
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const u32x4_t z = raw.row_codes(vs, n);
            bad |= nan_codes(z[0]) | nan_codes(z[1]) | nan_codes(z[2]) | nan_codes(z[3]);
        }
        const auto o = __builtin_amdgcn_permlane32_swap(bad, bad, false, false);
        bad = o[0] | o[1];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 32; ++n) {
        u32x4_t z = raw.row_codes(ks, n), f[2];
        if constexpr (CARE && CT == AMASS_E4M3) {
            if (bad) z = (u32x4_t){0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            widen4<DT, CT>(z[j], lo, hi);
            f[j >> 1][2 * (j & 1)] = lo;
            f[j >> 1][2 * (j & 1) + 1] = hi;
        }
        s = mfma32<DT>(f[0], q[2 * n], s);
        s = mfma32<DT>(f[1], q[2 * n + 1], s);
    }
}

// DT: the type of the weights; CARE: a NaN of V counts as zero (its key's score is NaN)
template <int DT, int CT, int D, bool CARE, int L>
__device__ __forceinline__ void few_values(uint32_t vs, const RawRows<D>& raw, const Weights<2, L>& wt,
                                           RowState<D>& st) {
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int z = 0; z < D / 32; ++z) {
            u32x2_t c = raw.column_codes(vs, z, y);
            u32x4_t f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t lo, hi;
                if constexpr (CARE && CT == AMASS_E4M3) c[j] &= ~((nan_codes(c[j]) >> 7) * 0xFFu);
                widen4<DT, CT>(c[j], lo, hi);
                f[2 * j] = lo;
                f[2 * j + 1] = hi;
            }
#pragma unroll
            for (int k = 0; k < L; ++k) st.o[z] = mfma32<DT>(f, wt.p[k][y], st.o[z]);
        }
}

// whether a row that is there needs all of it again with care
template <int D>
__device__ __forceinline__ bool needs_care(const RowState<D>& st, bool live, bool apart) {
    const bool far = st.m > -__FLT_MAX__ && fabsf(st.m) > QC_FAR;      // (it has seen something)
    float z[4] = {st.l * 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i & 3] = __builtin_fmaf(st.o[x][i], 0.f, z[i & 3]);
    return __any(live && (apart || far || !((z[0] + z[1]) + (z[2] + z[3]) == 0.f)));
}

// ------------------------------------------------------------------ results
// A wave's own rows (`group` of 32 of the row tile): normalised, or as a part.
template <int DT, int D, int UP>
__device__ __forceinline__ void finish_rows(const amass_chunk_args& a, const ChunkPlan& pl,
                                            const Item& it, int kh, const RowState<D>& st, float c,
                                            int row, int group, bool whole, int lane) {
    const float l = st.l + xor32_f(st.l);
    const RowOut ro = row_out(a, pl, it.q, kh, row);
    const float inv = row_scale<UP>(l);
    float* g = whole ? nullptr : slot_group<D>(a, pl, kh, it.slot, group);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = whole ? st.o[x][i] * ROW_UP<UP> * inv : st.o[x][i];
        if (whole) store_row<DT, D>(ro.out, x, o, lane);
        else save_tile<D>(g, x, o, lane);
    }
    if (whole) store_lse<DT, UP>(ro, st.m, l, c, lane);
    else save_stats<D>(g, st.m, l, lane);
}

// The rows that all waves share: their (m, l, O) through LDS, wave w takes d tile w of all of them.
// (The waves are past their last use of lds.kv.)
template <int DT, int D, int UP, class Lds>
__device__ __forceinline__ void finish_shared(const amass_chunk_args& a, const ChunkPlan& pl,
                                              const Item& it, int kh, const RowState<D>& st, Lds& lds,
                                              float c, int row, bool whole, int w, int lane) {
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
        const float inv = row_scale<UP>(l);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = o[i] * ROW_UP<UP> * inv;
        store_row<DT, D>(ro.out, w, o, lane);
        if (w == 0) store_lse<DT, UP>(ro, m, l, c, lane);
    } else {
        float* g = slot_group<D>(a, pl, kh, it.slot, 0);
        save_tile<D>(g, w, o, lane);
        if (w == 0) save_stats<D>(g, m, l, lane);
    }
}

template <int D>
struct __align__(1024) QuantLds {
    char kv[2 * 2 * CK_KEYS * 2 * D];              // widened tiles, then the waves' O
    float m[CK_WAVES][WAVE], l[CK_WAVES][WAVE];
    int bad[CK_WAVES];
};

// ------------------------------------------------------------------ kernel
// grid: as chunk_kernel.
template <int DT, int CT, int D>
__global__ __launch_bounds__(CK_WAVES * WAVE)
__attribute__((amdgpu_waves_per_eu(ck_wgs(D), ck_wgs(D)))) void
quant_chunk_kernel(const amass_chunk_args a, const Scales sc, const ChunkPlan pl) {
    __shared__ QuantLds<D> lds;
    constexpr int KB = CK_KEYS * 2 * D;            // bytes of a widened K (or V) tile
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
                      __builtin_amdgcn_readfirstlane(keys * (float)KB * (float)a.n_kv > QC_ONCE);
    const int group = few ? 0 : w;                 // 32-row group of this wave
    const int row = it.tile * CK_BM + 32 * group + (lane & 31);
    const int last = it.tile * CK_BM + min(rows, 32 * group + 32) - 1;    // of the wave
    const int start = it.q.len - it.q.n;
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
                              (int64_t)(kh * a.G + (row - tok * a.G)) * a.q_hs;
        const int h = lane >> 5;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {         // (in the order that K comes in: few_scores)
            const int at = few ? 32 * (i >> 1) + 16 * h + 8 * (i & 1) : 16 * i + 8 * h;
            q[i] = live ? *reinterpret_cast<const u32x4_t*>(src + at) : (u32x4_t){0u, 0u, 0u, 0u};
        }
    }
    // (here, not in the loop over the keys, where a wait would also wait for the next tile's loads)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(q[i]));
    const LdsLane<D> ll(lane);
    const Codes<D> cd((uint32_t)a.kv_st, lane);
    constexpr int LOADS = Codes<D>::LOADS;
    const uint8_t* k0 = (const uint8_t*)a.k + kh * a.kv_sh;
    const uint8_t* v0 = (const uint8_t*)a.v + kh * a.kv_sh;
    const auto page_at = [&](int id, int t) {      // offset of position t's row
        return (uint64_t)(uint32_t)id * (uint64_t)a.kv_sb + (uint32_t)(t & ((1 << pl.sh) - 1)) * (uint32_t)a.kv_st;
    };
    RowState<D> st;
    const auto look = [&](auto& lk, int t, int period) {
        lk.table = a.block_table + it.r * a.bt_st;
        lk.ks = sc.k + kh * sc.sh;
        lk.vs = sc.v + kh * sc.sh;
        lk.sb = sc.sb;
        lk.sh = pl.sh;
        lk.nb = a.nb;
        lk.last = sp.hi - 1;
        lk.c = a.scale * 1.44269504088896341f;
        lk.start(t, period);
    };

    if (!few) {
        // ---- many rows: the workgroup shares the tiles -------------------------------------
        // Wave w brings the 16 keys 64 j + 16 w .. of tile j: into registers during tile j - 2, widened into
        // LDS during tile j - 1.
        const uint32_t base = lds_addr(lds.kv);
        Lookup<DT, 4> lk;
        u32x4_t kr[LOADS], vr[LOADS];
        int lim = 16;                              // rows of the 16 that hold tokens
        const uint32_t own = base + 16 * w * 2 * D;
        uint64_t at = 0;                           // of the page in K and V
        const auto find = [&](int j, int s) {      // (a page without a block: block 0, whose V is cut off)
            const int t = CK_KEYS * (sp.lo + j) + 16 * w, id = lk.block(s, w);
            lim = id >= 0 ? len - t : 0;
            at = page_at(max(id, 0), t);
        };
        const auto request_k = [&] { cd.load(kr, k0 + at); };
        const auto request_v = [&] { cd.load(vr, v0 + at); };
        const auto put_k = [&](int buf, int i) {
            cd.template put<DT, CT>(own + 2 * KB * buf, i >> 1, i & 1, kr[i >> 1]);
        };
        const auto put_v = [&](int buf, int i, auto type) {
            cd.template put<type, CT>(own + 2 * KB * buf + KB, i >> 1, i & 1, vr[i >> 1]);
        };
        const auto clip = [&] {
            if (lim < 16) {
#pragma unroll
                for (int n = 0; n < LOADS; ++n) cd.clip(vr[n], n, lim);
            }
        };
        constexpr std::integral_constant<int, DT> usual;         // V's type in LDS
        constexpr std::integral_constant<int, CAREFUL_DT> careful;
        const auto put_all = [&](int buf, auto type) {
#pragma unroll
            for (int i = 0; i < 2 * LOADS; ++i) {
                put_k(buf, i);
                put_v(buf, i, type);
                step();
            }
        };
        const auto turn = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
        const auto seen = [&](int j) {             // by some row of the wave
            const int t0 = CK_KEYS * (sp.lo + j);
            return !idle && t0 < hi_hi && t0 + CK_KEYS > lo_lo;
        };
        reset(st);
        bool again = false;
        if (j0 < j1) {
            look(lk, CK_KEYS * (sp.lo + j0) + 16 * lane, 16 * WAVE);
            find(j0, 0);
            request_k();
            request_v();
            clip();
            put_all(0, usual);
            find(j0 + 1, 1);                       // (past the part: its keys are there or none are)
            request_k();
            request_v();
            // tiles [f0, f1) hold only keys that all of the wave's rows see
            const int f1 = idle ? j1 : min(j1, hi_lo / CK_KEYS - sp.lo);
            const int f0 = idle ? j1 : min(f1, max(j0, (lo_hi + CK_KEYS - 1) / CK_KEYS - sp.lo));
            int s = 0;
            const auto tile = [&](int j, auto masks) {
                const uint32_t ks = base + 2 * KB * ((j - j0) & 1);
                const int buf = (j + 1 - j0) & 1, t0 = CK_KEYS * (sp.lo + j);
                clip();
                find(j + 2, s + 2);
                const Factors<4> f(lk, s);
                ordered_tile<DT, D, masks>(
                    ks, ks + KB, ll, q, f, st, lo - t0, hi - t0, lane,
                    [&](int i) {
                        put_k(buf, i);
                        if (i == 2 * LOADS - 1) request_k();
                    },
                    [&](int i) { put_v(buf, i, usual); });
                request_v();
            };
            const auto pass = [&](int j) {         // a tile that none of the wave's rows see
                clip();
                put_all((j + 1 - j0) & 1, usual);
                find(j + 2, s + 2);
                request_k();
                request_v();
            };
            const auto next = [&] {
                if (++s == Lookup<DT, 4>::STEPS) {
                    lk.turn();
                    s = 0;
                }
            };
            const auto walk = [&](int j, int end, auto masks) {
                for (; j < end; ++j) {
                    turn();
                    lk.ahead(s);
                    if (!masks || seen(j)) tile(j, masks);
                    else pass(j);
                    next();
                }
            };
            walk(j0, f0, std::true_type());
            walk(max(f0, j0), f1, std::false_type());
            walk(max(f1, j0), j1, std::true_type());     // (f1 may lie before this part)
            const bool bad = needs_care(st, live, lk.apart());
            if (lane == 0) lds.bad[w] = bad;
            __syncthreads();
            again = __builtin_amdgcn_readfirstlane(lds.bad[0] | lds.bad[1] | lds.bad[2] | lds.bad[3]) != 0;
        }
        if (again) {
            float mo = 0.f;
            reset(st);
            look(lk, CK_KEYS * (sp.lo + j0) + 16 * lane, 16 * WAVE);
            for (int j = j0, s = 0; j < j1; ++j) {
                find(j, s);
                request_k();
                request_v();
                clip();
                if constexpr (CT == AMASS_E4M3) {
#pragma unroll
                    for (int n = 0; n < LOADS; ++n) cd.poison(kr[n], vr[n]);
                }
                put_all((j - j0) & 1, careful);
                turn();
                lk.ahead(s);
                if (seen(j)) {
                    const uint32_t ks = base + 2 * KB * ((j - j0) & 1);
                    const int t0 = CK_KEYS * (sp.lo + j);
                    const Factors<4> f(lk, s);
                    f32x16_t sc2[2];
                    Weights<4, LIMBS<DT>> wt;
                    scores<DT, D, 2>(ks, ll, q, sc2);
                    mask_scores<2>(sc2, lo - t0, hi - t0, lk.groups(s), lane);
                    weigh_careful<DT, D, 2>(sc2, f, st, mo, wt);
                    add_values<D, 2>(ks + KB, ll, wt, st);
                }
                if (++s == Lookup<DT, 4>::STEPS) {
                    lk.turn();
                    s = 0;
                }
            }
            careful_end(st, mo);
        }
        if (idle) return;
        finish_rows<DT, D, QC_UP>(a, pl, it, kh, st, 1.f, row, group, whole, lane);
        return;
    }
    // ---- few rows: each wave its own 32 keys, w + 4, w + 8, ... ------------------------
    // Codes go from HBM to LDS as they are, a step ahead, and are widened on their way into a matrix operand: no
    // wave shares a key with another here.  (Two steps ahead, 128 KB in flight a CU, 64 single tokens with 8k keys
    // took 2 to 3 % longer.)
    using Raw = RawRows<D>;
    constexpr int HALF = 32 * D, L = 2 * Raw::LOADS;     // bytes of 32 keys' K; its loads
    char* own = lds.kv + 2 * HALF * w;                   // K, then V
    const uint32_t base = lds_addr(own);
    const int b0 = 2 * (sp.lo + j0) + w, b1 = 2 * (sp.lo + j1);
    const Raw raw((uint32_t)a.kv_st, lane);
    Lookup<DT, 2> lk;
    // 32 keys of step s (b: their number); of V true if the usual number of loads is in flight
    const auto issue_k = [&](auto past, int b, int s) {
#pragma unroll
        for (int g = 0; g < 2; ++g)       // (a page without a block: block 0, whose weights are zero)
            raw.template load<past>(base + g * (HALF / 2), k0 + page_at(max(lk.block(s, g), 0), 32 * b + 16 * g));
    };
    const auto issue_v = [&](auto past, int b, int s) -> bool {
        const int id0 = lk.block(s, 0), id1 = lk.block(s, 1);
        const int64_t at0 = page_at(max(id0, 0), 32 * b), at1 = page_at(max(id1, 0), 32 * b + 16);
        if (id0 >= 0 && id1 >= 0 && 32 * b + 32 <= len) {
            raw.template load<past>(base + HALF, v0 + at0);
            raw.template load<past>(base + HALF + HALF / 2, v0 + at1);
            return true;
        }
        raw.load_part(own + HALF, base + HALF, v0 + at0, id0 >= 0 ? len - 32 * b : 0);
        raw.load_part(own + HALF + HALF / 2, base + HALF + HALF / 2, v0 + at1, id1 >= 0 ? len - 32 * b - 16 : 0);
        return false;
    };
    const auto walk = [&](auto past, auto care) {
        float mo = 0.f;
        reset(st);
        bool full = true;                          // the usual number of loads of V is in flight
        if (b0 < b1) {
            look(lk, 32 * (b0 + CK_WAVES * (lane >> 1)) + 16 * (lane & 1), 32 * 32 * CK_WAVES);
            issue_k(past, b0, 0);
            full = issue_v(past, b0, 0);
        }
        for (int b = b0, s = 0; b < b1; b += CK_WAVES) {
            const int t0 = 32 * b;
            const bool more = b + CK_WAVES < b1;
            const uint32_t ks = base, vs = base + HALF;
            if (!care && full) dma_wait<L>();      // (V may be on its way)
            else dma_wait<0>();
            f32x16_t sc1[1];
            Weights<2, care ? LIMBS<DT> : 1> wt;
            few_scores<DT, CT, D, care>(ks, vs, raw, q, sc1[0]);
            dma_wait<63>();                        // (the reads have returned)
            if (more) issue_k(past, b + CK_WAVES, s + 1);
            lk.ahead(s);
            const Factors<2> f(lk, s);
            if (care || t0 < lo_hi || t0 + 32 > hi_lo)
                mask_scores<1>(sc1, lo - t0, hi - t0, lk.groups(s), lane);
            if constexpr (care) weigh_careful<DT, D, 1>(sc1, f, st, mo, wt);
            else weigh_tile<DT, D, 1>(sc1, f, st, wt.p[0]);
            if (more && full) dma_wait<L>();       // (the next K may be)
            else dma_wait<0>();
            few_values<care ? CAREFUL_DT : DT, CT, D, care>(vs, raw, wt, st);
            dma_wait<63>();
            if (more) full = issue_v(past, b + CK_WAVES, s + 1);
            if (++s == Lookup<DT, 2>::STEPS) {
                lk.turn();
                s = 0;
            }
        }
        dma_wait<0>();
        if constexpr (care) careful_end(st, mo);
    };
    if (once) walk(std::true_type(), std::false_type());
    else walk(std::false_type(), std::false_type());
    if (needs_care(st, live, lk.apart())) walk(std::false_type(), std::true_type());      // (this wave alone)
    __syncthreads();
    finish_shared<DT, D, QC_UP>(a, pl, it, kh, st, lds, 1.f, row, whole, w, lane);
}

template <int DT, int D>
__global__ __launch_bounds__(CM_WAVES * WAVE) void quant_merge_kernel(const amass_chunk_args a,
                                                                      const ChunkPlan pl) {
    merge_parts<DT, D, QC_UP>(a, pl, 1.f);
}

// ------------------------------------------------------------------ host
static bool quant_empty(const amass_quant_chunk_args& a) { return a.n_tokens == 0 || a.n_req == 0; }

static int quant_check(const amass_quant_chunk_args& a) {
    if (quant_empty(a)) return AMASS_OK;
    if (!a.q || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.block_table || !a.seq_lens ||
        !a.query_start || !a.out)
        return AMASS_ERR_NULL;
    if ((a.dtype != AMASS_BF16 && a.dtype != AMASS_FP16) || (a.code != AMASS_INT8 && a.code != AMASS_E4M3) ||
        (a.d != 64 && a.d != 128))
        return AMASS_ERR_UNSUPPORTED;
    if (a.page < 16 || a.page > 1024 || (a.page & (a.page - 1))) return AMASS_ERR_GEOMETRY;
    if (a.n_req < 0 || a.n_tokens < 0 || a.n_kv < 1 || a.G < 1 || a.nb < 1 || a.max_pages < 1 ||
        a.window < 0 || !(a.scale > 0.f) || a.scale > 2e38f)
        return AMASS_ERR_GEOMETRY;
    if (a.n_kv > 4096 || a.G > 4096 || (int64_t)a.n_tokens * a.G > (1 << 30)) return AMASS_ERR_GEOMETRY;
    const auto off = [](const void* p) { return ((uintptr_t)p & 15) != 0; };
    if (off(a.q) || off(a.k_codes) || off(a.v_codes) || off(a.out) ||
        ((a.q_st | a.q_hs | a.o_st | a.o_hs) & 7) || ((a.c_sb | a.c_st | a.c_sh) & 15))
        return AMASS_ERR_GEOMETRY;
    // the kernel has 32 bits for a row's offset within its block
    if (a.c_sb < 0 || a.c_sb >= (1ll << 31) || a.c_st < 0 || a.c_st * a.page >= (1ll << 31))
        return AMASS_ERR_GEOMETRY;
    return AMASS_OK;
}

// the arguments that the plan and the results share with amass_chunk_attention
static amass_chunk_args chunk_args_of(const amass_quant_chunk_args& a) {
    amass_chunk_args c = {};
    c.q = a.q, c.q_st = a.q_st, c.q_hs = a.q_hs;
    c.k = a.k_codes, c.v = a.v_codes, c.kv_sb = a.c_sb, c.kv_st = a.c_st, c.kv_sh = a.c_sh;
    c.block_table = a.block_table, c.bt_st = a.bt_st;
    c.seq_lens = a.seq_lens, c.query_start = a.query_start;
    c.out = a.out, c.o_st = a.o_st, c.o_hs = a.o_hs;
    c.lse = a.lse, c.l_st = a.l_st, c.l_hs = a.l_hs;
    c.scratch = a.scratch, c.scratch_bytes = a.scratch_bytes;
    c.scale = a.scale, c.n_req = a.n_req, c.n_tokens = a.n_tokens, c.n_kv = a.n_kv, c.G = a.G;
    c.d = a.d, c.page = a.page, c.nb = a.nb, c.max_pages = a.max_pages;
    c.causal = a.causal, c.window = a.window, c.dtype = a.dtype;
    return c;
}

template <int DT, int CT, int D>
static int launch_quant(const amass_chunk_args& a, const Scales& sc, const ChunkPlan& p, hipStream_t s) {
    const int64_t items = (int64_t)p.items * a.n_kv;
    if (items * CK_WAVES * WAVE > 0xFFFFFFFFll) return AMASS_ERR_GEOMETRY;    // (threads of a launch)
    hipLaunchKernelGGL((quant_chunk_kernel<DT, CT, D>), dim3((unsigned)items), dim3(CK_WAVES * WAVE), 0, s, a,
                       sc, p);
    const int rc = check_launch();
    if (rc) return rc;
    // a cut tile has two slots at least
    const int cuts = p.tiles_max < (p.slots + 1) / 2 ? p.tiles_max : (p.slots + 1) / 2;
    hipLaunchKernelGGL((quant_merge_kernel<DT, D>), dim3(cuts * a.n_kv, p.slot_rows / 32, D / 32),
                       dim3(CM_WAVES * WAVE), 0, s, a, p);
    return check_launch();
}
template <int DT, int CT>
static int launch_quant(const amass_chunk_args& a, const Scales& sc, const ChunkPlan& p, hipStream_t s) {
    return a.d == 128 ? launch_quant<DT, CT, 128>(a, sc, p, s) : launch_quant<DT, CT, 64>(a, sc, p, s);
}

}  // namespace amass

using namespace amass;

extern "C" int64_t amass_quant_scratch_bytes(const amass_quant_chunk_args* a) {
    if (!a) return AMASS_ERR_NULL;
    const int rc = quant_check(*a);
    if (rc || quant_empty(*a)) return rc;
    const amass_chunk_args c = chunk_args_of(*a);
    return chunk_scratch(c, chunk_plan(c));
}

extern "C" int amass_quant_chunk_attention(const amass_quant_chunk_args* ain, void* stream) {
    if (!ain) return AMASS_ERR_NULL;
    const int rc = quant_check(*ain);
    if (rc) return rc;
    if (quant_empty(*ain)) return AMASS_OK;
    const amass_chunk_args a = chunk_args_of(*ain);
    if (!a.scratch) return AMASS_ERR_NULL;
    const ChunkPlan p = chunk_plan(a);
    if (((uintptr_t)a.scratch & 255) || a.scratch_bytes < chunk_scratch(a, p)) return AMASS_ERR_CAPACITY;
    const Scales sc = {ain->k_scale, ain->v_scale, ain->s_sb, ain->s_sh};
    hipStream_t s = (hipStream_t)stream;
    if (a.dtype == AMASS_BF16)
        return ain->code == AMASS_INT8 ? launch_quant<0, 0>(a, sc, p, s) : launch_quant<0, 1>(a, sc, p, s);
    return ain->code == AMASS_INT8 ? launch_quant<1, 0>(a, sc, p, s) : launch_quant<1, 1>(a, sc, p, s);
}
