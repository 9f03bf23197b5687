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
#include "chunk_core.h"

namespace amass {

// Keys that one row tile alone reads are loaded past the caches where the batch's row tiles read
// more bytes of K and V than this, half of the memory-side cache: 4 drafted tokens of 8 requests,
// 580 MB, 118 -> 103 us; 8 tokens with 8 heads per kv head, 164 MB, 43.7 -> 40.4; but 41 MB that the
// last call left there 24.1 -> 29.1 (1 kv head) and 21.8 -> 22.1 (8).
constexpr float CK_ONCE = 128e6f;
// maxima (times c) beyond this take the products with care: there a weight may be off by 2^(1/16);
// from 16 times as much on it may exceed fp16, from 2^11 times fp32
constexpr float CK_FAR = 0x1p20f;

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
            if (w == 0) store_lse<DT, 0>(ro, m, l, c, lane);
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
    if (whole) store_lse<DT, 0>(ro, st.m, l, c, lane);
    else save_stats<D>(g, st.m, l, lane);
}

template <int DT, int D>
__global__ __launch_bounds__(CM_WAVES * WAVE) void chunk_merge_kernel(const amass_chunk_args a,
                                                                      const ChunkPlan pl) {
    merge_parts<DT, D, 0>(a, pl, a.scale * 1.44269504088896341f);
}

// ------------------------------------------------------------------ host
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
