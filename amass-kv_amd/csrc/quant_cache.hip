// The paged cache in 8 bits for gfx950: the quantising write (amass_quant_write) and the reading back
// (amass_quant_read).
//
// Mathematics.  Write: a run of tokens in a block has one scale per half and head, s = max(step(max
// |x|), scale so far), and codes round(x / s).  K is turned first, as if in 64 bits: a product of an
// 8- or 11-bit number with an fp32 cosine is exact there and the difference rounded once, so that the 16-bit
// key, and with it the code, is the formula's and not one of the two beside it.  The int8 scales have
// 8 significant bits: then no quotient that is not half way between two codes lies nearer to it
// than 2^-17, so the fp32 quotient rounds to the code of the exact one.
//
// A run's numbers of one half and head stay in the registers of one wave (16 rows of 128: 32 a lane), of two
// where pages have 32 rows and of four beyond (a run of more than 64 rows is read twice), so the maximum is a chain
// of v_max, six exchanges and at most one barrier.  Runs are found in the slots: where a block
// starts or the one before is no neighbour.
// Read: 16 codes a thread, two 16-byte stores (two such units a thread took 86 us where one takes 82).
//
// HBM bounds both: a prompt of 8192 tokens (32 + 8 heads of 128, bf16, turned; 189 MB) 45 us, 4.2 TB/s where a copy
// reaches 4.8 to 5.1; its K and V alone, not turned, 13.5 us; three chunks of 1967 tokens, fp16 in pairs, 12.7 us among
// other calls, 13.9 in a graph over two batches in turn, the kernel alone 14.5 from an idle card; 16 single tokens 5 us,
// launch and two dependent rounds; 65536 tokens read back (403 MB) 81.5 us, 4.9 TB/s.
#include "quant_codes.h"

namespace amass {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ float half_f32(uint32_t w, int hi) {
    const uint32_t h = hi ? w >> 16 : w & 0xFFFFu;
    return DT == AMASS_BF16 ? bf16_to_f32((uint16_t)h) : fp16_to_f32((uint16_t)h);
}
template <int DT>
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {       // to nearest even
    if constexpr (DT == AMASS_BF16) return pack_bf16x2(lo, hi);
    else return (uint32_t)__half_as_ushort(__float2half_rn(lo)) |
                (uint32_t)__half_as_ushort(__float2half_rn(hi)) << 16;
}

// 16 channels of a head: 8 from c0 and 8 from c1
struct Chan {
    int c0, c1;
    bool turn;
};
__device__ __forceinline__ Chan channels(const amass_quant_write_args& a, int u, bool may_turn) {
    Chan c;
    c.turn = may_turn && 16 * u < a.rot;
    const bool apart = c.turn && !a.interleaved;
    c.c0 = apart ? 8 * u : 16 * u;
    c.c1 = apart ? (a.rot >> 1) + 8 * u : 16 * u + 8;
    return c;
}
// the 8 pairs of x (c0 ..) and y (c1 ..) turned: pair i is (x[i], y[i]), or interleaved two neighbours.
// EXACT: the 16-bit numbers that the products in 64 bits round to (through fp32).  The fp32 ones are off by less than
// 2^-22 (|f| + |g|) (|c| + |s|), so they round to others only that near to a border between two, once in thousands.
// fp16 asks 64 bits only there, bf16 always (us of three chunks of 1967 tokens in a graph: fp16 14.8 and paired 16.6
// with 64 bits always, 13.7 and 13.7 so; bf16 12.3 and 12.4 always, 12.7 and 12.8 so).
template <int DT, bool EXACT>
__device__ __forceinline__ void turn(const amass_quant_write_args& a, const float* tab, u32x4_t& x,
                                     u32x4_t& y) {
    const float4* tc = reinterpret_cast<const float4*>(tab);
    const float4* ts = reinterpret_cast<const float4*>(tab + (a.rot >> 1));
    const float4 c0 = tc[0], c1 = tc[1], s0 = ts[0], s1 = ts[1];
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    float f[8], g[8], p[8], r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = a.interleaved ? half_f32<DT>(i < 4 ? x[i] : y[i - 4], 0) : half_f32<DT>(x[i >> 1], i & 1);
        g[i] = a.interleaved ? half_f32<DT>(i < 4 ? x[i] : y[i - 4], 1) : half_f32<DT>(y[i >> 1], i & 1);
        if constexpr (EXACT && DT == AMASS_BF16) {
            p[i] = (float)((double)f[i] * cs[i] - (double)g[i] * sn[i]);
            r[i] = (float)((double)g[i] * cs[i] + (double)f[i] * sn[i]);
        } else {
            p[i] = f[i] * cs[i] - g[i] * sn[i];
            r[i] = g[i] * cs[i] + f[i] * sn[i];
        }
    }
    if constexpr (EXACT && DT == AMASS_FP16) {
        // the border within the fp32 numbers of one fp16 number; below the normal numbers they lie elsewhere
        const auto far = [](float v) {
            return fabsf(v - __uint_as_float((__float_as_uint(v) & ~0x1FFFu) | 0x1000u));
        };
        uint32_t near = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float off = 0x1p-22f * (fabsf(f[i]) + fabsf(g[i])) * (fabsf(cs[i]) + fabsf(sn[i]));
            near |= !(fminf(far(p[i]), far(r[i])) > off) || fminf(fabsf(p[i]), fabsf(r[i])) < 0x1p-14f ? 1u << i : 0u;
        }
        if (__any(near)) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (near >> i & 1) {
                    p[i] = (float)((double)f[i] * cs[i] - (double)g[i] * sn[i]);
                    r[i] = (float)((double)g[i] * cs[i] + (double)f[i] * sn[i]);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (a.interleaved) {
            x[i] = pack_half<DT>(p[i], r[i]);
            y[i] = pack_half<DT>(p[4 + i], r[4 + i]);
        } else {
            x[i] = pack_half<DT>(p[2 * i], p[2 * i + 1]);
            y[i] = pack_half<DT>(r[2 * i], r[2 * i + 1]);
        }
    }
}

constexpr int QW_THREADS = 256;
constexpr int QW_WAVES = QW_THREADS / WAVE;
constexpr int QW_ROWS = 16;              // rows that a wave holds
// Tokens that a workgroup looks for runs in: one, 4 or 16 by the batch's tokens.  The runs of a window follow each
// other, about 1 us each, and a workgroup that finds none costs as much of a place.  us in a graph with windows of
// 1 / 4 / 16 (32 + 8 heads of 128): 256 single tokens 6.3 / 8.8 / 28.5, a prompt of 256 7.7 / 5.1 / 4.6; 1024: 19.9
// / 17.5 / 32.0 and 17.2 / 10.5 / 7.1; 2048: 36.3 / 30.3 / 38.5 and 30.3 / 17.5 / 10.5.  The number of tokens is all that
// the host knows (which kind they are is in the slots), so each border weighs both: up to 256 the rule is single
// tokens' best, and costs a prompt 3 us; up to 1024 it is the least sum; beyond, a batch is a prompt's rather than
// thousands of single tokens, which take 8 us more by it.
constexpr int window_of(int tokens) { return tokens <= 256 ? 1 : tokens <= 1024 ? 4 : 16; }

template <int D>
constexpr int LPR_OF = D / 16;           // lanes a row

// 16 channels of a query a thread
template <int DT, int D>
__device__ __forceinline__ void turn_queries(const amass_quant_write_args& a, uint32_t e) {
    const uint32_t per = (uint32_t)a.n_heads * LPR_OF<D>, t = e / per;
    if (t >= (uint32_t)a.n_tokens) return;
    const uint32_t rest = e - t * per, head = rest / LPR_OF<D>, u = rest % LPR_OF<D>;
    const int pos = a.positions[t];
    if ((uint32_t)pos >= (uint32_t)a.max_pos) return;
    const Chan c = channels(a, u, true);
    const uint16_t* src = (const uint16_t*)a.q + t * a.q_st + head * a.q_hs;
    uint16_t* dst = (uint16_t*)a.q_out + t * a.qo_st + head * a.qo_hs;
    u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + c.c0);
    u32x4_t y = *reinterpret_cast<const u32x4_t*>(src + c.c1);
    if (c.turn) turn<DT, false>(a, a.table + pos * a.tab_st + 8 * u, x, y);
    *reinterpret_cast<u32x4_t*>(dst + c.c0) = x;
    *reinterpret_cast<u32x4_t*>(dst + c.c1) = y;
}

// Workgroups: `groups` for each window of tokens, then those of the queries.  A workgroup's waves are teams of
// TEAM, a team has a run's numbers of one half and head, QW_ROWS rows a wave.
template <int DT, int CT, int D, int TEAM>
__global__ __launch_bounds__(QW_THREADS) void quant_write_kernel(const amass_quant_write_args a, int sh,
                                                                 int window, int groups, int kv_wgs) {
    constexpr int LPR = LPR_OF<D>, RPL = WAVE / LPR, N = QW_ROWS / RPL;   // lanes a row, rows a load, loads
    constexpr int STEP = TEAM * QW_ROWS;
    __shared__ uint32_t tops[QW_WAVES];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= kv_wgs) {
        turn_queries<DT, D>(a, (blockIdx.x - kv_wgs) * QW_THREADS + threadIdx.x);
        return;
    }
    const int64_t end = (int64_t)a.nb << sh;
    const int t0 = blockIdx.x / groups * window;
    const int unit = (blockIdx.x % groups) * (QW_WAVES / TEAM) + w / TEAM, mate = w % TEAM;
    const bool is_k = unit < a.n_kv, works = unit < 2 * a.n_kv;
    const int head = is_k ? unit : unit - a.n_kv;
    const int lr = lane / LPR, u = lane % LPR;
    const Chan c = channels(a, u, is_k && a.table);

    // Lane i looks at token t0 + i (one round of memory): whether it enters a block, and as its
    // neighbour's successor in it.  Runs start where it is none.
    int64_t sl = -1, sl0 = -1;
    int ps = 0, ps0 = 0;
    if (t0 + lane < a.n_tokens) {
        sl = a.slots[t0 + lane];
        if (a.table) ps = a.positions[t0 + lane];
    }
    if (t0 > 0) {
        sl0 = a.slots[t0 - 1];
        if (a.table) ps0 = a.positions[t0 - 1];
    }
    const auto fits = [&](int64_t slot, int pos) {
        return (uint64_t)slot < (uint64_t)end && (!a.table || (uint32_t)pos < (uint32_t)a.max_pos);
    };
    const auto follows = [&](int64_t slot) { return (slot & ((1 << sh) - 1)) != 0; };
    const unsigned long long enter = __ballot(fits(sl, ps));
    const int64_t up = __shfl_up(sl, 1);         // (by all lanes)
    const int64_t before = lane == 0 ? sl0 : up;
    const bool neighbour = lane == 0 ? fits(sl0, ps0) : (enter >> (lane - 1)) & 1;
    const unsigned long long joins = __ballot(neighbour && sl == before + 1 && follows(sl)) & enter;
    for (unsigned long long left = enter & ~joins & ((2ull << (window - 1)) - 1); left; left &= left - 1) {
        const int i0 = __ffsll((long long)left) - 1, t = t0 + i0;
        const int64_t slot = (int64_t)readlane_u64((unsigned long long)sl, i0);
        const int first = (int)(slot & ((1 << sh) - 1));
        const int64_t blk = slot >> sh;
        // the run's length: the tokens behind the first that join, past the 64 a look at the next ones
        const unsigned long long rest = i0 < WAVE - 1 ? joins >> (i0 + 1) : 0;
        int n = ~rest ? __ffsll((long long)~rest) : WAVE;
        for (bool more = i0 + n == WAVE; more;) {
            const int i = n + lane, at = min(t + i, a.n_tokens - 1);
            const int64_t next = a.slots[at];
            const bool in = t + i < a.n_tokens && next == slot + i && follows(next) &&
                            fits(next, a.table ? a.positions[at] : 0);
            const unsigned long long out = ~__ballot(in);
            n += out ? __ffsll((long long)out) - 1 : WAVE;
            more = !out;
        }
        const uint16_t* src = is_k ? (const uint16_t*)a.k + t * a.k_st + head * a.k_hs
                                   : (const uint16_t*)a.v + t * a.v_st + head * a.v_hs;
        const int64_t src_st = is_k ? a.k_st : a.v_st;
        uint8_t* codes = (uint8_t*)(is_k ? a.k_codes : a.v_codes) + blk * a.c_sb + head * a.c_sh;
        float* scale = (is_k ? a.k_scale : a.v_scale) + blk * a.s_sb + head * a.s_sh;
        const float old = works && first > 0 ? *scale : 0.f;
        u32x4_t x[N], y[N];
        const auto load = [&](int r0) {                  // rows r0 .. r0 + 15 of the run
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = r0 + RPL * i + lr;
                x[i] = y[i] = (u32x4_t){0u, 0u, 0u, 0u};
                if (works && r < n) {
                    x[i] = *reinterpret_cast<const u32x4_t*>(src + r * src_st + c.c0);
                    y[i] = *reinterpret_cast<const u32x4_t*>(src + r * src_st + c.c1);
                }
            }
            if (is_k && a.table) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int r = r0 + RPL * i + lr;
                    int pos = __shfl(ps, (i0 + r) & (WAVE - 1));
                    if (r < n && i0 + r >= WAVE) pos = a.positions[t + r];
                    if (r < n && c.turn)
                        turn<DT, true>(a, a.table + (int64_t)pos * a.tab_st + 8 * u, x[i], y[i]);
                }
            }
        };
        // the largest magnitude as 16 bits, NaN above infinity above every number
        uint32_t top = 0;
        for (int r0 = mate * QW_ROWS; r0 < n; r0 += STEP) {
            load(r0);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t p = x[i][j] & 0x7FFF7FFFu, q = y[i][j] & 0x7FFF7FFFu;
                    top = max(top, max(max(p & 0xFFFFu, p >> 16), max(q & 0xFFFFu, q >> 16)));
                }
        }
        top = (uint32_t)wave_max_uniform((int)top);
        if constexpr (TEAM > 1) {
            if (lane == 0) tops[w] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TEAM; ++i) top = max(top, tops[w - mate + i]);
            top = __builtin_amdgcn_readfirstlane(top);
            __syncthreads();
        }
        if (!works) continue;
        const bool finite = top < (DT == AMASS_BF16 ? 0x7F80u : 0x7C00u);
        float s = __builtin_nanf("");
        if (finite) {
            const float step = step_of<CT>(half_f32<DT>(top, 0));
            s = step >= old ? step : old;                // (a NaN stays)
        }
        const bool keep = s < INFINITY;
        const float div = keep ? s : 1.f, inv = 1.f / div;
        for (int r0 = mate * QW_ROWS; r0 < n; r0 += STEP) {
            if (n > STEP) load(r0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = r0 + RPL * i + lr;
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t p = j < 2 ? x[i][2 * j] : y[i][2 * j - 4];
                    const uint32_t q = j < 2 ? x[i][2 * j + 1] : y[i][2 * j - 3];
                    o[j] = to_codes<CT>(quotient(half_f32<DT>(p, 0), div, inv), quotient(half_f32<DT>(p, 1), div, inv),
                                        quotient(half_f32<DT>(q, 0), div, inv), quotient(half_f32<DT>(q, 1), div, inv));
                    if (!keep) o[j] = 0u;
                }
                if (r < n) {
                    uint8_t* to = codes + (first + r) * a.c_st;
                    *reinterpret_cast<u32x2_t*>(to + c.c0) = (u32x2_t){o[0], o[1]};
                    *reinterpret_cast<u32x2_t*>(to + c.c1) = (u32x2_t){o[2], o[3]};
                }
            }
        }
        if (first > 0 && s > old) {                      // the rows before the run, by the new scale
            for (int r = mate * RPL + lr; r < first; r += TEAM * RPL) {
                u32x4_t* at = reinterpret_cast<u32x4_t*>(codes + r * a.c_st + 16 * u);
                u32x4_t z = *at;
#pragma unroll
                for (int j = 0; j < 4; ++j) z[j] = round_again<CT>(z[j], old, div, inv);
                *at = z;
            }
        }
        if (lane == 0 && mate == 0) *scale = s;
    }
}

// grid (entry, half and 256 units of 16 codes of the block)
constexpr int QR_THREADS = 256;

template <int DT, int CT, int D>
__global__ __launch_bounds__(QR_THREADS) void quant_read_kernel(const amass_quant_read_args a, int sh) {
    constexpr int LPR = LPR_OF<D>;
    const int src = a.src[blockIdx.x], dst = a.dst[blockIdx.x];
    if ((uint32_t)src >= (uint32_t)a.nb || (uint32_t)dst >= (uint32_t)a.nb_out) return;
    const bool is_k = !(blockIdx.y & 1);
    const int e = (blockIdx.y >> 1) * QR_THREADS + threadIdx.x;
    if (e >= (a.n_kv << sh) * LPR) return;
    const int rh = e / LPR, c = 16 * (e % LPR), row = rh / a.n_kv, head = rh - row * a.n_kv;
    const uint8_t* codes = (const uint8_t*)(is_k ? a.k_codes : a.v_codes) + src * a.c_sb;
    const u32x4_t z = *reinterpret_cast<const u32x4_t*>(codes + row * a.c_st + head * a.c_sh + c);
    const float s = (is_k ? a.k_scale : a.v_scale)[src * a.s_sb + head * a.s_sh];
    u32x4_t o[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 f = codes_f32<CT>(z[j]);
        o[j >> 1][2 * (j & 1)] = pack_half<DT>(f.x * s, f.y * s);
        o[j >> 1][2 * (j & 1) + 1] = pack_half<DT>(f.z * s, f.w * s);
    }
    uint16_t* to = (uint16_t*)(is_k ? a.k_cache : a.v_cache) + dst * a.o_sb + row * a.o_st + head * a.o_sh + c;
    reinterpret_cast<u32x4_t*>(to)[0] = o[0];
    reinterpret_cast<u32x4_t*>(to)[1] = o[1];
}

// ------------------------------------------------------------------ host
static bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
static int log2_of(int page) {
    int sh = 0;
    while ((1 << sh) < page) ++sh;
    return sh;
}
static int check_kind(int d, int page, int dtype, int code) {
    if ((dtype != AMASS_BF16 && dtype != AMASS_FP16) || (code != AMASS_INT8 && code != AMASS_E4M3) ||
        (d != 64 && d != 128))
        return AMASS_ERR_UNSUPPORTED;
    return page < 16 || page > 1024 || (page & (page - 1)) ? AMASS_ERR_GEOMETRY : AMASS_OK;
}

static int check_write(const amass_quant_write_args& a) {
    if (!a.k || !a.v || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.slots ||
        (a.q && (!a.q_out || !a.table)) || (a.table && !a.positions))
        return AMASS_ERR_NULL;
    const int rc = check_kind(a.d, a.page, a.dtype, a.code);
    if (rc) return rc;
    if (a.n_tokens < 0 || a.n_kv < 1 || a.n_kv > 4096 || a.nb < 1) return AMASS_ERR_GEOMETRY;
    if (misaligned(a.k) || misaligned(a.v) || misaligned(a.k_codes) || misaligned(a.v_codes) ||
        ((a.k_st | a.k_hs | a.v_st | a.v_hs) & 7) || ((a.c_sb | a.c_st | a.c_sh) & 15))
        return AMASS_ERR_GEOMETRY;
    if (a.table && (a.rot < 16 || (a.rot & 15) || a.rot > a.d || a.max_pos < 1 || misaligned(a.table) ||
                    (a.tab_st & 3)))
        return AMASS_ERR_GEOMETRY;
    if (a.q && (a.n_heads < 1 || a.n_heads > (1 << 16) || misaligned(a.q) || misaligned(a.q_out) ||
                ((a.q_st | a.q_hs | a.qo_st | a.qo_hs) & 7)))
        return AMASS_ERR_GEOMETRY;
    return AMASS_OK;
}
static int check_read(const amass_quant_read_args& a) {
    if (!a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.k_cache || !a.v_cache || !a.src || !a.dst)
        return AMASS_ERR_NULL;
    const int rc = check_kind(a.d, a.page, a.dtype, a.code);
    if (rc) return rc;
    if (a.n < 0 || a.n_kv < 1 || a.n_kv > 4096 || a.nb < 1 || a.nb_out < 1) return AMASS_ERR_GEOMETRY;
    if (misaligned(a.k_codes) || misaligned(a.v_codes) || misaligned(a.k_cache) || misaligned(a.v_cache) ||
        ((a.c_sb | a.c_st | a.c_sh) & 15) || ((a.o_sb | a.o_st | a.o_sh) & 7))
        return AMASS_ERR_GEOMETRY;
    return AMASS_OK;
}

template <int DT, int CT, int D, int TEAM>
static int launch_write(const amass_quant_write_args& a, hipStream_t s) {
    const int64_t window = window_of(a.n_tokens);
    const int64_t groups = (2 * a.n_kv * TEAM + QW_WAVES - 1) / QW_WAVES;
    const int64_t kv_wgs = (a.n_tokens + window - 1) / window * groups;
    const int64_t units = a.q ? (int64_t)a.n_tokens * a.n_heads * LPR_OF<D> : 0;
    const int64_t wgs = kv_wgs + (units + QW_THREADS - 1) / QW_THREADS;
    if (wgs * QW_THREADS > 0xFFFFFFFFll) return AMASS_ERR_GEOMETRY;          // (threads of a launch)
    hipLaunchKernelGGL((quant_write_kernel<DT, CT, D, TEAM>), dim3((unsigned)wgs), dim3(QW_THREADS), 0, s, a,
                       log2_of(a.page), (int)window, (int)groups, (int)kv_wgs);
    return check_launch();
}
template <int DT, int CT, int D>
static int launch_write(const amass_quant_write_args& a, hipStream_t s) {
    if (a.page == 16) return launch_write<DT, CT, D, 1>(a, s);
    return a.page == 32 ? launch_write<DT, CT, D, 2>(a, s) : launch_write<DT, CT, D, 4>(a, s);
}
template <int DT, int CT>
static int launch_write(const amass_quant_write_args& a, hipStream_t s) {
    return a.d == 128 ? launch_write<DT, CT, 128>(a, s) : launch_write<DT, CT, 64>(a, s);
}
template <int DT, int CT>
static int launch_read(const amass_quant_read_args& a, hipStream_t s) {
    const int sh = log2_of(a.page);
    const int64_t units = (int64_t)a.n_kv * a.page * (a.d / 16);
    const int64_t parts = 2 * ((units + QR_THREADS - 1) / QR_THREADS);
    if (parts > 65535 || (int64_t)a.n * QR_THREADS > 0xFFFFFFFFll) return AMASS_ERR_GEOMETRY;
    const dim3 grid(a.n, (unsigned)parts);
    if (a.d == 128)
        hipLaunchKernelGGL((quant_read_kernel<DT, CT, 128>), grid, dim3(QR_THREADS), 0, s, a, sh);
    else
        hipLaunchKernelGGL((quant_read_kernel<DT, CT, 64>), grid, dim3(QR_THREADS), 0, s, a, sh);
    return check_launch();
}

}  // namespace amass

using namespace amass;

extern "C" int amass_quant_write(const amass_quant_write_args* ain, void* stream) {
    if (!ain) return AMASS_ERR_NULL;
    const amass_quant_write_args& a = *ain;
    if (a.n_tokens == 0) return AMASS_OK;
    const int rc = check_write(a);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (a.dtype == AMASS_BF16)
        return a.code == AMASS_INT8 ? launch_write<0, 0>(a, s) : launch_write<0, 1>(a, s);
    return a.code == AMASS_INT8 ? launch_write<1, 0>(a, s) : launch_write<1, 1>(a, s);
}

extern "C" int amass_quant_read(const amass_quant_read_args* ain, void* stream) {
    if (!ain) return AMASS_ERR_NULL;
    const amass_quant_read_args& a = *ain;
    if (a.n == 0) return AMASS_OK;
    const int rc = check_read(a);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (a.dtype == AMASS_BF16)
        return a.code == AMASS_INT8 ? launch_read<0, 0>(a, s) : launch_read<0, 1>(a, s);
    return a.code == AMASS_INT8 ? launch_read<1, 0>(a, s) : launch_read<1, 1>(a, s);
}

extern "C" int amass_quant_abi_version(void) { return AMASS_QUANT_ABI_VERSION; }

extern "C" size_t amass_quant_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(amass_quant_write_args);
        case 1: return sizeof(amass_quant_read_args);
        case 2: return sizeof(amass_quant_chunk_args);
        default: return 0;
    }
}
