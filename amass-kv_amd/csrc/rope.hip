// Rotary positions and the paged K / V write for gfx950 (amass_rope_write).
//
// Mathematics.  With c_i and s_i = cos and sin of p w_i (times the table's amplitude) the pair
// (x, y) becomes (x c_i - y s_i, x s_i + y c_i), in fp32, rounded once to the element type.
//
// One pass: every element of q, k and v is read once and written once, so HBM bounds it
// (4 (H + 2 n_kv) d bytes per token in 16-bit types, 4 rot bytes of table beside them).  A thread
// owns 16 channels of one head of one token: 8 pairs (the 8 from channel 8u and the 8 from
// rot/2 + 8u, or 16 in a row when the pairs are interleaved), so both loads and both stores
// are 16 bytes and q may be turned in place.  The heads of a token share its table row
// through the L1.  A prompt of 8192 tokens (32 + 8 heads of 128, bf16; 206 MB) takes 42 us, 4.9
// TB/s, where a copy reaches 5.1; three chunks of 1800 tokens with 64 of 128 channels turned in
// pairs 10.8 us, 4.5 TB/s; 16 single tokens 2.8 us, launch and three dependent rounds.
// Shapes or addresses that 16-byte accesses do not fit take the same kernel with one pair per
// thread: the 8192 tokens, over and over in the caches, 66 us against 33.
#include "../../include/amass_chunk.h"
#include "common.h"

namespace amass {

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t h) {
    return DT == AMASS_BF16 ? bf16_to_f32(h) : fp16_to_f32(h);
}
template <int DT>
__device__ __forceinline__ uint16_t from_f32(float f) {     // to nearest even
    if (DT == AMASS_BF16) return (uint16_t)pack_bf16x2(f, 0.f);
    return __half_as_ushort(__float2half_rn(f));
}

template <int N>
struct __align__(2 * N) Vec16 {
    uint16_t e[N];
};
template <int N>
struct __align__(4 * (N < 4 ? N : 4)) VecF {
    float e[N];
};

constexpr int ROPE_THREADS = 256;

// grid (tokens, chunks of a token's units): unit e is head slot e / upt (q heads, k heads,
// v heads) and the 2 N channels e % upt of it.
template <int DT, int N, bool PAIRS>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const amass_rope_args a, int sh) {
    const int t = blockIdx.x;
    const int upt = a.d / (2 * N);
    const int e = blockIdx.y * blockDim.x + threadIdx.x;
    const int head = e / upt, u = e - head * upt;
    const int heads = a.n_heads + a.n_kv * (a.v ? 2 : 1);
    const int pos = a.positions[t];
    if (head >= heads || pos < 0 || pos >= a.max_pos) return;
    const int kind = head < a.n_heads ? 0 : head < a.n_heads + a.n_kv ? 1 : 2;
    const uint16_t* src;
    uint16_t* dst;
    if (kind == 0) {
        src = (const uint16_t*)a.q + t * a.q_st + head * a.q_hs;
        dst = (uint16_t*)a.q_out + t * a.qo_st + head * a.qo_hs;
    } else {
        const int64_t slot = a.slots[t];
        if (slot < 0 || slot >= (int64_t)a.nb << sh) return;
        const int64_t blk = slot >> sh, row = slot & ((1 << sh) - 1);
        if (kind == 1) {
            const int h = head - a.n_heads;
            src = (const uint16_t*)a.k + t * a.k_st + h * a.k_hs;
            dst = (uint16_t*)a.k_cache + blk * a.kc_sb + row * a.kc_st + h * a.kc_sh;
        } else {
            const int h = head - a.n_heads - a.n_kv;
            src = (const uint16_t*)a.v + t * a.v_st + h * a.v_hs;
            dst = (uint16_t*)a.v_cache + blk * a.vc_sb + row * a.vc_st + h * a.vc_sh;
        }
    }
    const int half = a.rot >> 1;
    const bool turn = kind < 2 && u * 2 * N < a.rot;
    const int c0 = !PAIRS && turn ? u * N : u * 2 * N;       // the two runs of N channels
    const int c1 = !PAIRS && turn ? half + u * N : c0 + N;
    Vec16<N> x = *reinterpret_cast<const Vec16<N>*>(src + c0);
    Vec16<N> y = *reinterpret_cast<const Vec16<N>*>(src + c1);
    if (turn) {
        const float* tab = a.table + (int64_t)pos * a.tab_st + u * N;
        const VecF<N> c = *reinterpret_cast<const VecF<N>*>(tab);
        const VecF<N> s = *reinterpret_cast<const VecF<N>*>(tab + half);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint16_t& p0 = !PAIRS ? x.e[i] : 2 * i < N ? x.e[(2 * i) % N] : y.e[(2 * i) % N];
            uint16_t& p1 = !PAIRS ? y.e[i] : 2 * i + 1 < N ? x.e[(2 * i + 1) % N] : y.e[(2 * i + 1) % N];
            const float f = to_f32<DT>(p0), g = to_f32<DT>(p1);
            p0 = from_f32<DT>(f * c.e[i] - g * s.e[i]);
            p1 = from_f32<DT>(g * c.e[i] + f * s.e[i]);
        }
    }
    *reinterpret_cast<Vec16<N>*>(dst + c0) = x;
    *reinterpret_cast<Vec16<N>*>(dst + c1) = y;
}

template <int DT, int N>
static int launch_rope(const amass_rope_args& a, hipStream_t s) {
    int sh = 0;
    while ((1 << sh) < a.page) ++sh;
    const int64_t units = (int64_t)(a.n_heads + a.n_kv * (a.v ? 2 : 1)) * (a.d / (2 * N));
    const int chunks = (int)((units + ROPE_THREADS - 1) / ROPE_THREADS);
    const int threads = (int)(((units + chunks - 1) / chunks + WAVE - 1) / WAVE) * WAVE;
    if (chunks > 65535 || (int64_t)a.n_tokens * threads > 0xFFFFFFFFll) return AMASS_ERR_GEOMETRY;
    const dim3 grid(a.n_tokens, chunks);
    if (a.interleaved)
        hipLaunchKernelGGL((rope_kernel<DT, N, true>), grid, dim3(threads), 0, s, a, sh);
    else
        hipLaunchKernelGGL((rope_kernel<DT, N, false>), grid, dim3(threads), 0, s, a, sh);
    return check_launch();
}

}  // namespace amass

using namespace amass;

extern "C" int amass_rope_write(const amass_rope_args* ain, void* stream) {
    if (!ain) return AMASS_ERR_NULL;
    const amass_rope_args& a = *ain;
    if (a.n_tokens == 0) return AMASS_OK;
    if (!a.q || !a.k || !a.q_out || !a.k_cache || !a.table || !a.positions || !a.slots ||
        (a.v && !a.v_cache))
        return AMASS_ERR_NULL;
    if (a.n_tokens < 0 || a.n_heads < 1 || a.n_kv < 1 || a.d < 2 || (a.d & 1) || a.rot < 2 ||
        (a.rot & 1) || a.rot > a.d || a.nb < 1 || a.max_pos < 1 || a.page < 1 ||
        a.page > (1 << 20) || (a.page & (a.page - 1)))
        return AMASS_ERR_GEOMETRY;
    if (a.n_heads > (1 << 16) || a.n_kv > (1 << 16) || a.d > (1 << 12)) return AMASS_ERR_GEOMETRY;
    if (a.dtype != AMASS_BF16 && a.dtype != AMASS_FP16) return AMASS_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    // 16-byte accesses: 8 channels, so every row and both runs of a unit start at one
    const auto off = [](const void* p) { return ((uintptr_t)p & 15) != 0; };
    const int64_t st = a.q_st | a.q_hs | a.k_st | a.k_hs | a.qo_st | a.qo_hs | a.kc_sb | a.kc_st |
                       a.kc_sh | (a.v ? a.v_st | a.v_hs | a.vc_sb | a.vc_st | a.vc_sh : 0);
    const bool wide = !(off(a.q) || off(a.k) || off(a.q_out) || off(a.k_cache) || off(a.table) ||
                        (a.v && (off(a.v) || off(a.v_cache)))) &&
                      !(st & 7) && !(a.d & 15) && !(a.rot & 15) && !(a.tab_st & 3);
    if (a.dtype == AMASS_BF16) return wide ? launch_rope<0, 8>(a, s) : launch_rope<0, 1>(a, s);
    return wide ? launch_rope<1, 8>(a, s) : launch_rope<1, 1>(a, s);
}
