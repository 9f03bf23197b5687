/*
 * amass_chunk.h -- C-ABI of the operators around a chunk of new tokens (gfx950).
 *
 * The same library (libamass_hip.so), status codes and calling rules as amass_hip.h: POD
 * argument structs of device pointers, ELEMENT strides and geometry, launches on `stream`,
 * no device allocation, no host synchronisation, nothing throws, fixed-shape launches that a
 * caller may capture in a HIP graph.  None of them has a counterpart in the reference, which
 * leaves prompts, slot maps and rotary positions to the serving engine.
 *
 * One step of a serving program brings n_req requests.  Request r brings the tokens (rows of
 * q, k, v, slots, ...) query_start[r] .. query_start[r+1]-1, the last ones of the seq_lens[r]
 * tokens it then has, so its row query_start[r] + i is at position
 * seq_lens[r] - (query_start[r+1] - query_start[r]) + i.  query_start has n_req + 1 ascending
 * entries; rows from query_start[n_req] to n_tokens-1 belong to no request (a padded batch).
 * Entries below 0 or above n_tokens are taken as those.  With entries that do not ascend a call
 * touches nothing outside its tensors, and what it leaves in them is not specified.  Position p
 * of request r is in block block_table[r][p / page], row p % page; `page` is a power of two.
 */
#ifndef AMASS_CHUNK_H
#define AMASS_CHUNK_H

#include "amass_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AMASS_CHUNK_ABI_VERSION 1

/* element types of q, k, v, out and the cache */
#define AMASS_BF16 0
#define AMASS_FP16 1

#define AMASS_MAX_STEP_REQS 4096    /* requests of one amass_extend / amass_release call */

/* ---- block tables and slot maps ---------------------------------------------------- */
/* Gives every page that a step's tokens enter a block, and every token its slot.  Request r
 * had have_r = ceil((seq_lens[r] - n_r) / page) pages before its n_r new tokens and needs
 * need_r = min(ceil(seq_lens[r] / page), max_pages) with them.  Its new pages have_r ..
 * need_r-1 take blocks off the end of the free list free_list[0 .. top[0]-1], in (request,
 * page) order: the k-th new page of the step takes free_list[top[0] - 1 - k].  Then
 *   block_table[r][page index]  the block, for every new page (other entries stay)
 *   positions[t]                the token's position, -1 for a row of no request and for the
 *                               rows before position 0 of a request shorter than its chunk
 *   slots[t]                    block * page + position % page; -1 where the position is -1,
 *                               at or past max_pages * page, or in a page without a block
 *   top_out[0]                  free blocks left; top_out[2]: new pages that got none (those
 *                               of the highest k: their table entries become -1)
 * A block outside [0, nb), in the table or the list, counts as none.  top_out may be top
 * itself (the step is taken) or another buffer (free_list and top stay as they are, so the
 * step may be dropped).  top[1] counts arriving workgroups: zero before, zero after. */
typedef struct amass_extend_args {
    int32_t*       block_table; int64_t bt_st;   /* (R, max_pages) */
    const int32_t* seq_lens;                     /* (R,) */
    const int32_t* query_start;                  /* (R+1,) */
    const int32_t* free_list;                    /* (capacity,) */
    int32_t*       top;                          /* (3,) free blocks, arrivals, short */
    int32_t*       top_out;                      /* (3,); word 1 is not written */
    int64_t*       slots;                        /* (n_tokens,) */
    int32_t*       positions;                    /* (n_tokens,) */
    int32_t n_req, n_tokens, max_pages, page, nb, capacity;
} amass_extend_args;
int amass_extend(const amass_extend_args* a, void* stream);

/* Puts the blocks of finished requests back: for every r with done[r] != 0, in (request,
 * page) order, the blocks of its first min(ceil(seq_lens[r] / page), max_pages) pages go
 * behind the free list, and their table entries become -1.  Entries outside [0, nb) are
 * passed over; blocks past the list's capacity are dropped and counted in top[2], which the
 * call sets.  A block belongs to one request: one that two of them hold would go back twice. */
typedef struct amass_release_args {
    int32_t*       block_table; int64_t bt_st;
    const int32_t* seq_lens;
    const uint8_t* done;                         /* (R,) */
    int32_t*       free_list;
    int32_t*       top;
    int32_t n_req, max_pages, page, nb, capacity;
} amass_release_args;
int amass_release(const amass_release_args* a, void* stream);

/* ---- rotary positions and the paged write -------------------------------------------- */
/* Turns q and k by their positions and writes k and v to their slots of the paged cache.
 * With c_i = table[p][i] and s_i = table[p][rot/2 + i] of the token's position p, the pair
 * (x, y) = (u[i], u[i + rot/2]) of a head (interleaved 0) or (u[2i], u[2i+1]) (interleaved 1)
 * becomes (x c_i - y s_i, x s_i + y c_i), computed in fp32 and rounded once; channels rot ..
 * d-1 are copied.  q_out may be q.  k_cache / v_cache are one layer's (NB, page, n_kv, d)
 * views; v NULL writes no V.  A token whose position is outside [0, max_pos) is passed over
 * (q_out and the cache keep what they have there); one whose slot is outside [0, nb * page)
 * only has its q turned.  Two tokens of one slot leave values of either there, in pieces.  q_out
 * is q or shares no memory with it. */
typedef struct amass_rope_args {
    const void* q;     int64_t q_st, q_hs;               /* (T,H,d)    */
    const void* k;     int64_t k_st, k_hs;               /* (T,n_kv,d) */
    const void* v;     int64_t v_st, v_hs;               /* (T,n_kv,d) or NULL */
    void*       q_out; int64_t qo_st, qo_hs;             /* (T,H,d)    */
    void*       k_cache; int64_t kc_sb, kc_st, kc_sh;
    void*       v_cache; int64_t vc_sb, vc_st, vc_sh;
    const float*   table; int64_t tab_st;                /* (max_pos, rot): cos | sin */
    const int32_t* positions;                            /* (T,) */
    const int64_t* slots;                                /* (T,) */
    int32_t n_tokens, n_heads, n_kv, d, rot, page, nb, max_pos, interleaved, dtype;
} amass_rope_args;
int amass_rope_write(const amass_rope_args* a, void* stream);

/* ---- attention of a chunk over the paged cache ------------------------------------------ */
/* For every row of a request, at position p, and query head h of kv head h / G, over the
 * visible positions j of its request: j < min(seq_lens[r], max_pages * page), j <= p if
 * causal, j > p - window if window > 0, and block_table[r][j / page] in [0, nb):
 *   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / l,  lse = m + ln l  (natural log)
 * with m = max_j s_j and l = sum_j e^(s_j - m), sums and statistics in fp32, the weights
 * e^(s_j - m) rounded to the element type for the second product.  What is not visible is
 * not used, whatever it holds (infinities and NaN among it).  A visible infinity in V
 * makes its channel that infinity (NaN beside the opposite one, or where the key's weight is below
 * fp32's least), a visible NaN makes it NaN; a key of score -inf counts as not visible.  A row
 * that sees no finite score (a position below 0, an empty request, only scores of -inf) gets zeros
 * and lse = -inf.  Rows of no request are left as they are.  out may be q.  0 < scale <= 2e38.
 * d 64 or 128, page >= 16, G >= 1; q, out and the K and V views 16-byte aligned with strides of
 * multiples of 8 elements (a block below 2^30 of them).
 *
 * scratch: amass_chunk_scratch_bytes(a) bytes, 256-byte aligned, for the parts of rows whose
 * keys several workgroups share.  It holds nothing between calls; calls that may run at the
 * same time need one each. */
typedef struct amass_chunk_args {
    const void*    q; int64_t q_st, q_hs;                /* (T,H,d) */
    const void*    k; const void* v;                     /* (NB,page,n_kv,d) views of */
    int64_t        kv_sb, kv_st, kv_sh;                  /* the same strides */
    const int32_t* block_table; int64_t bt_st;
    const int32_t* seq_lens;
    const int32_t* query_start;
    void*          out; int64_t o_st, o_hs;              /* (T,H,d) */
    float*         lse; int64_t l_st, l_hs;              /* (T,H) or NULL */
    void*          scratch; int64_t scratch_bytes;
    float   scale;
    int32_t n_req, n_tokens, n_kv, G, d, page, nb, max_pages, causal, window, dtype;
} amass_chunk_args;
int     amass_chunk_attention(const amass_chunk_args* a, void* stream);
int64_t amass_chunk_scratch_bytes(const amass_chunk_args* a);   /* negative: a status */

/* ---- introspection (host only) -------------------------------------------------------- */
int    amass_chunk_abi_version(void);
size_t amass_chunk_struct_size(int which);   /* 0 extend, 1 release, 2 rope, 3 chunk */

#ifdef __cplusplus
}
#endif
#endif /* AMASS_CHUNK_H */
