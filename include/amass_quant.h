/*
 * amass_quant.h -- C-ABI of the operators of a paged cache held in 8 bits (gfx950).
 *
 * The same library (libamass_hip.so), status codes and calling rules as amass_hip.h and
 * amass_chunk.h: POD argument structs of device pointers, ELEMENT strides and geometry, launches on
 * `stream`, no device allocation, no host synchronisation, nothing throws, fixed-shape launches
 * that a caller may capture in a HIP graph.  None of them has a counterpart in the reference.
 *
 * The cache holds a code for every number, int8 (-127 .. 127) or e4m3 (OCP: 448 at most, 0x7F and
 * 0xFF are NaN), in (NB, page, n_kv, d) views of K and V, and an fp32 scale for every block, half
 * (K, V) and kv head, in (NB, n_kv) views: number = code * scale.  `page` is a power of two from 16
 * to 1024, d 64 or 128; addresses and strides of codes are multiples of 16.
 */
#ifndef AMASS_QUANT_H
#define AMASS_QUANT_H

#include "amass_chunk.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AMASS_QUANT_ABI_VERSION 1

/* code types */
#define AMASS_INT8 0
#define AMASS_E4M3 1

/* ---- quantising write ------------------------------------------------------------------- */
/* Writes the tokens' k and v to their slots (slots[t] = block * page + row; amass_extend).  A
 * run is a longest sequence of consecutive tokens with consecutive slots in one block, rows a .. b-1 of
 * it.  For the run, each half and kv head, with m = max |x| over its numbers x:
 *   step(m)   int8: the smallest number of 8 significant bits (bf16) that is >= m / 127;
 *             e4m3: the smallest power of two with 448 step >= m;
 *             at least 2^-64, at most 2^121 (int8) or 2^119 (e4m3)
 *   s         step(m) where a = 0 (the block starts anew), else max(step(m), scale so far)
 *   rows < a  where s exceeds the scale so far: code = round(code * scale so far / s), an e4m3 NaN as it is
 *   the run   code = round(x / s)
 *   scale     s
 * Quotients are rounded to fp32, then half to even to a code, at most the largest code.  Rows behind
 * the run keep their codes, under the scale that is then the block's.  A number that is not finite
 * makes s NaN and the run's codes zero; the scale stays NaN until the block starts anew.
 *   x of V is v; x of K is k or, with `table` ((max_pos, rot): cos | sin, as amass_rope_write), k
 * turned by its position in 64 bits and rounded to fp32 and to the element type.  With q, q_out
 * receives q turned, as amass_rope_write turns it, for every token whose position is in the table.
 * A token whose slot is outside [0, nb * page) or, with a table, whose position is outside
 * [0, max_pos) is not written and ends a run.  A block that two runs of a call enter holds an
 * unspecified mixture of both and of what it held (nothing outside it is touched).  q_out is q or
 * shares no memory with it.  rot is a multiple of 16; k, v, q, q_out and table are 16-byte aligned
 * with strides of multiples of 8 elements (table: 4). */
typedef struct amass_quant_write_args {
    const void* k;     int64_t k_st, k_hs;               /* (T,n_kv,d) */
    const void* v;     int64_t v_st, v_hs;               /* (T,n_kv,d) */
    const void* q;     int64_t q_st, q_hs;               /* (T,H,d) or NULL */
    void*       q_out; int64_t qo_st, qo_hs;             /* (T,H,d) or NULL */
    void*       k_codes; void* v_codes;                  /* (NB,page,n_kv,d) views of */
    int64_t     c_sb, c_st, c_sh;                        /* the same strides */
    float*      k_scale; float* v_scale;                 /* (NB,n_kv) views of */
    int64_t     s_sb, s_sh;                              /* the same strides */
    const float*   table; int64_t tab_st;                /* (max_pos, rot) or NULL */
    const int32_t* positions;                            /* (T,) or NULL */
    const int64_t* slots;                                /* (T,) */
    int32_t n_tokens, n_heads, n_kv, d, rot, page, nb, max_pos, interleaved, dtype, code;
} amass_quant_write_args;
int amass_quant_write(const amass_quant_write_args* a, void* stream);

/* ---- reading back ------------------------------------------------------------------------- */
/* Block dst[i] of a 16-bit cache becomes code * scale (rounded to the element type) of block
 * src[i], K and V, whole blocks.  Entries with src outside [0, nb) or dst outside [0, nb_out) are
 * passed over; a block that two entries name holds either's numbers, in pieces. */
typedef struct amass_quant_read_args {
    const void*  k_codes; const void* v_codes; int64_t c_sb, c_st, c_sh;
    const float* k_scale; const float* v_scale; int64_t s_sb, s_sh;
    void*        k_cache; void* v_cache; int64_t o_sb, o_st, o_sh;   /* (NB_out,page,n_kv,d) views */
    const int32_t* src;                                  /* (n,) */
    const int32_t* dst;                                  /* (n,) */
    int32_t n, n_kv, d, page, nb, nb_out, dtype, code;
} amass_quant_read_args;
int amass_quant_read(const amass_quant_read_args* a, void* stream);

/* ---- attention of a chunk over the cache ------------------------------------------------------ */
/* amass_chunk_attention with k_j = code * scale and v_j = code * scale: the same rows, visible
 * positions, results (zeros and lse = -inf for a row that sees nothing) and scratch rules.  Codes
 * enter the products as they are, exact in the element type; K's scale multiplies the score, V's the
 * weight before its one rounding to the element type; sums and statistics are fp32.
 *   Scales are positive; V's count as at least 2^-64, and those of one request and kv head should lie
 * within 2^80 of each other (a weight that much below the largest is lost; pages of zeros, whose scale
 * the write makes 2^-64, count in full beside V of up to 2^40).  A scale that is not finite makes NaN of
 * the rows that see its page; a code that is NaN makes NaN of the rows that see its key.  What is not
 * visible is not used, whatever it holds.  q is finite. */
typedef struct amass_quant_chunk_args {
    const void*    q; int64_t q_st, q_hs;                /* (T,H,d) */
    const void*    k_codes; const void* v_codes;         /* (NB,page,n_kv,d) views of */
    int64_t        c_sb, c_st, c_sh;                     /* the same strides */
    const float*   k_scale; const float* v_scale;        /* (NB,n_kv) views of */
    int64_t        s_sb, s_sh;                           /* the same strides */
    const int32_t* block_table; int64_t bt_st;
    const int32_t* seq_lens;
    const int32_t* query_start;
    void*          out; int64_t o_st, o_hs;              /* (T,H,d) */
    float*         lse; int64_t l_st, l_hs;              /* (T,H) or NULL */
    void*          scratch; int64_t scratch_bytes;
    float   scale;
    int32_t n_req, n_tokens, n_kv, G, d, page, nb, max_pages, causal, window, dtype, code;
} amass_quant_chunk_args;
int     amass_quant_chunk_attention(const amass_quant_chunk_args* a, void* stream);
int64_t amass_quant_scratch_bytes(const amass_quant_chunk_args* a);   /* negative: a status */

/* ---- introspection (host only) ---------------------------------------------------------------- */
int    amass_quant_abi_version(void);
size_t amass_quant_struct_size(int which);   /* 0 write, 1 read, 2 chunk */

#ifdef __cplusplus
}
#endif
#endif /* AMASS_QUANT_H */
