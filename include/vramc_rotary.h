/*
 * vramc_rotary.h -- C ABI of the rotation by positions in librans_hip.so: RMS
 * norms of queries and keys for each head and the rotation in one pass, into
 * tensors or straight into the pages of a key-value cache (vramc_kv.h).  No
 * reference counterpart.
 *
 * Conventions are those of vramc_rans.h: device pointers owned by the caller,
 * launches asynchronous on the caller's stream, return value 0, a hipError_t or
 * a negative RANS_E* code.
 */
#ifndef VRAMC_ROTARY_H
#define VRAMC_ROTARY_H

#include "vramc_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The first 2 * pairs columns of a head rotate: column i with column i + pairs, or,
 * interleaved, 2i with 2i + 1, by positions[t] * turns[i] full turns. */
typedef struct vramc_rotary {
    int32_t head_dim;     /* 64, 96, 128, 192 or 256 */
    int32_t pairs;        /* a multiple of 8, at most head_dim / 2 */
    int32_t interleaved;
    float amplitude;      /* of cosine and sine */
    const double* turns;  /* [pairs] */
} vramc_rotary;

/* The queries and keys of `tokens` tokens, q[t*q_token + h*q_head + d] of dtype
 * (RANS_X_*; k likewise; strides in values, not negative; heads may be 0), and what
 * they are multiplied by: y = x * w / sqrt(mean(x^2) + eps) over a head's columns
 * where there is a weight w ([head_dim] of weight_dtype: dtype or f32), x else. */
typedef struct vramc_rotary_rows {
    const void *q, *k;
    int64_t q_token, q_head, k_token, k_head;
    int32_t q_heads, k_heads;
    const void *q_weight, *k_weight;  /* or NULL */
    int32_t dtype, weight_dtype;
    float eps;
    const int32_t* positions;         /* [tokens] */
    int64_t tokens;
} vramc_rotary_rows;

/* q_out, k_out: [tokens][heads][head_dim] of dtype, 16-byte aligned, sharing no
 * memory with each other or what is read (RANS_EARG).  Everything is computed in f32
 * (the angle in 64 bits up to its whole turns, for f32 rows up to its sine) and rounded
 * once; the norm of a head whose squares leave f32 is no number of use. */
int vramc_rotary_apply(const vramc_rotary* r, const vramc_rotary_rows* x, void* q_out, void* k_out,
                       hipStream_t stream);

/* The same, with the keys rounded to dtype and written, as vramc_kv_append writes
 * them, into the slots of a cache of the same dtype, head_dim and k_heads heads,
 * with the values v; where it has them, the slot's mass becomes 0 and its position
 * the token's.  k of x stays as it is.  The cache's tensors share no memory with what
 * is read or q_out (RANS_EARG). */
int vramc_rotary_append(const vramc_rotary* r, const vramc_rotary_rows* x, const vramc_kv_cache* c,
                        const void* v, int64_t v_token, int64_t v_head, const int64_t* slots,
                        void* q_out, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* VRAMC_ROTARY_H */
