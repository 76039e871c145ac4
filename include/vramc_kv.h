/*
 * vramc_kv.h -- C ABI of the key-value cache in librans_hip.so: pages of keys
 * and values in the model's type or in microscaled 4-bit floating point, the
 * attention of one new token over them, eviction by accumulated weight, and the
 * choice of the pages that a query attends to.  No reference counterpart:
 * snuri00/vram-compression stops at the weights; this is the other part of a
 * served model's memory.
 *
 * Conventions are those of vramc_rans.h: every pointer in the descriptor is a
 * device pointer owned by the caller, launches are asynchronous on the
 * caller's stream, nothing synchronises or allocates, and the return value is
 * 0, a hipError_t, or a negative RANS_E* code for arguments refused before
 * anything is launched (RANS_EUNSUPPORTED: a type or size without a kernel,
 * RANS_EWORKSPACE: workspace missing or too small, RANS_EARG: a null pointer,
 * a size out of range, a pointer less aligned than its kernel reads, or an
 * output over what the call reads where that is said to be refused).
 *
 * Layout.  Keys and values are [pages][kv_heads][page_size][head_dim],
 * contiguous.  With mx = 0 they are values of dtype.  With mx = 1 they are
 * 4-bit codes, two to a byte (the even column in the low half), with one scale
 * byte for every 32 columns in k_scale / v_scale, [pages][kv_heads][page_size]
 * [head_dim / 32]: the OCP Microscaling format MXFP4.  A code's bits are sign,
 * two of exponent, one of mantissa: the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6;
 * a scale byte s stands for 2^(s-127), 255 for NaN.  A slot is a place of the
 * cache: page * page_size + place within the page.
 */
#ifndef VRAMC_KV_H
#define VRAMC_KV_H

#include "vramc_rans.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct vramc_kv_cache {
    int32_t pages, kv_heads;
    int32_t page_size;    /* tokens of a page: 16, 32, 64, 128 or 256 */
    int32_t head_dim;     /* 64, 96, 128, 192 or 256 */
    int32_t dtype;        /* of keys, values, queries and outputs, RANS_X_* */
    int32_t mx;           /* 1: 4-bit storage (dtype bf16 or f16) */
    void *k, *v;          /* 16-byte aligned */
    uint8_t *k_scale, *v_scale; /* mx only */
    float* mass;          /* [pages][kv_heads][page_size] accumulated weight, or NULL */
    int32_t* position;    /* [pages][kv_heads][page_size] token positions, or NULL
                             (present where mass is); both 16-byte aligned */
} vramc_kv_cache;

/* Writes `tokens` keys and values into their slots: k[t*k_token + h*k_head + d]
 * (strides in values) for every kv head h and column d goes to slot slots[t],
 * v likewise.  A slot outside the cache is skipped, which is how padding is
 * marked (-1); no two tokens may have the same slot.  In 4-bit storage a block
 * of 32 columns gets the exponent floor(log2(largest magnitude)) - 2 (at least
 * -127, at most 125), every value is rounded to the nearest code, ties to the
 * even one, beyond 6 to 6; a block with a value that is not finite becomes
 * NaN.  Where the cache has mass and position, the slot's mass becomes 0 and
 * its position positions[t]. */
int vramc_kv_append(const vramc_kv_cache* c, const void* k, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_token, int64_t v_head, const int64_t* slots,
                    const int32_t* positions, int64_t tokens, hipStream_t stream);

/* The keys and values of `tokens` slots, [tokens][kv_heads][head_dim] of dtype
 * each; zeros for a slot outside the cache. */
int vramc_kv_read(const vramc_kv_cache* c, const int64_t* slots, int64_t tokens, void* k_out,
                  void* v_out, hipStream_t stream);

/* Attention of one query token of each sequence over its cached tokens:
 *   out[b,h] = sum_j p_j v[j], p = softmax_j(scale * q[b,h] . k[j])
 * over tokens j < lengths[b], token j at place j % page_size of page
 * table[b*table_row + j/page_size], kv head h / (q_heads/kv_heads).  Sums and
 * softmax are in f32, out ([batch][q_heads][head_dim]) is rounded once.  A value
 * that is not finite, or so large that 256 times its column's sum of magnitudes
 * leaves f32, makes its column of its sequences' outputs NaN or infinite; a
 * token of weight 0 counts there too.  Tokens
 * whose table entry is no page of the cache are left out; a sequence without
 * tokens gets zeros.  lengths beyond table_width * page_size are cut to it.
 * With track, mass[token] of each kv head increases by the sum of p over the
 * query heads of that kv head.  q[b*q_seq + h*q_head + d], strides in values.
 * workspace: vramc_kv_attend_workspace bytes (negative: a RANS_E* code), no
 * content expected, 16-byte aligned. */
int64_t vramc_kv_attend_workspace(const vramc_kv_cache* c, int q_heads, int table_width, int batch,
                                  int track);
int vramc_kv_attend(const vramc_kv_cache* c, const void* q, int64_t q_seq, int64_t q_head,
                    int q_heads, const int32_t* table, int64_t table_row, int table_width,
                    const int32_t* lengths, int batch, float scale, int track, void* out,
                    void* workspace, int64_t workspace_bytes, hipStream_t stream);

/* Cuts every sequence longer than `budget` to that many tokens, each kv head
 * by itself: kept first are the tokens with position >= seen[b] - recent, then
 * those of the largest mass (NaN counts as -infinity), ties to the lower
 * index.  Tokens whose table entry is no page of the cache are never kept, and
 * places whose entry is none are never filled: where some of the first
 * min(lengths[b], budget) places are such, as many fewer tokens are kept.  With
 * into = NULL the kept tokens stay where they are and those at index >= budget,
 * in order, move into the places that became free below it, in order: pages
 * that other sequences share must not be passed.  Otherwise the kept tokens of
 * every sequence, also of one within the budget, are copied, in order, to the
 * places of the pages into[b*into_row + i/page_size], which must be none of the
 * sequences' own.  Keys, values, mass and position move together.
 * new_lengths[b] = min(lengths[b], budget), or with into, where there are fewer
 * tokens than places, the place behind the last that is filled; it must share no
 * memory with lengths, seen, table or into (RANS_EARG).  workspace as above. */
int64_t vramc_kv_evict_workspace(const vramc_kv_cache* c, int table_width, int batch, int budget,
                                 int into);
int vramc_kv_evict(const vramc_kv_cache* c, const int32_t* table, int64_t table_row,
                   int table_width, const int32_t* lengths, const int32_t* seen, int batch,
                   int budget, int recent, const int32_t* into, int64_t into_row, int into_width,
                   int32_t* new_lengths, void* workspace, int64_t workspace_bytes,
                   hipStream_t stream);

/* The smallest and largest key of each column of n pages (a number that is no page
 * of the cache is skipped): bounds[page][kv_head][0 and 1][head_dim] of dtype,
 * 16-byte aligned, over all places of the page; NaN in both where a column has a
 * key that is not finite.  They share no memory with the cache's tensors or the list
 * (RANS_EARG). */
int vramc_kv_bound(const vramc_kv_cache* c, const int32_t* pages, int64_t n, void* bounds,
                   hipStream_t stream);

/* The pages of each sequence that its query attends to, for each kv head by itself:
 * all of them where there are at most `count`, or else the first `first`, the last
 * `last` and those of the largest score,
 *   score = max over the kv head's query heads of sum_d max(q_d lo_d, q_d hi_d),
 * which no q . k of the page exceeds, lo and hi its bounds; ties to the lower index, a
 * score that is not a number before all others, an entry that is no page behind all
 * (any pages where a query is not finite).  Sums are in 64 bits and of the larger
 * products alone, in one order for all pages of a call: pages with the same products
 * tie, others whose scores differ by less than that rounding may change places.
 * 0 <= first, 1 <= last, first + last <= count.  lengths are cut to 0 and
 * table_width * page_size.
 * chosen[b*kv_heads + h][count]: the pages in order of the sequence's, page * kv_heads
 * + h (a page of the same tensors taken as a cache of pages * kv_heads pages of one
 * head), -1 for an entry that is none and behind the last; held[b*kv_heads + h]: the
 * tokens in them, so that vramc_kv_attend takes both as table and lengths.
 * workspace: vramc_kv_select_workspace bytes, no content expected, 16-byte aligned,
 * private to the call until its kernels have run.  chosen, held and the workspace share
 * no memory with one another or with what is read (RANS_EARG). */
int64_t vramc_kv_select_workspace(const vramc_kv_cache* c, int q_heads, int table_width, int batch,
                                  int count);
int vramc_kv_select(const vramc_kv_cache* c, const void* bounds, const void* q, int64_t q_seq,
                    int64_t q_head, int q_heads, const int32_t* table, int64_t table_row,
                    int table_width, const int32_t* lengths, int batch, int count, int first,
                    int last, int32_t* chosen, int32_t* held, void* workspace,
                    int64_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* VRAMC_KV_H */
