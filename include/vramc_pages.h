/*
 * vramc_pages.h -- C ABI of the page pool in librans_hip.so: which pages of a
 * key-value cache (vramc_kv.h) are free, kept on the GPU, so that a step's block
 * table and slots are made there from the sequences' lengths.  No reference
 * counterpart.
 *
 * Conventions are those of vramc_rans.h: device pointers owned by the caller,
 * launches asynchronous on the caller's stream, return value 0, a hipError_t or
 * a negative RANS_E* code.  A pool is a stack: free[0 .. count[0]) are its pages,
 * taken from the top.  Calls that change a pool must be ordered (one stream, or
 * events between them).
 */
#ifndef VRAMC_PAGES_H
#define VRAMC_PAGES_H

#include "vramc_rans.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct vramc_pages {
    int32_t pages;      /* of the cache, and entries of `free` */
    int32_t page_size;  /* tokens of a page: 16, 32, 64, 128 or 256 */
    int32_t* free;
    int32_t* count;     /* one */
    int32_t* ticket;    /* one, 0 before the first call; the calls keep it so */
} vramc_pages;

/* Room for `fresh[b]` new tokens behind the lengths[b] that sequence b holds (rows
 * of `table`, [batch][table_width], table_row apart; at most 4096 sequences).  The
 * new tokens of all sequences lie behind each other in `tokens` rows:
 *   starts[b], starts[batch]   sums of fresh, cut to `tokens`;
 *   slots[t]                   where row t goes, page * page_size + place; -1 where
 *                              it is no token, its sequence got no room, or the
 *                              table names no page of the cache for it;
 *   positions[t]               (seen ? seen : lengths)[b] + t - starts[b], 0 where it
 *                              is no token;
 *   filled[t]                  the page whose last place it takes, -1 for none;
 *   new_lengths[b]             with the new tokens, or as before without room.
 * A sequence gets room whose tokens fit its row of the table, lie among the rows,
 * and whose pages, with those that sequences before it want, are all in the pool.
 * New pages come from the top of the stack in order and are written behind the
 * ceil(length / page_size) entries that the length takes up.  Negative numbers
 * count as 0, lengths beyond the row as its end.  Outputs, the table and the pool's
 * tensors share no memory with one another or with what is read, rows of the table
 * none with each other (RANS_EARG). */
int vramc_pages_extend(const vramc_pages* p, int32_t* table, int64_t table_row, int table_width,
                       const int32_t* lengths, const int32_t* fresh, const int32_t* seen, int batch,
                       int64_t tokens, int64_t* slots, int32_t* positions, int32_t* filled,
                       int32_t* starts, int32_t* new_lengths, hipStream_t stream);

/* Puts the pages of entries at ceil(lengths[b] / page_size) and behind on the stack,
 * in order of the sequences and entries, and -1 in their place.  Entries that are
 * no page become -1 and go nowhere; what would not fit the stack (a page given back
 * twice) is dropped.  Table, lengths, workspace and the pool's tensors share no memory
 * (RANS_EARG).  workspace: vramc_pages_release_workspace bytes, no content expected,
 * 16-byte aligned, private to the call until its kernels have run. */
int64_t vramc_pages_release_workspace(const vramc_pages* p, int table_width, int batch);
int vramc_pages_release(const vramc_pages* p, int32_t* table, int64_t table_row, int table_width,
                        const int32_t* lengths, int batch, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* VRAMC_PAGES_H */
