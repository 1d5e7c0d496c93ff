/*
 * C ABI of the bookkeeping of a paged cache's pages on the device, in the library of fmha_mxfp8_abi.h: page tables, lengths, positions and slot maps from the numbers of new tokens, for
 * the caches of fmha_kv4_abi.h and fmha_kv8_abi.h alike.
 *
 * Free pages are a stack in device memory: int32 free[4 + pages], free[0] how many there are, free[1] to free[3] 0 between calls, free[4 + i] the page numbers, the next to be handed out
 * at i = free[0] - 1. Whoever uses a stack, its table or its lengths uses one stream, or waits.
 *
 * Enqueued on `stream`; allocates nothing and waits for nothing. Returns 0, > 0 FMHA_MXFP8_E_ARG with a message in `err`, < 0 minus a cudaError_t.
 */
#ifndef FMHA_PAGES_ABI_H
#define FMHA_PAGES_ABI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct fmha_pages {
    int32_t* free;
    int32_t* table;      /* [B][table_width] */
    int32_t* lengths;    /* [B] */
    uint32_t pages;      /* that the stack has room for */
    uint32_t B, page, table_width;
    uint32_t pool_pages; /* of the pool that the table's entries are pages of: others below 0 or from there on name none. 0: not known, all from 0 on do */
} fmha_pages;

/*
 * take: sequence b asks for counts[b] new tokens (below 0: none). It needs the pages that length + counts[b] tokens take and it does not have; sequences are served in order. One is
 *   granted all of its tokens, or none where its table has no room for them, or where it needs pages and the pages needed by it and the sequences in front of it (those without room
 *   aside) are more than are free. granted[b] = counts[b] or 0; the new pages go from the stack to the table, in order; lengths[b] grows by granted[b].
 *   positions: NULL or int32 [B][S] (int64 with positions_64): of row i < granted[b] the token it becomes, length (before) + i; -1 in other rows.
 *   slots: NULL or int64 [B][S]: page * (tokens of a page) + place within the page of that token; -1 in other rows and where the table names no page.
 *     (Rows are all that the maps have: a sequence may be granted more than S tokens.)
 *   starts: NULL or int32 [B + 1]: sums of granted in front of each sequence, and of all. (pages + B) * page is below 2^31 then.
 *   granted, positions, slots and starts share no memory with counts, the stack, the table, the lengths or one another.
 * cut: lengths[b] becomes min(length, max(keep[b], 0)); pages without tokens go back to the stack, their table entries become -1. The last sequence's last page goes onto it first: a cut
 *   to the lengths before a take leaves stack, table and lengths as they were before it. Entries that name no page give none back. Pages that the stack has no room for are dropped. keep shares
 *   no memory with the others.
 *   Nobody counts a page's users: every page behind keep goes back, and is handed out again. Pages that other sequences hold too (a prefix in common) have to lie in front of keep; they, and the
 *   last sequence that holds them, are the caller's to look after.
 */
int fmha_pages_take(const fmha_pages* p, const int32_t* counts, int32_t* granted, void* positions, int positions_64, int64_t* slots, int32_t* starts, uint32_t S, void* stream, char* err, size_t cap);
int fmha_pages_cut(const fmha_pages* p, const int32_t* keep, void* stream, char* err, size_t cap);

#ifdef __cplusplus
}
#endif
#endif /* FMHA_PAGES_ABI_H */
