/*
 * infiniop_paged.h - the C ABI exported by libinfiniop_paged.so: operators of a
 * key/value cache that many sequences share page by page and that is held in 8
 * bits.  The reference library has none of them; they live in a library of
 * their own beside libinfiniop.so, whose entry points stay the reference's.
 * Handles and tensor descriptors are those of infiniop.h, and so is the calling
 * convention (create a descriptor, ask for the workspace size, call, destroy):
 * all checks of shapes, strides and types at creation, every call enqueues on
 * `stream` and returns without synchronising, nothing is allocated on the GPU,
 * descriptors are immutable, calls may be captured into a graph.
 *
 * The cache of one layer is four tensors:
 *   k_cache, v_cache  [pages, kv_heads, page, dim]           I8 or F8E4M3 codes
 *   k_scale, v_scale  [pages, kv_heads, page / block]        F32
 * and stands for code * scale, one scale (not below 0) for each `block` tokens of a head.
 * page and block are multiples of 16 (block divides page), dim is a multiple of
 * 16 up to 256.  The innermost strides are 1, the others free: codes in
 * multiples of 16, so the pages of all heads may lie in any order, e.g. as
 * slices of one pool.  Codes at addresses that are multiples of 16.
 *
 * The sequences are the rows of a batch, the same for every layer (all I32):
 *   table    [rows, cols]  page t / page of the row holds its token t; what is
 *                          outside 0..pages-1 is no page: nothing is stored
 *                          there, and attention sees no tokens there
 *   lengths  [rows]        tokens of the row in the cache, the call's own with them
 *   offsets  [rows + 1]    the call's own tokens of row r are tokens
 *                          offsets[r] .. offsets[r + 1] - 1 of q, k, v and out, and
 *                          the last ones of the row; rows without one are left out
 *   refcount [pages]       how often the page stands in the table; 0: it is free
 * These are read on the GPU by each call, so a captured graph serves whatever
 * they hold when it is replayed.  Lengths beyond cols * page are taken as that.
 *
 * Every call of one step: PageTableUpdate (once), then for each layer KVCacheCopy
 * (what was copied on write), KVCacheAppend, PagedAttention.
 */
#ifndef INFINIOP_AMD_INFINIOP_PAGED_H
#define INFINIOP_AMD_INFINIOP_PAGED_H

#include "infiniop.h"

/* 8-bit floating point with 4 bits of exponent and 3 of mantissa, largest value 448, no infinities */
static const DataLayout F8E4M3 = INFINIOP_DT(1, 1, 1, 3, 4);

/* ======================================================================== *
 * KVCacheAppend:  stores the new tokens of every row.  k, v: [tokens, kv_heads,
 * dim], F16 or BF16, unit innermost strides, the others free (so slices of a
 * fused qkv buffer will do).  Token i of the n new ones of row r goes to place
 * lengths[r] - n + i of the row.  For each block of tokens and head, with top
 * the largest finite magnitude of the new values in it (0 if below 2^-96):
 *     scale = top / 127                     I8
 *     scale = the smallest power of two with top <= 448 scale       F8E4M3
 * and, where the block holds older tokens of the row, at least the scale that
 * it has; their codes are brought to a scale that grew,
 *     code = round(code * (old scale / scale)).
 * New values become round(x * (1 / scale)), in fp32, to nearest even, what is
 * beyond the codes (infinities too) the largest of its sign, NaN 0 (and 0 where the scale is 0).  The places
 * behind a row's last token keep what they hold.  Two rows that call may not store
 * into one page (a page that rows share is copied on write by PageTableUpdate).
 * ======================================================================== */
typedef struct KVCacheAppendDescriptor {
    Device device;
} KVCacheAppendDescriptor;
typedef KVCacheAppendDescriptor *infiniopKVCacheAppendDescriptor_t;

INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopCreateKVCacheAppendDescriptor(
    infiniopHandle_t handle, infiniopKVCacheAppendDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
    infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
    infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets, infiniopTensorDescriptor_t lengths);
/* always 0 bytes */
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopGetKVCacheAppendWorkspaceSize(infiniopKVCacheAppendDescriptor_t desc, uint64_t *size);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopKVCacheAppend(
    infiniopKVCacheAppendDescriptor_t desc, void *workspace, uint64_t workspace_size,
    void *k_cache, void *v_cache, void *k_scale, void *v_scale, void const *k, void const *v,
    void const *table, void const *offsets, void const *lengths, void *stream);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopDestroyKVCacheAppendDescriptor(infiniopKVCacheAppendDescriptor_t desc);

/* ======================================================================== *
 * PagedAttention:  out[t][h] = sum_j softmax_j(scale * q[t][h] . K[j]) V[j]
 * over the places j <= lengths[r] - n + i of the row r that token t is the i-th
 * of n new ones of, K and V those of head h / (heads / kv_heads).  q, out:
 * [tokens, heads, dim], F16 or BF16, unit innermost strides, the others free;
 * heads a multiple of kv_heads.  A token that sees nothing gets zeros; what of
 * `out` belongs to no row is left as it was.  No row may have more than
 * max_tokens new tokens (what it has beyond is not computed): 1 for plain
 * decoding, which lets the call pass by the kernels for prompts.  scale is
 * usually 1 / sqrt(dim).  q and what the cache holds for a row's places have to
 * be finite, and so has scale * q K in fp32; behind lengths[r] it may hold anything.
 * Scores, sums and results are fp32 (rounded once, to nearest even); q is rounded to
 * fp16 relative to the largest element of its row, by at most 2^-25 of that, and the
 * weights, each times its V scale, to fp16 (11 bits, none below 2^-35 of the largest of
 * the same query row).  In chunks of many tokens a V scale below 2^-80 of the
 * largest that neighbouring tokens see may count as 2^-80 of that.
 * ======================================================================== */
typedef struct PagedAttentionDescriptor {
    Device device;
} PagedAttentionDescriptor;
typedef PagedAttentionDescriptor *infiniopPagedAttentionDescriptor_t;

INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopCreatePagedAttentionDescriptor(
    infiniopHandle_t handle, infiniopPagedAttentionDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t out, infiniopTensorDescriptor_t q,
    infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
    infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets, infiniopTensorDescriptor_t lengths,
    uint64_t max_tokens, float scale);
/* room for what the workgroups that share a long row hand on, as far as the table is long enough for that: for decoding
 * up to 16 to 33 MiB, for prompts up to 65 (one row) or 200 MiB, more only with more than 256 K/V heads, and 16 bytes where
 * no row is long enough; a call with less is refused with STATUS_MEMORY_NOT_ALLOCATED.  It may be shared by all calls that run one after the other. */
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopGetPagedAttentionWorkspaceSize(infiniopPagedAttentionDescriptor_t desc, uint64_t *size);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopPagedAttention(
    infiniopPagedAttentionDescriptor_t desc, void *workspace, uint64_t workspace_size,
    void *out, void const *q, void const *k_cache, void const *v_cache, void const *k_scale, void const *v_scale,
    void const *table, void const *offsets, void const *lengths, void *stream);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopDestroyPagedAttentionDescriptor(infiniopPagedAttentionDescriptor_t desc);

/* ======================================================================== *
 * KVCacheCopy:  for every pair (source, destination) of pairs [count, 2] I32,
 * page `destination` of the cache becomes a copy of page `source`, codes and
 * scales.  A pair in which either is no page of the cache, e.g. -1, is passed
 * over.  Destinations are distinct, and none is a source of the same call.
 * ======================================================================== */
typedef struct KVCacheCopyDescriptor {
    Device device;
} KVCacheCopyDescriptor;
typedef KVCacheCopyDescriptor *infiniopKVCacheCopyDescriptor_t;

INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopCreateKVCacheCopyDescriptor(
    infiniopHandle_t handle, infiniopKVCacheCopyDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
    infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t pairs);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopKVCacheCopy(
    infiniopKVCacheCopyDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale,
    void const *pairs, void *stream);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopDestroyKVCacheCopyDescriptor(infiniopKVCacheCopyDescriptor_t desc);

/* ======================================================================== *
 * PageTableUpdate:  row r becomes what row source[r] was before the call (its
 * pages are then shared), or empty where source[r] is no row, e.g. -1; then it
 * grows by grow[r] tokens (less than 0: by none).  So source[r] = r decodes on,
 * -1 frees the row's pages, another row forks it, a permutation reorders beams.
 * Where a row grows inside its last page and that page is shared after the first
 * part, the row gets a fresh page in its place and pairs[r] = (shared, fresh),
 * to be copied in every layer before tokens are appended; otherwise pairs[r] =
 * (-1, -1).  Fresh pages are the free ones of the lowest numbers, in the order of
 * the rows, for each its copy first.  Where the pages do not suffice or a row
 * would need more than cols, no row grows: result = {pages lacking, rows too
 * wide}, both 0 if all grew.  Entries of new_table behind a row's pages are -1
 * where source[r] != r, and those of table elsewhere.
 * table, new_table [rows, cols], lengths, new_lengths, source, grow [rows],
 * refcount, new_refcount [pages], pairs [rows, 2], result [2], all I32; a new_
 * tensor may be its old one (same address, same strides), but not overlap it
 * otherwise.  The entries that a row's length covers have to be pages of it
 * (others are passed over).  rows <= 8192.
 * ======================================================================== */
typedef struct PageTableUpdateDescriptor {
    Device device;
} PageTableUpdateDescriptor;
typedef PageTableUpdateDescriptor *infiniopPageTableUpdateDescriptor_t;

INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopCreatePageTableUpdateDescriptor(
    infiniopHandle_t handle, infiniopPageTableUpdateDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t new_table, infiniopTensorDescriptor_t new_lengths, infiniopTensorDescriptor_t new_refcount,
    infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount,
    infiniopTensorDescriptor_t source, infiniopTensorDescriptor_t grow, uint64_t page_size);
/* a copy of the table and a few words for each row and page; a call with less is refused with
 * STATUS_MEMORY_NOT_ALLOCATED */
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopGetPageTableUpdateWorkspaceSize(infiniopPageTableUpdateDescriptor_t desc, uint64_t *size);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopPageTableUpdate(
    infiniopPageTableUpdateDescriptor_t desc, void *workspace, uint64_t workspace_size,
    void *new_table, void *new_lengths, void *new_refcount, void *pairs, void *result,
    void const *table, void const *lengths, void const *refcount, void const *source, void const *grow, void *stream);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopDestroyPageTableUpdateDescriptor(infiniopPageTableUpdateDescriptor_t desc);

/* ======================================================================== *
 * PageTableCompact:  renumbers pages so that the `used` ones in use are pages
 * 0 .. used-1: the i-th (from the lowest) of the used pages above takes the i-th
 * of the free ones below, pairs[i] = (above, below), -1 behind; the table and the
 * counts follow, and KVCacheCopy of pairs moves each layer's data.  result =
 * {used, moved}.  table, new_table [rows, cols], lengths [rows], refcount,
 * new_refcount [pages], pairs [count >= pages / 2, 2], result [2], all I32; a new_
 * tensor may be its old one (same address, same strides).
 * ======================================================================== */
typedef struct PageTableCompactDescriptor {
    Device device;
} PageTableCompactDescriptor;
typedef PageTableCompactDescriptor *infiniopPageTableCompactDescriptor_t;

INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopCreatePageTableCompactDescriptor(
    infiniopHandle_t handle, infiniopPageTableCompactDescriptor_t *desc_ptr,
    infiniopTensorDescriptor_t new_table, infiniopTensorDescriptor_t new_refcount,
    infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount, uint64_t page_size);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopGetPageTableCompactWorkspaceSize(infiniopPageTableCompactDescriptor_t desc, uint64_t *size);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopPageTableCompact(
    infiniopPageTableCompactDescriptor_t desc, void *workspace, uint64_t workspace_size,
    void *new_table, void *new_refcount, void *pairs, void *result,
    void const *table, void const *lengths, void const *refcount, void *stream);
INFINIOP_C INFINIOP_EXPORT infiniopStatus_t infiniopDestroyPageTableCompactDescriptor(infiniopPageTableCompactDescriptor_t desc);

#endif /* INFINIOP_AMD_INFINIOP_PAGED_H */
