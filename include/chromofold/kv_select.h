/* kv_select.h — ADDITIVE: reading and keeping only a part of a long batched cache (kv_codec_ext.h). No counterpart in
 * the reference, whose attention reads every page of a sequence (include/chromofold/kv_cuda.h) and whose caches drop
 * pages only from the ends (integrations/llama.cpp/chromofold_kv_adapter.h:66-75, seq_rm).
 *
 *   cf_kv_key_bounds_async                 while sealing: an 8-bit bound on the keys of every group
 *   cf_kv_select_groups_async              each step: the groups whose keys can give a query its largest scores
 *   cf_kv_paged_attention_selected_async   each step: attention over those groups (or all), and each group's share of the
 *                                          attention weight
 *   cf_kv_evict_groups_async               now and then: the groups of least accumulated weight leave the page tables
 *
 * Tables are those of cf_kv_batched_desc: group_offsets [seq_count, kv_head_count, max_groups], group g of a (sequence,
 * KV head) holding tokens 64 g .. 64 g + 63. Arrays "per group" below have the same shape. A "unit" is what is selected or
 * evicted as one: unit_groups = 1 group, or unit_groups = 2, the groups 2u and 2u + 1, which share a rANS chain in a
 * RANS_HYBRID pool sealed with chain pairs (seal with continues = NULL to use single groups there).
 *
 * Limits (beyond them CF_ERR_UNSUPPORTED): max_groups and a selection's max_units below 2^25, seq_count and kv_head_count up
 * to 65535. Tokens past 64 * max_groups do not count.
 *
 * Every array is device memory on the current device; calls are asynchronous on `stream`, allocate nothing and never
 * synchronise, and may be captured into a graph. Calls that may overlap need a workspace each. Results repeat bit for bit.
 */
#ifndef CHROMOFOLD_KV_SELECT_H
#define CHROMOFOLD_KV_SELECT_H

#include <stdint.h>

#include "chromofold/chromofold.h"
#include "chromofold/kv_codec_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CF_KV_SELECT_ABI_VERSION 1u
#define CF_KV_NO_UNIT 0xFFFFFFFFu      /* fills a selection behind its last unit */
#define CF_KV_SELECT_MAX_GQA 16u       /* query heads per KV head (attention over RANS_HYBRID pools: 4) */

/* ---- key bounds ------------------------------------------------------------------------------------------------
 * Record of a group, head_dim D: scale s = max |k| / 127 over its tokens and channels (rounded up where s is subnormal: to
 * nearest, 127 s could be far below the maximum); 2 D codes,
 *   codes[d]     = min(127, ceil( max_t k[t][d] / s))      an upper bound on channel d in steps of s
 *   codes[D + d] = min(127, ceil(-min_t k[t][d] / s))      a lower bound, negated
 * (IEEE fp32 quotients; codes are in [-127, 127]). A group of zeros has scale 0 and codes 0; one that holds an infinity or
 * a NaN has scale +inf and codes 127, so that it is selected and what is wrong with it shows in the output.
 *
 * The group arguments are those of cf_kv_encode_groups_async, so that sealing calls both: keys page-major
 * [*][16][head_dim] fp32, 16-byte aligned; group i = page_counts[i] (1..4) pages from page first_page[i], token_counts per
 * page (1..16; NULL: all 16). Group i's record goes to index slots[i] (NULL: i) of codes [slot_count][2 D] (16-byte
 * aligned) and scales [slot_count]; a slot past slot_count is skipped. Slots are meant to differ: of two groups with one
 * slot either may leave its record's parts. A group with a bad page or token count is not read and gets the record of
 * a group that holds a NaN. head_dim 64 or 128. */
cf_status cf_kv_key_bounds_async(const float *keys, uint64_t ngroups, const uint64_t *first_page,
                                 const uint32_t *page_counts, const uint32_t *token_counts, uint32_t head_dim,
                                 const uint64_t *slots, int8_t *codes, float *scales, uint64_t slot_count,
                                 void *stream);

/* ---- selection -------------------------------------------------------------------------------------------------
 * Score of group g for KV head j of sequence s, over the query heads h of j, with step_h = max |q_h| / 127 and
 * a_h = rint(q_h / step_h) (0 where step_h is 0):
 *   score = max_h(step_h * sum_d (a_hd >= 0 ? a_hd * codes[d] : -a_hd * codes[D + d])) * scale
 * The sum is a whole number below 2^24; each of the two products is rounded to fp32 once, so that scores, and with them the
 * selection, are the same wherever they are computed. It bounds q_h . k over the group's tokens (for the rounded queries;
 * a positive softmax scale is assumed). Of a query head, elements that are NaN count as 0; heads with an infinity are passed
 * over (with no other head the score is -inf * scale). A unit has the larger score of its groups; a NaN counts as the largest.
 *
 * Of the n units that hold a visible token (64 * unit_groups tokens each; visible = min(seq_tokens, query_pos + 1)), the
 * first keep_first and the last keep_last are selected whatever their scores, then the best, min(n, max_units) in all;
 * among equal scores the lower index. units [seq_count, kv_head_count, max_units] receives them in ascending order, the
 * rest of a row CF_KV_NO_UNIT. keep_first + keep_last <= max_units. Rows of sequences without tokens are all
 * CF_KV_NO_UNIT. */
typedef struct cf_kv_select_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    uint32_t seq_count;
    uint32_t kv_head_count;
    uint32_t query_head_count;
    uint32_t head_dim;             /* 64 or 128 */
    uint32_t max_groups;
    uint32_t unit_groups;
    uint32_t max_units;
    uint32_t keep_first;
    uint32_t keep_last;
    uint32_t reserved;
    const int8_t *codes;           /* per group, 2 head_dim each; 16-byte aligned */
    const float *scales;           /* per group */
    const uint32_t *seq_tokens;
    const uint32_t *query_pos;
    const float *queries;          /* [seq_count, query_head_count, head_dim] */
    uint32_t *units;
    void *workspace;               /* cf_kv_select_workspace_bytes(), 16-byte aligned */
    uint64_t workspace_bytes;
} cf_kv_select_desc;

cf_status cf_kv_validate_select_desc(const cf_kv_select_desc *desc);  /* host only; not the workspace */
uint64_t cf_kv_select_workspace_bytes(const cf_kv_select_desc *desc); /* 0 for a bad descriptor */
cf_status cf_kv_select_groups_async(const cf_kv_select_desc *desc, void *stream);

/* ---- attention over selected groups ------------------------------------------------------------------------------
 * cf_kv_paged_attention_batched_async over the listed units of each (sequence, KV head). units [seq_count, kv_head_count,
 * max_units] ascends strictly up to the first CF_KV_NO_UNIT, which only CF_KV_NO_UNIT follows, as
 * cf_kv_select_groups_async writes it; a row that does not becomes NaN (its output, and the weights of the groups it
 * lists). Of a row the first min(max_units, n) entries are read, n being its units with a visible token: more cannot be
 * listed. Units without a visible token are passed over; units = NULL takes every group (max_units and unit_groups are then
 * ignored). Rows with nothing to attend are 0; rows whose visible scores are all -inf (as a K scale of +inf can make them) are
 * NaN, as their softmax is. As in the batched call, with splits = 0 a row's fp32 rounding may depend on the other rows' lengths. As there, V is added up in units of the
 * largest V scale of a group's visible pages, but pages without any visible V other than 0 do not count, whatever their
 * scale: pages with a scale down to 2^-10 of that keep 22 bits, smaller ones fewer, below 2^-31 none (RANS_HYBRID: 2^-18
 * and 2^-39).
 *
 * weights_out (may be NULL), per group, is fp32: weights_out = decay * weights_in + the softmax weight of the group's
 * tokens summed over the KV head's query heads (0 for a group not attended). All max_groups entries of a row are written.
 * weights_in may be NULL (zeros) or weights_out itself; otherwise the two must not overlap.
 *
 * Pools: INT8 with at most CF_KV_SELECT_MAX_GQA query heads per KV head, RANS_HYBRID (raw groups in it too) with at most 4;
 * more is CF_ERR_UNSUPPORTED. In an INT8 pool a listed group whose header is not an INT8 group of this head_dim makes its
 * row NaN. desc->splits as in the batched call (0 = choose; 1 is the faster choice for many whole rows that the caller knows
 * to be of one length, INT8, max_groups times query heads per KV head up to 2048: the lengths are device memory, and the
 * cut that is chosen suits unlike ones). desc->workspace must hold
 * cf_kv_selected_workspace_bytes() bytes, 16-byte aligned. */
typedef struct cf_kv_selection {
    uint32_t struct_size;
    uint32_t abi_version;
    uint32_t unit_groups;
    uint32_t max_units;
    const uint32_t *units;
    const float *weights_in;
    float *weights_out;
    float decay;                   /* finite */
    uint32_t reserved;
} cf_kv_selection;

cf_status cf_kv_validate_selection(const cf_kv_batched_desc *desc, const cf_kv_selection *sel);
uint64_t cf_kv_selected_workspace_bytes(const cf_kv_batched_desc *desc, const cf_kv_selection *sel);
cf_status cf_kv_paged_attention_selected_async(const cf_kv_batched_desc *desc, const cf_kv_selection *sel,
                                               void *stream);

/* ---- eviction ----------------------------------------------------------------------------------------------------
 * A sequence of n units (its last one may hold fewer groups and tokens) keeps, per KV head, budget_units of them if it has
 * more: the first keep_first, the last keep_last, then those of the largest weight; among equal weights the lower index; a
 * NaN counts as the largest. A unit's weight is the fp32 sum of its groups'. Kept groups move down in order; since every
 * head keeps as many, the sequence is then one of seq_tokens - 64 * unit_groups * (units dropped) tokens for every call that
 * takes these tables (the keys keep the rotary positions they were sealed with; set query_pos accordingly).
 * keep_last >= 1 and keep_first + keep_last <= budget_units.
 *
 * Outputs, per group: group_offsets_out, and where given codes_out / scales_out (moved records of cf_kv_key_bounds_async)
 * are written for the groups that stay, entries behind them left as they were; weights_out (may be NULL) is 0 there.
 * dropped (may be NULL) receives the offsets of the groups that went, in order, the rest CF_KV_NO_UNIT: blobs that may be
 * reused once no other table refers to them. seq_tokens_out [seq_count]. Each output may be the input of the same kind
 * (eviction in place) and must not overlap any other array. */
typedef struct cf_kv_evict_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    uint32_t seq_count;
    uint32_t kv_head_count;
    uint32_t head_dim;             /* of the records; 64 or 128 */
    uint32_t max_groups;
    uint32_t unit_groups;
    uint32_t budget_units;
    uint32_t keep_first;
    uint32_t keep_last;
    const uint32_t *group_offsets;
    const uint32_t *seq_tokens;
    const float *weights;
    const int8_t *codes;           /* with codes_out, scales and scales_out, or all four NULL; 16-byte aligned */
    const float *scales;
    uint32_t *group_offsets_out;
    uint32_t *seq_tokens_out;
    float *weights_out;
    int8_t *codes_out;
    float *scales_out;
    uint32_t *dropped;
} cf_kv_evict_desc;

cf_status cf_kv_validate_evict_desc(const cf_kv_evict_desc *desc);
cf_status cf_kv_evict_groups_async(const cf_kv_evict_desc *desc, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* CHROMOFOLD_KV_SELECT_H */
