/*
 * libgsage.so -- operators around learning and ranking on the embeddings and
 * neighborhoods of gsage.h: attention over neighbors (the aggregation beside mean
 * and max), log probabilities over a catalog of items (the loss and the ranking
 * beside the link head), and dropout whose mask is never stored.  The reference
 * has none of them; conventions (ownership, streams, return codes) are gsage.h's.
 *
 * Tables come as fp32, bf16 or fp16 (`dtype` below: one type for all tables of a
 * call, contiguous, aligned to their element); sums, statistics and losses are
 * fp32 whatever the tables' type.
 */
#ifndef GSAGE_OPS_H_
#define GSAGE_OPS_H_

#include "gsage.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GS_F32   0
#define GS_BF16  1
#define GS_F16   2

/*
 * Dropout: out[i] = x[i] / share where element i is kept, else 0 (also where x is
 * not finite).  With t = floor(rate * 2^16), i is kept where the 16-bit piece
 * i % 8 (word (i % 8) / 2, low half first) of
 *     Philox4x32-10(counter = (b lo, b hi, 0x50000000, 0), key = seed),
 *     b = offset + i / 8
 * is >= t; share = 1 - t / 2^16.  The mask is drawn again wherever it is needed:
 * the gradient is the same call on the gradient of out.
 *   x, out       device [n]; out may be x, else the two do not overlap
 *   rate         0 <= rate, t < 2^16
 *   seed_device  nullable device uint64[1]: read in place of `seed`, so that a
 *                captured graph draws other masks when the caller changes it
 *   offset       blocks of eight used by earlier calls under this seed
 */
int gs_dropout(const void *x, int64_t n, int dtype, double rate, uint64_t seed, const uint64_t *seed_device,
               uint64_t offset, void *out, void *stream);

/*
 * The neighbors of n_parents parents: edges 0 .. n_edges - 1, those of parent p
 * being consecutive,
 *   indptr == NULL: p * n_child .. (p + 1) * n_child - 1 (n_edges = n_parents * n_child)
 *   indptr != NULL: device int64[n_parents + 1], not decreasing, indptr[p] ..
 *                   indptr[p + 1] - 1; edges before the first or from the last on belong to no parent
 * Edge e reads table row ids[e] - id_offset (ids device int32[n_edges]), or row e
 * when ids is NULL; an edge whose row lies outside [0, n_rows) is no neighbor.
 */
typedef struct gs_neighbors {
    const int64_t *indptr;
    int64_t        n_parents;
    int64_t        n_child;
    const int32_t *ids;
    int64_t        n_edges;       /* < 2^31 */
    int64_t        id_offset;
    int64_t        n_rows;
} gs_neighbors;

/*
 * Attention of every parent over its neighbors, head by head (heads a multiple of
 * kv_heads; heads h * kv_heads / heads share keys and values):
 *     s_e = scale * <q[p][h], k[row(e)][j]>,  P = softmax of s over p's edges,
 *     out[p][h] = sum_e P_e v[row(e)][j],  lse[p][h] = log sum_e exp(s_e)
 * and zeros / -inf for a parent without neighbors.
 *   q, out   device [n_parents][heads][dim]      k, v  device [n_rows][kv_heads][dim]
 *   v        NULL: the keys are the values
 *   lse      device float[n_parents][heads]
 *   workspace of gs_neighbor_attention_workspace(...) bytes (may be 0), 16-byte aligned
 * 1 <= dim <= 256; parents, edges and rows below 2^31, else GS_ELIMIT.
 */
size_t gs_neighbor_attention_workspace(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype);
int gs_neighbor_attention_fwd(const void *q, const void *k, const void *v, const gs_neighbors *nb, int heads,
                              int kv_heads, int dim, int dtype, float scale, void *out, float *lse,
                              void *workspace, size_t workspace_bytes, void *stream);

/*
 * Its gradients; the probabilities are computed again from lse.
 *   out, lse   what the forward call left;  g_out device [n_parents][heads][dim]
 *   g_q        device [n_parents][heads][dim], NULL: not wanted
 *   g_k, g_v   device [n_rows][kv_heads][dim], NULL: not wanted (g_v is ignored when v
 *              is NULL: g_k then takes both parts).  Every row is written, rows that
 *              no parent reads as zeros, except rows (ids == NULL) whose edge belongs
 *              to no parent: these are left as they are
 *   inv_indptr / inv_edges  with ids, where g_k or g_v is wanted: the edges that read
 *              row r are inv_edges[inv_indptr[r] .. inv_indptr[r + 1]) (device
 *              int64[n_rows + 1], int32[n_inv]), each edge once.  Sums run in their order: the
 *              result does not depend on timing.  NULL without ids
 */
size_t gs_neighbor_attention_bwd_workspace(const gs_neighbors *nb, int heads, int kv_heads, int dim, int dtype,
                                           int64_t n_inv);
int gs_neighbor_attention_bwd(const void *q, const void *k, const void *v, const gs_neighbors *nb, int heads,
                              int kv_heads, int dim, int dtype, float scale, const void *out, const float *lse,
                              const void *g_out, const int64_t *inv_indptr, const int32_t *inv_edges, int64_t n_inv,
                              void *g_q, void *g_k, void *g_v, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Users against every item of a catalog: z[n][j] = scale * <user[n], item[j]> + bias[j],
 *     log_prob[n] = z[n][targets[n]] - lse[n],  lse = log sum_j exp(z),
 *     entropy[n]  = -sum_j p_j log p_j,  p = exp(z - lse)
 * and the top_k items by z, the scores compared in 64 bits, the lower index first where two
 * are equal.  The scores never pass through memory.
 *   user device [n_users][dim], item device [n_items][dim] of `dtype`
 *   bias     nullable device float[n_items]; below -1e10 (-inf, the type's lowest value): the item is
 *            not on offer, and its row is never looked at.  A user for whom nothing is on offer: lse -inf, entropy 0
 *   targets  nullable device int32[n_users]; outside [0, n_items): no target, log_prob 0;
 *            a target that is not on offer: log_prob -inf
 *   scores   are held in fp32; one below -6.9e11 (-1e12 in units of log 2) counts as not on offer
 *   log_prob, entropy, lse  device float[n_users], each nullable
 *   top_log_prob / top_ids  device float / int32 [n_users][top_k], with top_k > 0;
 *            places beyond the items on offer hold -inf / -1
 *   workspace of gs_catalog_workspace(...) bytes, 256-byte aligned
 * scale > 0 and finite; 1 <= dim <= 256, top_k <= 64, n_users and n_items < 2^31 - 512, else GS_ELIMIT.
 */
size_t gs_catalog_workspace(int64_t n_users, int64_t n_items, int dim, int dtype, int top_k);
int gs_catalog_fwd(const void *user, int64_t n_users, const void *item, int64_t n_items, int dim, int dtype,
                   const float *bias, float scale, const int32_t *targets, float *log_prob, float *entropy, float *lse,
                   int top_k, float *top_log_prob, int32_t *top_ids, void *workspace, size_t workspace_bytes,
                   void *stream);

/*
 * Its gradients for g_log_prob and g_entropy (device float[n_users], each nullable, lse and
 * entropy from the forward call):
 *     dz_j = g_log_prob ([j = target] - p_j) - g_entropy p_j (log p_j + entropy)
 * into g_user [n_users][dim], g_item [n_items][dim] (of `dtype`) and g_bias float[n_items],
 * each nullable.  An item that is not on offer gets zeros.  The order of every sum is fixed.
 * n_users + n_items < 2^31, else GS_ELIMIT.
 * For the tables' gradients dz_j is cut to the bits of the tables' type (bf16: below 2^-8, fp16: below 2^-14 of a term left
 * out), except the target's, of which nothing is left out: g (1 - p) of a well predicted target is as exact as p is in
 * fp32.  g_bias takes every dz_j whole.
 */
size_t gs_catalog_bwd_workspace(int64_t n_users, int64_t n_items, int dim, int dtype);
int gs_catalog_bwd(const void *user, int64_t n_users, const void *item, int64_t n_items, int dim, int dtype,
                   const float *bias, float scale, const int32_t *targets, const float *lse, const float *entropy,
                   const float *g_log_prob, const float *g_entropy, void *g_user, void *g_item, float *g_bias,
                   void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GSAGE_OPS_H_ */
