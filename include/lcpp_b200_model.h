/*
 * lcpp_b200_model.h -- the ragged bookkeeping of one language-model step:
 * block tables and slot maps of a paged cache, expert routing with its
 * balance loss, and the grouping of token rows by expert, the last two with
 * their gradients.
 *
 * No counterpart in the reference: its users assemble these steps from
 * scans, reductions by key and radix sorts.  The conventions of lcpp_b200.h
 * hold: device pointers owned by the caller, no allocation, work enqueued on
 * the given stream without host synchronisation, a status code on misuse.
 * Every pointer must be aligned to its element.  Row strides count elements.
 * Row dtypes ("rows" and logits) are LCPP_F32, LCPP_F16 and LCPP_BF16; sums,
 * softmax statistics and weights are held in 32 bits.  Results do not depend
 * on the order in which blocks run: equal inputs give equal bits.
 */
#ifndef LCPP_B200_MODEL_H
#define LCPP_B200_MODEL_H

#include "lcpp_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * DeviceBlockTable: pages of a paged cache for the tokens of one step
 * ------------------------------------------------------------------------ */

/* Largest num_requests of lcpp_block_table_extend. */
#define LCPP_MAX_REQUESTS (1u << 20)

typedef struct lcpp_block_table_args {
    const int32_t* context_lens;  /* [num_requests] tokens already in the cache (below 0: 0) */
    const int32_t* new_lens;      /* [num_requests] tokens to add (below 0: 0); NULL: one each */
    int32_t* block_table;         /* [num_requests][table_stride] page ids, extended in place */
    uint64_t table_stride;        /* elements from row to row, >= table_width */
    uint32_t table_width;         /* pages a request can hold */
    uint32_t num_requests;
    uint32_t block_size;          /* tokens a page holds, >= 1 */
    uint32_t num_free;            /* entries of free_blocks */
    const int32_t* free_blocks;   /* [num_free] ids of free pages, taken from the front */
    const int32_t* free_used;     /* [1] entries of free_blocks taken by earlier steps; NULL: 0 */
    int32_t* free_used_out;       /* [1] the same after this step; not free_used itself */
    int32_t* seq_lens_out;        /* [num_requests] tokens in the cache after this step */
    int32_t* query_starts_out;    /* [num_requests + 1] exclusive sums of new_lens (at most 2^31 - 1) */
    int64_t* slots_out;           /* [max_tokens] page id * block_size + offset in the page */
    int32_t* positions_out;       /* [max_tokens] position in the request's sequence, or NULL */
    int32_t* token_request_out;   /* [max_tokens] request of the token, or NULL */
    uint64_t max_tokens;          /* entries of the three arrays above, below 2^31 - 1 */
} lcpp_block_table_args;

lcpp_status lcpp_block_table_temp_bytes(uint64_t num_requests, uint64_t max_tokens, size_t* temp_bytes);

/* Lays out the step's tokens, request after request: request r's token i (of
 * new_lens[r]) is number query_starts_out[r] + i, has position
 * context_lens[r] + i, and lies in page position / block_size of its row of
 * the block table.  Pages the row does not hold yet are taken from
 * free_blocks in request order and written into the row.
 *
 * A request is refused when its tokens end past max_tokens, its sequence
 * needs more than table_width pages (or is longer than 2^31 - 1), or
 * free_blocks ends before its pages.  A refused request takes no page, its
 * row stays as it is, seq_lens_out keeps its context length, and its tokens
 * that lie below max_tokens are marked like the entries past the step's last
 * token: slot -1, position 0, request -1.  Requests after it that need no new
 * page are still served; those that need one are refused too when free_blocks
 * is what ended.  A negative page id in the row gives slot -1.
 *
 * The outputs, temp storage and the table must not overlap one another or the
 * inputs: a step's outputs are the next one's inputs through two sets of
 * buffers.  Zero requests give one start, no pages and marked entries. */
lcpp_status lcpp_block_table_extend(void* temp, size_t temp_bytes, const lcpp_block_table_args* args,
                                    lcpp_stream_t stream);

/* ------------------------------------------------------------------------
 * DeviceRouter: experts of each token, their weights, counts and balance loss
 * ------------------------------------------------------------------------ */

#define LCPP_MAX_EXPERTS 1024
#define LCPP_MAX_TOP_K 32

typedef enum lcpp_router_score {
    LCPP_SCORE_SOFTMAX = 0, /* s = softmax of the token's logits */
    LCPP_SCORE_SIGMOID = 1  /* s = 1 / (1 + exp(-logit)) */
} lcpp_router_score;

/* Added to the score: a bias is added to s instead of the logit. */
#define LCPP_BIAS_ON_SCORE 0x10

typedef struct lcpp_router_config {
    uint32_t num_experts; /* 1 to LCPP_MAX_EXPERTS */
    uint32_t top_k;       /* 1 to min(num_experts, LCPP_MAX_TOP_K) */
    int32_t score;        /* lcpp_router_score, + LCPP_BIAS_ON_SCORE */
    int32_t renormalize;  /* nonzero: a token's weights are divided by their sum */
    float weight_scale;   /* factor of every weight */
    float loss_coef;      /* factor of the balance loss */
} lcpp_router_config;

lcpp_status lcpp_router_temp_bytes(uint64_t num_tokens, uint32_t num_experts, size_t* temp_bytes);

/* For each token t: the top_k experts with the largest logit + bias, or s + bias
 * with LCPP_BIAS_ON_SCORE (the selection bias of models that balance their
 * experts without a loss; s is then rounded to 32 bits first), added in 32 bits,
 * equal sums to the lower expert, in descending order, and
 *   weights[t][j] = weight_scale * s[e_j] (/ sum_i s[e_i] when renormalised).
 * The bias (NULL: none) only takes part in the choice; +inf and NaN in it count
 * as the largest finite number.  An expert whose logit, bias or sum is -inf is
 * never chosen; entries left over hold expert -1, weight 0.
 * A token with a negative token_request (NULL: none has), or with no expert
 * to choose, is left out: all its entries are -1 and 0, and it takes no part
 * in the counts or the loss.  With T' tokens that took part (d_num_routed_out)
 * and counts[e] entries that name expert e:
 *   loss = loss_coef * E * sum_e counts[e] / (top_k T') * mean_t s[t][e] / sum_i s[t][i]
 * (0 when T' is 0).  NaN logits order above +inf, and NaN (and +inf under
 * softmax) go into the token's weights and the loss as the formulas say; a
 * token that is left out passes nothing on.  The outputs and temp storage must
 * not overlap one another or the inputs. */
lcpp_status lcpp_router_forward(void* temp, size_t temp_bytes, const void* d_logits, uint64_t logits_stride,
                                lcpp_dtype logits_dtype, const float* d_bias, const int32_t* d_token_request,
                                float* d_weights_out, int32_t* d_experts_out, int32_t* d_counts_out,
                                int32_t* d_num_routed_out, float* d_loss_out, uint64_t num_tokens,
                                const lcpp_router_config* config, lcpp_stream_t stream);

/* The gradient of sum(weights * grad_weights) + loss * grad_loss with respect
 * to the logits, the counts held constant.  d_experts, d_counts and
 * d_num_routed are forward's outputs; d_grad_weights [num_tokens][top_k] and
 * d_grad_loss [1] may be NULL (zero).  Tokens whose first expert is -1 get
 * zeros.  d_grad_logits_out has the logits' dtype and may be d_logits itself
 * when the strides agree; else it must not overlap the inputs. */
lcpp_status lcpp_router_backward(const void* d_logits, uint64_t logits_stride, lcpp_dtype logits_dtype,
                                 const int32_t* d_experts, const int32_t* d_counts, const int32_t* d_num_routed,
                                 const float* d_grad_weights, const float* d_grad_loss, void* d_grad_logits_out,
                                 uint64_t grad_logits_stride, uint64_t num_tokens,
                                 const lcpp_router_config* config, lcpp_stream_t stream);

/* ------------------------------------------------------------------------
 * DeviceDispatch: token rows grouped by expert, and back
 * ------------------------------------------------------------------------ */

lcpp_status lcpp_dispatch_temp_bytes(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, size_t* temp_bytes);

/* Rows that hold any choice of num_tokens * top_k experts when segments start
 * at multiples of row_align: pairs + min(num_experts, pairs) * (row_align - 1). */
lcpp_status lcpp_dispatch_max_rows(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, uint32_t row_align,
                                   uint64_t* max_rows);

/* Groups the pairs p = t * top_k + j of d_experts [num_tokens][top_k] by
 * expert, in the order of p.  Expert e's rows start at
 * d_expert_starts_out[e], a multiple of row_align; d_expert_starts_out
 * [num_experts] is the end of the last segment.  d_row_of_out[p] = the pair's
 * row, d_pair_of_out[row] = the row's pair, -1 for rows that pad a segment or
 * lie past the last one.  Pairs whose expert is not in [0, num_experts), or
 * whose row would lie past max_rows, get row -1; the starts are not cut off
 * there.  num_tokens * top_k, max_rows and lcpp_dispatch_max_rows' answer stay
 * below 2^31.  The outputs of this call and the next three must not overlap one
 * another, temp storage or the inputs, except where it says so. */
lcpp_status lcpp_dispatch_plan(void* temp, size_t temp_bytes, const int32_t* d_experts, int32_t* d_expert_starts_out,
                               int32_t* d_row_of_out, int32_t* d_pair_of_out, uint64_t num_tokens, uint32_t top_k,
                               uint32_t num_experts, uint32_t row_align, uint64_t max_rows, lcpp_stream_t stream);

/* d_rows_out[row_of(t, j)] = d_x[t]; rows that pad a segment get zeros, rows
 * past the last segment (d_expert_starts[num_experts]) are not written.  Its
 * gradient with respect to x is lcpp_dispatch_combine without weights. */
lcpp_status lcpp_dispatch_gather(const void* d_x, uint64_t x_stride, const int32_t* d_row_of,
                                 const int32_t* d_pair_of, const int32_t* d_expert_starts, void* d_rows_out,
                                 uint64_t rows_stride, uint64_t num_tokens, uint32_t top_k, uint32_t num_experts,
                                 uint64_t max_rows, uint64_t hidden, lcpp_dtype dtype, lcpp_stream_t stream);

/* d_out[t] = sum_j weights[t][j] * d_rows[row_of(t, j)], added in 32 bits in
 * the order of j and rounded once; d_weights NULL: weights of 1.  Pairs
 * without a row add nothing. */
lcpp_status lcpp_dispatch_combine(const void* d_rows, uint64_t rows_stride, const int32_t* d_row_of,
                                  const float* d_weights, void* d_out, uint64_t out_stride, uint64_t num_tokens,
                                  uint32_t top_k, uint64_t max_rows, uint64_t hidden, lcpp_dtype dtype,
                                  lcpp_stream_t stream);

/* The gradient of combine with weights: d_grad_rows_out[row_of(t, j)] =
 * weights[t][j] * d_grad_out[t], d_grad_weights_out[t][j] = the dot product of
 * d_grad_out[t] and d_rows[row_of(t, j)] (0 without a row).  Padding rows of
 * d_grad_rows_out get zeros, rows past the last segment are not written.
 * d_grad_rows_out may be d_rows itself when the strides agree, and
 * d_grad_weights_out may be d_weights itself. */
lcpp_status lcpp_dispatch_combine_backward(const void* d_grad_out, uint64_t grad_out_stride, const void* d_rows,
                                           uint64_t rows_stride, const int32_t* d_row_of, const int32_t* d_pair_of,
                                           const int32_t* d_expert_starts, const float* d_weights,
                                           void* d_grad_rows_out, uint64_t grad_rows_stride,
                                           float* d_grad_weights_out, uint64_t num_tokens, uint32_t top_k,
                                           uint32_t num_experts, uint64_t max_rows, uint64_t hidden,
                                           lcpp_dtype dtype, lcpp_stream_t stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* LCPP_B200_MODEL_H */
