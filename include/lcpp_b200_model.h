/*
 * lcpp_b200_model.h -- the ragged steps of a language model: block tables and
 * slot maps of a paged cache, rotary positions with the write of keys and
 * values into it, attention of one new token over its pages, eviction from it
 * by attention weight, expert routing with its balance loss, and the grouping
 * of token rows by expert; rotary positions, routing and grouping with their
 * gradients.
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
 * DeviceRotary: rotary positions, and the write into a paged cache
 * ------------------------------------------------------------------------ */

/* Largest head_dim of the operators below. */
#define LCPP_MAX_HEAD_DIM 256

typedef enum lcpp_rotary_layout {
    LCPP_ROTARY_HALF = 0,       /* pairs (i, i + rotary_dim / 2) */
    LCPP_ROTARY_INTERLEAVED = 1 /* pairs (2 i, 2 i + 1) */
} lcpp_rotary_layout;

typedef enum lcpp_rotary_scaling {
    LCPP_ROTARY_PLAIN = 0,       /* f_i = base^(-2 i / rotary_dim) */
    LCPP_ROTARY_LINEAR = 1,      /* f_i / factor */
    LCPP_ROTARY_BASE = 2,        /* f_i of base * factor^(rotary_dim / (rotary_dim - 2)) */
    LCPP_ROTARY_BY_ROTATIONS = 3 /* f_i / factor where f_i turns at most low times in the original
                                    context, f_i where it turns at least high times, and between
                                    them the mean weighted by the number of turns */
} lcpp_rotary_scaling;

/* Writes rotary_dim / 2 frequencies (radians per position) to HOST memory; the
 * operators read them from the device, in 64 bits, because angles of far
 * positions lose their fractions in 32.  rotary_dim is even, base above 0 and
 * finite, factor at least 1; original_context, low and high (0 < low < high)
 * count only for LCPP_ROTARY_BY_ROTATIONS.  Any other table serves as well. */
lcpp_status lcpp_rotary_frequencies(double* frequencies_out, uint32_t rotary_dim, double base, int32_t scaling,
                                    double factor, double original_context, double low, double high);

/* A tensor's element (token, head, column) is in[token * in_token_stride +
 * head * in_head_stride + column]; strides count elements. */
typedef struct lcpp_head_rows {
    const void* in;
    void* out;
    uint64_t in_token_stride, in_head_stride;
    uint64_t out_token_stride, out_head_stride;
    uint32_t num_heads; /* 0: the tensor is left out */
} lcpp_head_rows;

/* Pages of keys and values: element (page, token in the page, head, column) is
 * k[page * page_stride + token * token_stride + head * head_stride + column],
 * and v the same; strides count elements, so both memory orders of tokens and
 * heads, and pages that hold keys and values side by side, are the same to the
 * operators.  The slot of a token is page * block_size + token in the page. */
typedef struct lcpp_kv_cache {
    void* k;
    void* v;
    uint64_t page_stride, token_stride, head_stride;
    uint32_t num_pages;    /* num_pages * block_size below 2^40 */
    uint32_t block_size;   /* tokens a page holds, >= 1 */
    uint32_t num_kv_heads; /* >= 1 */
    uint32_t head_dim;     /* 1 to LCPP_MAX_HEAD_DIM */
    lcpp_dtype dtype;      /* a row dtype */
} lcpp_kv_cache;

typedef struct lcpp_rotary_args {
    lcpp_head_rows q, k;            /* turned by the same angles */
    const int32_t* positions;       /* [num_tokens] */
    const int32_t* token_request;   /* [num_tokens], or NULL; tokens outside [0, num_requests) are left out */
    const int32_t* position_offset; /* [num_requests] added to the positions of a request's tokens, or NULL */
    const double* frequencies;      /* [rotary_dim / 2] radians per position */
    uint64_t num_tokens;            /* below 2^31 */
    uint32_t num_requests;          /* entries of position_offset; counts only with token_request */
    uint32_t head_dim;              /* 1 to LCPP_MAX_HEAD_DIM */
    uint32_t rotary_dim;            /* even, at most head_dim: columns that are turned, the first ones */
    int32_t layout;                 /* lcpp_rotary_layout */
    float scale;                    /* factor of cosine and sine (1 unless the model's scaling has one) */
    lcpp_dtype dtype;               /* of q and k, a row dtype */
} lcpp_rotary_args;

/* For the pairs (a, b) of every head, with angle = position * f_i:
 *   a' = scale * (a cos(angle) - b sin(angle)),  b' = scale * (b cos(angle) + a sin(angle));
 * columns from rotary_dim on are copied.  Computed in 32 bits (an angle's fraction
 * of a turn in 64, cosine and sine of it in 32), rounded once.  `out` may be `in` itself with the same strides; else outputs
 * must not overlap inputs or one another.  Tokens that are left out are neither
 * read nor written. */
lcpp_status lcpp_rotary_forward(const lcpp_rotary_args* args, lcpp_stream_t stream);

/* The gradient: in = the gradient of forward's output, out = that of its input
 * (a = scale * (a' cos + b' sin), b = scale * (b' cos - a' sin)). */
lcpp_status lcpp_rotary_backward(const lcpp_rotary_args* args, lcpp_stream_t stream);

typedef struct lcpp_cache_append_args {
    lcpp_kv_cache cache;
    const void* v; /* [num_tokens][num_kv_heads][head_dim] with strides */
    uint64_t v_token_stride, v_head_stride;
    const int64_t* slots;    /* [num_tokens]; tokens whose slot lies outside the cache are left out */
    int32_t* slot_positions; /* [num_pages * block_size] gets the tokens' positions with their offsets, or NULL */
    float* slot_scores;      /* [num_pages * block_size] gets zeros for the tokens, or NULL */
} lcpp_cache_append_args;

/* lcpp_rotary_forward for q; k is turned into the keys of the tokens' slots and
 * v copied to their values (k.out is not used, k.num_heads = num_kv_heads).
 * Tokens that are left out keep their row of q's output and touch no slot.  The
 * slots of one call's tokens have to differ.  The cache must not overlap other
 * arrays of the call. */
lcpp_status lcpp_rotary_append(const lcpp_rotary_args* args, const lcpp_cache_append_args* append,
                               lcpp_stream_t stream);

/* ------------------------------------------------------------------------
 * DevicePagedAttention: one new token of each request over its pages
 * ------------------------------------------------------------------------ */

typedef struct lcpp_paged_attention_args {
    lcpp_kv_cache cache;
    const void* q; /* [num_requests][num_heads][head_dim] with strides, of the cache's dtype */
    uint64_t q_request_stride, q_head_stride;
    void* out; /* the same */
    uint64_t out_request_stride, out_head_stride;
    const int32_t* block_table; /* [num_requests][table_stride] page ids */
    uint64_t table_stride;      /* elements from row to row, >= table_width */
    uint32_t table_width;       /* pages a request can hold */
    uint32_t num_requests;      /* at most LCPP_MAX_REQUESTS */
    const int32_t* seq_lens;    /* [num_requests] tokens in the cache, the new one among them */
    uint32_t num_heads;         /* a multiple of num_kv_heads: query head h reads kv head h / (num_heads / num_kv_heads) */
    uint32_t window;            /* only the last `window` tokens are looked at; 0: all */
    float scale;                /* factor of the dot products */
    float softcap;              /* above 0: logits x become softcap * tanh(x / softcap); scale / softcap has to be finite, and
                                   1.45 times scale and softcap */
    float* lse_out;             /* [num_requests][num_heads] logarithm of the sum of exponentials, or NULL */
    const float* slot_scores;   /* [num_pages * block_size]; NULL: zeros */
    float* slot_scores_out;     /* the same after this step, may be slot_scores itself; NULL: not wanted */
    float score_decay;          /* factor of slot_scores */
} lcpp_paged_attention_args;

/* score_slots: num_pages * block_size when slot_scores_out is wanted, else 0.
 * Scores take 4 bytes for each of these slots and each query head (rounded up to
 * whole units of the kernel): they are the logits of the call's tokens. */
lcpp_status lcpp_paged_attention_temp_bytes(uint32_t num_requests, uint32_t num_heads, uint32_t num_kv_heads,
                                            uint32_t head_dim, uint64_t score_slots, size_t* temp_bytes);

/* For request r and head h, over its tokens t in the cache (position t of the
 * sequence lies in page t / block_size of the request's row):
 *   x_t = scale * q . k_t,  p = softmax of x,  out = sum_t p_t v_t,
 *   slot_scores_out[slot of t] = score_decay * slot_scores[slot of t] + sum_h p_t.
 * Statistics and sums are held in 32 bits, p as two numbers of the cache's
 * type where that has 16 bits (bfloat16: 16 digits; float16: 22, but to 2^-32
 * of the row's largest p, below which p counts as 0); the output is rounded
 * once.  A row that has
 * weights but did not end as finite numbers that way is computed again with p
 * as one number and sums in 64 bits: large values whose mean is a number give
 * that number, infinities and NaN among the values act as in the formula (a
 * block takes about 0.13 ms for 1000 tokens of such a row).  Lengths outside
 * [0, table_width * block_size] count as its ends; tokens whose page id is
 * outside [0, num_pages) are not looked at and have no score.  A row without
 * tokens, or whose logits are all -inf, gets zeros and lse -inf; keys and values
 * outside the request are never used, whatever they hold.  Tokens before the
 * window keep score_decay * slot_scores; slots of no request are not written.
 * Requests may share pages unless scores are wanted: the score of a shared slot
 * would depend on which request came first, and where the requests have more
 * tokens in all than num_pages * block_size, those whose logits find no room in
 * temp storage leave the scores of their slots as they are.  A request's bits depend on the lengths of the
 * call's requests, which the work is divided by, not on their values.
 * out, lse_out, slot_scores_out and temp storage must not overlap one another
 * or the inputs (slot_scores_out may be slot_scores). */
lcpp_status lcpp_paged_attention_decode(void* temp, size_t temp_bytes, const lcpp_paged_attention_args* args,
                                        lcpp_stream_t stream);

/* ------------------------------------------------------------------------
 * DeviceCacheEviction: requests cut down to their heaviest tokens
 * ------------------------------------------------------------------------ */

typedef struct lcpp_cache_evict_args {
    const int32_t* seq_lens;     /* [num_requests] tokens in the cache */
    const int32_t* block_table;  /* [num_requests][table_stride] page ids */
    uint64_t table_stride;       /* elements from row to row, >= table_width */
    uint32_t table_width;        /* pages a request can hold */
    uint32_t num_requests;       /* at most LCPP_MAX_REQUESTS */
    uint32_t num_pages;          /* num_pages * block_size below 2^40 */
    uint32_t block_size;         /* >= 1 */
    const float* slot_scores;    /* [num_pages * block_size] */
    const int32_t* slot_positions; /* [num_pages * block_size] positions in the sequences; NULL: places in the cache */
    const int32_t* evicted;      /* [num_requests] tokens that left a request before; NULL: 0 */
    uint32_t budget;             /* tokens that a cut request keeps, >= 1, below 2^31 */
    uint32_t trigger;            /* requests longer than this are cut, >= budget */
    uint32_t keep_first;         /* positions below this are kept */
    uint32_t keep_recent;        /* the last positions are kept; keep_first + keep_recent <= budget */
    uint32_t max_moves;          /* moves_out's entries of a request; min(budget, longest - budget) hold any */
    int32_t* seq_lens_out;       /* [num_requests] */
    int32_t* evicted_out;        /* [num_requests], or NULL; may be evicted itself */
    int32_t* move_counts_out;    /* [num_requests] */
    int64_t* moves_out;          /* [num_requests][moves_stride][2] slots, from and to */
    uint64_t moves_stride;       /* pairs from request to request, >= max_moves */
    int32_t* free_blocks;        /* [num_free] the list that lcpp_block_table_extend takes pages from, or NULL */
    const int32_t* free_used;    /* [1] its entries that are taken */
    int32_t* free_used_out;      /* [1] the same after the pages came back; not free_used itself */
    uint32_t num_free;
} lcpp_cache_evict_args;

/* Cuts every request longer than trigger to budget tokens: those whose position
 * is below keep_first or among the last keep_recent of its seq_lens + evicted
 * positions (without slot_positions: whose place is among the first keep_first
 * or the last keep_recent of its seq_lens), then the heaviest by slot_scores,
 * equal ones by their place in the cache, earlier ones first (NaN counts as
 * heavier than +inf, both zeros as equal; should more than budget positions be
 * protected, the earlier places are kept).  The kept tokens come to lie in the first budget places: the i-th kept
 * token past them goes to the i-th place among them whose token is not kept, so
 * at most as many move as leave.  moves_out holds the slots; entries past
 * move_counts_out are not written.  This call moves nothing:
 * lcpp_cache_evict_move does, for each layer's cache.  Attention does not mind
 * the order of the tokens (a window does: it counts places).
 *
 * No page may belong to two requests: its tokens would be moved and its page given
 * back for one of them while the other still uses it.
 *
 * A request whose row holds a page id outside [0, num_pages), or that has more
 * moves than max_moves, is left as it is (0 moves, its length).  Lengths count as
 * in lcpp_paged_attention_decode.  Pages of a cut request that hold no
 * token any more go back to the free list, request by request, page by page:
 * with n of them, free_used_out = free_used - n and they are written from
 * free_blocks[free_used_out] on (where free_used, at most num_free, is less than
 * n, the first n - free_used of them do not fit and are dropped). */
lcpp_status lcpp_cache_evict_plan(const lcpp_cache_evict_args* args, lcpp_stream_t stream);

/* Copies keys and values, and where given scores and positions, of the first
 * min(move_counts[r], max_moves) pairs of moves[r] from slot to slot.  The slots
 * of one call have to differ, as a plan's do; moves from or to a slot outside
 * the cache are left out. */
lcpp_status lcpp_cache_evict_move(const lcpp_kv_cache* cache, const int64_t* moves, uint64_t moves_stride,
                                  uint32_t max_moves, const int32_t* move_counts, uint32_t num_requests,
                                  float* slot_scores, int32_t* slot_positions, lcpp_stream_t stream);

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
