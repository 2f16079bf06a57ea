// router.cu -- DeviceRouter's C entry points (include/lcpp_b200_model.h); the
// kernels are in router.cuh.
#include "router.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace lcpp {
namespace router {

__global__ void __launch_bounds__(kThreads) clear_kernel(uint32_t* words, uint32_t n)
{
    let_next_start();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) words[i] = 0;
}

}  // namespace router
}  // namespace lcpp

namespace {

size_t temp_size(uint32_t experts) { return align_up(router::cleared_bytes(experts), kTempAlign); }

// Bytes of the widest copy that every row's start and length are a multiple of.
uint32_t copy_unit(const void* logits, uint64_t stride, uint32_t experts, int size)
{
    const uint64_t bits = reinterpret_cast<uintptr_t>(logits) | stride * size | uint64_t(experts) * size | 16;
    return uint32_t(bits & (~bits + 1));
}

int32_t score_of(const lcpp_router_config* c) { return c->score & ~LCPP_BIAS_ON_SCORE; }

lcpp_status check_config(const lcpp_router_config* c, uint64_t tokens, uint64_t stride)
{
    if (!c || !c->num_experts || c->num_experts > LCPP_MAX_EXPERTS || !c->top_k || c->top_k > c->num_experts ||
        c->top_k > LCPP_MAX_TOP_K || (score_of(c) != LCPP_SCORE_SOFTMAX && score_of(c) != LCPP_SCORE_SIGMOID))
        return LCPP_ERR_INVALID_ARG;
    // counts are 32-bit, and rows are addressed with 64-bit element offsets
    if (tokens * c->top_k >= uint64_t(1) << 31 || tokens >> 31 || (tokens > 1 && stride < c->num_experts) || stride >> 32)
        return LCPP_ERR_INVALID_ARG;
    return LCPP_OK;
}

lcpp_status forward(void* temp, size_t temp_bytes, const void* logits, uint64_t stride, lcpp_dtype dtype,
                    const float* bias, const int32_t* token_request, float* weights, int32_t* experts,
                    int32_t* counts, int32_t* num_routed, float* loss, uint64_t tokens, const lcpp_router_config* c,
                    cudaStream_t s)
{
    lcpp_status st = check_config(c, tokens, stride);
    if (st != LCPP_OK) return st;
    const int size = row_dtype_bytes(dtype);
    if (!size) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!temp || misaligned(temp, kTempAlign) || !counts || !num_routed || !loss ||
        (tokens && (!logits || !weights || !experts)))
        return LCPP_ERR_INVALID_ARG;
    const void* words[] = {bias, token_request, weights, experts, counts, num_routed, loss};
    for (const void* w : words)
        if (misaligned(w, 4)) return LCPP_ERR_INVALID_ARG;
    if (misaligned(logits, size)) return LCPP_ERR_INVALID_ARG;
    if (temp_bytes < temp_size(c->num_experts)) return LCPP_ERR_TEMP_TOO_SMALL;
    const uint64_t pairs = tokens * c->top_k, n = c->num_experts;
    const Array arrays[] = {{bias, n * 4, false},     {token_request, tokens * 4, false}, {weights, pairs * 4, true},
                            {experts, pairs * 4, true}, {counts, n * 4, true},            {num_routed, 4, true},
                            {loss, 4, true},            {temp, temp_size(uint32_t(n)), true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
    for (const Array& o : arrays)
        if (o.written && overlap_rows(logits, tokens, stride, n, size, o.p, o.bytes)) return LCPP_ERR_INVALID_ARG;

    unsigned char* t = static_cast<unsigned char*>(temp);
    router::Params p{};
    p.logits = logits;
    p.stride = stride;
    p.bias = bias;
    p.token_request = token_request;
    p.weights = weights;
    p.experts = experts;
    p.counts = counts;
    p.num_routed = num_routed;
    p.loss = loss;
    p.tokens = tokens;
    p.num_experts = c->num_experts;
    p.top_k = c->top_k;
    p.renormalize = c->renormalize != 0;
    p.weight_scale = c->weight_scale;
    p.loss_coef = c->loss_coef;
    p.bias_on_score = (c->score & LCPP_BIAS_ON_SCORE) != 0;
    p.unit = copy_unit(logits, stride, c->num_experts, size);
    p.ctrl = reinterpret_cast<uint32_t*>(t);
    p.share_total = reinterpret_cast<unsigned long long*>(t + router::kShareOffset);
    p.count_total = reinterpret_cast<uint32_t*>(p.share_total + router::kShareScales * c->num_experts);
    const bool sigmoid = score_of(c) == LCPP_SCORE_SIGMOID;
    diag::KernelTimer timer(kTimerRouter, tokens * c->num_experts, s);
    switch (dtype) {
    case LCPP_F32: return router::forward_f32(p, sigmoid, s);
    case LCPP_F16: return router::forward_f16(p, sigmoid, s);
    default: return router::forward_bf16(p, sigmoid, s);
    }
}

lcpp_status backward(const void* logits, uint64_t stride, lcpp_dtype dtype, const int32_t* experts,
                     const int32_t* counts, const int32_t* num_routed, const float* grad_weights,
                     const float* grad_loss, void* grad_logits, uint64_t grad_stride, uint64_t tokens,
                     const lcpp_router_config* c, cudaStream_t s)
{
    lcpp_status st = check_config(c, tokens, stride);
    if (st == LCPP_OK) st = check_config(c, tokens, grad_stride);
    if (st != LCPP_OK) return st;
    const int size = row_dtype_bytes(dtype);
    if (!size) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!tokens) return LCPP_OK;
    if (!logits || !experts || !counts || !num_routed || !grad_logits) return LCPP_ERR_INVALID_ARG;
    const void* words[] = {experts, counts, num_routed, grad_weights, grad_loss};
    for (const void* w : words)
        if (misaligned(w, 4)) return LCPP_ERR_INVALID_ARG;
    if (misaligned(logits, size) || misaligned(grad_logits, size)) return LCPP_ERR_INVALID_ARG;
    // in place: each warp writes a row after it has read it
    const bool in_place = logits == grad_logits && stride == grad_stride;
    if (!in_place && overlap(logits, span_bytes(tokens, stride, c->num_experts, size), grad_logits,
                             span_bytes(tokens, grad_stride, c->num_experts, size)))
        return LCPP_ERR_INVALID_ARG;
    const uint64_t pairs = tokens * c->top_k;
    const Array inputs[] = {{experts, pairs * 4, false}, {counts, uint64_t(c->num_experts) * 4, false},
                            {num_routed, 4, false},      {grad_weights, pairs * 4, false},
                            {grad_loss, 4, false}};
    for (const Array& i : inputs)
        if (overlap_rows(grad_logits, tokens, grad_stride, c->num_experts, size, i.p, i.bytes)) return LCPP_ERR_INVALID_ARG;

    router::BackParams p{};
    p.logits = logits;
    p.stride = stride;
    p.experts = experts;
    p.counts = counts;
    p.num_routed = num_routed;
    p.grad_weights = grad_weights;
    p.grad_loss = grad_loss;
    p.grad_logits = grad_logits;
    p.grad_stride = grad_stride;
    p.tokens = tokens;
    p.num_experts = c->num_experts;
    p.top_k = c->top_k;
    p.renormalize = c->renormalize != 0;
    p.weight_scale = c->weight_scale;
    p.loss_coef = c->loss_coef;
    p.unit = copy_unit(logits, stride, c->num_experts, size);
    p.wide_stores = rows_16b(grad_logits, grad_stride, size);
    const bool sigmoid = score_of(c) == LCPP_SCORE_SIGMOID;
    diag::KernelTimer timer(kTimerRouter, tokens * c->num_experts, s);
    switch (dtype) {
    case LCPP_F32: return router::backward_f32(p, sigmoid, s);
    case LCPP_F16: return router::backward_f16(p, sigmoid, s);
    default: return router::backward_bf16(p, sigmoid, s);
    }
}

}  // namespace

extern "C" {

lcpp_status lcpp_router_temp_bytes(uint64_t num_tokens, uint32_t num_experts, size_t* temp_bytes)
{
    if (!temp_bytes || num_tokens >> 31 || !num_experts || num_experts > LCPP_MAX_EXPERTS) return LCPP_ERR_INVALID_ARG;
    *temp_bytes = temp_size(num_experts);
    return LCPP_OK;
}

lcpp_status lcpp_router_forward(void* temp, size_t temp_bytes, const void* d_logits, uint64_t logits_stride,
                                lcpp_dtype logits_dtype, const float* d_bias, const int32_t* d_token_request,
                                float* d_weights_out, int32_t* d_experts_out, int32_t* d_counts_out,
                                int32_t* d_num_routed_out, float* d_loss_out, uint64_t num_tokens,
                                const lcpp_router_config* config, lcpp_stream_t stream)
{
    return guarded("lcpp_router_forward", [&] {
        return forward(temp, temp_bytes, d_logits, logits_stride, logits_dtype, d_bias, d_token_request, d_weights_out,
                       d_experts_out, d_counts_out, d_num_routed_out, d_loss_out, num_tokens, config,
                       reinterpret_cast<cudaStream_t>(stream));
    });
}

lcpp_status lcpp_router_backward(const void* d_logits, uint64_t logits_stride, lcpp_dtype logits_dtype,
                                 const int32_t* d_experts, const int32_t* d_counts, const int32_t* d_num_routed,
                                 const float* d_grad_weights, const float* d_grad_loss, void* d_grad_logits_out,
                                 uint64_t grad_logits_stride, uint64_t num_tokens,
                                 const lcpp_router_config* config, lcpp_stream_t stream)
{
    return guarded("lcpp_router_backward", [&] {
        return backward(d_logits, logits_stride, logits_dtype, d_experts, d_counts, d_num_routed, d_grad_weights,
                        d_grad_loss, d_grad_logits_out, grad_logits_stride, num_tokens, config,
                        reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
