/*
 * lcpp_b200_model.hpp -- C++ surface of the model-step operators
 * (lcpp_b200_model.h) in the style of lcpp_b200.hpp: views of device buffers,
 * the stream first, misuse throws lcpp_b200::Error.  Header-only; every call
 * forwards to the C ABI.  No counterpart in the reference.
 */
#ifndef LCPP_B200_MODEL_HPP
#define LCPP_B200_MODEL_HPP

#include "lcpp_b200.hpp"
#include "lcpp_b200_model.h"

namespace lcpp_b200 {

/// Rows of LCPP_F32, LCPP_F16 or LCPP_BF16 elements; `stride` counts elements.
template <typename Void>
struct BasicRowsView {
    Void* ptr = nullptr;
    uint64_t rows = 0, columns = 0, stride = 0;
    lcpp_dtype dtype = LCPP_NONE;

    BasicRowsView() = default;
    BasicRowsView(Void* p, uint64_t num_rows, uint64_t num_columns, lcpp_dtype type, uint64_t row_stride = 0) noexcept
        : ptr(p), rows(num_rows), columns(num_columns), stride(row_stride ? row_stride : num_columns), dtype(type)
    {
    }
    template <typename Other>
    BasicRowsView(const BasicRowsView<Other>& o) noexcept
        : ptr(o.ptr), rows(o.rows), columns(o.columns), stride(o.stride), dtype(o.dtype)
    {
    }
};
using RowsView = BasicRowsView<void>;
using ConstRowsView = BasicRowsView<const void>;

namespace detail {

inline void require_rows(bool ok) { require(ok, "view of too few rows or columns, or of another element type"); }

}  // namespace detail

/// Block tables and slot maps of a paged cache, from request lengths.
class DeviceBlockTable {
public:
    static size_t GetTempStorageBytes(uint64_t num_requests, uint64_t max_tokens)
    {
        size_t b = 0;
        detail::check(lcpp_block_table_temp_bytes(num_requests, max_tokens, &b), "GetTempStorageBytes");
        return b;
    }

    /// Gives the step's tokens their pages and slots (lcpp_block_table_extend).
    void Extend(lcpp_stream_t stream, BufferView<uint32_t> temp_storage, const lcpp_block_table_args& args)
    {
        detail::check(lcpp_block_table_extend(temp_storage.data(), detail::temp_bytes(temp_storage), &args, stream),
                      "Extend");
    }
};

/// Experts of each token, their weights, per-expert counts and the balance
/// loss, with the gradient.
class DeviceRouter {
public:
    static size_t GetTempStorageBytes(uint64_t num_tokens, uint32_t num_experts)
    {
        size_t b = 0;
        detail::check(lcpp_router_temp_bytes(num_tokens, num_experts, &b), "GetTempStorageBytes");
        return b;
    }

    /// lcpp_router_forward; empty `bias` and `token_request` views: none.
    void Forward(lcpp_stream_t stream, BufferView<uint32_t> temp_storage, ConstRowsView logits,
                 BufferView<const float> bias, BufferView<const int32_t> token_request, BufferView<float> weights_out,
                 BufferView<int32_t> experts_out, BufferView<int32_t> counts_out, BufferView<int32_t> num_routed_out,
                 BufferView<float> loss_out, uint64_t num_tokens, const lcpp_router_config& config)
    {
        const uint64_t pairs = num_tokens * config.top_k;
        detail::require_rows(logits.rows >= num_tokens && logits.columns >= config.num_experts);
        detail::require(weights_out.size() >= pairs && experts_out.size() >= pairs &&
                            counts_out.size() >= config.num_experts && num_routed_out.size() >= 1 &&
                            loss_out.size() >= 1 && (!bias.data() || bias.size() >= config.num_experts) &&
                            (!token_request.data() || token_request.size() >= num_tokens),
                        "Forward: a view is too short");
        detail::check(lcpp_router_forward(temp_storage.data(), detail::temp_bytes(temp_storage), logits.ptr,
                                          logits.stride, logits.dtype, bias.data(), token_request.data(),
                                          weights_out.data(), experts_out.data(), counts_out.data(),
                                          num_routed_out.data(), loss_out.data(), num_tokens, &config, stream),
                      "Forward");
    }

    /// lcpp_router_backward; empty `grad_weights` and `grad_loss` views: zero.
    void Backward(lcpp_stream_t stream, ConstRowsView logits, BufferView<const int32_t> experts,
                  BufferView<const int32_t> counts, BufferView<const int32_t> num_routed,
                  BufferView<const float> grad_weights, BufferView<const float> grad_loss, RowsView grad_logits_out,
                  uint64_t num_tokens, const lcpp_router_config& config)
    {
        const uint64_t pairs = num_tokens * config.top_k;
        detail::require_rows(logits.rows >= num_tokens && logits.columns >= config.num_experts &&
                             grad_logits_out.rows >= num_tokens && grad_logits_out.columns >= config.num_experts &&
                             grad_logits_out.dtype == logits.dtype);
        detail::require(experts.size() >= pairs && counts.size() >= config.num_experts && num_routed.size() >= 1 &&
                            (!grad_weights.data() || grad_weights.size() >= pairs) &&
                            (!grad_loss.data() || grad_loss.size() >= 1),
                        "Backward: a view is too short");
        detail::check(lcpp_router_backward(logits.ptr, logits.stride, logits.dtype, experts.data(), counts.data(),
                                           num_routed.data(), grad_weights.data(), grad_loss.data(),
                                           grad_logits_out.ptr, grad_logits_out.stride, num_tokens, &config, stream),
                      "Backward");
    }
};

/// Token rows grouped by expert and summed back, with the gradients.
class DeviceDispatch {
public:
    static size_t GetTempStorageBytes(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts)
    {
        size_t b = 0;
        detail::check(lcpp_dispatch_temp_bytes(num_tokens, top_k, num_experts, &b), "GetTempStorageBytes");
        return b;
    }

    /// Rows that hold any choice when segments start at multiples of row_align.
    static uint64_t MaxRows(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, uint32_t row_align = 1)
    {
        uint64_t rows = 0;
        detail::check(lcpp_dispatch_max_rows(num_tokens, top_k, num_experts, row_align, &rows), "MaxRows");
        return rows;
    }

    /// lcpp_dispatch_plan; pair_of_out's length is max_rows.
    void Plan(lcpp_stream_t stream, BufferView<uint32_t> temp_storage, BufferView<const int32_t> experts,
              BufferView<int32_t> expert_starts_out, BufferView<int32_t> row_of_out, BufferView<int32_t> pair_of_out,
              uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, uint32_t row_align = 1)
    {
        detail::require(experts.size() >= num_tokens * top_k && row_of_out.size() >= num_tokens * top_k &&
                            expert_starts_out.size() >= uint64_t(num_experts) + 1,
                        "Plan: a view is too short");
        detail::check(lcpp_dispatch_plan(temp_storage.data(), detail::temp_bytes(temp_storage), experts.data(),
                                         expert_starts_out.data(), row_of_out.data(), pair_of_out.data(), num_tokens,
                                         top_k, num_experts, row_align, pair_of_out.size(), stream),
                      "Plan");
    }

    /// lcpp_dispatch_gather: token rows to their experts' rows.
    void Gather(lcpp_stream_t stream, ConstRowsView x, BufferView<const int32_t> row_of,
                BufferView<const int32_t> pair_of, BufferView<const int32_t> expert_starts, RowsView rows_out,
                uint64_t num_tokens, uint32_t top_k, uint32_t num_experts)
    {
        detail::require_rows(x.rows >= num_tokens && rows_out.rows >= pair_of.size() &&
                             rows_out.columns >= x.columns && rows_out.dtype == x.dtype);
        detail::require(row_of.size() >= num_tokens * top_k && expert_starts.size() >= uint64_t(num_experts) + 1,
                        "Gather: a view is too short");
        detail::check(lcpp_dispatch_gather(x.ptr, x.stride, row_of.data(), pair_of.data(), expert_starts.data(),
                                           rows_out.ptr, rows_out.stride, num_tokens, top_k, num_experts,
                                           pair_of.size(), x.columns, x.dtype, stream),
                      "Gather");
    }

    /// lcpp_dispatch_combine: sums of the tokens' rows; an empty `weights` view: weights of 1.
    void Combine(lcpp_stream_t stream, ConstRowsView rows, BufferView<const int32_t> row_of,
                 BufferView<const float> weights, RowsView out, uint64_t num_tokens, uint32_t top_k)
    {
        detail::require_rows(out.rows >= num_tokens && rows.columns >= out.columns && rows.dtype == out.dtype);
        detail::require(row_of.size() >= num_tokens * top_k && (!weights.data() || weights.size() >= num_tokens * top_k),
                        "Combine: a view is too short");
        detail::check(lcpp_dispatch_combine(rows.ptr, rows.stride, row_of.data(), weights.data(), out.ptr, out.stride,
                                            num_tokens, top_k, rows.rows, out.columns, out.dtype, stream),
                      "Combine");
    }

    /// lcpp_dispatch_combine_backward: gradients of Combine with weights.
    void CombineBackward(lcpp_stream_t stream, ConstRowsView grad_out, ConstRowsView rows,
                         BufferView<const int32_t> row_of, BufferView<const int32_t> pair_of,
                         BufferView<const int32_t> expert_starts, BufferView<const float> weights,
                         RowsView grad_rows_out, BufferView<float> grad_weights_out, uint64_t num_tokens,
                         uint32_t top_k, uint32_t num_experts)
    {
        detail::require_rows(grad_out.rows >= num_tokens && rows.rows >= pair_of.size() &&
                             grad_rows_out.rows >= pair_of.size() && rows.columns >= grad_out.columns &&
                             grad_rows_out.columns >= grad_out.columns && rows.dtype == grad_out.dtype &&
                             grad_rows_out.dtype == grad_out.dtype);
        detail::require(row_of.size() >= num_tokens * top_k && weights.size() >= num_tokens * top_k &&
                            grad_weights_out.size() >= num_tokens * top_k &&
                            expert_starts.size() >= uint64_t(num_experts) + 1,
                        "CombineBackward: a view is too short");
        detail::check(lcpp_dispatch_combine_backward(grad_out.ptr, grad_out.stride, rows.ptr, rows.stride,
                                                     row_of.data(), pair_of.data(), expert_starts.data(),
                                                     weights.data(), grad_rows_out.ptr, grad_rows_out.stride,
                                                     grad_weights_out.data(), num_tokens, top_k, num_experts,
                                                     pair_of.size(), grad_out.columns, grad_out.dtype, stream),
                      "CombineBackward");
    }
};

}  // namespace lcpp_b200

#endif /* LCPP_B200_MODEL_HPP */
