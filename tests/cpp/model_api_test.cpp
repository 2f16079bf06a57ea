// C++ caller of include/lcpp_b200_model.hpp: one step of a paged, sparsely
// routed model (block table, router, dispatch, combine, the gradients) with
// float rows, checked against host loops.  Built and run by
// tests/test_model_step_cpp.py on a GPU box; also compiled (not run) on the CPU.
// Prints "OK <checks>" and exits 0 on success.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "lcpp_b200_model.hpp"

using namespace lcpp_b200;

namespace {

int g_checks = 0;

#define CHECK(cond)                                                                  \
    do {                                                                             \
        ++g_checks;                                                                  \
        if (!(cond)) {                                                               \
            std::fprintf(stderr, "FAILED %s at %s:%d\n", #cond, __FILE__, __LINE__); \
            std::exit(1);                                                            \
        }                                                                            \
    } while (0)

template <typename T>
struct DeviceArray {
    T* p = nullptr;
    size_t n = 0;
    explicit DeviceArray(size_t count) : n(count)
    {
        CHECK(cudaMalloc(&p, std::max<size_t>(count, 1) * sizeof(T)) == cudaSuccess);
    }
    explicit DeviceArray(const std::vector<T>& h) : DeviceArray(h.size())
    {
        CHECK(cudaMemcpy(p, h.data(), n * sizeof(T), cudaMemcpyHostToDevice) == cudaSuccess);
    }
    DeviceArray(const DeviceArray&) = delete;
    DeviceArray& operator=(const DeviceArray&) = delete;
    ~DeviceArray() { cudaFree(p); }
    BufferView<T> view() const { return {p, n}; }
    BufferView<const T> in() const { return {p, n}; }
    RowsView rows(uint64_t columns) const { return {p, n / columns, columns, LCPP_F32}; }
    std::vector<T> download() const
    {
        std::vector<T> h(n);
        CHECK(cudaMemcpy(h.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess);
        return h;
    }
};

std::vector<float> normal(std::mt19937& rng, size_t n)
{
    std::normal_distribution<float> d;
    std::vector<float> v(n);
    for (auto& x : v) x = d(rng);
    return v;
}

bool near(double a, double b, double scale) { return std::abs(a - b) <= 1e-5 * scale + 1e-7; }

void step(lcpp_stream_t s)
{
    std::mt19937 rng(7);
    // three requests: a prompt of 20 tokens, a decode on 30, one without room in its row
    const int block = 16, width = 4, capacity = 32;
    const std::vector<int32_t> context{0, 30, 60}, fresh{20, 1, 9};
    std::vector<int32_t> table(3 * width, -1);
    table[1 * width] = 40, table[1 * width + 1] = 41;
    for (int i = 0; i < 4; ++i) table[2 * width + i] = 50 + i;
    DeviceArray<int32_t> d_context(context), d_fresh(fresh), d_table(table), d_free(std::vector<int32_t>{7, 5, 9}),
        d_used(1), d_seq(3), d_starts(4), d_positions(capacity), d_request(capacity);
    DeviceArray<int64_t> d_slots(capacity);
    DeviceArray<uint32_t> temp(bytes_to_uint_count(std::max(
        {DeviceBlockTable::GetTempStorageBytes(3, capacity), DeviceRouter::GetTempStorageBytes(capacity, 8),
         DeviceDispatch::GetTempStorageBytes(capacity, 2, 8)})));
    lcpp_block_table_args args{};
    args.context_lens = d_context.p;
    args.new_lens = d_fresh.p;
    args.block_table = d_table.p;
    args.table_stride = width;
    args.table_width = width;
    args.num_requests = 3;
    args.block_size = block;
    args.num_free = 3;
    args.free_blocks = d_free.p;
    args.free_used_out = d_used.p;
    args.seq_lens_out = d_seq.p;
    args.query_starts_out = d_starts.p;
    args.slots_out = d_slots.p;
    args.positions_out = d_positions.p;
    args.token_request_out = d_request.p;
    args.max_tokens = capacity;
    DeviceBlockTable().Extend(s, temp.view(), args);
    const auto slots = d_slots.download();
    const auto request = d_request.download();
    for (int t = 0; t < capacity; ++t) {
        if (t < 20) CHECK(slots[t] == (t < 16 ? 7 : 5) * block + t % block && request[t] == 0);
        else if (t == 20) CHECK(slots[t] == 41 * block + 14 && request[t] == 1);
        else CHECK(slots[t] == -1 && request[t] == -1);
    }
    CHECK((d_seq.download() == std::vector<int32_t>{20, 31, 60}));
    CHECK((d_starts.download() == std::vector<int32_t>{0, 20, 21, 30}));
    CHECK(d_used.download()[0] == 2);

    // the marked tokens are not routed
    const uint32_t experts = 8, k = 2, hidden = 12, align = 4;
    const lcpp_router_config config{experts, k, LCPP_SCORE_SOFTMAX, 1, 1.f, 0.5f};
    const auto logits = normal(rng, capacity * experts);
    DeviceArray<float> d_logits(logits), d_weights(capacity * k), d_loss(1);
    DeviceArray<int32_t> d_experts(capacity * k), d_counts(experts), d_routed(1);
    DeviceRouter().Forward(s, temp.view(), d_logits.rows(experts), {}, d_request.in(), d_weights.view(),
                           d_experts.view(), d_counts.view(), d_routed.view(), d_loss.view(), capacity, config);
    const auto chosen = d_experts.download();
    const auto weights = d_weights.download();
    CHECK(d_routed.download()[0] == 21);
    for (int t = 0; t < capacity; ++t) {
        const float* x = logits.data() + t * experts;
        if (t >= 21) {
            CHECK(chosen[t * k] == -1 && chosen[t * k + 1] == -1 && weights[t * k] == 0.f);
            continue;
        }
        const int first = int(std::max_element(x, x + experts) - x);
        CHECK(chosen[t * k] == first);
        const double a = std::exp(double(x[chosen[t * k + 1]] - x[first]));
        CHECK(near(weights[t * k], 1 / (1 + a), 1) && near(weights[t * k + 1], a / (1 + a), 1));
    }

    // rows there and back; the experts double them
    const uint64_t max_rows = DeviceDispatch::MaxRows(capacity, k, experts, align);
    DeviceArray<int32_t> d_expert_starts(experts + 1), d_row_of(capacity * k), d_pair_of(max_rows);
    const auto x = normal(rng, capacity * hidden);
    DeviceArray<float> d_x(x), d_rows(max_rows * hidden), d_out(capacity * hidden);
    DeviceDispatch d;
    d.Plan(s, temp.view(), d_experts.in(), d_expert_starts.view(), d_row_of.view(), d_pair_of.view(), capacity, k,
           experts, align);
    d.Gather(s, d_x.rows(hidden), d_row_of.in(), d_pair_of.in(), d_expert_starts.in(), d_rows.rows(hidden), capacity, k,
             experts);
    const auto starts = d_expert_starts.download();
    const auto row_of = d_row_of.download();
    const auto pair_of = d_pair_of.download();
    auto rows = d_rows.download();
    for (uint32_t e = 0; e < experts; ++e) CHECK(starts[e] % align == 0);
    for (int r = 0; r < starts[experts]; ++r)
        for (uint32_t h = 0; h < hidden; ++h)
            CHECK(rows[r * hidden + h] == (pair_of[r] < 0 ? 0.f : x[pair_of[r] / k * hidden + h]));
    DeviceArray<float> d_doubled(max_rows * hidden);
    for (auto& v : rows) v *= 2;
    CHECK(cudaMemcpy(d_doubled.p, rows.data(), rows.size() * 4, cudaMemcpyHostToDevice) == cudaSuccess);
    d.Combine(s, d_doubled.rows(hidden), d_row_of.in(), d_weights.in(), d_out.rows(hidden), capacity, k);
    const auto out = d_out.download();
    for (int t = 0; t < capacity; ++t)
        for (uint32_t h = 0; h < hidden; ++h)
            CHECK(near(out[t * hidden + h], t < 21 ? 2 * double(x[t * hidden + h]) : 0.0, 4));

    // gradients: rows get w dy, weights <dy, row>, logits sum to zero over the experts
    const auto dy = normal(rng, capacity * hidden);
    DeviceArray<float> d_dy(dy), d_grad_rows(max_rows * hidden), d_grad_weights(capacity * k),
        d_grad_logits(capacity * experts), d_one(std::vector<float>{1.f});
    d.CombineBackward(s, d_dy.rows(hidden), d_doubled.rows(hidden), d_row_of.in(), d_pair_of.in(),
                      d_expert_starts.in(), d_weights.in(), d_grad_rows.rows(hidden), d_grad_weights.view(), capacity,
                      k, experts);
    const auto grad_rows = d_grad_rows.download();
    const auto grad_weights = d_grad_weights.download();
    for (int p = 0; p < 21 * int(k); ++p) {
        double dot = 0, size = 0;
        for (uint32_t h = 0; h < hidden; ++h) {
            CHECK(near(grad_rows[row_of[p] * hidden + h], double(weights[p]) * dy[p / k * hidden + h], 4));
            dot += 2.0 * x[p / k * hidden + h] * dy[p / k * hidden + h];
            size += std::abs(2.0 * x[p / k * hidden + h] * dy[p / k * hidden + h]);
        }
        CHECK(near(grad_weights[p], dot, size));
    }
    DeviceRouter().Backward(s, d_logits.rows(experts), d_experts.in(), d_counts.in(), d_routed.in(),
                            d_grad_weights.in(), d_one.in(), d_grad_logits.rows(experts), capacity, config);
    const auto grad_logits = d_grad_logits.download();
    for (int t = 0; t < capacity; ++t) {
        double sum = 0, size = 0;
        for (uint32_t e = 0; e < experts; ++e) {
            sum += grad_logits[t * experts + e];
            size += std::abs(grad_logits[t * experts + e]);
        }
        CHECK(t < 21 ? size > 0 && near(sum, 0, size) : size == 0);
    }

    bool threw = false;
    try {
        d.Combine(s, d_rows.rows(hidden), d_row_of.in(), {}, {d_out.p, 4, hidden, LCPP_F32}, capacity, k);
    } catch (const Error& e) {
        threw = e.status() == LCPP_ERR_INVALID_ARG;
    }
    CHECK(threw);
}

}  // namespace

int main()
{
    cudaStream_t stream;
    CHECK(cudaStreamCreate(&stream) == cudaSuccess);
    step(reinterpret_cast<lcpp_stream_t>(stream));
    CHECK(cudaStreamDestroy(stream) == cudaSuccess);
    std::printf("OK %d\n", g_checks);
    return 0;
}
