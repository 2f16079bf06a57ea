// C++ caller of the paged cache's classes in include/lcpp_b200_model.hpp: tokens
// turned and written to their slots, attention over the pages with scores, the
// lightest tokens evicted and the pages given back, checked against host loops in
// 64 bits.  Built and run by tests/test_cache_ops_cpp.py on a GPU box; also compiled
// (not run) on the CPU.  Prints "OK <checks>" and exits 0 on success.
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
        CHECK(cudaMemset(p, 0, std::max<size_t>(count, 1) * sizeof(T)) == cudaSuccess);
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
    HeadsView heads(uint32_t heads, uint32_t dim) const { return {p, n / heads / dim, heads, dim, LCPP_F32}; }
    std::vector<T> download() const
    {
        std::vector<T> h(n);
        CHECK(cudaDeviceSynchronize() == cudaSuccess);
        CHECK(cudaMemcpy(h.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess);
        return h;
    }
};

bool near(double a, double b, double scale) { return std::abs(a - b) <= 3e-5 * scale + 1e-7; }

void run(lcpp_stream_t s)
{
    std::mt19937 rng(3);
    std::normal_distribution<float> normal;
    const auto draw = [&](size_t n) {
        std::vector<float> v(n);
        for (auto& x : v) x = normal(rng);
        return v;
    };
    // two requests of 21 and 9 tokens in pages of 8
    const uint32_t heads = 4, kv = 2, dim = 12, rotary = 8, pages = 7, block = 8, width = 3, tokens = 30;
    const std::vector<int32_t> table{5, 1, 4, 2, 6, -1}, lens{21, 9};
    std::vector<int64_t> slots;
    std::vector<int32_t> positions;
    for (int r = 0; r < 2; ++r)
        for (int t = 0; t < lens[r]; ++t) {
            slots.push_back(table[r * width + t / block] * block + t % block);
            positions.push_back(t);
        }
    std::vector<double> f(rotary / 2);
    DeviceRotary::Frequencies(f.data(), rotary, 100.0);
    CHECK(f[0] == 1.0 && std::abs(f[1] - std::pow(100.0, -0.25)) < 1e-15);
    const auto q = draw(tokens * heads * dim), k = draw(tokens * kv * dim), v = draw(tokens * kv * dim);
    DeviceArray<float> d_q(q), d_k(k), d_v(v), d_turned(q.size()), d_keys(pages * block * kv * dim),
        d_values(d_keys.n), d_scores(pages * block), d_scores_out(pages * block);
    DeviceArray<int64_t> d_slots(slots);
    DeviceArray<int32_t> d_positions(positions), d_where(pages * block), d_table(table), d_lens(lens);
    DeviceArray<double> d_f(f);
    lcpp_kv_cache cache{d_keys.p, d_values.p, block * kv * dim, kv * dim, dim, pages, block, kv, dim, LCPP_F32};
    Rotation rotation;
    rotation.positions = d_positions.in();
    rotation.frequencies = d_f.in();
    DeviceRotary().Append(s, d_q.heads(heads, dim), d_k.heads(kv, dim), d_v.heads(kv, dim), d_turned.heads(heads, dim),
                          cache, d_slots.in(), rotation, tokens, d_where.view(), d_scores.view());
    const auto turned = d_turned.download(), keys = d_keys.download(), values = d_values.download();
    const auto turn = [&](const float* x, int position, int c) {  // column c of a head
        if (c >= int(rotary)) return double(x[c]);
        const int i = c % (rotary / 2), other = c < int(rotary / 2) ? c + rotary / 2 : c - rotary / 2;
        const double a = position * f[i];
        return x[c] * std::cos(a) + (c < int(rotary / 2) ? -1 : 1) * x[other] * std::sin(a);
    };
    for (uint32_t t = 0; t < tokens; ++t)
        for (uint32_t c = 0; c < dim; ++c) {
            for (uint32_t h = 0; h < heads; ++h)
                CHECK(near(turned[(t * heads + h) * dim + c], turn(&q[(t * heads + h) * dim], positions[t], c), 4));
            for (uint32_t h = 0; h < kv; ++h) {
                CHECK(near(keys[(slots[t] * kv + h) * dim + c], turn(&k[(t * kv + h) * dim], positions[t], c), 4));
                CHECK(values[(slots[t] * kv + h) * dim + c] == v[(t * kv + h) * dim + c]);
            }
        }
    // the gradient undoes the turn
    DeviceArray<float> d_back(q.size());
    DeviceRotary().Backward(s, d_turned.heads(heads, dim), {}, d_back.heads(heads, dim), {}, rotation, tokens);
    const auto back = d_back.download();
    for (size_t i = 0; i < q.size(); ++i) CHECK(near(back[i], q[i], 4));

    // the last tokens' attention
    std::vector<float> last(2 * heads * dim);
    for (int r = 0; r < 2; ++r)
        std::copy_n(&turned[(r ? 29 : 20) * heads * dim], heads * dim, &last[r * heads * dim]);
    DeviceArray<float> d_last(last), d_out(last.size()), d_lse(2 * heads);
    DeviceArray<uint32_t> temp(bytes_to_uint_count(
        DevicePagedAttention::GetTempStorageBytes(2, heads, kv, dim, pages * block)));
    lcpp_paged_attention_args a{};
    a.cache = cache;
    a.q = d_last.p;
    a.out = d_out.p;
    a.q_request_stride = a.out_request_stride = heads * dim;
    a.q_head_stride = a.out_head_stride = dim;
    a.block_table = d_table.p;
    a.table_stride = a.table_width = width;
    a.num_requests = 2;
    a.seq_lens = d_lens.p;
    a.num_heads = heads;
    a.scale = 0.3f;
    a.lse_out = d_lse.p;
    a.slot_scores = d_scores.p;
    a.slot_scores_out = d_scores_out.p;
    a.score_decay = 1.f;
    DevicePagedAttention().Decode(s, temp.view(), a);
    const auto out = d_out.download(), lse = d_lse.download(), scores = d_scores_out.download();
    std::vector<double> mass(pages * block);
    for (int r = 0, first = 0; r < 2; first += lens[r++])
        for (uint32_t h = 0; h < heads; ++h) {
            std::vector<double> x(lens[r]), o(dim), size(dim);
            double top = -1e300, sum = 0;
            for (int t = 0; t < lens[r]; ++t) {
                for (uint32_t c = 0; c < dim; ++c)
                    x[t] += 0.3 * last[(r * heads + h) * dim + c] * keys[(slots[first + t] * kv + h / 2) * dim + c];
                top = std::max(top, x[t]);
            }
            for (double e : x) sum += std::exp(e - top);
            for (int t = 0; t < lens[r]; ++t) {
                const double share = std::exp(x[t] - top) / sum;
                mass[slots[first + t]] += share;
                for (uint32_t c = 0; c < dim; ++c) {
                    o[c] += share * values[(slots[first + t] * kv + h / 2) * dim + c];
                    size[c] += share * std::abs(values[(slots[first + t] * kv + h / 2) * dim + c]);
                }
            }
            CHECK(near(lse[r * heads + h], top + std::log(sum), 1 + std::abs(top)));
            for (uint32_t c = 0; c < dim; ++c) CHECK(near(out[(r * heads + h) * dim + c], o[c], size[c]));
        }
    for (int64_t slot : slots) CHECK(near(scores[slot], mass[slot], mass[slot]));

    // the longer request keeps its first token, its last three and the heaviest of the others
    DeviceArray<int32_t> d_cut(2), d_gone(2), d_counts(2), d_free(std::vector<int32_t>{9, 9, 9, 9, 9, 0, 3}),
        d_used(std::vector<int32_t>{5}), d_used_out(1);
    DeviceArray<int64_t> d_moves(2 * 12 * 2);
    lcpp_cache_evict_args e{};
    e.seq_lens = d_lens.p;
    e.block_table = d_table.p;
    e.table_stride = e.table_width = width;
    e.num_requests = 2;
    e.num_pages = pages;
    e.block_size = block;
    e.slot_scores = d_scores_out.p;
    e.slot_positions = d_where.p;
    e.budget = 12;
    e.trigger = 15;
    e.keep_first = 1;
    e.keep_recent = 3;
    e.max_moves = 12;
    e.seq_lens_out = d_cut.p;
    e.evicted_out = d_gone.p;
    e.move_counts_out = d_counts.p;
    e.moves_out = d_moves.p;
    e.moves_stride = 12;
    e.free_blocks = d_free.p;
    e.free_used = d_used.p;
    e.free_used_out = d_used_out.p;
    e.num_free = 7;
    DeviceCacheEviction().Plan(s, e);
    const auto moves = d_moves.download();
    std::vector<int> order(21);
    for (int t = 0; t < 21; ++t) order[t] = t;
    const auto weight = [&](int t) { return t < 1 || t >= 18 ? 1e30f : scores[slots[t]]; };
    std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return weight(i) > weight(j); });
    std::vector<bool> kept(21);
    for (int i = 0; i < 12; ++i) kept[order[i]] = true;
    size_t n = 0;
    for (int hole = 0, filler = 12; hole < 12; ++hole) {
        if (kept[hole]) continue;
        while (!kept[filler]) ++filler;
        CHECK(moves[2 * n] == slots[filler] && moves[2 * n + 1] == slots[hole]);
        ++filler, ++n;
    }
    CHECK((d_counts.download() == std::vector<int32_t>{int32_t(n), 0}));
    CHECK((d_cut.download() == std::vector<int32_t>{12, 9}) && (d_gone.download() == std::vector<int32_t>{9, 0}));
    CHECK(d_used_out.download()[0] == 4 && d_free.download()[4] == 4);  // the third page came back
    DeviceCacheEviction().Move(s, cache, d_moves.in(), 12, 12, d_counts.in(), 2, d_scores_out.view(), d_where.view());
    const auto keys_after = d_keys.download(), scores_after = d_scores_out.download();
    const auto where = d_where.download();
    for (size_t i = 0; i < n; ++i) {
        const int64_t from = moves[2 * i], to = moves[2 * i + 1];
        for (uint32_t c = 0; c < kv * dim; ++c) CHECK(keys_after[to * kv * dim + c] == keys[from * kv * dim + c]);
        CHECK(scores_after[to] == scores[from] && slots[where[to]] == from);
    }

    bool threw = false;
    try {
        DeviceRotary().Forward(s, d_q.heads(heads, dim), {}, d_k.heads(kv, dim), {}, rotation, tokens);
    } catch (const Error& error) {
        threw = error.status() == LCPP_ERR_INVALID_ARG;
    }
    CHECK(threw);
}

}  // namespace

int main()
{
    cudaStream_t stream;
    CHECK(cudaStreamCreate(&stream) == cudaSuccess);
    run(reinterpret_cast<lcpp_stream_t>(stream));
    CHECK(cudaStreamDestroy(stream) == cudaSuccess);
    std::printf("OK %d\n", g_checks);
    return 0;
}
