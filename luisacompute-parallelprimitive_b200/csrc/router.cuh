// router.cuh -- DeviceRouter's kernels (include/lcpp_b200_model.h).
//
// A row of logits is spread over LANES lanes, C elements each, and stays in
// registers from its one read to its last use; a warp works on 32 / LANES rows
// at a time.  Element i of lane l is expert ((i / V) * LANES + l) * V + i % V,
// V elements being 16 bytes, so that aligned rows are read in 16-byte vectors
// and a row's lanes read consecutive ones.
//
// Choice.  Each biased logit becomes one 32-bit word whose unsigned order is
// (value, lower expert first): the float's order-preserving bits with their
// low IB bits replaced by the complement of the expert, IB = log2(LANES * C).
// The words of a row differ, so the next largest below `best` is the maximum
// of (word - best) mod 2^32: words below `best` wrap to the top of the range
// and those already taken stay at its bottom, and nothing has to be marked as
// taken.  One round is C subtract-and-max steps and log2(LANES) shuffles.
//
// The dropped bits matter only where two of the first top_k + 1 words agree in
// all kept bits and their logits do not.  16-bit logits without a bias have no
// such bits (at most 19 bits of a float are in use); for the others a row whose
// choice could depend on them is chosen again from the full values (rows of
// continuous 32-bit logits: about one in a thousand at 256 experts).
#pragma once

#include "model.cuh"

namespace lcpp {
namespace router {

using namespace lcpp::model;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr float kNegInf = -INFINITY;
// Under this largest logit every sigmoid of the row equals exp(logit) to 32
// bits and their sum may underflow, so shares are taken as a softmax instead.
constexpr float kDeepSigmoid = -60.f;

struct Params {
    const void* logits;
    uint64_t stride;
    const float* bias;
    const int32_t* token_request;
    float* weights;
    int32_t* experts;
    int32_t* counts;
    int32_t* num_routed;
    float* loss;
    uint64_t tokens;
    uint32_t num_experts;
    uint32_t top_k;
    int32_t renormalize;
    float weight_scale;
    float loss_coef;
    uint32_t aligned;
    // temp storage, cleared before a launch of several blocks
    uint32_t* ctrl;                  // [0] blocks done, [1] error word, [2] a share was not finite, [3] tokens routed
    unsigned long long* share_total; // [num_experts] sums of shares in units of 2^-32
    uint32_t* count_total;           // [num_experts]
};

struct BackParams {
    const void* logits;
    uint64_t stride;
    const int32_t* experts;
    const int32_t* counts;
    const int32_t* num_routed;
    const float* grad_weights;
    const float* grad_loss;
    void* grad_logits;
    uint64_t grad_stride;
    uint64_t tokens;
    uint32_t num_experts;
    uint32_t top_k;
    int32_t renormalize;
    float weight_scale;
    float loss_coef;
    uint32_t aligned;
};

constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }
constexpr int ceil_log2(int v) { return log2_of(2 * v - 1); }

template <typename T, int LANES, int C>
struct Tile {
    static constexpr int kV = Vec<T>::kN;
    static constexpr int kRows = kWarp / LANES;  // rows of a warp
    static constexpr int kSpan = LANES * C;      // experts that fit
    static constexpr int kIndexBits = ceil_log2(kSpan);
    static_assert(C % kV == 0, "whole vectors");

    static __device__ __forceinline__ uint32_t expert(int lane, int i)
    {
        return uint32_t(((i / kV) * LANES + lane) * kV + i % kV);
    }

    // The row's elements of this lane; -inf past num_experts.  `rest` and the
    // row must be valid memory only for experts below num_experts.
    static __device__ __forceinline__ void load(const T* row, int lane, uint32_t n, bool aligned, float (&x)[C])
    {
#pragma unroll
        for (int v = 0; v < C / kV; ++v) {
            const uint32_t e0 = expert(lane, v * kV);
            if (aligned && e0 + kV <= n) {
                float part[kV];
                Vec<T>::unpack(*reinterpret_cast<const uint4*>(row + e0), part);
#pragma unroll
                for (int i = 0; i < kV; ++i) x[v * kV + i] = part[i];
            } else {
#pragma unroll
                for (int i = 0; i < kV; ++i) x[v * kV + i] = e0 + i < n ? to_float(row[e0 + i]) : kNegInf;
            }
        }
    }
};

template <int LANES, typename V, typename Op>
__device__ __forceinline__ V row_all(V v, Op op)
{
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) v = op(v, __shfl_xor_sync(~0u, v, d));
    return v;
}

struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
    __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
struct Add {
    __device__ float operator()(float a, float b) const { return a + b; }
};
struct Or {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a | b; }
};

// Order-preserving bits of f; both zeros alike, every NaN above +inf.
__device__ __forceinline__ uint32_t ordered(float f)
{
    const uint32_t b = __float_as_uint(f + 0.f);  // -0 + 0 = +0; a NaN becomes the positive one
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

// x (in place) becomes the row's shares s / sum s; returns the factor that a
// score is to be multiplied with to give its share, and the row's largest
// logit in `top`.
template <bool SIGMOID, int LANES, int C>
__device__ __forceinline__ void shares(float (&x)[C], float& top, float& sum)
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < C; ++i) m = fmaxf(m, x[i]);
    m = row_all<LANES>(m, Max{});
    float z = 0.f;
    if (SIGMOID && m >= kDeepSigmoid) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            x[i] = sigmoid(x[i]);
            z += x[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            x[i] = __expf(x[i] - m);
            z += x[i];
        }
    }
    top = m;
    sum = row_all<LANES>(z, Add{});
}

// The score of a chosen logit before any division, on the scale `shares` used.
template <bool SIGMOID>
__device__ __forceinline__ float score_of(float x, float top)
{
    return SIGMOID && top >= kDeepSigmoid ? sigmoid(x) : __expf(x - top);
}

// The exact choice of a warp's rows from the full values, one composite word
// {ordered value, complement of the expert} per element: rare, so it reads the
// logits again instead of keeping them.
template <typename T, int LANES, int C>
__device__ __noinline__ void choose_exactly(const T* row, const float* bias, int lane, uint32_t n, uint32_t k,
                                            uint32_t* chosen)
{
    using L = Tile<T, LANES, C>;
    uint64_t last = ~0ull;
    for (uint32_t j = 0; j < k; ++j) {
        uint64_t best = 0;
        for (int i = 0; i < C; ++i) {
            const uint32_t e = L::expert(lane, i);
            if (e >= n) continue;
            const float x = to_float(row[e]);
            const float f = bias ? x + bias[e] : x;
            if (x == kNegInf || f == kNegInf) continue;
            const uint64_t word = uint64_t(ordered(f)) << 32 | (0xffffffffu - e);
            if (word < last && word > best) best = word;
        }
        best = row_all<LANES>(best, Max{});
        if (lane == 0) chosen[j] = best ? 0xffffffffu - uint32_t(best) : ~0u;
        last = best;
    }
    __syncwarp();
}

// A block's share of an expert, at most 2^31 tokens, in units of 2^-32: whole
// numbers add up to the same total in any order, and 2^-32 is far below the
// rounding of the 32-bit sums that go in.
constexpr double kShareUnit = 4294967296.0;

// Writes the counts and, from sum_e share_e * count_e, the loss.
template <typename Share, typename Count>
__device__ void finish(const Params& p, uint32_t routed_tokens, bool broken, double* scratch, Share share, Count count)
{
    double dot = 0.0;
    for (uint32_t e = threadIdx.x; e < p.num_experts; e += kThreads) {
        const uint32_t c = count(e);
        p.counts[e] = int32_t(c);
        dot += share(e) * double(c);
    }
    scratch[threadIdx.x] = dot;
    __syncthreads();
    for (int d = kThreads / 2; d > 0; d /= 2) {
        if (threadIdx.x < unsigned(d)) scratch[threadIdx.x] += scratch[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double routed = routed_tokens;
        *p.num_routed = int32_t(routed_tokens);
        float loss = 0.f;
        if (routed_tokens) loss = float(double(p.loss_coef) * p.num_experts * scratch[0] / (p.top_k * routed * routed));
        *p.loss = broken ? NAN : loss;
    }
}

template <typename T, int LANES, int C, bool SIGMOID, bool BIAS>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Params p)
{
    using L = Tile<T, LANES, C>;
    constexpr uint32_t kMask = (1u << L::kIndexBits) - 1;
    constexpr bool kExact = sizeof(T) == 2 && !BIAS;
    const uint32_t n = p.num_experts, k = p.top_k;
    const int warp = threadIdx.x / kWarp, wl = threadIdx.x % kWarp, lane = wl % LANES, sub = wl / LANES;

    extern __shared__ float dynamic[];
    float* share_sum = dynamic;                                               // [kWarps][n]
    uint32_t* count = reinterpret_cast<uint32_t*>(share_sum + kWarps * n);    // [n]
    float* bias = reinterpret_cast<float*>(count + n);                        // [n]
    __shared__ uint32_t chosen_all[kWarps][L::kRows][LCPP_MAX_TOP_K];
    __shared__ float value_all[kWarps][L::kRows][LCPP_MAX_TOP_K];
    __shared__ double scratch[kThreads];
    __shared__ uint32_t routed_block;
    __shared__ bool is_last;
    uint32_t* chosen = chosen_all[warp][sub];
    float* value = value_all[warp][sub];
    for (uint32_t e = threadIdx.x; e < n; e += kThreads) {
        count[e] = 0;
        if (BIAS) bias[e] = p.bias[e];
    }
    if (threadIdx.x == 0) routed_block = 0;
    __syncthreads();

    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    int routed = 0;

    const uint64_t step = uint64_t(gridDim.x) * kWarps * L::kRows;
    for (uint64_t t0 = (uint64_t(blockIdx.x) * kWarps + warp) * L::kRows; t0 < p.tokens; t0 += step) {
        const uint64_t t = t0 + sub;
        const bool inside = t < p.tokens;
        const bool wanted = inside && (!p.token_request || p.token_request[t] >= 0);
        const T* row = static_cast<const T*>(p.logits) + (inside ? t : t0) * p.stride;
        float x[C];
        L::load(row, lane, n, p.aligned, x);

        uint32_t word[C], low = 0;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const uint32_t e = L::expert(lane, i);
            float f = x[i];
            if (BIAS) f += e < n ? bias[e] : 0.f;
            const uint32_t o = ordered(f);
            if (!kExact) low |= __float_as_uint(f);
            word[i] = x[i] == kNegInf || f == kNegInf ? 0u : (o & ~kMask) | (kMask - e);
        }
        // choice
        uint32_t best = 0, found = 0;
        bool unsure = false;
        const uint32_t rounds = kExact ? k : min(k + 1, n);
        for (uint32_t j = 0; j < rounds; ++j) {
            uint32_t next = word[0] - best;
#pragma unroll
            for (int i = 1; i < C; ++i) next = max(next, word[i] - best);
            next = row_all<LANES>(next, Max{}) + best;
            if (j && best == 0) next = 0;
            if (!kExact) unsure |= next && j && (next & ~kMask) == (best & ~kMask);
            if (j < k) {
                found += next != 0;
                if (lane == 0) chosen[j] = next ? kMask - (next & kMask) : ~0u;
            }
            best = next;
        }
        __syncwarp();
        if (!kExact) {
            // logits whose dropped bits are all zero were compared in full
            low = row_all<LANES>(low & kMask, Or{});
            unsure = unsure && low;
            if (__any_sync(~0u, unsure)) choose_exactly<T, LANES, C>(row, BIAS ? bias : nullptr, lane, n, k, chosen);
        }
        const bool live = wanted && found;

        float top, sum;
        shares<SIGMOID, LANES>(x, top, sum);
        const float inv = live ? 1.f / sum : 0.f;
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] = live ? fmaf(x[i], inv, acc[i]) : acc[i];

        // weights of the chosen
        float most = kNegInf;
        for (uint32_t j = lane; j < k; j += LANES) {
            const uint32_t e = chosen[j];
            const float v = e < n ? to_float(row[e]) : kNegInf;
            value[j] = v;
            most = fmaxf(most, v);
        }
        if (p.renormalize) most = row_all<LANES>(most, Max{});
        else most = top;
        float total = 0.f;
        for (uint32_t j = lane; j < k; j += LANES) {
            const float s = chosen[j] < n ? score_of<SIGMOID>(value[j], most) : 0.f;
            value[j] = s;
            total += s;
        }
        float scale = p.weight_scale;
        if (p.renormalize) scale /= row_all<LANES>(total, Add{});
        else if (!SIGMOID) scale /= sum;
        else if (top < kDeepSigmoid) scale *= __expf(top);
        if (inside) {
            for (uint32_t j = lane; j < k; j += LANES) {
                const uint32_t e = live ? chosen[j] : ~0u;
                p.weights[t * k + j] = e < n ? value[j] * scale : 0.f;
                p.experts[t * k + j] = e < n ? int32_t(e) : -1;
                if (e < n) atomicAdd(count + e, 1u);
            }
        }
        routed += live && lane == 0;
        __syncwarp();
    }

    // the block's sums
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
        for (int d = LANES; d < kWarp; d *= 2) acc[i] += __shfl_xor_sync(~0u, acc[i], d);
        const uint32_t e = L::expert(lane, i);
        if (sub == 0 && e < n) share_sum[warp * n + e] = acc[i];
    }
    if (routed) atomicAdd(&routed_block, uint32_t(routed));
    __syncthreads();
    const auto block_share = [&](uint32_t e) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += share_sum[w * n + e];
        return sum;
    };
    if (gridDim.x == 1) {
        if (threadIdx.x == 0) p.ctrl[1] = 0;
        finish(p, routed_block, false, scratch, [&](uint32_t e) { return double(block_share(e)); },
               [&](uint32_t e) { return count[e]; });
        return;
    }
    for (uint32_t e = threadIdx.x; e < n; e += kThreads) {
        const float sum = block_share(e);
        if (!(sum < INFINITY)) atomicOr(p.ctrl + 2, 1u);
        else if (sum > 0.f) atomicAdd(p.share_total + e, (unsigned long long)(__double2ull_rn(double(sum) * kShareUnit)));
        if (count[e]) atomicAdd(p.count_total + e, count[e]);
    }
    if (threadIdx.x == 0 && routed_block) atomicAdd(p.ctrl + 3, routed_block);
    // the block that gets here last has everyone's sums
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) is_last = atomicAdd(p.ctrl, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    finish(p, __ldcg(p.ctrl + 3), __ldcg(p.ctrl + 2) != 0, scratch,
           [&](uint32_t e) { return double(__ldcg(p.share_total + e)) / kShareUnit; },
           [&](uint32_t e) { return __ldcg(p.count_total + e); });
}

template <typename T, int LANES, int C, bool SIGMOID, bool RENORM>
__global__ void __launch_bounds__(kThreads) backward_kernel(const BackParams p)
{
    // Softmax weights as they are: the chosen experts' slopes join the loss's
    // before the row's mean is taken off; else they are added afterwards.
    constexpr bool kJoined = !SIGMOID && !RENORM;
    using L = Tile<T, LANES, C>;
    const uint32_t n = p.num_experts, k = p.top_k;
    const int warp = threadIdx.x / kWarp, wl = threadIdx.x % kWarp, lane = wl % LANES, sub = wl / LANES;
    __shared__ float score_all[kWarps][L::kRows][LCPP_MAX_TOP_K], upstream_all[kWarps][L::kRows][LCPP_MAX_TOP_K];
    float* score = score_all[warp][sub];
    float* upstream = upstream_all[warp][sub];
    extern __shared__ float dynamic[];
    float* pull = dynamic;                                                            // [kSpan]
    float* extra = dynamic + L::kSpan * (1 + warp * L::kRows + sub);                  // [kSpan] of this row
    for (int e = wl; e < L::kSpan * L::kRows; e += kWarp) dynamic[L::kSpan * (1 + warp * L::kRows) + e] = 0.f;
    {
        // the loss's slope by an expert's share, grad_loss coef E counts / (k T'^2).
        // Only its differences between experts matter (the shares add up to 1),
        // so an even share of the counts is taken off first: what is left of a
        // balanced batch keeps its digits.
        const float routed = float(max(*p.num_routed, 1));
        const float scale = p.grad_loss ? *p.grad_loss * p.loss_coef * float(n) / (float(k) * routed * routed) : 0.f;
        const float even = float(k) * routed / float(n);
        for (int e = threadIdx.x; e < L::kSpan; e += kThreads)
            pull[e] = p.grad_loss && uint32_t(e) < n ? scale * (float(p.counts[e]) - even) : 0.f;
    }
    __syncthreads();

    const uint64_t step = uint64_t(gridDim.x) * kWarps * L::kRows;
    for (uint64_t t0 = (uint64_t(blockIdx.x) * kWarps + warp) * L::kRows; t0 < p.tokens; t0 += step) {
        const uint64_t t = t0 + sub;
        const bool inside = t < p.tokens;
        const uint64_t tt = inside ? t : t0;
        const T* row = static_cast<const T*>(p.logits) + tt * p.stride;
        T* out = static_cast<T*>(p.grad_logits) + tt * p.grad_stride;
        float x[C];
        L::load(row, lane, n, p.aligned & 1, x);
        float top, sum;
        shares<SIGMOID, LANES>(x, top, sum);
        const float inv = 1.f / sum;
        const bool deep = SIGMOID && top < kDeepSigmoid;

        const bool live = p.experts[tt * k] >= 0;
        // the chosen experts' scores and upstream gradients
        float most = top;
        if (RENORM) {
            most = kNegInf;
            for (uint32_t j = lane; j < k; j += LANES) {
                const uint32_t e = uint32_t(p.experts[tt * k + j]);
                if (e < n) most = fmaxf(most, to_float(row[e]));
            }
            most = row_all<LANES>(most, Max{});
        }
        float total = 0.f;
        for (uint32_t j = lane; j < k; j += LANES) {
            const uint32_t e = uint32_t(p.experts[tt * k + j]);
            const float s = e < n ? score_of<SIGMOID>(to_float(row[e]), most) : 0.f;
            score[j] = s;
            upstream[j] = p.grad_weights && e < n ? p.grad_weights[tt * k + j] : 0.f;
            total += s;
        }
        if (RENORM) total = row_all<LANES>(total, Add{});
        __syncwarp();
        // The expert that has most of the row's share, among the chosen: slopes
        // are taken relative to its own, so that the mean of a row that one
        // expert dominates is not the difference of two equal numbers.
        uint32_t lead = 0;
        for (uint32_t j = 1; j < k; ++j) lead = score[j] > score[lead] ? j : lead;
        const uint32_t lead_expert = uint32_t(p.experts[tt * k + lead]);
        const float pull0 = lead_expert < n ? pull[lead_expert] : 0.f, up0 = upstream[lead];
        // one addend per chosen expert
        const float c = p.weight_scale;
        for (uint32_t j = lane; j < k; j += LANES) {
            const uint32_t e = uint32_t(p.experts[tt * k + j]);
            if (e >= n) continue;
            const float s = score[j], g = upstream[j];
            float a = g;
            if (!kJoined) {
                const float slope = SIGMOID && !deep ? sigmoid(-to_float(row[e])) : 1.f;
                if (RENORM) {
                    // g_j - sum_i r_i g_i, as a sum of differences for the same reason
                    float apart = 0.f;
                    for (uint32_t i = 0; i < k; ++i) apart = fmaf(score[i], g - upstream[i], apart);
                    a = c * slope * (s / total) * (apart / total);
                } else {
                    a = c * g * slope * (deep ? s * __expf(top) : s);
                }
            }
            extra[e] = a;
        }
        __syncwarp();
        // every expert's part
        const auto slope_of = [&](uint32_t e) {
            const float h = pull[e] - pull0;
            return kJoined ? fmaf(c, extra[e] - up0, h) : h;
        };
        float mean = 0.f;
#pragma unroll
        for (int v = 0; v < C / L::kV; ++v) {
            const uint32_t e0 = L::expert(lane, v * L::kV);
#pragma unroll
            for (int i = 0; i < L::kV; ++i) mean = fmaf(x[v * L::kV + i] * inv, slope_of(e0 + i), mean);
        }
        mean = row_all<LANES>(mean, Add{});
#pragma unroll
        for (int v = 0; v < C / L::kV; ++v) {
            const uint32_t e0 = L::expert(lane, v * L::kV);
            float g[L::kV];
#pragma unroll
            for (int i = 0; i < L::kV; ++i) {
                const float s = x[v * L::kV + i];
                const float factor = SIGMOID && !deep ? 1.f - s : 1.f;
                const float d = fmaf(factor * s * inv, slope_of(e0 + i) - mean, kJoined ? 0.f : extra[e0 + i]);
                g[i] = live ? d : 0.f;
            }
            if (inside) {
                if ((p.aligned & 2) && e0 + L::kV <= n) {
                    *reinterpret_cast<uint4*>(out + e0) = Vec<T>::pack(g);
                } else {
#pragma unroll
                    for (int i = 0; i < L::kV; ++i)
                        if (e0 + i < n) out[e0 + i] = from_float<T>(g[i]);
                }
            }
        }
        __syncwarp();
        for (uint32_t j = lane; j < k; j += LANES) {
            const uint32_t e = uint32_t(p.experts[tt * k + j]);
            if (e < n) extra[e] = 0.f;
        }
        __syncwarp();
    }
}

// Temp storage: the control words, the share totals, the count totals.
constexpr size_t kShareOffset = kTempAlign;
inline size_t cleared_bytes(uint32_t experts) { return kShareOffset + size_t(experts) * 12; }

// Blocks for `tokens` rows: as many as are resident at once, fewer for few rows.
inline unsigned grid_for(const void* kernel, size_t smem, uint64_t tokens, int rows_per_block)
{
    const uint64_t most = uint64_t(device_sm_count()) * resident_blocks(kernel, kThreads, smem);
    return unsigned(std::max<uint64_t>(1, std::min(most, ceil_div(tokens, rows_per_block))));
}

template <typename T, int LANES, int C>
lcpp_status forward_shape(const Params& p, bool sigmoid, cudaStream_t s)
{
    const size_t smem = (size_t(kWarps) + 2) * p.num_experts * 4;
    void (*kernel)(Params) =
        sigmoid ? (p.bias ? forward_kernel<T, LANES, C, true, true> : forward_kernel<T, LANES, C, true, false>)
                : (p.bias ? forward_kernel<T, LANES, C, false, true> : forward_kernel<T, LANES, C, false, false>);
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, (size_t(kWarps) + 2) * LANES * C * 4);
    const unsigned grid = grid_for(f, smem, p.tokens, kWarps * kWarp / LANES);
    if (grid > 1) LCPP_CUDA_TRY(cudaMemsetAsync(p.ctrl, 0, cleared_bytes(p.num_experts), s));
    kernel<<<grid, kThreads, smem, s>>>(p);
    return launched();
}

template <typename T, int LANES, int C>
lcpp_status backward_shape(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    const size_t smem = size_t(LANES) * C * (1 + kWarps * (kWarp / LANES)) * 4;
    void (*kernel)(BackParams) =
        sigmoid ? (p.renormalize ? backward_kernel<T, LANES, C, true, true> : backward_kernel<T, LANES, C, true, false>)
                : (p.renormalize ? backward_kernel<T, LANES, C, false, true> : backward_kernel<T, LANES, C, false, false>);
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, smem);
    kernel<<<grid_for(f, smem, p.tokens, kWarps * kWarp / LANES), kThreads, smem, s>>>(p);
    return launched();
}

// The smallest shape that holds the experts.
template <typename T>
lcpp_status forward_rows(const Params& p, bool sigmoid, cudaStream_t s)
{
    const uint32_t n = p.num_experts;
    if (n <= 32) return forward_shape<T, 4, 8>(p, sigmoid, s);
    if (n <= 128) return forward_shape<T, 8, 16>(p, sigmoid, s);
    if (n <= 256) return forward_shape<T, 8, 32>(p, sigmoid, s);
    if (n <= 512) return forward_shape<T, 16, 32>(p, sigmoid, s);
    return forward_shape<T, 32, 32>(p, sigmoid, s);
}

template <typename T>
lcpp_status backward_rows(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    const uint32_t n = p.num_experts;
    if (n <= 32) return backward_shape<T, 4, 8>(p, sigmoid, s);
    if (n <= 128) return backward_shape<T, 8, 16>(p, sigmoid, s);
    if (n <= 256) return backward_shape<T, 8, 32>(p, sigmoid, s);
    if (n <= 512) return backward_shape<T, 16, 32>(p, sigmoid, s);
    return backward_shape<T, 32, 32>(p, sigmoid, s);
}

// One translation unit per logits dtype.
lcpp_status forward_f32(const Params& p, bool sigmoid, cudaStream_t s);
lcpp_status forward_f16(const Params& p, bool sigmoid, cudaStream_t s);
lcpp_status forward_bf16(const Params& p, bool sigmoid, cudaStream_t s);
lcpp_status backward_f32(const BackParams& p, bool sigmoid, cudaStream_t s);
lcpp_status backward_f16(const BackParams& p, bool sigmoid, cudaStream_t s);
lcpp_status backward_bf16(const BackParams& p, bool sigmoid, cudaStream_t s);

}  // namespace router
}  // namespace lcpp
