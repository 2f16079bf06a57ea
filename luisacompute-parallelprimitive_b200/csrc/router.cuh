// router.cuh -- DeviceRouter's kernels (include/lcpp_b200_model.h).
//
// A row of logits is spread over LANES lanes, C elements each; a warp works on
// 32 / LANES rows at a time.  Element i of lane l is expert
// ((i / V) * LANES + l) * V + i % V, V elements being 16 bytes, so a row's lanes
// read consecutive vectors.  Every lane copies its own vectors of the next rows
// into shared memory (cp.async) while the warp works on the present ones, and
// reads them from there: no registers are held for loads in flight, and a
// chosen expert's logit can be had by any lane.
//
// Choice.  Each biased logit becomes one 32-bit word whose unsigned order is
// (value, lower expert first): the float's order-preserving bits with their
// low IB bits replaced by the complement of the expert, IB = log2(LANES * C).
// The words of a row differ, so the next largest below `best` is the maximum
// of (word - best) mod 2^32: words below `best` wrap to the top of the range
// and those already taken stay at its bottom, and nothing has to be marked as
// taken.  Each lane finds the kHeads largest of its own words that way, then
// the lanes of a row hand out their heads, the largest first; a lane that has
// handed out all of them looks for its next one (8 lanes rarely hold 4 of a
// row's 8 largest).  The part of the expert that is the lane joins a head only,
// so a word's low bits are constants of its register.
//
// 16-bit logits without a bias fit the upper half of the word (Packed below):
// two words come from one 32-bit register in five instructions, the first
// round's winner is the row's maximum, and a chosen word holds its own logit.
// For the others the dropped bits matter only where two of the first top_k + 1
// words agree in all kept bits and their sums do not; a row whose choice could
// depend on them is chosen again from the full values (rows of continuous
// 32-bit logits: about one in a thousand at 256 experts).
#pragma once

#include "model.cuh"

namespace lcpp {
namespace router {

using namespace lcpp::model;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr float kNegInf = -INFINITY;
// Where a row's sigmoids are all below this, each equals exp(logit) to 32 bits
// and their sum may underflow: shares are taken as a softmax instead.
constexpr float kDeepSigmoid = 1e-20f;
constexpr float kDeepLogit = -60.f;  // the same for the largest chosen logit
constexpr int kHeads = 4;

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
    uint32_t unit;  // bytes of a copy: 16, 8, 4, or 2 (plain loads)
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
    uint32_t unit;         // bytes of a copy: 16, 8, 4, or 2 (plain loads)
    uint32_t wide_stores;  // gradient rows start on 16-byte boundaries
};

constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from)
{
    const uint32_t smem = uint32_t(__cvta_generic_to_shared(to));
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(from) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest group of this thread's copies have landed.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

template <typename T, int LANES, int C>
struct Tile {
    static constexpr int kV = Vec<T>::kN;
    static constexpr int kVecs = C / kV;
    static constexpr int kRows = kWarp / LANES;  // rows of a warp
    static constexpr int kSpan = LANES * C;      // experts that fit
    static constexpr int kIndexBits = log2_of(kSpan);
    static constexpr uint32_t kMask = kSpan - 1;
    static_assert(C % kV == 0 && (kSpan & (kSpan - 1)) == 0, "whole vectors, a power of two of experts");

    static __host__ __device__ constexpr uint32_t expert(int lane, int i)
    {
        return uint32_t(((i / kV) * LANES + lane) * kV + i % kV);
    }
    // The complement of the expert in a word's low bits, as the register's and
    // the lane's part.
    static __host__ __device__ constexpr uint32_t register_bits(int i) { return kMask - expert(LANES - 1, i); }
    static __device__ __forceinline__ uint32_t lane_bits(int lane) { return uint32_t(LANES - 1 - lane) * kV; }

    // A warp's rows in shared memory: vector v of warp lane wl is slot
    // v * 32 + wl.  What lies past num_experts is set to -inf once.
    static constexpr int kSlots = kVecs * kWarp;
    static __device__ __forceinline__ void clear(uint4* tile, int wl)
    {
        T part[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) part[i] = from_float<T>(kNegInf);
        uint4 raw;
        memcpy(&raw, part, 16);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) tile[v * kWarp + wl] = raw;
    }
    // Starts copying the lane's vectors of `row`; `unit` divides the row's
    // start, its stride and num_experts elements, so no copy is cut off.
    static __device__ __forceinline__ void fetch(uint4* tile, const T* row, int wl, uint32_t n, uint32_t unit)
    {
        const int lane = wl % LANES;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const uint32_t e0 = expert(lane, v * kV);
            uint4* slot = tile + v * kWarp + wl;
            if (unit == 16) {
                if (e0 < n) copy_async<16>(slot, row + e0);
            } else if (unit >= 4) {
#pragma unroll
                for (int b = 0; b < 16; b += 4) {
                    if (e0 + b / int(sizeof(T)) >= n) break;
                    if (unit == 8 && b % 8 == 0) copy_async<8>(reinterpret_cast<char*>(slot) + b, row + e0 + b / sizeof(T));
                    if (unit == 4) copy_async<4>(reinterpret_cast<char*>(slot) + b, row + e0 + b / sizeof(T));
                }
            } else {
#pragma unroll
                for (int i = 0; i < kV; ++i)
                    if (e0 + i < n) reinterpret_cast<T*>(slot)[i] = row[e0 + i];
            }
        }
    }
    static __device__ __forceinline__ void unpack(const uint4* tile, int wl, float (&x)[C])
    {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            float part[kV];
            Vec<T>::unpack(tile[v * kWarp + wl], part);
#pragma unroll
            for (int i = 0; i < kV; ++i) x[v * kV + i] = part[i];
        }
    }
    // Expert e's element of the row that sub-warp `sub` works on.
    static __device__ __forceinline__ T* element(uint4* tile, int sub, uint32_t e)
    {
        const uint32_t vec = e / kV;
        return reinterpret_cast<T*>(tile + (vec / LANES) * kWarp + sub * LANES + vec % LANES) + e % kV;
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

// ordered() backwards.
__device__ __forceinline__ float unordered(uint32_t o)
{
    return __uint_as_float(o ^ (uint32_t(int32_t(~o) >> 31) | 0x80000000u));
}

// Pairs of 16-bit logits as order-preserving 16-bit halves and back.
template <typename T>
struct Packed;
template <>
struct Packed<__half> {
    static __device__ __forceinline__ uint32_t plus_zero(uint32_t v)
    {
        const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(0.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kLowestChoice = 0x04000000u;  // above -inf
    static __device__ __forceinline__ float value(uint32_t bits) { return __half2float(__ushort_as_half(uint16_t(bits))); }
};
template <>
struct Packed<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t plus_zero(uint32_t v)
    {
        const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(0.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kLowestChoice = 0x00800000u;
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Packed<float> {  // never packed
    static __device__ __forceinline__ uint32_t plus_zero(uint32_t v) { return v; }
    static constexpr uint32_t kLowestChoice = 0x00800000u;
    static __device__ __forceinline__ float value(uint32_t) { return 0.f; }
};

template <typename T>
__device__ __forceinline__ uint32_t ordered_pair(uint32_t v)
{
    v = Packed<T>::plus_zero(v);  // as in ordered()
    uint32_t sign;                // 0xffff in each negative half
    asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(sign) : "r"(v));
    return v ^ (sign | 0x80008000u);
}

// The logit in the upper half of a word.
template <typename T>
__device__ __forceinline__ float word_value(uint32_t word)
{
    const uint32_t o = word >> 16;
    return Packed<T>::value(o & 0x8000u ? o ^ 0x8000u : ~o & 0xffffu);
}

// exp(x) for x <= 0 and its sigmoid; results below 2^-126 become 0.
__device__ __forceinline__ float exp_of(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + exp_of(-x)); }

template <int C>
__device__ __forceinline__ float lane_max(const float (&x)[C])
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < C; ++i) m = fmaxf(m, x[i]);
    return m;
}

// x (in place) becomes the lane's scores; returns their sum over the lane.
// Softmax scores are taken relative to `top`, as are sigmoids of a deep row.
template <bool SIGMOID, int C>
__device__ __forceinline__ float scores(float (&x)[C], float top, bool deep)
{
    float z[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
        x[i] = SIGMOID && !deep ? sigmoid(x[i]) : exp_of(x[i] - top);
        z[i % 2] += x[i];
    }
    return z[0] + z[1];
}

// The score that a chosen expert's weight is made of, `most` being the largest
// chosen logit where weights are renormalised and the row's largest otherwise.
template <bool SIGMOID>
__device__ __forceinline__ float weight_score(float x, float most, bool renormalize)
{
    if (SIGMOID) return renormalize && most < kDeepLogit ? exp_of(x - most) : sigmoid(x);
    return exp_of(x - most);
}

// The exact choice of a warp's rows from the full values, one composite word
// {ordered value, complement of the expert} per element: rare, so it reads the
// logits again instead of keeping them.  Writes words whose upper part says
// only whether an expert was chosen.
template <typename T, int LANES, int C>
__device__ __noinline__ void choose_exactly(const uint4* tile, const float* bias, int wl, uint32_t n, uint32_t k,
                                            uint32_t* chosen)
{
    using L = Tile<T, LANES, C>;
    uint64_t last = ~0ull;
    for (uint32_t j = 0; j < k; ++j) {
        uint64_t best = 0;
        for (int i = 0; i < C; ++i) {
            const uint32_t e = L::expert(wl % LANES, i);
            if (e >= n) continue;
            const float x = to_float(reinterpret_cast<const T*>(tile + i / L::kV * kWarp + wl)[i % L::kV]);
            const float f = bias ? x + bias[e] : x;
            if (f == kNegInf) continue;
            const uint64_t word = uint64_t(ordered(f)) << 32 | (0xffffffffu - e);
            if (word < last && word > best) best = word;
        }
        best = row_all<LANES>(best, Max{});
        if (wl % LANES == 0) chosen[j] = best ? ~L::kMask | (uint32_t(best) & L::kMask) : 0u;
        last = best;
    }
    __syncwarp();
}

// Largest of the words below `below` (mod 2^32; 0: of all).  Half of the words
// take the fused add-and-max, half an add on the FMA pipe and a three-way max,
// so that neither pipe waits for the other.
template <int C>
__device__ __forceinline__ uint32_t largest_below(const uint32_t (&word)[C], uint32_t below)
{
    uint32_t a = 0, b = 0, c = 0;
#pragma unroll
    for (int i = 0; i < C; i += 4) {
        a = __viaddmax_u32(word[i], -below, a);
        b = __viaddmax_u32(word[i + 1], -below, b);
        c = __vimax3_u32(word[i + 2] - below, word[i + 3] - below, c);
    }
    return __vimax3_u32(a, b, c) + below;
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
__global__ void __launch_bounds__(kThreads, C > 16 ? 2 : C > 8 ? 3 : 5) forward_kernel(const Params p)
{
    using L = Tile<T, LANES, C>;
    constexpr uint32_t kMask = L::kMask;
    constexpr bool kExact = sizeof(T) == 2 && !BIAS;  // words hold all of a logit
    constexpr uint32_t kLowest = kExact ? Packed<T>::kLowestChoice : 0x00800000u;
    const uint32_t n = p.num_experts, k = p.top_k;
    const int warp = threadIdx.x / kWarp, wl = threadIdx.x % kWarp, lane = wl % LANES, sub = wl / LANES;

    // the warps' two tiles; after the last row the shares' sums of every warp
    extern __shared__ uint4 dynamic[];
    uint4* tiles = dynamic + warp * 2 * L::kSlots;
    float* share_sum = reinterpret_cast<float*>(dynamic);                              // [kWarps][n]
    uint32_t* count = reinterpret_cast<uint32_t*>(dynamic + kWarps * 2 * L::kSlots);   // [n]
    float* bias = reinterpret_cast<float*>(count + n);                                 // [n]
    static_assert(2 * L::kSlots * 16 >= L::kSpan * 4, "the sums fit in the tiles");
    __shared__ uint32_t chosen_all[kWarps][L::kRows][LCPP_MAX_TOP_K];
    __shared__ float value_all[kWarps][L::kRows][LCPP_MAX_TOP_K];
    __shared__ double scratch[kThreads];
    __shared__ uint32_t routed_block;
    __shared__ bool is_last;
    uint32_t* chosen = chosen_all[warp][sub];
    float* value = value_all[warp][sub];
    for (uint32_t e = threadIdx.x; e < n; e += kThreads) {
        count[e] = 0;
        // finite, so that a logit of -inf stays -inf; NaN counts as the largest too
        if (BIAS) bias[e] = fminf(p.bias[e], 3.402823466e38f);
    }
    if (threadIdx.x == 0) routed_block = 0;
    L::clear(tiles, wl);
    L::clear(tiles + L::kSlots, wl);
    __syncthreads();

    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    uint32_t routed = 0;

    // lanes past the last token work on its row and write nothing
    const T* logits = static_cast<const T*>(p.logits);
    const uint32_t tokens = uint32_t(p.tokens), step = gridDim.x * kWarps * L::kRows;
    uint32_t t0 = (blockIdx.x * kWarps + warp) * L::kRows;
    if (t0 < tokens) L::fetch(tiles, logits + min(t0 + sub, tokens - 1) * p.stride, wl, n, p.unit);
    copies_commit();
    for (int stage = 0; t0 < tokens; t0 += step, stage ^= 1) {
        const uint32_t t = t0 + sub;
        const bool inside = t < tokens;
        uint4* tile = tiles + stage * L::kSlots;
        if (t0 + step < tokens)
            L::fetch(tiles + (stage ^ 1) * L::kSlots, logits + min(t + step, tokens - 1) * p.stride, wl, n, p.unit);
        copies_commit();
        const bool wanted = inside && (!p.token_request || p.token_request[t] >= 0);
        copies_wait();

        uint32_t word[C], low = 0;
        if constexpr (kExact) {
#pragma unroll
            for (int v = 0; v < L::kVecs; ++v) {
                const uint4 raw = tile[v * kWarp + wl];
                const uint32_t pair[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = v * L::kV + 2 * i;
                    const uint32_t o = ordered_pair<T>(pair[i]);
                    word[at] = o * 65536u + L::register_bits(at);
                    word[at + 1] = (o & 0xffff0000u) | L::register_bits(at + 1);
                }
            }
        } else {
            float x[C];
            L::unpack(tile, wl, x);
#pragma unroll
            for (int i = 0; i < C; ++i) {
                float f = x[i];
                // read where it is used: the biases would fill the registers otherwise
                if (BIAS) f += *static_cast<const volatile float*>(bias + min(L::expert(lane, i), n - 1));
                low |= __float_as_uint(f);
                word[i] = (ordered(f) & ~kMask) | L::register_bits(i);
            }
        }
        // The lane's largest words, then the row's: words below kLowest are
        // those of -inf.
        const uint32_t rounds = kExact ? k : min(k + 1, n);
        uint32_t head[kHeads], tail = 0;  // tail: the last word found so far
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            head[h] = 0;
            if (uint32_t(h) < rounds) head[h] = tail = largest_below(word, tail);
        }
        const uint32_t lane_bits = L::lane_bits(lane);
        uint32_t best = 0, handed = 0;
        bool found = false, unsure = false;
        for (uint32_t j = 0; j < rounds; ++j) {
            const uint32_t mine = head[0] + lane_bits;
            const uint32_t next = row_all<LANES>(mine, Max{});
            if (!kExact) unsure |= j && next >= kLowest && (next & ~kMask) == (best & ~kMask);
            best = next;
            if (j == 0) found = best >= kLowest;
            if (j < k && lane == 0) chosen[j] = best;
            const bool out = mine == next;
#pragma unroll
            for (int h = 0; h + 1 < kHeads; ++h) head[h] = out ? head[h + 1] : head[h];
            if (out) head[kHeads - 1] = 0;
            handed += out;
            const bool empty = head[0] == 0 && handed < C;
            if (__any_sync(~0u, empty) && j + 1 < rounds) {
                const uint32_t more = largest_below(word, tail);
                if (empty) head[0] = tail = more;
            }
        }
        __syncwarp();
        if (!kExact) {
            // logits whose dropped bits are all zero were compared in full
            low = row_all<LANES>(low & kMask, Or{});
            unsure = unsure && low;
            if (__any_sync(~0u, unsure)) choose_exactly<T, LANES, C>(tile, BIAS ? bias : nullptr, wl, n, k, chosen);
        }
        const bool live = wanted && found;

        float x[C], top = 0.f;
        L::unpack(tile, wl, x);
        if (!SIGMOID) top = kExact ? word_value<T>(chosen[0]) : row_all<LANES>(lane_max(x), Max{});
        float sum = row_all<LANES>(scores<SIGMOID>(x, top, false), Add{});
        if (SIGMOID) {
            const bool deep = sum < kDeepSigmoid;
            if (__any_sync(~0u, deep)) {
                L::unpack(tile, wl, x);
                top = row_all<LANES>(lane_max(x), Max{});
                sum = row_all<LANES>(scores<SIGMOID>(x, top, deep), Add{});
            }
        }
        const float inv = live ? __fdividef(1.f, sum) : 0.f;
        if (live) {
#pragma unroll
            for (int i = 0; i < C; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
        }

        // weights of the chosen
        float most = kNegInf;
        for (uint32_t j = lane; j < k; j += LANES) {
            const uint32_t w = chosen[j], e = kMask - (w & kMask);
            const float v = w < kLowest ? kNegInf : kExact ? word_value<T>(w) : to_float(*L::element(tile, sub, e));
            value[j] = v;
            most = fmaxf(most, v);
        }
        if (p.renormalize) most = row_all<LANES>(most, Max{});
        else most = top;
        float total = 0.f;
        for (uint32_t j = lane; j < k; j += LANES) {
            const float s = chosen[j] >= kLowest ? weight_score<SIGMOID>(value[j], most, p.renormalize) : 0.f;
            value[j] = s;
            total += s;
        }
        float scale = p.weight_scale;
        if (p.renormalize) scale = __fdividef(scale, row_all<LANES>(total, Add{}));
        else if (!SIGMOID) scale = __fdividef(scale, sum);
        if (inside) {
            for (uint32_t j = lane; j < k; j += LANES) {
                const uint32_t w = chosen[j], e = kMask - (w & kMask);
                const bool is = live && w >= kLowest;
                p.weights[uint64_t(t) * k + j] = is ? value[j] * scale : 0.f;
                p.experts[uint64_t(t) * k + j] = is ? int32_t(e) : -1;
                if (is) atomicAdd(count + e, 1u);
            }
        }
        routed += live && lane == 0;
        __syncwarp();
    }

    // the block's sums, in the tiles' memory
    __syncthreads();
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

// The logits' gradient.  The chosen experts of a row are taken out of it first
// (their logits in the tile become -inf): the dense part of a row then has one
// formula, and each chosen expert's entry is computed by a lane of its own and
// stored after the dense ones.
template <typename T, int LANES, int C, bool SIGMOID, bool RENORM>
__global__ void __launch_bounds__(kThreads, C > 16 ? 2 : 3) backward_kernel(const BackParams p)
{
    using L = Tile<T, LANES, C>;
    // Softmax weights as they are: the chosen experts' slopes join the loss's
    // before the row's mean is taken off; else they are added afterwards.
    constexpr bool kJoined = !SIGMOID && !RENORM;
    const uint32_t n = p.num_experts, k = p.top_k;
    const int warp = threadIdx.x / kWarp, wl = threadIdx.x % kWarp, lane = wl % LANES, sub = wl / LANES;
    extern __shared__ uint4 dynamic[];
    uint4* tiles = dynamic + warp * 2 * L::kSlots;
    float* pull = reinterpret_cast<float*>(dynamic + kWarps * 2 * L::kSlots);  // [kSpan]
    // this row's chosen experts and upstream gradients, twice, and their logits: [kRows][k] each
    const uint32_t row_k = L::kRows * k;
    uint32_t* ids = reinterpret_cast<uint32_t*>(pull + L::kSpan) + warp * 5 * row_k + sub * k;
    float* ups = reinterpret_cast<float*>(ids + 2 * row_k);
    float* values = ups + 2 * row_k;
    L::clear(tiles, wl);
    L::clear(tiles + L::kSlots, wl);
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

    const T* logits = static_cast<const T*>(p.logits);
    const uint32_t tokens = uint32_t(p.tokens), step = gridDim.x * kWarps * L::kRows;
    const auto fetch = [&](uint32_t t, int stage) {
        const uint32_t tt = min(t, tokens - 1);
        L::fetch(tiles + stage * L::kSlots, logits + tt * p.stride, wl, n, p.unit);
        for (uint32_t j = lane; j < k; j += LANES) {
            copy_async<4>(ids + stage * row_k + j, p.experts + uint64_t(tt) * k + j);
            if (p.grad_weights) copy_async<4>(ups + stage * row_k + j, p.grad_weights + uint64_t(tt) * k + j);
            else ups[stage * row_k + j] = 0.f;
        }
    };
    uint32_t t0 = (blockIdx.x * kWarps + warp) * L::kRows;
    if (t0 < tokens) fetch(t0 + sub, 0);
    copies_commit();
    for (int stage = 0; t0 < tokens; t0 += step, stage ^= 1) {
        const uint32_t t = t0 + sub;
        const bool inside = t < tokens;
        uint4* tile = tiles + stage * L::kSlots;
        const uint32_t* id = ids + stage * row_k;
        const float* up = ups + stage * row_k;
        if (t0 + step < tokens) fetch(t + step, stage ^ 1);
        copies_commit();
        copies_wait();
        __syncwarp();

        const bool live = int32_t(id[0]) >= 0;
        float chosen_top = kNegInf;
        for (uint32_t j = lane; j < k; j += LANES) {
            float v = kNegInf;
            if (id[j] < n) {
                T* at = L::element(tile, sub, id[j]);
                v = to_float(*at);
                *at = from_float<T>(kNegInf);
            }
            values[j] = v;
            chosen_top = fmaxf(chosen_top, v);
        }
        if (RENORM || !SIGMOID) chosen_top = row_all<LANES>(chosen_top, Max{});
        __syncwarp();
        // The expert with most of the row's share, among the chosen: slopes are
        // taken relative to its own, so that the mean of a row that one expert
        // dominates is not the difference of two equal numbers.
        uint32_t lead = 0;
        for (uint32_t j = 1; j < k; ++j) lead = values[j] > values[lead] ? j : lead;
        const float up0 = up[lead], c = p.weight_scale;
        const float pull0 = id[lead] < n ? pull[id[lead]] : 0.f;
        const float base = kJoined ? fmaf(c, up0, pull0) : pull0;

        float x[C], top = 0.f;
        L::unpack(tile, wl, x);
        if (!SIGMOID) top = fmaxf(row_all<LANES>(lane_max(x), Max{}), chosen_top);
        float sum = scores<SIGMOID>(x, top, false), weights = 0.f;
        for (uint32_t j = lane; j < k; j += LANES) {
            sum += SIGMOID ? sigmoid(values[j]) : exp_of(values[j] - top);
            if (RENORM) weights += id[j] < n ? weight_score<SIGMOID>(values[j], chosen_top, true) : 0.f;
        }
        sum = row_all<LANES>(sum, Add{});
        if (RENORM) weights = row_all<LANES>(weights, Add{});
        bool deep = false;
        if (SIGMOID) {
            deep = sum < kDeepSigmoid;
            if (__any_sync(~0u, deep)) {
                L::unpack(tile, wl, x);
                float most = lane_max(x);
                for (uint32_t j = lane; j < k; j += LANES) most = fmaxf(most, values[j]);
                top = row_all<LANES>(most, Max{});
                sum = scores<SIGMOID>(x, top, deep);
                for (uint32_t j = lane; j < k; j += LANES) sum += deep ? exp_of(values[j] - top) : sigmoid(values[j]);
                sum = row_all<LANES>(sum, Add{});
            }
        }
        const float inv = __fdividef(1.f, sum);
        const auto share_of = [&](float v) { return (SIGMOID && !deep ? sigmoid(v) : exp_of(v - top)) * inv; };
        const auto slope_at = [&](uint32_t j) {
            const float h = pull[id[j]] - pull0;
            return kJoined ? fmaf(c, up[j] - up0, h) : h;
        };
        float mean = 0.f;
#pragma unroll
        for (int v = 0; v < L::kVecs; ++v) {
            const float* h = pull + L::expert(lane, v * L::kV);
#pragma unroll
            for (int i = 0; i < L::kV; ++i) mean = fmaf(x[v * L::kV + i], h[i] - base, mean);
        }
        mean *= inv;
        for (uint32_t j = lane; j < k; j += LANES)
            if (id[j] < n) mean = fmaf(share_of(values[j]), slope_at(j), mean);
        mean = row_all<LANES>(mean, Add{});

        T* out = static_cast<T*>(p.grad_logits) + uint64_t(t) * p.grad_stride;
        const float rest = base + mean;
#pragma unroll
        for (int v = 0; v < L::kVecs; ++v) {
            const uint32_t e0 = L::expert(lane, v * L::kV);
            float g[L::kV];
#pragma unroll
            for (int i = 0; i < L::kV; ++i) {
                const float s = x[v * L::kV + i];
                g[i] = s * inv * (pull[e0 + i] - rest);
                if (SIGMOID && !deep) g[i] *= 1.f - s;
            }
            uint4 raw = Vec<T>::pack(g);
            if (!live) raw = uint4{0, 0, 0, 0};
            if (inside && p.wide_stores && e0 + L::kV <= n) {
                *reinterpret_cast<uint4*>(out + e0) = raw;
            } else if (inside) {
                T part[L::kV];
                memcpy(part, &raw, 16);
#pragma unroll
                for (int i = 0; i < L::kV; ++i)
                    if (e0 + i < n) out[e0 + i] = part[i];
            }
        }
        __syncwarp();
        for (uint32_t j = lane; j < k; j += LANES) {
            if (id[j] >= n || !inside) continue;
            const float v = values[j], g = up[j];
            const float flat = SIGMOID ? sigmoid(-v) : 1.f;  // 1 - s
            float d = flat * share_of(v) * (slope_at(j) - mean);
            if (RENORM) {
                // g_j - sum_i r_i g_i as a sum of differences, for the same reason
                float apart = 0.f;
                for (uint32_t i = 0; i < k; ++i)
                    if (id[i] < n)
                        apart = fmaf(weight_score<SIGMOID>(values[i], chosen_top, true), g - up[i], apart);
                d += c * flat * __fdividef(weight_score<SIGMOID>(v, chosen_top, true), weights) * __fdividef(apart, weights);
            } else if (SIGMOID) {
                d = fmaf(c * g * flat, sigmoid(v), d);
            }
            out[id[j]] = from_float<T>(d);
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
    using L = Tile<T, LANES, C>;
    const size_t smem = size_t(kWarps) * 2 * L::kSlots * 16 + size_t(p.num_experts) * 8;
    void (*kernel)(Params) =
        sigmoid ? (p.bias ? forward_kernel<T, LANES, C, true, true> : forward_kernel<T, LANES, C, true, false>)
                : (p.bias ? forward_kernel<T, LANES, C, false, true> : forward_kernel<T, LANES, C, false, false>);
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, size_t(kWarps) * 2 * L::kSlots * 16 + L::kSpan * 8);
    const unsigned grid = grid_for(f, smem, p.tokens, kWarps * L::kRows);
    if (grid > 1) LCPP_CUDA_TRY(cudaMemsetAsync(p.ctrl, 0, cleared_bytes(p.num_experts), s));
    kernel<<<grid, kThreads, smem, s>>>(p);
    return launched();
}

template <typename T, int LANES, int C>
lcpp_status backward_shape(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    using L = Tile<T, LANES, C>;
    const size_t fixed = size_t(kWarps) * 2 * L::kSlots * 16 + L::kSpan * 4;
    const size_t smem = fixed + size_t(kWarps) * 5 * L::kRows * p.top_k * 4;
    void (*kernel)(BackParams) =
        sigmoid ? (p.renormalize ? backward_kernel<T, LANES, C, true, true> : backward_kernel<T, LANES, C, true, false>)
                : (p.renormalize ? backward_kernel<T, LANES, C, false, true> : backward_kernel<T, LANES, C, false, false>);
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, fixed + size_t(kWarps) * 5 * L::kRows * LCPP_MAX_TOP_K * 4);
    kernel<<<grid_for(f, smem, p.tokens, kWarps * L::kRows), kThreads, smem, s>>>(p);
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
