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
// words agree in all kept bits and their sums do not; such a row's words (and
// those past them that agree too) are put in the order of their full values
// (about one row in 300 of continuous 32-bit logits at 256 experts); only where
// more than kMoreRounds agree is the row chosen again from the full values.
//
// What has to move is a row's logits once (and, backward, its gradient) and 8
// bytes a choice.  131072 rows of 256 bfloat16 logits, top 8: forward 44 us, of
// which the copy rate would take 11.8, gradient 40 us (22.2; sigmoid scores).
// Neither memory nor a pipe is what bounds them, but dependent steps and too few
// warps to fill the time: forward issues 830 instructions per four rows in 59 % of
// the issue slots (integer pipe 57 %, 24 warps an SM), about 170 of them the lanes'
// heads and 180 the rounds, each of which waits for shuffles of the one before; the
// gradient 725 in 58 % (exponential unit 47 %, 16 warps an SM).  65536 rows of 256
// 32-bit logits: forward 36 us (11.1), gradient 26 us (21.6).
#pragma once

#include "model.cuh"

namespace lcpp {
namespace router {

using namespace lcpp::model;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr float kNegInf = -INFINITY;
// Where the sum of a row's sigmoids is below this, each equals exp(logit) to 32
// bits (they differ by a factor of 1 + exp(logit)), and smaller ones may underflow
// beside it: shares are taken as a softmax instead.
constexpr float kDeepSigmoid = 1e-8f;
constexpr float kDeepLogit = -18.5f;  // the same for the largest chosen logit
constexpr int kHeads = 4;
constexpr int kMoreRounds = 6;  // words past top_k that a tie is followed for

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
    bool bias_on_score;  // else on the logit
    uint32_t unit;  // bytes of a copy: 16, 8, 4, or 2 (plain loads)
    // temp storage, cleared before a launch of several blocks
    uint32_t* ctrl;                  // [0] blocks done, [1] error word, [2] a share was not finite, [3] tokens routed
    unsigned long long* share_total; // [kShareScales][num_experts] sums of shares
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
// Read each time it is used: loop-invariant values would fill the registers.
__device__ __forceinline__ float4 shared_load4(const float* from)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(uint32_t(__cvta_generic_to_shared(from))));
    return v;
}
// All but the newest group of this thread's copies have landed.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

template <typename T, int LANES, int C>
struct Tile {
    static constexpr int kV = Vec<T>::kN;
    static constexpr int kVecs = C / kV;
    static constexpr int kRows = kWarp / LANES;  // rows of a warp
    static constexpr int kSpan = LANES * C;      // experts that fit
    static constexpr int kMaxTopK = kSpan < LCPP_MAX_TOP_K ? kSpan : LCPP_MAX_TOP_K;
    static constexpr int kPlaces = kMaxTopK / LANES;  // a lane's entries of a row are j = lane, lane + LANES, ...
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
        if (unit == 16) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v)
                if (expert(lane, v * kV) < n) copy_async<16>(tile + v * kWarp + wl, row + expert(lane, v * kV));
            return;
        }
#pragma unroll 1
        for (int v = 0; v < kVecs; ++v) {
            const uint32_t e0 = expert(lane, v * kV);
            T* slot = reinterpret_cast<T*>(tile + v * kWarp + wl);
            const uint32_t step = unit >= 4 ? unit / sizeof(T) : 1;
            for (uint32_t i = 0; i < kV && e0 + i < n; i += step) {
                if (unit == 8) copy_async<8>(slot + i, row + e0 + i);
                else if (unit == 4) copy_async<4>(slot + i, row + e0 + i);
                else slot[i] = row[e0 + i];
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

// 2^x and exp(x); results below 2^-126 become 0.
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * kLog2E); }

__device__ __forceinline__ float reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float sigmoid(float x)
{
    return reciprocal(1.f + exp_of(-x));
}

// Two sums or products in one instruction: forward 895 -> 826 instructions per
// four rows of 256 (45 -> 44 us), sigmoid gradient 900 -> 745 (43 -> 42 us; 128
// experts, softmax 13.9 -> 12.9 us).
__device__ __forceinline__ float2 both(float x) { return {x, x}; }
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
template <int C>
__device__ __forceinline__ float2 pair_of(const float (&x)[C], int i)
{
    return {x[i], x[i + 1]};
}

template <int C>
__device__ __forceinline__ float lane_max(const float (&x)[C])
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < C; ++i) m = fmaxf(m, x[i]);
    return m;
}

// What a row's softmax scores are taken relative to: exp(x - top), as one
// multiply-add and 2^x where `top` is of ordinary size.  The rounding of
// top log2(e) is then a factor common to all scores of the row, which are only
// used as quotients; past 10^6 the factor itself could overflow.
struct Reference {
    float top, scaled;
    bool wide, any_rare;  // this row; it or another rarity in any row of the warp
    __device__ __forceinline__ Reference() : top(0.f), scaled(0.f), wide(false), any_rare(false) {}
    __device__ __forceinline__ explicit Reference(float t, bool rare = false)
        : top(t), scaled(t * -kLog2E), wide(!(fabsf(t) < 1e6f)), any_rare(__any_sync(~0u, wide || rare))
    {
    }
    __device__ __forceinline__ float score(float x) const
    {
        return any_rare && wide ? exp_of(x - top) : exp2_of(fmaf(x, kLog2E, scaled));
    }
};

// x (in place) becomes the lane's scores; returns their sum over the lane.
template <int C>
__device__ __forceinline__ float softmax_scores(float (&x)[C], const Reference& ref)
{
    float2 z = both(0.f);
    if (ref.any_rare) {
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] = ref.score(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            const float2 at = fma2(pair_of(x, i), both(kLog2E), both(ref.scaled));
            x[i] = exp2_of(at.x);
            x[i + 1] = exp2_of(at.y);
        }
    }
#pragma unroll
    for (int i = 0; i < C; i += 2) z = add2(z, pair_of(x, i));
    return z.x + z.y;
}

// exp(-x) of two logits; where `deep`, exp(x - top).
template <bool DEEP>
__device__ __forceinline__ float2 two_parts(float2 x, float top, bool deep)
{
    if (DEEP) x = add2(x, both(deep ? -top : 0.f));
    x = mul2(x, both(DEEP && deep ? kLog2E : -kLog2E));
    return {exp2_of(x.x), exp2_of(x.y)};
}

// For the gradient: x becomes the sigmoid's slope s (1 - s), whose second factor
// is e s of e = exp(-x), for near 1 a subtraction would leave nothing of it; where
// `deep`, the score exp(x - top), which is its own slope.  Returns the lane's sum
// of scores, `mean` that of s (pull - base).
constexpr float kLargestPart = 3e38f;  // s is 0 there: keeps infinity times that 0
template <typename L, bool DEEP, int C>
__device__ __forceinline__ float sigmoid_slopes(float (&x)[C], const float* pull, int lane, float base, float top,
                                                bool deep, float& mean)
{
    float2 z = both(0.f), m = both(0.f);
#pragma unroll
    for (int q = 0; q < C; q += 4) {
        const float4 h = shared_load4(pull + L::expert(lane, q));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float2 e = two_parts<DEEP>(pair_of(x, q + i), top, deep), sum = add2(e, both(1.f));
            float2 s = {reciprocal(sum.x), reciprocal(sum.y)};
            float2 slope = mul2(mul2({fminf(e.x, kLargestPart), fminf(e.y, kLargestPart)}, s), s);
            if (DEEP && deep) s = slope = e;
            x[q + i] = slope.x;
            x[q + i + 1] = slope.y;
            z = add2(z, s);
            m = fma2(s, add2(i ? float2{h.z, h.w} : float2{h.x, h.y}, both(-base)), m);
        }
    }
    mean = m.x + m.y;
    return z.x + z.y;
}

// The scores of sigmoids; where `deep`, exp(x - top).
template <bool DEEP, int C>
__device__ __forceinline__ float sigmoid_scores(float (&x)[C], float top, bool deep)
{
    float2 z = both(0.f);
#pragma unroll
    for (int i = 0; i < C; i += 2) {
        float2 s = two_parts<DEEP>(pair_of(x, i), top, deep);
        if (!(DEEP && deep)) {
            s = add2(s, both(1.f));
            s = {reciprocal(s.x), reciprocal(s.y)};
        }
        x[i] = s.x;
        x[i + 1] = s.y;
        z = add2(z, s);
    }
    return z.x + z.y;
}

// What a chosen expert's renormalised weight is made of, `most` being the
// largest chosen logit.
template <bool SIGMOID>
__device__ __forceinline__ float weight_score(float x, float most)
{
    return SIGMOID && !(most < kDeepLogit) ? sigmoid(x) : exp_of(x - most);
}

// What the choice goes by: logits, logits + bias, or scores + bias.  Scores are
// computed for the choice and again for the sums (131072 rows of 256 bfloat16,
// sigmoid: 48, 72 and 84 us).
enum Choice { kByLogit, kByBiasedLogit, kByBiasedScore };

// The 32-bit value an expert is chosen by.  All that compare two of them go
// through here and get the same bits: rounded sums and products, no contraction.
template <bool SIGMOID, Choice BY>
struct ChoiceKey {
    const float* bias;
    Reference ref;  // scores only: the row's, and the inverse of its scores' sum
    float inv;
    __device__ __forceinline__ float operator()(float x, float b) const
    {
        if (BY == kByLogit) return x;
        if (BY == kByBiasedLogit) return __fadd_rn(x, b);
        const float s = SIGMOID ? sigmoid(x) : __fmul_rn(ref.score(x), inv);
        return x == kNegInf ? kNegInf : __fadd_rn(s, b);
    }
    // -inf also for an expert that is switched off
    __device__ __forceinline__ float of(float x, uint32_t e) const
    {
        if (BY == kByLogit) return x;
        return bias[e] == kNegInf ? kNegInf : (*this)(x, bias[e]);
    }
};

// The exact choice of a warp's rows from the full values, one composite word
// {ordered value, complement of the expert} per element: rare, so it reads the
// logits again instead of keeping them.  Writes words whose upper part says
// only whether an expert was chosen.
template <typename T, int LANES, int C, typename Key>
__device__ __noinline__ void choose_exactly(const uint4* tile, const Key key, int wl, uint32_t n, uint32_t k,
                                            uint32_t* chosen)
{
    using L = Tile<T, LANES, C>;
    uint64_t last = 0;
    for (uint32_t j = 0; j < k; ++j) {
        uint64_t best = 0;
        for (int i = 0; i < C; ++i) {
            const uint32_t e = L::expert(wl % LANES, i);
            if (e >= n) continue;
            const float f = key.of(to_float(reinterpret_cast<const T*>(tile + i / L::kV * kWarp + wl)[i % L::kV]), e);
            if (f == kNegInf) continue;
            const uint64_t word = uint64_t(ordered(f)) << 32 | (0xffffffffu - e);
            if ((j == 0 || word < last) && word > best) best = word;  // the first may be all ones
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

// Blocks' shares of an expert are added up as whole numbers, whose total is the
// same in any order: in units of 2^-32 those from 2^-8 up (at most 2^31 tokens in
// all), smaller ones in totals of their own with units of 2^-60, 2^-88, 2^-116 and
// 2^-144, of which a 32-bit sum is a multiple there (below 2^-121 it is rounded to
// one) and at most 2^52.
constexpr int kShareScales = 5;
__device__ __forceinline__ int share_scale(float share)
{
    return (share < 0x1p-8f) + (share < 0x1p-36f) + (share < 0x1p-64f) + (share < 0x1p-92f);
}
// 2^(+-(32 + 28 scale)): units in a share of 1, and a unit.
__device__ __forceinline__ double share_units(int scale, int sign)
{
    return __hiloint2double((1023 + sign * (32 + 28 * scale)) << 20, 0);
}

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

template <typename T, int LANES, int C, bool SIGMOID, Choice BY>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 && C > 16 ? 2 : 3) forward_kernel(const Params p)
{
    using L = Tile<T, LANES, C>;
    constexpr uint32_t kMask = L::kMask;
    constexpr bool BIAS = BY != kByLogit;
    constexpr bool kExact = sizeof(T) == 2 && !BIAS;  // words hold all of a logit
    constexpr int kPlaces = L::kPlaces;
    constexpr uint32_t kLowest = kExact ? Packed<T>::kLowestChoice : 0x00800000u;
    const uint32_t n = p.num_experts, k = p.top_k;
    const int warp = threadIdx.x / kWarp, wl = threadIdx.x % kWarp, lane = wl % LANES, sub = wl / LANES;

    // The warps' two tiles, and every lane's sums of its experts' shares: they
    // are touched once a row, and in registers they would cost a third of the
    // resident warps.
    extern __shared__ uint4 dynamic[];
    uint4* tiles = dynamic + warp * 2 * L::kSlots;
    float4* all_sums = reinterpret_cast<float4*>(dynamic + kWarps * 2 * L::kSlots);    // [kWarps][C / 4][32]
    float4* sums = all_sums + warp * (C / 4) * kWarp + wl;
    float* bias = reinterpret_cast<float*>(all_sums + kWarps * (C / 4) * kWarp);  // [kSpan]
    uint32_t* count = reinterpret_cast<uint32_t*>(bias + (BIAS ? L::kSpan : 0));   // [n]
    __shared__ uint32_t chosen_all[kExact ? 1 : kWarps][kExact ? 1 : L::kRows][L::kMaxTopK];
    __shared__ uint32_t lists[kExact ? 1 : kWarps][kExact ? 1 : L::kRows][L::kMaxTopK + kMoreRounds];
    double* scratch = reinterpret_cast<double*>(dynamic);  // [kThreads], after the last row
    static_assert(kWarps * 2 * L::kSlots * 16 >= kThreads * 8, "the tiles hold it");
    __shared__ uint32_t routed_block;
    __shared__ bool is_last;
    uint32_t* chosen = chosen_all[kExact ? 0 : warp][kExact ? 0 : sub];
    for (uint32_t e = threadIdx.x; e < n; e += kThreads) count[e] = 0;
    bool off = false;  // a bias of -inf, which no logit outweighs
    if (BIAS) {
        // not +inf, so that a logit of -inf stays -inf; NaN counts as the largest too
        for (uint32_t e = threadIdx.x; e < L::kSpan; e += kThreads) {
            bias[e] = e < n ? fminf(p.bias[e], 3.402823466e38f) : 0.f;
            off |= bias[e] == kNegInf;
        }
    }
    if (threadIdx.x == 0) routed_block = 0;
    L::clear(tiles, wl);
    L::clear(tiles + L::kSlots, wl);
    const bool any_off = __syncthreads_or(off);

#pragma unroll
    for (int q = 0; q < C / 4; ++q) sums[q * kWarp] = float4{0.f, 0.f, 0.f, 0.f};
    uint32_t routed = 0;

    // a row past the last token works on what its tile holds and writes nothing
    const uint32_t tokens = uint32_t(p.tokens), step = gridDim.x * kWarps * L::kRows;
    uint32_t t = (blockIdx.x * kWarps + warp) * L::kRows + sub;
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    const uint64_t row_step = step * p.stride;
    int32_t request = 0, request_ahead = 0;
    if (t < tokens) {
        L::fetch(tiles, row, wl, n, p.unit);
        if (p.token_request) request_ahead = p.token_request[t];
    }
    copies_commit();
    for (int stage = 0; t - sub < tokens; t += step, stage ^= 1) {
        const bool inside = t < tokens;
        uint4* tile = tiles + stage * L::kSlots;
        row += row_step;
        request = request_ahead;
        if (t + step < tokens) {
            L::fetch(tiles + (stage ^ 1) * L::kSlots, row, wl, n, p.unit);
            if (p.token_request) request_ahead = p.token_request[t + step];
        }
        copies_commit();
        copies_wait();
        if (!kExact) __syncwarp();  // a chosen logit may be another lane's copy

        uint32_t word[C], low = 0;
        ChoiceKey<SIGMOID, BY> key{bias, Reference(), 0.f};
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
            if constexpr (BY == kByBiasedScore && !SIGMOID) {
                key.ref = Reference(row_all<LANES>(lane_max(x), Max{}));
                key.inv = __fdividef(1.f, row_all<LANES>(softmax_scores(x, key.ref), Add{}));
                L::unpack(tile, wl, x);
            }
#pragma unroll
            for (int q = 0; q < C; q += 4) {
                float4 b{0.f, 0.f, 0.f, 0.f};
                if (BIAS) b = shared_load4(bias + L::expert(lane, q));
                const float f[4] = {key(x[q], b.x), key(x[q + 1], b.y), key(x[q + 2], b.z), key(x[q + 3], b.w)};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    low |= __float_as_uint(f[i]);
                    word[q + i] = (ordered(f[i]) & ~kMask) | L::register_bits(q + i);
                }
            }
            if (BIAS && any_off) {
#pragma unroll
                for (int i = 0; i < C; ++i)
                    if (bias[L::expert(lane, i)] == kNegInf) word[i] = (kLowest - 1 & ~kMask) | L::register_bits(i);
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
        // each lane keeps those of its places j = lane, lane + LANES, ...
        const uint32_t lane_bits = L::lane_bits(lane);
        uint32_t picked[kPlaces + 1], best = 0, handed = 0;
        bool unsure = false, tie = false;
        // the row's largest head
        const auto hand_out = [&] {
            const uint32_t mine = head[0] + lane_bits, next = row_all<LANES>(mine, Max{});
            const bool out = mine == next;
#pragma unroll
            for (int h = 0; h + 1 < kHeads; ++h) head[h] = out ? head[h + 1] : head[h];
            if (out) head[kHeads - 1] = 0;
            handed += out;
            return next;
        };
        // a head for lanes that have handed out all they had found
        const auto refill = [&] {
            const bool empty = head[0] == 0 && handed < C;
            if (__any_sync(~0u, empty)) {
                const uint32_t more = largest_below(word, tail);
                if (empty) head[0] = tail = more;
            }
        };
#pragma unroll
        for (int s = 0; s < kPlaces + !kExact; ++s) {
            picked[s] = 0;
            if (uint32_t(s * LANES) >= rounds) break;
            for (uint32_t i = 0, j = s * LANES; i < LANES && j < rounds; ++i, ++j) {
                if (j >= kHeads) refill();
                const uint32_t next = hand_out();
                tie = next >= kLowest && (next & ~kMask) == (best & ~kMask);
                unsure |= tie;
                best = next;
                if (uint32_t(lane) == i) picked[s] = next;
            }
        }
        if (!kExact) {
            // logits whose dropped bits are all zero were compared in full
            low = row_all<LANES>(low & kMask, Or{});
            if (__any_sync(~0u, unsure && low)) {
                // Words that tie with the last one are handed out too, then all
                // are put in the order of their full values.
                uint32_t* list = lists[warp][sub];
                const auto full = [&](uint32_t w) -> uint64_t {
                    if (w < kLowest) return 0;
                    const uint32_t e = kMask - (w & kMask);
                    return uint64_t(ordered(key.of(to_float(*L::element(tile, sub, e)), e))) << 32 | (0xffffffffu - e);
                };
                __syncwarp();
#pragma unroll
                for (int s = 0; s <= kPlaces; ++s)
                    if (uint32_t(s * LANES + lane) < rounds) list[s * LANES + lane] = picked[s];
                uint32_t m = rounds;
                for (; m < min(n, k + kMoreRounds) && __any_sync(~0u, tie); ++m) {
                    refill();
                    const uint32_t next = hand_out();
                    tie = next >= kLowest && (next & ~kMask) == (best & ~kMask);
                    best = next;
                    if (lane == 0) list[m] = next;
                }
                for (uint32_t j = lane; j < k; j += LANES) chosen[j] = 0;
                __syncwarp();
                if (__any_sync(~0u, tie && m < n)) {
                    choose_exactly<T, LANES, C>(tile, key, wl, n, k, chosen);
                } else {
                    for (uint32_t j = lane; j < m; j += LANES) {
                        const uint64_t mine = full(list[j]);
                        uint32_t rank = 0;
                        for (uint32_t i = 0; i < m; ++i) rank += full(list[i]) > mine;
                        if (mine && rank < k) chosen[rank] = list[j];
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int s = 0; s < kPlaces; ++s)
                    if (uint32_t(s * LANES + lane) < k) picked[s] = chosen[s * LANES + lane];
            }
        }
        const uint32_t first = __shfl_sync(~0u, picked[0], sub * LANES);
        const bool live = inside && request >= 0 && first >= kLowest;

        float x[C], top = 0.f;
        L::unpack(tile, wl, x);
        if (!SIGMOID) top = kExact ? word_value<T>(first) : row_all<LANES>(lane_max(x), Max{});
        const Reference ref(top);
        float sum = row_all<LANES>(SIGMOID ? sigmoid_scores<false>(x, 0.f, false) : softmax_scores(x, ref), Add{});
        if (SIGMOID) {
            const bool deep = sum < kDeepSigmoid;
            if (__any_sync(~0u, deep)) {
                L::unpack(tile, wl, x);
                top = row_all<LANES>(lane_max(x), Max{});
                sum = row_all<LANES>(sigmoid_scores<true>(x, top, deep), Add{});
            }
        }
        const float inv = live ? __fdividef(1.f, sum) : 0.f;
        if (live) {
#pragma unroll
            for (int q = 0; q < C / 4; ++q) {
                const float4 v = sums[q * kWarp];
                const float2 low = fma2(pair_of(x, 4 * q), both(inv), {v.x, v.y});
                const float2 high = fma2(pair_of(x, 4 * q + 2), both(inv), {v.z, v.w});
                sums[q * kWarp] = {low.x, low.y, high.x, high.y};
            }
        }

        // weights of the chosen
        float value[kPlaces], most = kNegInf, total = 0.f;
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            if (uint32_t(s * LANES + lane) >= k) picked[s] = 0;
            const uint32_t w = picked[s];
            value[s] = kNegInf;
            if (w >= kLowest) value[s] = kExact ? word_value<T>(w) : to_float(*L::element(tile, sub, kMask - (w & kMask)));
            most = fmaxf(most, value[s]);
        }
        if (p.renormalize) most = row_all<LANES>(most, Max{});
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            float v = 0.f;
            if (picked[s] >= kLowest) {
                if (p.renormalize) v = weight_score<SIGMOID>(value[s], most);
                else v = SIGMOID ? sigmoid(value[s]) : ref.score(value[s]);
            }
            value[s] = v;
            total += v;
        }
        float scale = p.weight_scale;
        if (p.renormalize) scale = __fdividef(scale, row_all<LANES>(total, Add{}));
        else if (!SIGMOID) scale = __fdividef(scale, sum);
        // a NaN among the logits is in every score, also where a bias kept its expert out
        if (BIAS && !SIGMOID && sum != sum) scale = sum;
        const uint32_t at = t * k + lane;
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            if (inside && uint32_t(s * LANES + lane) < k) {
                const bool is = live && picked[s] >= kLowest;
                const uint32_t e = kMask - (picked[s] & kMask);
                p.weights[at + s * LANES] = is ? value[s] * scale : 0.f;
                p.experts[at + s * LANES] = is ? int32_t(e) : -1;
                if (is) atomicAdd(count + e, 1u);
            }
        }
        routed += live && lane == 0;
        __syncwarp();
    }

    if (routed) atomicAdd(&routed_block, uint32_t(routed));
    __syncthreads();
    // an expert's sum over the block: its register of its lane in every row of every warp
    const auto block_share = [&](uint32_t e) {
        const uint32_t vec = e / L::kV, of_lane = vec % LANES, i = vec / LANES * L::kV + e % L::kV;
        const float* at = reinterpret_cast<const float*>(all_sums + (i / 4) * kWarp + of_lane) + i % 4;
        float sum = 0.f;
        for (int w = 0; w < kWarps; ++w)
#pragma unroll
            for (int r = 0; r < L::kRows; ++r) sum += at[(w * (C / 4) * kWarp + r * LANES) * 4];
        return sum;
    };
    if (gridDim.x == 1) {
        if (threadIdx.x == 0) p.ctrl[1] = 0;
        finish(p, routed_block, false, scratch, [&](uint32_t e) { return double(block_share(e)); },
               [&](uint32_t e) { return count[e]; });
        return;
    }
    // the totals are cleared by the launch before this one, which may still run
    wait_for_previous();
    for (uint32_t e = threadIdx.x; e < n; e += kThreads) {
        const float sum = block_share(e);
        if (!(sum < INFINITY)) atomicOr(p.ctrl + 2, 1u);
        else if (sum > 0.f) {
            const int scale = share_scale(sum);
            atomicAdd(p.share_total + scale * n + e, (unsigned long long)(__double2ull_rn(double(sum) * share_units(scale, 1))));
        }
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
           [&](uint32_t e) {
               double share = 0.0;
#pragma unroll
               for (int scale = kShareScales - 1; scale >= 0; --scale)
                   share += double(__ldcg(p.share_total + scale * n + e)) * share_units(scale, -1);
               return share;
           },
           [&](uint32_t e) { return __ldcg(p.count_total + e); });
}

// The first lane of the row that says it leads (its first lane, if none does).
template <int LANES>
__device__ __forceinline__ int leading_lane(bool leads, int sub)
{
    const uint32_t lanes = __ballot_sync(~0u, leads) >> (sub * LANES) & uint32_t((uint64_t(1) << LANES) - 1);
    return sub * LANES + (lanes ? __ffs(lanes) - 1 : 0);
}

// The largest logit left in a row's tile and its slope.  Rarely needed, so it
// reads the tile again instead of keeping it; out of line, it also takes the
// pressure off the sigmoid kernels' registers (131072 rows of 256 bfloat16: 160
// bytes of spills and 41.4 us before, none and 39.7 now).
template <typename T, int LANES, int C>
__device__ __noinline__ float2 leader_left(const uint4* tile, const float* pull, int wl)
{
    using L = Tile<T, LANES, C>;
    const int lane = wl % LANES, sub = wl / LANES;
    float top = kNegInf, slope = 0.f;
#pragma unroll 4
    for (int i = 0; i < C; ++i) {
        const float x = to_float(reinterpret_cast<const T*>(tile + i / L::kV * kWarp + wl)[i % L::kV]);
        if (x > top) {
            top = x;
            slope = pull[L::expert(lane, i)];
        }
    }
    const float row_top = row_all<LANES>(top, Max{});
    return {row_top, __shfl_sync(~0u, slope, leading_lane<LANES>(top == row_top, sub))};
}

// With a sigmoid of 0.03 or more among the chosen, of which the others are at most
// 34 times, a row's slopes lose little by being taken relative to a chosen one's:
// the largest of the others is looked for below this logit only.
constexpr float kLedLogit = -3.5f;

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
    constexpr int kPlaces = L::kPlaces;
    extern __shared__ uint4 dynamic[];
    uint4* tiles = dynamic + warp * 2 * L::kSlots;
    float* pull = reinterpret_cast<float*>(dynamic + kWarps * 2 * L::kSlots);  // [kSpan]
    // the rows' chosen experts and upstream gradients, twice: [kRows][k] each
    const uint32_t row_k = L::kRows * k;
    uint32_t* ids = reinterpret_cast<uint32_t*>(pull + L::kSpan) + warp * 4 * row_k + sub * k + lane;
    float* ups = reinterpret_cast<float*>(ids + 2 * row_k);
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

    // a row past the last token works on what its tile holds and writes nothing
    const uint32_t tokens = uint32_t(p.tokens), step = gridDim.x * kWarps * L::kRows;
    uint32_t t = (blockIdx.x * kWarps + warp) * L::kRows + sub;
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    T* out = static_cast<T*>(p.grad_logits) + t * p.grad_stride;
    const uint64_t row_step = step * p.stride, out_step = step * p.grad_stride;
    const auto fetch = [&](uint32_t token, int stage) {
        L::fetch(tiles + stage * L::kSlots, row, wl, n, p.unit);
        const uint32_t at = token * k + lane;
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            if (uint32_t(s * LANES + lane) < k) {
                copy_async<4>(ids + stage * row_k + s * LANES, p.experts + at + s * LANES);
                if (p.grad_weights) copy_async<4>(ups + stage * row_k + s * LANES, p.grad_weights + at + s * LANES);
            }
        }
    };
    if (t < tokens) fetch(t, 0);
    copies_commit();
    for (int stage = 0; t - sub < tokens; t += step, stage ^= 1, out += out_step) {
        const bool inside = t < tokens;
        uint4* tile = tiles + stage * L::kSlots;
        row += row_step;
        if (t + step < tokens) fetch(t + step, stage ^ 1);
        copies_commit();
        copies_wait();
        __syncwarp();

        // the chosen experts leave the tile
        uint32_t id[kPlaces];
        float value[kPlaces], up[kPlaces], chosen_top = kNegInf;
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            id[s] = ~0u;
            value[s] = kNegInf;
            up[s] = 0.f;
            if (uint32_t(s * LANES) >= k) break;
            if (inside && uint32_t(s * LANES + lane) < k) id[s] = ids[stage * row_k + s * LANES];
            if (id[s] < n) {
                T* at = L::element(tile, sub, id[s]);
                value[s] = to_float(*at);
                *at = from_float<T>(kNegInf);
                if (p.grad_weights) up[s] = ups[stage * row_k + s * LANES];
            }
            chosen_top = fmaxf(chosen_top, value[s]);
        }
        const bool live = int32_t(__shfl_sync(~0u, id[0], sub * LANES)) >= 0;
        // The expert with most of the row's share: slopes and upstream gradients
        // are taken relative to its own, so that what is left of a row that one
        // expert dominates is not the difference of two nearly equal numbers.
        // Here the one with most of it among the chosen; where a bias kept a
        // larger one out, that one's slope takes its place below.
        const float lane_top = chosen_top;
        chosen_top = row_all<LANES>(chosen_top, Max{});
        float pull0 = 0.f, up0 = 0.f;
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            if (id[s] < n && value[s] == lane_top) {
                pull0 = pull[id[s]];
                up0 = up[s];
            }
        }
        const int lead = leading_lane<LANES>(lane_top == chosen_top, sub);
        pull0 = __shfl_sync(~0u, pull0, lead);
        up0 = __shfl_sync(~0u, up0, lead);
        const float c = p.weight_scale;

        __syncwarp();
        float x[C], top = 0.f;
        L::unpack(tile, wl, x);
        bool outside = false;
        float lane_left = 0.f, left = 0.f;
        if (!SIGMOID) {
            lane_left = lane_max(x);
            left = row_all<LANES>(lane_left, Max{});
            outside = left > chosen_top;
            top = fmaxf(left, chosen_top);
        }
        const Reference ref(top, outside);
        if constexpr (!SIGMOID) {
            if (ref.any_rare) {
                float slope = 0.f;
#pragma unroll
                for (int i = 0; i < C; ++i)
                    if (x[i] == left) slope = pull[L::expert(lane, i)];
                slope = __shfl_sync(~0u, slope, leading_lane<LANES>(lane_left == left, sub));
                if (outside) pull0 = slope;
                if (kJoined && outside) up0 = 0.f;  // the leader has no weight
            }
        }
        float base = kJoined ? fmaf(c, up0, pull0) : pull0;
        // the scores' sum, and the mean slope before it is divided by that
        float mean = 0.f, score[kPlaces], sum;
        if constexpr (SIGMOID) {
            sum = sigmoid_slopes<L, false>(x, pull, lane, base, 0.f, false, mean);
        } else {
            sum = softmax_scores(x, ref);
            float2 m = both(0.f);
#pragma unroll
            for (int q = 0; q < C; q += 4) {
                const float4 h = shared_load4(pull + L::expert(lane, q));
                m = fma2(pair_of(x, q), add2({h.x, h.y}, both(-base)), m);
                m = fma2(pair_of(x, q + 2), add2({h.z, h.w}, both(-base)), m);
            }
            mean = m.x + m.y;
        }
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            score[s] = SIGMOID ? sigmoid(value[s]) : ref.score(value[s]);
            sum += score[s];
        }
        sum = row_all<LANES>(sum, Add{});
        bool deep = false;
        if constexpr (SIGMOID) {
            deep = sum < kDeepSigmoid;
            bool again = deep;
            const bool led = live && chosen_top < kLedLogit;
            if (__any_sync(~0u, led)) {
                const float2 leader = leader_left<T, LANES, C>(tile, pull, wl);
                if (led && leader.x > chosen_top) {
                    base = pull0 = leader.y;
                    again = true;
                }
            }
            if (__any_sync(~0u, again)) {
                L::unpack(tile, wl, x);
                top = row_all<LANES>(fmaxf(lane_max(x), lane_top), Max{});
                sum = sigmoid_slopes<L, true>(x, pull, lane, base, top, deep, mean);
#pragma unroll
                for (int s = 0; s < kPlaces; ++s) {
                    if (uint32_t(s * LANES) >= k) break;
                    score[s] = deep ? exp_of(value[s] - top) : sigmoid(value[s]);
                    sum += score[s];
                }
                sum = row_all<LANES>(sum, Add{});
            }
        }
        const float inv = __fdividef(1.f, sum);

        // a chosen expert's slope of the loss (and, joined, of its weight)
        float slope[kPlaces];
        float weights = 0.f, dot = 0.f, share[kPlaces];  // of renormalised weights: sum r, sum r (g - g0)
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            slope[s] = share[s] = 0.f;
            if (kJoined || RENORM) up[s] -= up0;
            if (id[s] < n) {
                slope[s] = pull[id[s]] - pull0;
                if (kJoined) slope[s] = fmaf(c, up[s], slope[s]);
                mean = fmaf(score[s], slope[s], mean);
                if (RENORM) {
                    share[s] = weight_score<SIGMOID>(value[s], chosen_top);
                    weights += share[s];
                    dot = fmaf(share[s], up[s], dot);
                }
            }
        }
        mean = row_all<LANES>(mean, Add{}) * inv;
        if (RENORM) {
            weights = row_all<LANES>(weights, Add{});
            dot = row_all<LANES>(dot, Add{});
        }

#pragma unroll
        for (int v = 0; v < L::kVecs; ++v) {
            const uint32_t e0 = L::expert(lane, v * L::kV);
            float g[L::kV];
#pragma unroll
            for (int q = 0; q < L::kV; q += 4) {
                const float4 h = shared_load4(pull + e0 + q);
                const float2 low = add2(add2({h.x, h.y}, both(-base)), both(-mean));
                const float2 high = add2(add2({h.z, h.w}, both(-base)), both(-mean));
                const float2 g0 = mul2(mul2(pair_of(x, v * L::kV + q), both(inv)), low);
                const float2 g1 = mul2(mul2(pair_of(x, v * L::kV + q + 2), both(inv)), high);
                g[q] = g0.x;
                g[q + 1] = g0.y;
                g[q + 2] = g1.x;
                g[q + 3] = g1.y;
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
#pragma unroll
        for (int s = 0; s < kPlaces; ++s) {
            if (uint32_t(s * LANES) >= k) break;
            if (id[s] >= n || !live) continue;  // a token without its first choice has zeros, stored above
            const float flat = SIGMOID ? sigmoid(-value[s]) : 1.f;  // 1 - s
            float d = flat * score[s] * inv * (slope[s] - mean);
            if (RENORM) {
                const float part = __fdividef(share[s], weights);
                d = fmaf(c * flat * part, up[s] - __fdividef(dot, weights), d);
            } else if (SIGMOID) {
                d = fmaf(c * up[s] * flat, sigmoid(value[s]), d);
            }
            out[id[s]] = from_float<T>(d);
        }
        __syncwarp();
    }
}

// Temp storage: the control words, the share totals, the count totals.
constexpr size_t kShareOffset = kTempAlign;
inline size_t cleared_bytes(uint32_t experts) { return kShareOffset + size_t(experts) * (kShareScales * 8 + 4); }

__global__ void __launch_bounds__(kThreads) clear_kernel(uint32_t* words, uint32_t n);

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
    const size_t fixed = size_t(kWarps) * (2 * L::kSlots * 16 + kWarp * C * 4), smem = fixed + (p.bias ? L::kSpan : 0) * 4 + size_t(p.num_experts) * 4;
    const auto by = [&](auto is_sigmoid) -> void (*)(Params) {
        constexpr bool kSigmoid = decltype(is_sigmoid)::value;
        if (!p.bias) return forward_kernel<T, LANES, C, kSigmoid, kByLogit>;
        return p.bias_on_score ? forward_kernel<T, LANES, C, kSigmoid, kByBiasedScore>
                               : forward_kernel<T, LANES, C, kSigmoid, kByBiasedLogit>;
    };
    void (*kernel)(Params) = sigmoid ? by(std::true_type{}) : by(std::false_type{});
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, fixed + L::kSpan * 8);
    const unsigned grid = grid_for(f, smem, p.tokens, kWarps * L::kRows);
    if (grid == 1) {
        kernel<<<1, kThreads, smem, s>>>(p);
        return launched();
    }
    // The totals are cleared by a small launch of their own, which the kernel
    // only waits for before it first adds to them.
    clear_kernel<<<1, kThreads, 0, s>>>(p.ctrl, uint32_t(cleared_bytes(p.num_experts) / 4));
    return launch_early(kernel, grid, kThreads, smem, s, p);
}

template <typename T, int LANES, int C>
lcpp_status backward_shape(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    using L = Tile<T, LANES, C>;
    const size_t fixed = size_t(kWarps) * 2 * L::kSlots * 16 + L::kSpan * 4;
    const size_t smem = fixed + size_t(kWarps) * 4 * L::kRows * p.top_k * 4;
    void (*kernel)(BackParams) =
        sigmoid ? (p.renormalize ? backward_kernel<T, LANES, C, true, true> : backward_kernel<T, LANES, C, true, false>)
                : (p.renormalize ? backward_kernel<T, LANES, C, false, true> : backward_kernel<T, LANES, C, false, false>);
    const void* f = reinterpret_cast<const void*>(kernel);
    set_max_dynamic_smem(f, fixed + size_t(kWarps) * 4 * L::kRows * LCPP_MAX_TOP_K * 4);
    kernel<<<grid_for(f, smem, p.tokens, kWarps * L::kRows), kThreads, smem, s>>>(p);
    return launched();
}

// The smallest shape that holds the experts, of those that measured best
// (bfloat16; lanes x elements): few lanes share a round's shuffles among more
// rows, many elements take registers.  131072 rows of 256: 8 x 32 44 us, 16 x 16
// 64, 4 x 64 62; of 64: 4 x 16 20, 8 x 8 23, 8 x 16 29; of 8: 1 x 8 8, 4 x 8 12.
template <typename T>
lcpp_status forward_rows(const Params& p, bool sigmoid, cudaStream_t s)
{
    const uint32_t n = p.num_experts;
    if (n <= 8) return forward_shape<T, 1, 8>(p, sigmoid, s);
    if (n <= 16) return forward_shape<T, 2, 8>(p, sigmoid, s);
    if (n <= 32) return forward_shape<T, 4, 8>(p, sigmoid, s);
    if (n <= 64) return forward_shape<T, 4, 16>(p, sigmoid, s);
    if (n <= 128) return forward_shape<T, 8, 16>(p, sigmoid, s);
    if (n <= 256) return forward_shape<T, 8, 32>(p, sigmoid, s);
    if (n <= 512) return forward_shape<T, 16, 32>(p, sigmoid, s);
    return forward_shape<T, 32, 32>(p, sigmoid, s);
}

// The same for the gradient.  131072 rows of 256: 8 x 32 42 us (40 now), 16 x 16 47, 32 x 8
// 61; of 64: 8 x 8 17, 4 x 16 17 (but 47 against 29 for 61 experts, whose rows
// allow no wide access), 8 x 16 23; 65536 of 512: 16 x 32 36, 32 x 16 38.
template <typename T>
lcpp_status backward_rows(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    const uint32_t n = p.num_experts;
    if (n <= 8) return backward_shape<T, 1, 8>(p, sigmoid, s);
    if (n <= 16) return backward_shape<T, 2, 8>(p, sigmoid, s);
    if (n <= 32) return backward_shape<T, 4, 8>(p, sigmoid, s);
    if (n <= 64) return backward_shape<T, 8, 8>(p, sigmoid, s);
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
