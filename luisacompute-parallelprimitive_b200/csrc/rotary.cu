// rotary.cu -- DeviceRotary (include/lcpp_b200_model.h): queries and keys turned
// by their positions, and keys and values written to their slots of a paged cache.
//
// A pair (a, b) at angle t = position * f becomes scale * (a cos t - b sin t,
// b cos t + a sin t); the gradient is the same with -t.  The angle is taken in
// 64 bits as a number of turns, whose fraction alone goes to sincospi in 32: a
// position of 10^6 leaves a 32-bit angle 4 bits of fraction.  A block takes a
// few tokens, computes their cosines and sines once into shared memory (half a
// head's columns each, next to nothing beside the heads that use them), and its
// threads turn vectors of pairs; a thread's first loads are on their way while
// it works on the angles.
//
// Bound by memory: every element is read once and written once.
#include "cache.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;                 // vectors that a thread loads before the angles are ready
constexpr int kMaxTokens = 16;            // tokens of a block
constexpr uint32_t kItemsPerBlock = kThreads * kAhead;

struct Section {
    const void* in;
    void* out;
    uint64_t in_token, in_head, out_token, out_head;
    uint32_t items;  // vectors of all heads of a token
    uint32_t copied; // 0: the columns past rotary_dim are in place already
};

struct Params {
    Section s[3];  // q, k, v
    const int32_t* positions;
    const int32_t* token_request;
    const int32_t* position_offset;
    const double* frequencies;
    const int64_t* slots;
    int32_t* slot_positions;
    float* slot_scores;
    uint64_t num_slots;
    uint64_t page_stride;
    uint32_t block_size;
    uint32_t tokens, requests;
    uint32_t half;       // rotary_dim / 2
    uint32_t turned;     // vectors (of pairs) of a head that are turned
    uint32_t per_head;   // and those with the ones that are copied
    uint32_t plain;      // vectors of a head of v
    uint32_t items;      // vectors of a token
    uint32_t per_block;  // tokens of a block
    float scale, sign;
};

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = unsigned short; };

// N adjacent elements.
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T e[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load(const T* p)
{
    using R = typename Raw<N * int(sizeof(T))>::type;
    union {
        R raw;
        Pack<T, N> pack;
    } u;
    u.raw = *reinterpret_cast<const R*>(p);
    return u.pack;
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Pack<T, N>& v)
{
    using R = typename Raw<N * int(sizeof(T))>::type;
    union {
        R raw;
        Pack<T, N> pack;
    } u;
    u.pack = v;
    *reinterpret_cast<R*>(p) = u.raw;
}

// One order of roundings, so that a pair's bits do not depend on the vector it is part of.
template <typename T>
__device__ __forceinline__ void turn_pair(float2 cs, float x, float y, T& a, T& b)
{
    a = from_float<T>(fmaf(x, cs.x, -__fmul_rn(y, cs.y)));
    b = from_float<T>(fmaf(y, cs.x, __fmul_rn(x, cs.y)));
}

// One vector's work: where it comes from and goes to, and its first angle.
// kHalf: N pairs (i, i + half), two vectors apart; else N / 2 adjacent pairs, or
// for N = 1 one pair as two elements.
template <typename T>
struct Item {
    const T* in;
    T* out;
    int angle;  // in the block's table; below 0: copied
    bool live;
};

template <typename T, int N, bool kHalf, bool kAppend>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Params p)
{
    extern __shared__ float2 turn[];  // [per_block][half] cosine and sine with the scale
    __shared__ int64_t place_of[kMaxTokens];  // elements from the cache's start; below 0: the token is left out
    constexpr int kElements = kHalf ? N : (N == 1 ? 2 : N);
    const uint32_t first = blockIdx.x * p.per_block, tokens = min(p.per_block, p.tokens - first);

    if (threadIdx.x < tokens) {
        const uint32_t t = first + threadIdx.x;
        int64_t slot = 0;
        if (kAppend) {
            slot = p.slots[t];
            if (uint64_t(slot) >= p.num_slots) slot = -1;
        }
        int64_t position = p.positions[t];
        if (p.token_request) {
            const int32_t r = p.token_request[t];
            if (uint32_t(r) >= p.requests) slot = -1;
            else if (p.position_offset) position += p.position_offset[r];
        }
        int64_t place = slot;
        if (kAppend && slot >= 0) {
            const uint64_t page = uint64_t(slot) / p.block_size;
            place = int64_t(page * p.page_stride + (uint64_t(slot) - page * p.block_size) * p.s[1].out_token);
        }
        place_of[threadIdx.x] = place;
        if (kAppend && slot >= 0) {
            if (p.slot_positions) p.slot_positions[slot] = int32_t(position);
            if (p.slot_scores) p.slot_scores[slot] = 0.f;
        }
    }
    __syncthreads();

    const auto item_at = [&](uint32_t i) {
        Item<T> item{nullptr, nullptr, -1, false};
        if (i >= tokens * p.items) return item;
        const uint32_t t = i / p.items;
        uint32_t rest = i - t * p.items;
        const int64_t place = place_of[t];
        if (place < 0) return item;
        int s = 0;
        if (rest >= p.s[0].items) {
            rest -= p.s[0].items;
            s = 1;
            if (kAppend && rest >= p.s[1].items) {
                rest -= p.s[1].items;
                s = 2;
            }
        }
        const Section& c = p.s[s];
        const uint32_t wide = kAppend && s == 2 ? p.plain : p.per_head;
        const uint32_t head = rest / wide;
        uint32_t j = rest - head * wide;
        uint32_t column;
        if ((!kAppend || s < 2) && j < p.turned) {
            item.angle = int(t * p.half + (kHalf ? j * N : j * (kElements / 2)));
            column = kHalf ? j * N : j * kElements;
        } else {
            if (!c.copied) return item;
            column = kAppend && s == 2 ? j * N : 2 * p.half + (j - p.turned) * N;
        }
        item.live = true;
        item.in = static_cast<const T*>(c.in) + uint64_t(first + t) * c.in_token + head * c.in_head + column;
        const uint64_t to = kAppend && s > 0 ? uint64_t(place) : uint64_t(first + t) * c.out_token;
        item.out = static_cast<T*>(c.out) + to + head * c.out_head + column;
        return item;
    };
    using P = Pack<T, N>;
    const auto fetch = [&](const Item<T>& item, P& a, P& b) {
        if (!item.live) return;
        a = load<T, N>(item.in);
        if (item.angle >= 0) {
            if (kHalf) b = load<T, N>(item.in + p.half);
            else if (N == 1) b = load<T, N>(item.in + 1);
        }
    };
    const auto finish = [&](const Item<T>& item, P a, P b) {
        if (!item.live) return;
        if (item.angle < 0) {
            store<T, N>(item.out, a);
            return;
        }
        if (kHalf || N == 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 cs = turn[item.angle + i];
                const float x = to_float(a.e[i]), y = to_float(b.e[i]);
                turn_pair(cs, x, y, a.e[i], b.e[i]);
            }
            store<T, N>(item.out, a);
            store<T, N>(item.out + (kHalf ? p.half : 1), b);
        } else {
#pragma unroll
            for (int i = 0; i + 1 < N; i += 2) {
                const float2 cs = turn[item.angle + i / 2];
                const float x = to_float(a.e[i]), y = to_float(a.e[i + 1]);
                turn_pair(cs, x, y, a.e[i], a.e[i + 1]);
            }
            store<T, N>(item.out, a);
        }
    };

    Item<T> item[kAhead];
    P a[kAhead], b[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        item[i] = item_at(threadIdx.x + i * kThreads);
        fetch(item[i], a[i], b[i]);
    }
    for (uint32_t i = threadIdx.x; i < tokens * p.half; i += kThreads) {
        const uint32_t t = i / p.half;
        int64_t position = p.positions[first + t];
        if (p.position_offset) {
            const int32_t r = p.token_request[first + t];
            if (uint32_t(r) < p.requests) position += p.position_offset[r];
        }
        // turns = position * f / 2 pi, whose whole part is dropped before 32 bits
        const double turns = double(position) * (p.frequencies[i - t * p.half] * 0.15915494309189533577);
        float sine, cosine;
        sincospif(2.f * float(turns - rint(turns)), &sine, &cosine);
        turn[i] = make_float2(p.scale * cosine, p.sign * sine);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) finish(item[i], a[i], b[i]);
    for (uint32_t i = threadIdx.x + kItemsPerBlock; i < tokens * p.items; i += kThreads) {
        const Item<T> more = item_at(i);
        P x, y;
        fetch(more, x, y);
        finish(more, x, y);
    }
}

Strided rows_in(const lcpp_head_rows& r, uint64_t tokens, uint32_t dim, int e)
{
    return Strided(r.in, e, dim, {{tokens, r.in_token_stride}, {r.num_heads, r.in_head_stride}});
}
Strided rows_out(const lcpp_head_rows& r, uint64_t tokens, uint32_t dim, int e)
{
    return Strided(r.out, e, dim, {{tokens, r.out_token_stride}, {r.num_heads, r.out_head_stride}});
}
Strided flat(const void* p, uint64_t n, int e) { return Strided(p, e, n, {}); }

template <typename T, int N, bool kHalf>
lcpp_status launch(const Params& p, bool append, cudaStream_t s)
{
    const unsigned grid = unsigned(ceil_div(p.tokens, p.per_block));
    const size_t smem = size_t(p.per_block) * p.half * sizeof(float2);
    if (append) rotary_kernel<T, N, kHalf, true><<<grid, kThreads, smem, s>>>(p);
    else rotary_kernel<T, N, kHalf, false><<<grid, kThreads, smem, s>>>(p);
    return launched();
}

template <typename T, int N>
lcpp_status launch(Params& p, const lcpp_rotary_args& a, bool append, cudaStream_t s)
{
    const bool half = a.layout == LCPP_ROTARY_HALF;
    const uint32_t in_vector = half ? N : (N == 1 ? 2 : N);
    p.turned = (half ? p.half : 2 * p.half) / in_vector;
    p.per_head = p.turned + (a.head_dim - a.rotary_dim) / N;
    p.plain = a.head_dim / N;
    p.s[0].items = a.q.num_heads * p.per_head;
    p.s[1].items = a.k.num_heads * p.per_head;
    p.s[2].items = append ? a.k.num_heads * p.plain : 0;
    p.items = p.s[0].items + p.s[1].items + p.s[2].items;
    // as many tokens as the loads ahead cover, when there are tokens for every SM
    const uint32_t fit = std::max<uint32_t>(1, kItemsPerBlock / std::max<uint32_t>(1, p.items));
    const uint32_t spread = uint32_t(ceil_div(p.tokens, uint64_t(device_sm_count()) * 4));
    p.per_block = std::min<uint32_t>({fit, std::max<uint32_t>(spread, 1), uint32_t(kMaxTokens)});
    return half ? launch<T, N, true>(p, append, s) : launch<T, N, false>(p, append, s);
}

lcpp_status run(const lcpp_rotary_args* a, const lcpp_cache_append_args* c, float sign, cudaStream_t s)
{
    if (!a || !a->head_dim || a->head_dim > LCPP_MAX_HEAD_DIM || a->rotary_dim % 2 || a->rotary_dim > a->head_dim ||
        a->num_tokens >= uint64_t(1) << 31 || (a->layout != LCPP_ROTARY_HALF && a->layout != LCPP_ROTARY_INTERLEAVED))
        return LCPP_ERR_INVALID_ARG;
    const int e = row_dtype_bytes(a->dtype);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    const uint64_t n = a->num_tokens;
    const lcpp_head_rows* rows[2] = {&a->q, &a->k};
    // a head is at most 256 columns; the vectors of a token are counted in 32 bits
    if (uint64_t(a->q.num_heads) + 2 * uint64_t(a->k.num_heads) > uint64_t(1) << 22) return LCPP_ERR_INVALID_ARG;
    for (const lcpp_head_rows* r : rows)
        if (r->in_token_stride > kMostStride || r->in_head_stride > kMostStride || r->out_token_stride > kMostStride ||
            r->out_head_stride > kMostStride)
            return LCPP_ERR_INVALID_ARG;
    if (c) {
        if (!sane_cache(c->cache) || c->cache.num_kv_heads != a->k.num_heads || c->cache.head_dim != a->head_dim ||
            c->cache.dtype != a->dtype || c->v_token_stride > kMostStride || c->v_head_stride > kMostStride)
            return LCPP_ERR_INVALID_ARG;
    }
    if (a->position_offset && !a->token_request) return LCPP_ERR_INVALID_ARG;
    if (!n || (!a->q.num_heads && !a->k.num_heads)) return LCPP_OK;
    if (!a->positions || (a->rotary_dim && !a->frequencies)) return LCPP_ERR_INVALID_ARG;
    if (misaligned(a->positions, 4) || misaligned(a->token_request, 4) || misaligned(a->position_offset, 4) ||
        misaligned(a->frequencies, 8))
        return LCPP_ERR_INVALID_ARG;

    // what is read, and what is written
    std::vector<Strided> in{flat(a->positions, n, 4), flat(a->token_request, n, 4),
                            flat(a->position_offset, a->position_offset ? a->num_requests : 0, 4),
                            flat(a->frequencies, a->rotary_dim / 2, 8)};
    std::vector<Strided> out;
    for (int i = 0; i < 2; ++i) {
        const lcpp_head_rows& r = *rows[i];
        if (!r.num_heads) continue;
        const bool written = !c || i == 0;
        if (!r.in || misaligned(r.in, e) || (written && (!r.out || misaligned(r.out, e)))) return LCPP_ERR_INVALID_ARG;
        const Strided from = rows_in(r, n, a->head_dim, e);
        if (!from.sane()) return LCPP_ERR_INVALID_ARG;
        if (written) {
            const Strided to = rows_out(r, n, a->head_dim, e);
            if (!to.sane() || !to.distinct()) return LCPP_ERR_INVALID_ARG;
            out.push_back(to);
        }
        const bool in_place = written && r.in == r.out && r.in_token_stride == r.out_token_stride &&
                              r.in_head_stride == r.out_head_stride;
        if (!in_place) in.push_back(from);
    }
    Params p{};
    if (c) {
        const uint64_t slots = uint64_t(c->cache.num_pages) * c->cache.block_size;
        if (!c->v || !c->slots || misaligned(c->v, e) || misaligned(c->slots, 8) || misaligned(c->slot_positions, 4) ||
            misaligned(c->slot_scores, 4))
            return LCPP_ERR_INVALID_ARG;
        if (slots && (!c->cache.k || !c->cache.v || misaligned(c->cache.k, e) || misaligned(c->cache.v, e) ||
                      !writable_cache(c->cache)))
            return LCPP_ERR_INVALID_ARG;
        const Strided v(c->v, e, a->head_dim, {{n, c->v_token_stride}, {a->k.num_heads, c->v_head_stride}});
        if (!v.sane()) return LCPP_ERR_INVALID_ARG;
        in.push_back(v);
        in.push_back(flat(c->slots, n, 8));
        // k and v of a page may lie side by side: they are checked against each other above
        const Strided pages[] = {pages_of(c->cache, c->cache.k), pages_of(c->cache, c->cache.v)};
        const Strided arrays[] = {flat(c->slot_positions, c->slot_positions ? slots : 0, 4),
                                  flat(c->slot_scores, c->slot_scores ? slots : 0, 4)};
        for (const Strided& page : pages) {
            for (const Strided& x : in)
                if (overlap(page.p, page.bytes(), x.p, x.bytes())) return LCPP_ERR_INVALID_ARG;
            for (const Strided& x : out)
                if (overlap(page.p, page.bytes(), x.p, x.bytes())) return LCPP_ERR_INVALID_ARG;
            for (const Strided& x : arrays)
                if (overlap(page.p, page.bytes(), x.p, x.bytes())) return LCPP_ERR_INVALID_ARG;
        }
        for (const Strided& x : arrays) out.push_back(x);
        p.slots = c->slots;
        p.slot_positions = c->slot_positions;
        p.slot_scores = c->slot_scores;
        p.num_slots = slots;
        p.page_stride = c->cache.page_stride;
        p.block_size = c->cache.block_size;
        p.s[2] = Section{c->v, c->cache.v, c->v_token_stride, c->v_head_stride, c->cache.token_stride,
                         c->cache.head_stride, 0, 1};
    }
    for (size_t i = 0; i < out.size(); ++i) {
        for (const Strided& x : in)
            if (may_share(out[i], x)) return LCPP_ERR_INVALID_ARG;
        for (size_t j = 0; j < i; ++j)
            if (may_share(out[i], out[j])) return LCPP_ERR_INVALID_ARG;
    }

    for (int i = 0; i < 2; ++i) {
        const lcpp_head_rows& r = *rows[i];
        const bool cached = c && i == 1;
        p.s[i] = Section{r.in,
                         cached ? c->cache.k : r.out,
                         r.in_token_stride,
                         r.in_head_stride,
                         cached ? c->cache.token_stride : r.out_token_stride,
                         cached ? c->cache.head_stride : r.out_head_stride,
                         0,
                         uint32_t(cached || r.in != r.out)};
    }
    p.positions = a->positions;
    p.token_request = a->token_request;
    p.position_offset = a->position_offset;
    p.frequencies = a->frequencies;
    p.tokens = uint32_t(n);
    p.requests = a->token_request ? a->num_requests : 0;
    p.half = a->rotary_dim / 2;
    p.scale = a->scale;
    p.sign = sign * a->scale;

    // the widest vectors that all rows, the turned part and the rest allow
    const auto fits = [&](int count) {
        const size_t bytes = size_t(count) * e;
        const uint32_t unit = a->layout == LCPP_ROTARY_HALF ? p.half : a->rotary_dim;
        if (unit % count || a->head_dim % count) return false;
        for (int i = 0; i < 2; ++i) {
            const Section& x = p.s[i];
            if (rows[i]->num_heads && (!rows_aligned(x.in, {x.in_token, x.in_head}, e, bytes) ||
                                       !rows_aligned(x.out, {x.out_token, x.out_head}, e, bytes)))
                return false;
        }
        return !c || (rows_aligned(p.s[2].in, {p.s[2].in_token, p.s[2].in_head}, e, bytes) &&
                      rows_aligned(p.s[2].out, {p.s[2].out_token, p.s[2].out_head}, e, bytes) &&
                      rows_aligned(nullptr, {p.page_stride}, e, bytes));
    };
    diag::KernelTimer timer(kTimerRotary, n, s);
    return with_row_type(a->dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int kMost = 16 / int(sizeof(T));
        if (kMost == 8 && fits(8)) return launch<T, kMost>(p, *a, c, s);
        if (fits(4)) return launch<T, 4>(p, *a, c, s);
        if (fits(2)) return launch<T, 2>(p, *a, c, s);
        return launch<T, 1>(p, *a, c, s);
    });
}

}  // namespace

extern "C" {

lcpp_status lcpp_rotary_frequencies(double* out, uint32_t rotary_dim, double base, int32_t scaling, double factor,
                                    double original_context, double low, double high)
{
    if (!out || rotary_dim % 2 || rotary_dim > LCPP_MAX_HEAD_DIM || !(base > 0) || !std::isfinite(base) ||
        scaling < LCPP_ROTARY_PLAIN || scaling > LCPP_ROTARY_BY_ROTATIONS)
        return LCPP_ERR_INVALID_ARG;
    if (scaling != LCPP_ROTARY_PLAIN && (!(factor >= 1) || !std::isfinite(factor))) return LCPP_ERR_INVALID_ARG;
    if (scaling == LCPP_ROTARY_BASE && rotary_dim == 2) return LCPP_ERR_INVALID_ARG;
    if (scaling == LCPP_ROTARY_BY_ROTATIONS &&
        (!(original_context > 0) || !std::isfinite(original_context) || !(low > 0) || !(low < high) || !std::isfinite(high)))
        return LCPP_ERR_INVALID_ARG;
    if (scaling == LCPP_ROTARY_BASE) base *= std::pow(factor, double(rotary_dim) / (rotary_dim - 2.0));
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (scaling == LCPP_ROTARY_LINEAR) f /= factor;
        if (scaling == LCPP_ROTARY_BY_ROTATIONS) {
            const double turns = original_context * f * 0.15915494309189533577;
            const double whole = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            f = (1 - whole) * f / factor + whole * f;
        }
        out[i] = f;
    }
    return LCPP_OK;
}

lcpp_status lcpp_rotary_forward(const lcpp_rotary_args* args, lcpp_stream_t stream)
{
    return guarded("lcpp_rotary_forward", [&] { return run(args, nullptr, 1.f, reinterpret_cast<cudaStream_t>(stream)); });
}

lcpp_status lcpp_rotary_backward(const lcpp_rotary_args* args, lcpp_stream_t stream)
{
    return guarded("lcpp_rotary_backward",
                   [&] { return run(args, nullptr, -1.f, reinterpret_cast<cudaStream_t>(stream)); });
}

lcpp_status lcpp_rotary_append(const lcpp_rotary_args* args, const lcpp_cache_append_args* append, lcpp_stream_t stream)
{
    return guarded("lcpp_rotary_append", [&] {
        if (!append) return LCPP_ERR_INVALID_ARG;
        return run(args, append, 1.f, reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
