// rotary.cu -- DeviceRotary (include/lcpp_b200_model.h): queries and keys turned
// by their positions, and keys and values written to their slots of a paged cache.
//
// A pair (a, b) at angle t = position * f becomes scale * (a cos t - b sin t,
// b cos t + a sin t); the gradient is the same with -t.  The angle is taken in
// 64 bits as a number of turns, whose fraction alone goes to sincospi in 32: a
// position of 10^6 leaves a 32-bit angle 4 bits of fraction.
//
// A team of 1 to 8 warps takes a token: each warp puts the token's cosines and
// sines into shared memory of its own (half a head's columns each, next to
// nothing beside the heads that use them) while its lanes' first vectors of pairs
// are on their way, and turns its share of the vectors.  No warp waits for
// another.
//
// Bound by memory: every element is read once and written once.  Turned columns and
// copied ones are walked one after the other, each with the widest access that its
// own start allows (together with the narrower one's: 32768 tokens of 40 heads of
// 128 whose first 42 columns are turned 444 us, apart 211).  32768 tokens of 40 heads
// of 128 in bfloat16: 107 us, 6.3 TB/s (a copy reaches 6.5); queries and the append
// of keys and values of as many tokens: 82 us for 537 MB; 64 tokens: 4.1 us.
#include "cache.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / kWarp;

// Vectors of a token that are turned or copied: of all heads, per_head of each.
struct Section {
    const void* in;
    void* out;
    uint64_t in_token, in_head, out_token, out_head;
    // From a lane's vector to its next one, 32 * team on, in elements; and what
    // is added where that lies in the next head.
    int64_t in_step, in_wrap, out_step, out_wrap;
    uint32_t vectors;         // of a token
    uint32_t step, per_head;  // a lane's step past whole heads, and a head's vectors
};

struct Params {
    Section turn[2];  // of q and k
    Section copy[3];  // their columns past rotary_dim, and v
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
    uint32_t turned;     // vectors of pairs of a head
    uint32_t team;       // warps that share a token, a power of two
    float scale, sign;
};

// N adjacent elements, as the 32-bit words of one access (two bytes in the low half of one).
template <typename T, int N>
struct Pack {
    static constexpr int kBytes = N * int(sizeof(T)), kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];
};
template <typename T, int N>
__device__ __forceinline__ void load(Pack<T, N>& v, const T* p)
{
    if constexpr (Pack<T, N>::kBytes == 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        v.w[0] = x.x, v.w[1] = x.y, v.w[2] = x.z, v.w[3] = x.w;
    } else if constexpr (Pack<T, N>::kBytes == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v.w[0] = x.x, v.w[1] = x.y;
    } else if constexpr (Pack<T, N>::kBytes == 4) {
        v.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        v.w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Pack<T, N>& v)
{
    if constexpr (Pack<T, N>::kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    else if constexpr (Pack<T, N>::kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(v.w[0], v.w[1]);
    else if constexpr (Pack<T, N>::kBytes == 4) *reinterpret_cast<uint32_t*>(p) = v.w[0];
    else *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(v.w[0]);
}
template <typename T, int N>
__device__ __forceinline__ void floats_of(const Pack<T, N>& v, float (&out)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) out[i] = __uint_as_float(v.w[i]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            out[i] = __uint_as_float(i % 2 ? v.w[i / 2] & 0xffff0000u : v.w[i / 2] << 16);
        else out[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(i % 2 ? v.w[i / 2] >> 16 : v.w[i / 2])));
    }
}
template <typename T, int N>
__device__ __forceinline__ void pack(Pack<T, N>& v, const float (&in)[N])
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) v.w[i] = __float_as_uint(in[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float high = N > 1 ? in[(i + 1) % N] : 0.f;
            if constexpr (std::is_same<T, __nv_bfloat16>::value)
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.w[i / 2]) : "f"(high), "f"(in[i]));
            else
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v.w[i / 2]) : "f"(high), "f"(in[i]));
        }
    }
}

// One order of roundings, so that a pair's bits do not depend on the vector it is part of.
__device__ __forceinline__ void turn_pair(float2 cs, float& a, float& b)
{
    const float x = a, y = b;
    a = fmaf(x, cs.x, -__fmul_rn(y, cs.y));
    b = fmaf(y, cs.x, __fmul_rn(x, cs.y));
}

// N: elements of an access to pairs, kCopy: to columns that are copied.
template <typename T, int N, bool kHalf, bool kAppend, int kCopy>
__global__ void __launch_bounds__(kThreads, kHalf && kAppend && Pack<T, N>::kBytes < 16 ? 3 : 4) rotary_kernel(const Params p)
{
    // kHalf: vectors of N pairs (i, i + half) in two places; else of N / 2 adjacent
    // pairs, or for N = 1 of one pair as two elements
    constexpr bool kTwo = kHalf || N == 1;  // a pair's second half is loaded by itself
    constexpr int kPairs = kHalf ? N : N == 1 ? 1 : N / 2;
    constexpr int kColumns = kHalf ? N : N == 1 ? 2 : N;  // from vector to vector
    // Vectors that a lane has under way: enough that loads cover the latency, few
    // enough that nothing spills. 32768 tokens of 32 + 8 heads of 128 in bfloat16:
    // halves 107 us with one (two loads each) and 118 with two; the first 42 columns
    // by elements 211 us with four and 242 with two; an interleaved append of 8191 tokens
    // 38.5 us with two, 41 with one, 47 with four.  Copied columns of 32768 appended
    // tokens of 192 columns, 64 turned: 134 us with two, 127.5 with three; without the
    // append (32 of 128 turned) 119 with two, 129 with three.
    constexpr bool kWide = Pack<T, N>::kBytes == 16, kNarrow = !kAppend && Pack<T, N>::kBytes <= 4;
    constexpr int kAhead = kHalf && kWide ? 1 : kNarrow ? 4 : 2, kCopies = kNarrow ? 4 : kAppend ? 3 : 2;
    extern __shared__ __align__(16) float2 tables[];  // [warp][half] cosine and sine with the scale
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    float2* turn = tables + warp * ((p.half + 1) / 2 * 2);
    const uint32_t worker = blockIdx.x * kWarps + warp, part = worker & (p.team - 1);
    const uint32_t teams = gridDim.x * kWarps / p.team;
    const uint32_t start = part * kWarp + lane;  // the lane's first vector

    for (uint32_t t = worker / p.team; t < p.tokens; t += teams) {
        int64_t position = p.positions[t], place = 0;
        bool live = true;
        if (kAppend) {
            const int64_t slot = p.slots[t];
            live = uint64_t(slot) < p.num_slots;
            if (live) {
                const uint64_t page = uint64_t(slot) / p.block_size;
                place = int64_t(page * p.page_stride + (uint64_t(slot) - page * p.block_size) * p.turn[1].out_token);
            }
        }
        if (p.token_request) {
            const int32_t r = p.token_request[t];
            if (uint32_t(r) >= p.requests) live = false;
            else if (p.position_offset) position += p.position_offset[r];
        }
        if (!live) continue;
        if (kAppend && part == 0 && lane == 0) {
            const int64_t slot = p.slots[t];
            if (p.slot_positions) p.slot_positions[slot] = int32_t(position);
            if (p.slot_scores) p.slot_scores[slot] = 0.f;
        }
        // The first vectors of q, or of k, are loaded before the angles are worked out.
        bool ready = false;
        const auto turn_all = [&](const Section& c, uint64_t to) {
            const uint32_t head = start / c.per_head;
            uint32_t j = start - head * c.per_head;
            const T* in = static_cast<const T*>(c.in) + t * c.in_token + head * c.in_head + j * kColumns;
            T* out = static_cast<T*>(c.out) + to + head * c.out_head + j * kColumns;
            for (uint32_t v = start; v - lane < c.vectors;) {  // the warp's lanes together
                Pack<T, N> a[kAhead], b[kAhead];
                T* at[kAhead];
                uint32_t angle[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    at[u] = nullptr;
                    angle[u] = j;
                    if (v < c.vectors) {
                        at[u] = out;
                        load(a[u], in);
                        if (kTwo) load(b[u], in + (kHalf ? p.half : 1));
                    }
                    v += p.team * kWarp;
                    in += c.in_step;
                    out += c.out_step;
                    j += c.step;
                    if (j >= c.per_head) {
                        j -= c.per_head;
                        in += c.in_wrap;
                        out += c.out_wrap;
                    }
                }
                if (!ready) {
                    for (uint32_t i = lane; i < p.half; i += kWarp) {
                        // turns = position * f / 2 pi, whose whole part is dropped before 32 bits
                        const double of = double(position) * (p.frequencies[i] * 0.15915494309189533577);
                        float sine, cosine;
                        sincospif(2.f * float(of - rint(of)), &sine, &cosine);
                        // two pairs of a vector together, those of the lanes' vectors side by side
                        const uint32_t to = kPairs == 1 ? i : (i % kPairs / 2 * p.turned + i / kPairs) * 2 + i % 2;
                        turn[to] = make_float2(p.scale * cosine, p.sign * sine);
                    }
                    __syncwarp();
                    ready = true;
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (!at[u]) continue;
                    float x[N], y[N];
                    floats_of(a[u], x);
                    if constexpr (kTwo) floats_of(b[u], y);
                    if constexpr (kPairs == 1) {
                        const float2 cs = turn[angle[u]];
                        if constexpr (kTwo) turn_pair(cs, x[0], y[0]);
                        else turn_pair(cs, x[0], x[1 % N]);
                    } else {
#pragma unroll
                        for (int i = 0; i < kPairs; i += 2) {
                            const float4 cs = *reinterpret_cast<const float4*>(turn + (i / 2 * p.turned + angle[u]) * 2);
                            if constexpr (kTwo) {
                                turn_pair(make_float2(cs.x, cs.y), x[i], y[i]);
                                turn_pair(make_float2(cs.z, cs.w), x[i + 1], y[i + 1]);
                            } else {
                                turn_pair(make_float2(cs.x, cs.y), x[i * 2], x[i * 2 + 1]);
                                turn_pair(make_float2(cs.z, cs.w), x[i * 2 + 2], x[i * 2 + 3]);
                            }
                        }
                    }
                    if constexpr (kTwo) {
                        pack(b[u], y);
                        store(at[u] + (kHalf ? p.half : 1), b[u]);
                    }
                    pack(a[u], x);
                    store(at[u], a[u]);
                }
            }
        };
        const auto copy_all = [&](const Section& c, uint64_t to) {
            const uint32_t head = start / c.per_head;
            uint32_t j = start - head * c.per_head;
            const T* in = static_cast<const T*>(c.in) + t * c.in_token + head * c.in_head + j * kCopy;
            T* out = static_cast<T*>(c.out) + to + head * c.out_head + j * kCopy;
            for (uint32_t v = start; v < c.vectors;) {
                Pack<T, kCopy> x[kCopies];
                T* at[kCopies];
#pragma unroll
                for (int u = 0; u < kCopies; ++u) {
                    at[u] = nullptr;
                    if (v < c.vectors) {
                        at[u] = out;
                        load(x[u], in);
                    }
                    v += p.team * kWarp;
                    in += c.in_step;
                    out += c.out_step;
                    j += c.step;
                    if (j >= c.per_head) {
                        j -= c.per_head;
                        in += c.in_wrap;
                        out += c.out_wrap;
                    }
                }
#pragma unroll
                for (int u = 0; u < kCopies; ++u)
                    if (at[u]) store(at[u], x[u]);
            }
        };
#pragma unroll 1
        for (int i = 0; i < 2; ++i) turn_all(p.turn[i], kAppend && i ? uint64_t(place) : t * p.turn[i].out_token);
#pragma unroll 1
        for (int i = 0; i < (kAppend ? 3 : 2); ++i)
            copy_all(p.copy[i], kAppend && i ? uint64_t(place) : t * p.copy[i].out_token);
        __syncwarp();  // the table is free
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

template <typename T, int N, bool kHalf, int kCopy>
lcpp_status launch(const Params& p, bool append, cudaStream_t s)
{
    auto kernel = append ? rotary_kernel<T, N, kHalf, true, kCopy> : rotary_kernel<T, N, kHalf, false, kCopy>;
    const size_t smem = size_t(kWarps) * align_up(p.half, 2) * sizeof(float2);
    // as for the longest tables, so that few launch shapes are looked up and kept
    const size_t room = size_t(kWarps) * (LCPP_MAX_HEAD_DIM / 2) * sizeof(float2);
    const uint64_t most = uint64_t(device_sm_count()) * resident_blocks(reinterpret_cast<const void*>(kernel), kThreads, room);
    const unsigned grid = unsigned(std::min<uint64_t>(most, ceil_div(uint64_t(p.tokens) * p.team, kWarps)));
    kernel<<<grid, kThreads, smem, s>>>(p);
    return launched();
}

template <typename T, int N>
lcpp_status launch(Params& p, const lcpp_rotary_args& a, int copy, bool append, cudaStream_t s)
{
    const bool half = a.layout == LCPP_ROTARY_HALF;
    const uint32_t columns = half ? N : N == 1 ? 2 : N, heads[2] = {a.q.num_heads, a.k.num_heads};
    p.turned = (half ? p.half : 2 * p.half) / columns;
    const uint32_t rest = (a.head_dim - a.rotary_dim) / copy;
    for (int i = 0; i < 2; ++i) {
        p.turn[i].per_head = std::max<uint32_t>(p.turned, 1);
        p.turn[i].vectors = heads[i] * p.turned;
        p.copy[i].per_head = std::max<uint32_t>(rest, 1);
        p.copy[i].vectors = p.copy[i].in == p.copy[i].out ? 0 : heads[i] * rest;  // in place
    }
    const uint32_t value = append ? a.head_dim / copy : 0;  // vectors of a head of v
    p.copy[2].per_head = std::max<uint32_t>(value, 1);
    p.copy[2].vectors = append ? a.k.num_heads * value : 0;
    // Warps to a token: of 1, 2, 4 and 8 the number that takes the shortest time, which
    // is the rounds of 32 warps on every SM times what one takes: its vectors' turns
    // and two more for the start and the table.  40 heads of 128 in bfloat16, 1 / 2 / 4
    // / 8 warps: 64 tokens 7.9 / 5.6 / 4.7 / 4.2 us (with the append), 1024 tokens 6.8 /
    // 5.6 / 5.5 / 7.5, 4096 tokens 17.7 / 17.8 / 19.6 / 25.4, 5003 tokens 26.0 / 22.9 /
    // 23.5 / 30.0, 32768 tokens 107 / 108 / 123 / 180.
    uint64_t least = ~0ull;
    for (uint32_t team = 1; team <= kWarps; team *= 2) {
        uint64_t turns = 2;
        for (const Section& c : p.turn) turns += ceil_div(c.vectors, team * kWarp);
        for (const Section& c : p.copy) turns += ceil_div(c.vectors, team * kWarp);
        const uint64_t time = ceil_div(uint64_t(p.tokens) * team, uint64_t(device_sm_count()) * 32) * turns;
        if (time < least) {
            least = time;
            p.team = team;
        }
    }
    const auto steps = [&](Section& c, uint32_t in_vector) {
        const uint32_t step = p.team * kWarp;
        c.step = step % c.per_head;
        const int64_t over = step / c.per_head;
        c.in_step = over * int64_t(c.in_head) + int64_t(c.step) * in_vector;
        c.out_step = over * int64_t(c.out_head) + int64_t(c.step) * in_vector;
        c.in_wrap = int64_t(c.in_head) - int64_t(c.per_head) * in_vector;
        c.out_wrap = int64_t(c.out_head) - int64_t(c.per_head) * in_vector;
    };
    for (Section& c : p.turn) steps(c, columns);
    for (Section& c : p.copy) steps(c, copy);
    constexpr int kWide = 16 / int(sizeof(T));
    if (copy == kWide) return half ? launch<T, N, true, kWide>(p, append, s) : launch<T, N, false, kWide>(p, append, s);
    if (copy == 4 / int(sizeof(T)) && copy > 1)
        return half ? launch<T, N, true, 4 / int(sizeof(T))>(p, append, s) : launch<T, N, false, 4 / int(sizeof(T))>(p, append, s);
    return half ? launch<T, N, true, 1>(p, append, s) : launch<T, N, false, 1>(p, append, s);
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
        p.copy[2].in = c->v;
        p.copy[2].out = c->cache.v;
        p.copy[2].in_token = c->v_token_stride;
        p.copy[2].in_head = c->v_head_stride;
        p.copy[2].out_token = c->cache.token_stride;
        p.copy[2].out_head = c->cache.head_stride;
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
        Section& x = p.turn[i];
        x.in = r.in;
        x.out = cached ? c->cache.k : r.out;
        x.in_token = r.in_token_stride;
        x.in_head = r.in_head_stride;
        x.out_token = cached ? c->cache.token_stride : r.out_token_stride;
        x.out_head = cached ? c->cache.head_stride : r.out_head_stride;
        p.copy[i] = x;
        if (r.num_heads) {
            p.copy[i].in = static_cast<const char*>(x.in) + size_t(a->rotary_dim) * e;
            p.copy[i].out = static_cast<char*>(x.out) + size_t(a->rotary_dim) * e;
        }
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

    // the widest accesses that the rows of pairs allow, and those of the columns that are copied
    const auto rows_fit = [&](const Section& x, size_t bytes) {
        return rows_aligned(x.in, {x.in_token, x.in_head}, e, bytes) && rows_aligned(x.out, {x.out_token, x.out_head}, e, bytes) &&
               (!c || rows_aligned(nullptr, {p.page_stride}, e, bytes));
    };
    const auto pairs_fit = [&](int count) {
        if ((a->layout == LCPP_ROTARY_HALF ? p.half : a->rotary_dim) % count) return false;
        for (int i = 0; i < 2; ++i)
            if (rows[i]->num_heads && !rows_fit(p.turn[i], size_t(count) * e)) return false;
        return true;
    };
    const auto copies_fit = [&](int count) {
        if ((a->head_dim - a->rotary_dim) % count || (c && a->head_dim % count)) return false;
        for (int i = 0; i < 2; ++i)
            if (rows[i]->num_heads && a->head_dim > a->rotary_dim && !rows_fit(p.copy[i], size_t(count) * e)) return false;
        return !c || rows_fit(p.copy[2], size_t(count) * e);
    };
    diag::KernelTimer timer(kTimerRotary, n, s);
    return with_row_type(a->dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int kMost = 16 / int(sizeof(T)), kWord = 4 / int(sizeof(T));
        const int copy = copies_fit(kMost) ? kMost : copies_fit(kWord) ? kWord : 1;
        if (kMost == 8 && pairs_fit(8)) return launch<T, kMost>(p, *a, copy, c, s);
        if (pairs_fit(4)) return launch<T, 4>(p, *a, copy, c, s);
        if (pairs_fit(2)) return launch<T, 2>(p, *a, copy, c, s);
        return launch<T, 1>(p, *a, copy, c, s);
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
