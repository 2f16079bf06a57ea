// block_table.cu -- DeviceBlockTable (include/lcpp_b200_model.h): pages, slots
// and positions of one step's tokens, from the requests' lengths.
//
// With B the page size, ctx and new a request's lengths, it holds
// ceil(ctx / B) pages and needs ceil((ctx + new) / B); two exclusive sums over
// the requests (new tokens, new pages) give each its place in the packed
// tokens and in the free list.  A token of position p reads one page id, from
// the request's row when p / B is a page it holds and from the free list
// otherwise, and the token at a new page's first position writes the id into
// the row: new pages start past ctx, so that token is always part of the step.
//
// Up to kFusedRequests requests one launch does all: every block sums the
// lengths itself (they come from L2; 8 bytes per request) and then lays out
// its own range of tokens from the sums in shared memory.  Beyond that, the
// sums take two small launches (tile totals, then each tile's scan on top of
// the totals before it) and the third lays out the tokens.
#include "model.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / kWarp;
constexpr int kItems = 8;                      // requests per thread of one scan tile
constexpr int kTile = kThreads * kItems;       // requests of one scan tile
constexpr uint32_t kFusedRequests = kTile;
constexpr uint32_t kMaxStart = 0x7fffffffu;    // starts saturate here, past any token

struct Params {
    const int32_t* context;
    const int32_t* fresh;
    int32_t* table;
    uint64_t table_stride;
    uint32_t width;
    uint32_t requests;
    uint32_t block_size;
    uint32_t num_free;
    const int32_t* free_blocks;
    const int32_t* free_used;
    int32_t* free_used_out;
    int32_t* seq_lens;
    int32_t* starts;
    int64_t* slots;
    int32_t* positions;
    int32_t* token_request;
    uint32_t tokens;        // entries of slots
    uint32_t div_mul;       // p / block_size == (p * div_mul) >> div_shift for p < 2^31
    uint32_t div_shift;
    uint32_t tokens_per_warp;
    uint32_t* ctrl;
};

// Lengths of one request and what follows from them.
struct Request {
    uint32_t context;
    uint32_t fresh;
    uint32_t held;   // pages in the row
    uint32_t need;   // pages to take
    bool in_row;
};

__device__ __forceinline__ uint32_t divide(const Params& p, uint32_t v)
{
    return uint32_t((uint64_t(v) * p.div_mul) >> p.div_shift);
}

__device__ __forceinline__ Request request_at(const Params& p, uint32_t r)
{
    Request q{0, 0, 0, 0, true};
    if (r >= p.requests) return q;
    q.context = uint32_t(max(p.context[r], 0));
    q.fresh = p.fresh ? uint32_t(max(p.fresh[r], 0)) : 1u;
    const uint32_t end = q.context + q.fresh;  // below 2^32
    // ceil(v / B) as (v - 1) / B + 1, which stays below 2^31 for v <= 2^31
    q.held = q.context ? divide(p, q.context - 1) + 1 : 0;
    const uint32_t total = end - 1 < 0x7fffffffu ? divide(p, end - 1) + 1 : (end ? 0xffffffffu : 0);
    q.in_row = end <= 0x7fffffffu && total <= p.width;
    q.need = q.in_row ? total - q.held : 0;
    return q;
}

// Inclusive sums of two counts over the block, per thread.
struct Sums {
    uint64_t tokens, pages;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

__device__ __forceinline__ Sums shfl_up(Sums v, int d)
{
    return {__shfl_up_sync(~0u, v.tokens, d), __shfl_up_sync(~0u, v.pages, d)};
}

// Exclusive sum of `mine` over the block's threads; `total` over all of them.
__device__ Sums block_exclusive(Sums mine, Sums* warp_sums, Sums& total)
{
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    Sums inc = mine;
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
        const Sums o = shfl_up(inc, d);
        if (lane >= d) inc = inc + o;
    }
    if (lane == kWarp - 1) warp_sums[warp] = inc;
    __syncthreads();
    Sums before{0, 0};
    total = {0, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before = total;
        total = total + warp_sums[w];
    }
    __syncthreads();
    return {before.tokens + inc.tokens - mine.tokens, before.pages + inc.pages - mine.pages};
}

__device__ __forceinline__ uint32_t used_before(const Params& p) { return p.free_used ? uint32_t(max(*p.free_used, 0)) : 0u; }

// What laying out a request's tokens needs, by request: its first token, its
// context length (-1: refused) and the free-list index of page 0 had all its
// pages come from there (modulo 2^32; page >= held makes it exact).
struct Plan {
    uint32_t* start;
    int32_t* context;
    uint32_t* free_base;
};

// Scans one tile of requests on top of `before` into the plan (indexed from
// the tile's first request) and, where `write`, the outputs.  Returns the pages
// in use after the thread's last request that was served with new ones.
template <int ITEMS>
__device__ uint64_t scan_tile(const Params& p, uint32_t first, Sums before, Plan plan, bool write, Sums* warp_sums,
                              Sums& total)
{
    Request q[ITEMS];
    Sums mine{0, 0};
    const uint32_t r0 = first + threadIdx.x * ITEMS;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        q[i] = request_at(p, r0 + i);
        mine = mine + Sums{q[i].fresh, q[i].need};
    }
    Sums at = before + block_exclusive(mine, warp_sums, total);
    const uint64_t used = used_before(p);
    uint64_t used_after = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t r = r0 + i;
        if (r < p.requests) {
            const Sums end = at + Sums{q[i].fresh, q[i].need};
            const bool fits = q[i].in_row && end.tokens <= p.tokens &&
                              (q[i].need == 0 || used + end.pages <= p.num_free);
            const uint32_t start = uint32_t(min(at.tokens, uint64_t(kMaxStart)));
            const uint32_t slot = r - first;
            plan.start[slot] = start;
            plan.context[slot] = fits ? int32_t(q[i].context) : -1;
            plan.free_base[slot] = uint32_t(used + at.pages) - q[i].held;
            if (write) {
                p.starts[r] = int32_t(start);
                if (r == p.requests - 1) p.starts[r + 1] = int32_t(min(end.tokens, uint64_t(kMaxStart)));
                p.seq_lens[r] = int32_t(fits ? q[i].context + q[i].fresh : q[i].context);
                if (fits && q[i].need) used_after = used + end.pages;
            }
            at = end;
        }
    }
    return used_after;
}

// Last request of [lo, hi] that starts at or before token t; start[lo] <= t.
__device__ __forceinline__ uint32_t find(const uint32_t* start, uint32_t lo, uint32_t hi, uint32_t t)
{
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (start[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Lays out tokens [first, last) of the warp.  `plan` is indexed from request
// `base`; `end` is the step's token count.  Tokens go 32 at a time; where one
// request covers all 32 (prompts) nothing is searched, else each lane searches
// between the group's first request and the warp's last.
__device__ void lay_out(const Params& p, const Plan& plan, uint32_t base, uint32_t lo, uint32_t hi, uint32_t first,
                        uint32_t last, uint32_t end)
{
    const uint32_t lane = threadIdx.x % kWarp;
    const uint32_t inside = min(last, end);
    uint32_t r = lo;
    if (first < inside) {
        r = find(plan.start, lo, hi, first);
        hi = find(plan.start, r, hi, inside - 1);
    }
    for (uint32_t t0 = first; t0 < last; t0 += kWarp) {
        const uint32_t t = t0 + lane;
        if (t0 < inside) {
            const uint32_t t_last = min(t0 + kWarp, inside) - 1;
            uint32_t mine = r;
            if (r < hi && plan.start[r + 1] <= t_last) mine = find(plan.start, r, hi, min(t, t_last));
            r = __shfl_sync(~0u, mine, kWarp - 1);
            if (t >= last) continue;
            const int32_t context = plan.context[mine];
            if (t < inside && context >= 0) {
                const uint32_t position = uint32_t(context) + (t - plan.start[mine]);
                const uint32_t page = divide(p, position);
                const uint32_t offset = position - page * p.block_size;
                const uint64_t row = uint64_t(base + mine) * p.table_stride;
                int32_t id;
                if (page * p.block_size >= uint32_t(context)) {  // a page the row did not hold
                    id = p.free_blocks[plan.free_base[mine] + page];
                    if (offset == 0) p.table[row + page] = id;
                } else {
                    id = p.table[row + page];
                }
                p.slots[t] = id < 0 ? -1 : int64_t(id) * p.block_size + offset;
                if (p.positions) p.positions[t] = int32_t(position);
                if (p.token_request) p.token_request[t] = int32_t(base + mine);
                continue;
            }
        }
        if (t < last) {
            p.slots[t] = -1;
            if (p.positions) p.positions[t] = 0;
            if (p.token_request) p.token_request[t] = -1;
        }
    }
}

__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* shared)
{
    if (threadIdx.x == 0) *shared = 0;
    __syncthreads();
    if (v) atomicMax(reinterpret_cast<unsigned long long*>(shared), static_cast<unsigned long long>(v));
    __syncthreads();
    return *shared;
}

template <int ITEMS>
__global__ void __launch_bounds__(kThreads) fused_kernel(const Params p)
{
    __shared__ Sums warp_sums[kWarps];
    __shared__ uint64_t top;
    extern __shared__ uint32_t dynamic[];
    const uint32_t n = p.requests;
    const Plan plan{dynamic, reinterpret_cast<int32_t*>(dynamic) + n, dynamic + 2 * n};
    Sums total;
    const bool writer = blockIdx.x == 0;
    const uint64_t used_after = scan_tile<ITEMS>(p, 0, Sums{0, 0}, plan, writer, warp_sums, total);
    if (writer) {
        const uint64_t most = block_max(used_after, &top);
        if (threadIdx.x == 0) {
            *p.free_used_out = int32_t(max(most, uint64_t(used_before(p))));
            p.ctrl[0] = p.ctrl[1] = 0;
        }
    }
    __syncthreads();
    const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / kWarp;
    const uint64_t first = uint64_t(warp) * p.tokens_per_warp;
    if (first >= p.tokens) return;
    lay_out(p, plan, 0, 0, n - 1, uint32_t(first), uint32_t(min(first + p.tokens_per_warp, uint64_t(p.tokens))),
            uint32_t(min(total.tokens, uint64_t(kMaxStart))));
}

// The three launches for many requests.
__global__ void __launch_bounds__(kThreads) totals_kernel(const Params p, Sums* tile_sums)
{
    __shared__ Sums warp_sums[kWarps];
    Sums mine{0, 0}, total;
    // the tile's sums only: lane-consecutive requests, so that loads coalesce
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const Request q = request_at(p, blockIdx.x * kTile + i * kThreads + threadIdx.x);
        mine = mine + Sums{q.fresh, q.need};
    }
    block_exclusive(mine, warp_sums, total);
    if (threadIdx.x == 0) {
        tile_sums[blockIdx.x] = total;
        if (blockIdx.x == 0) {
            *p.free_used_out = int32_t(used_before(p));
            p.ctrl[0] = p.ctrl[1] = 0;
        }
    }
}

__global__ void __launch_bounds__(kThreads) starts_kernel(const Params p, const Sums* tile_sums, Plan plan)
{
    __shared__ Sums warp_sums[kWarps];
    __shared__ uint64_t top;
    Sums before{0, 0}, mine{0, 0}, total;
    for (uint32_t i = threadIdx.x; i < blockIdx.x; i += kThreads) mine = mine + tile_sums[i];
    block_exclusive(mine, warp_sums, before);
    const uint32_t first = blockIdx.x * kTile;
    const Plan here{plan.start + first, plan.context + first, plan.free_base + first};
    const uint64_t used_after = scan_tile<kItems>(p, first, before, here, true, warp_sums, total);
    const uint64_t most = block_max(used_after, &top);
    if (threadIdx.x == 0 && most) atomicMax(p.free_used_out, int32_t(most));
}

__global__ void __launch_bounds__(kThreads) tokens_kernel(const Params p, const Plan plan)
{
    const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / kWarp;
    const uint64_t first = uint64_t(warp) * p.tokens_per_warp;
    if (first >= p.tokens) return;
    lay_out(p, plan, 0, 0, p.requests - 1, uint32_t(first),
            uint32_t(min(first + p.tokens_per_warp, uint64_t(p.tokens))), uint32_t(p.starts[p.requests]));
}

// No requests: one start and marked entries.
__global__ void __launch_bounds__(kThreads) empty_kernel(const Params p)
{
    const uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i == 0) {
        p.starts[0] = 0;
        *p.free_used_out = int32_t(used_before(p));
        p.ctrl[0] = p.ctrl[1] = 0;
    }
    if (i < p.tokens) {
        p.slots[i] = -1;
        if (p.positions) p.positions[i] = 0;
        if (p.token_request) p.token_request[i] = -1;
    }
}

struct Layout {
    size_t sums, start, context, free_base, bytes;
};

Layout layout(uint64_t requests)
{
    Layout l{};
    l.bytes = kTempAlign;
    if (requests <= kFusedRequests) return l;
    const auto take = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += align_up(bytes, kTempAlign);
        return at;
    };
    l.sums = take(ceil_div(requests, kTile) * sizeof(Sums));
    l.start = take(requests * 4);
    l.context = take(requests * 4);
    l.free_base = take(requests * 4);
    return l;
}

lcpp_status run(void* temp, size_t temp_bytes, const lcpp_block_table_args* a, cudaStream_t s)
{
    if (!a || !a->block_size || a->max_tokens >> 31 || a->num_requests > LCPP_MAX_REQUESTS ||
        a->table_stride < a->table_width)
        return LCPP_ERR_INVALID_ARG;
    const uint64_t n = a->num_requests;
    if (!temp || misaligned(temp, kTempAlign) || !a->free_used_out || !a->query_starts_out ||
        (a->max_tokens && !a->slots_out) || (a->num_free && !a->free_blocks))
        return LCPP_ERR_INVALID_ARG;
    if (n && (!a->context_lens || !a->seq_lens_out || (a->table_width && !a->block_table)))
        return LCPP_ERR_INVALID_ARG;
    if (misaligned(a->slots_out, 8)) return LCPP_ERR_INVALID_ARG;
    const void* words[] = {a->context_lens, a->new_lens,       a->block_table,   a->free_blocks,      a->free_used,
                           a->free_used_out, a->seq_lens_out,  a->query_starts_out, a->positions_out, a->token_request_out};
    for (const void* w : words)
        if (misaligned(w, 4)) return LCPP_ERR_INVALID_ARG;
    // blocks read the inputs while one of them writes these
    const struct { const void* p; uint64_t bytes; } outputs[] = {{a->free_used_out, 4}, {a->seq_lens_out, n * 4}},
        inputs[] = {{a->context_lens, n * 4}, {a->new_lens, n * 4}, {a->free_used, 4},
                    {a->free_blocks, uint64_t(a->num_free) * 4}};
    for (const auto& o : outputs)
        for (const auto& i : inputs)
            if (overlap(o.p, o.bytes, i.p, i.bytes)) return LCPP_ERR_INVALID_ARG;
    const Layout l = layout(n);
    if (temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;

    Params p{};
    p.context = a->context_lens;
    p.fresh = a->new_lens;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.width = a->table_width;
    p.requests = a->num_requests;
    p.block_size = a->block_size;
    // num_free past 2^31 - 1 cannot be counted in free_used; the rest is not used
    p.num_free = std::min(a->num_free, 0x7fffffffu);
    p.free_blocks = a->free_blocks;
    p.free_used = a->free_used;
    p.free_used_out = a->free_used_out;
    p.seq_lens = a->seq_lens_out;
    p.starts = a->query_starts_out;
    p.slots = a->slots_out;
    p.positions = a->positions_out;
    p.token_request = a->token_request_out;
    p.tokens = uint32_t(a->max_tokens);
    // division of p < 2^31 by B through a multiplication: with l = ceil(log2 B)
    // and m = floor(2^(31+l) / B) + 1, p / B == (p * m) >> (31 + l).  m has at
    // most 32 bits; a page size past 2^31 divides every position to page 0.
    uint32_t log = 0;
    while (log < 32 && (uint64_t(1) << log) < a->block_size) ++log;
    p.div_shift = 31 + log;
    p.div_mul = log >= 32 ? 0u : uint32_t((uint64_t(1) << p.div_shift) / a->block_size + 1);
    p.ctrl = static_cast<uint32_t*>(temp);

    diag::KernelTimer timer(kTimerBlockTable, a->max_tokens, s);
    if (n == 0) {
        empty_kernel<<<unsigned(std::max<uint64_t>(1, ceil_div(p.tokens, kThreads))), kThreads, 0, s>>>(p);
        return launched();
    }
    // tokens in equal contiguous runs over the warps of at most three blocks per SM
    const uint64_t most_warps = uint64_t(device_sm_count()) * 3 * kWarps;
    p.tokens_per_warp = uint32_t(align_up(ceil_div(std::max(p.tokens, 1u), most_warps), kWarp));
    const unsigned grid = unsigned(std::max<uint64_t>(1, ceil_div(ceil_div(p.tokens, p.tokens_per_warp), kWarps)));
    if (n <= kFusedRequests) {
        const size_t smem = n * 12;
        auto kernel = n <= kThreads ? fused_kernel<1> : n <= 2 * kThreads ? fused_kernel<2> : fused_kernel<kItems>;
        if (n > 2 * kThreads)  // up to 48 KB beside the static arrays
            set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), size_t(kFusedRequests) * 12);
        kernel<<<grid, kThreads, smem, s>>>(p);
        return launched();
    }
    unsigned char* t = static_cast<unsigned char*>(temp);
    const Plan plan{reinterpret_cast<uint32_t*>(t + l.start), reinterpret_cast<int32_t*>(t + l.context),
                    reinterpret_cast<uint32_t*>(t + l.free_base)};
    Sums* sums = reinterpret_cast<Sums*>(t + l.sums);
    const unsigned tiles = unsigned(ceil_div(n, kTile));
    totals_kernel<<<tiles, kThreads, 0, s>>>(p, sums);
    starts_kernel<<<tiles, kThreads, 0, s>>>(p, sums, plan);
    tokens_kernel<<<grid, kThreads, 0, s>>>(p, plan);
    return launched();
}

}  // namespace

extern "C" {

lcpp_status lcpp_block_table_temp_bytes(uint64_t num_requests, uint64_t max_tokens, size_t* temp_bytes)
{
    if (!temp_bytes || num_requests > LCPP_MAX_REQUESTS || max_tokens >> 31) return LCPP_ERR_INVALID_ARG;
    *temp_bytes = layout(num_requests).bytes;
    return LCPP_OK;
}

lcpp_status lcpp_block_table_extend(void* temp, size_t temp_bytes, const lcpp_block_table_args* args,
                                    lcpp_stream_t stream)
{
    return guarded("lcpp_block_table_extend",
                   [&] { return run(temp, temp_bytes, args, reinterpret_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
