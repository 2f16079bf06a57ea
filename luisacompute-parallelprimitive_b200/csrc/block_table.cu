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
// sums take two small launches (totals of 512 requests, then each 512's scan on
// top of the totals before it) and the third lays out the tokens.
//
// What has to move is 8 bytes a request in, and out 16 bytes a token, 8 a
// request and 4 a new page.  A step of 64 single tokens takes 2.9 us and one of
// 7001 mixed tokens 3.3 us, a launch and its dependent loads.  4.0 M tokens of
// 6001 requests in pages of 64 take 25 us (67 MB written at 2.6 TB/s; the copy
// rate would be 10.5 us): the layout kernel, 20 us of it, is bound by the latency
// of a run's chain (search, page load, stores: 5.2 warps wait for a load per
// instruction issued, in 54 % of the issue slots), not by memory, for all it writes
// stays in L2.
#include "model.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / kWarp;
constexpr int kItems = 8;                      // requests per thread of the fused kernel, at most
// One launch up to here, whose blocks hold 12 bytes a request in shared memory and
// all sum all lengths.  Single tokens for 3000 and 4096 requests take 6.9 and 7.1 us
// in one launch, 7.3 and 7.4 in three; for 4097 and 8000 (16 requests a thread,
// 96 KB) 10.5 and 11.5 us in one, 7.6 and 8.2 in three.
constexpr uint32_t kFusedRequests = kThreads * kItems;
constexpr uint32_t kWindow = 1024;             // requests of a block's tokens held in shared memory
constexpr uint32_t kMost = 0x7fffffffu;        // sums saturate here, past every token and page

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
    uint32_t tokens_per_block;
    uint32_t wide;          // token arrays start on 16-byte boundaries
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

// Tokens and pages, added up to at most kMost: what saturates is past every
// array, and saturating sums may be taken in any order.
struct Sums {
    uint32_t tokens, pages;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b)
{
    return {min(a.tokens + b.tokens, kMost), min(a.pages + b.pages, kMost)};
}

// Sum of the values of the lanes before this one, and of all lanes.
__device__ __forceinline__ Sums warp_exclusive(Sums v, Sums& total)
{
    const int lane = threadIdx.x % kWarp;
    Sums inc = v;
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
        const Sums o{__shfl_up_sync(~0u, inc.tokens, d), __shfl_up_sync(~0u, inc.pages, d)};
        if (lane >= d) inc = inc + o;
    }
    total = {__shfl_sync(~0u, inc.tokens, kWarp - 1), __shfl_sync(~0u, inc.pages, kWarp - 1)};
    const Sums before{__shfl_up_sync(~0u, inc.tokens, 1), __shfl_up_sync(~0u, inc.pages, 1)};
    return lane ? before : Sums{0, 0};
}

// Sum of the warps' values before this warp, and of all warps.
__device__ __forceinline__ Sums warps_exclusive(Sums of_warp, Sums* shared, Sums& total)
{
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    if (lane == 0) shared[warp] = of_warp;
    __syncthreads();
    const Sums before = warp_exclusive(lane < kWarps ? shared[lane] : Sums{0, 0}, total);
    __syncthreads();
    return {__shfl_sync(~0u, before.tokens, warp), __shfl_sync(~0u, before.pages, warp)};
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

// Scans the block's ITEMS * kThreads requests from `first` on, on top of
// `before`, into the plan (indexed from `first`).  Each warp has ITEMS * 32 of
// them in a row and takes 32 at a time, so that all accesses are coalesced.
// Returns the pages in use after the last request that this thread saw served
// with new ones; `total` includes `before`.
template <int ITEMS>
__device__ uint32_t scan_tile(const Params& p, uint32_t first, Sums before, Plan plan, Sums* shared, Sums& total)
{
    const uint32_t lane = threadIdx.x % kWarp, slot0 = threadIdx.x / kWarp * kWarp * ITEMS + lane;
    Request q[ITEMS];
    Sums at[ITEMS], of_warp{0, 0};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) q[i] = request_at(p, first + slot0 + i * kWarp);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        Sums of_row;
        at[i] = of_warp + warp_exclusive(Sums{q[i].fresh, q[i].need}, of_row);
        of_warp = of_warp + of_row;
    }
    const Sums base = before + warps_exclusive(of_warp, shared, total);
    total = before + total;
    const uint32_t used = used_before(p);
    uint32_t used_after = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t slot = slot0 + i * kWarp;
        if (first + slot < p.requests) {
            const Sums start = base + at[i], end = start + Sums{q[i].fresh, q[i].need};
            const bool fits = q[i].in_row && end.tokens <= p.tokens &&
                              (q[i].need == 0 || (used <= p.num_free && end.pages <= p.num_free - used));
            plan.start[slot] = start.tokens;
            plan.context[slot] = fits ? int32_t(q[i].context) : -1;
            plan.free_base[slot] = used + start.pages - q[i].held;
            if (fits && q[i].need) used_after = used + end.pages;
        }
    }
    return used_after;
}

// The outputs by request: i of the plan is request `first` + i.
__device__ __forceinline__ void write_request(const Params& p, const Plan& plan, uint32_t first, uint32_t i)
{
    const uint32_t r = first + i;
    p.starts[r] = int32_t(plan.start[i]);
    const Request q = request_at(p, r);
    p.seq_lens[r] = int32_t(plan.context[i] < 0 ? q.context : q.context + q.fresh);
}

// Number of the first `n` starts at or below t, found by all threads of the
// block together: each round narrows the range kThreads-fold.
__device__ uint32_t block_count_starts(const uint32_t* start, uint32_t n, uint32_t t)
{
    uint32_t lo = 0;  // starts known to be at or below t
    while (n > 0) {
        const uint32_t step = (n + kThreads - 1) / kThreads;
        const uint32_t at = threadIdx.x * step + step - 1;  // last of the thread's stretch
        const uint32_t whole = uint32_t(__syncthreads_count(at < n && start[lo + at] <= t));
        lo += whole * step;
        if (step == 1) break;
        n = min(step - 1, n - whole * step);
    }
    return lo;
}

// Last request of the plan's first `window` that starts at or before token t
// (the first one does).
__device__ __forceinline__ uint32_t request_of(const Plan& plan, uint32_t window, uint32_t t)
{
    uint32_t r = 0;
    for (uint32_t half = 1u << (31 - __clz(max(window, 2u) - 1)); half > 0; half /= 2) {
        const uint32_t at = r + half;
        if (at < window && plan.start[at] <= t) r = at;
    }
    return r;
}

// The G tokens from t on of request r, all of them served or none.  They lie in
// one page or two: G is 1 or at most the page size.
template <int G>
__device__ __forceinline__ void lay_out_run(const Params& p, const Plan& plan, uint32_t base, uint32_t r, bool in_step,
                                            uint32_t t)
{
    const int32_t context = in_step ? plan.context[r] : -1;
    const bool served = context >= 0;
    uint32_t position = 0;
    int64_t slot[G];
#pragma unroll
    for (int i = 0; i < G; ++i) slot[i] = -1;
    if (served) {
        position = uint32_t(context) + (t - plan.start[r]);
        const uint32_t page = divide(p, position), offset = position - page * p.block_size;
        const bool two = G > 1 && offset + G > p.block_size;
        // pages the row did not hold come from the free list
        const bool fresh0 = page * p.block_size >= uint32_t(context);
        const bool fresh1 = two && (page + 1) * p.block_size >= uint32_t(context);
        int32_t* row = p.table + uint64_t(base + r) * p.table_stride + page;
        const uint32_t at0 = plan.free_base[r] + page, at1 = at0 + 1;  // modulo 2^32, before they index
        const int32_t id0 = fresh0 ? p.free_blocks[at0] : row[0];
        const int32_t id1 = two ? (fresh1 ? p.free_blocks[at1] : row[1]) : -1;
        if (fresh0 && offset == 0) row[0] = id0;
        if (fresh1) row[1] = id1;
        const int64_t slot0 = int64_t(id0) * p.block_size + offset;
        const int64_t slot1 = (int64_t(id1) - 1) * p.block_size + offset;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const bool second = G > 1 && offset + i >= p.block_size;
            if ((second ? id1 : id0) >= 0) slot[i] = (second ? slot1 : slot0) + i;
        }
    }
    const int32_t request = served ? int32_t(base + r) : -1;
    if (G == 4 && p.wide) {
        longlong2* s = reinterpret_cast<longlong2*>(p.slots + t);
        s[0] = make_longlong2(slot[0], slot[1 % G]);
        s[1] = make_longlong2(slot[2 % G], slot[3 % G]);
        const int32_t q = int32_t(position);
        if (p.positions)
            *reinterpret_cast<int4*>(p.positions + t) = served ? make_int4(q, q + 1, q + 2, q + 3) : make_int4(0, 0, 0, 0);
        if (p.token_request) *reinterpret_cast<int4*>(p.token_request + t) = make_int4(request, request, request, request);
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            p.slots[t + i] = slot[i];
            if (p.positions) p.positions[t + i] = served ? int32_t(position + i) : 0;
            if (p.token_request) p.token_request[t + i] = request;
        }
    }
}

// Lays out tokens [first, last) of the block, whose requests are among
// [0, window) of the plan, the first of them numbered `base`; `end` is the
// step's token count.  A thread takes G tokens at a time: where one request has
// them all they cost one search, one division and, mostly, one page (G = 4
// against 1 at 4.0 M tokens: 26 against 28 us).
template <int G>
__device__ void lay_out(const Params& p, const Plan& plan, uint32_t base, uint32_t window, uint32_t first,
                        uint32_t last, uint32_t end)
{
    for (uint32_t t = first + threadIdx.x * G; t < last; t += kThreads * G) {
        const uint32_t r = request_of(plan, window, t);
        const uint32_t next = r + 1 < window ? min(plan.start[r + 1], end) : end;
        if (G == 1 || (t + G <= last && (t + G <= next || t >= end))) {
            lay_out_run<G>(p, plan, base, r, t < end, t);
        } else {
            for (uint32_t i = t; i < min(t + G, last); ++i)
                lay_out_run<1>(p, plan, base, i == t ? r : request_of(plan, window, i), i < end, i);
        }
    }
}

template <int ITEMS, int G>
__global__ void __launch_bounds__(kThreads) fused_kernel(const Params p)
{
    __shared__ Sums shared[kWarps];
    __shared__ uint32_t used_after;
    extern __shared__ uint32_t dynamic[];
    const uint32_t n = p.requests;
    const Plan plan{dynamic, reinterpret_cast<int32_t*>(dynamic) + n, dynamic + 2 * n};
    if (threadIdx.x == 0) used_after = used_before(p);
    Sums total;
    const uint32_t used = scan_tile<ITEMS>(p, 0, Sums{0, 0}, plan, shared, total);
    if (used) atomicMax(&used_after, used);
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *p.free_used_out = int32_t(used_after);
        p.starts[n] = int32_t(total.tokens);
        p.ctrl[0] = p.ctrl[1] = 0;
    }
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < n; i += gridDim.x * kThreads)
        write_request(p, plan, 0, i);
    const uint32_t first = min(blockIdx.x * p.tokens_per_block, p.tokens);
    lay_out<G>(p, plan, 0, n, first, min(first + p.tokens_per_block, p.tokens), total.tokens);
}

// The three launches for many requests.
__global__ void __launch_bounds__(kThreads) totals_kernel(const Params p, Sums* tile_sums)
{
    let_next_start();
    __shared__ Sums shared[kWarps];
    const Request q = request_at(p, blockIdx.x * kThreads + threadIdx.x);
    Sums of_warp, total;
    warp_exclusive(Sums{q.fresh, q.need}, of_warp);
    warps_exclusive(of_warp, shared, total);
    if (threadIdx.x == 0) {
        tile_sums[blockIdx.x] = total;
        if (blockIdx.x == 0) {
            *p.free_used_out = int32_t(used_before(p));
            p.ctrl[0] = p.ctrl[1] = 0;
        }
    }
}

__global__ void __launch_bounds__(kThreads) starts_kernel(const Params p, const Sums* tile_sums, const Plan all)
{
    __shared__ Sums shared[kWarps];
    __shared__ uint32_t used_after;
    if (threadIdx.x == 0) used_after = 0;
    let_next_start();
    wait_for_previous();
    Sums mine{0, 0}, of_warp, before, total;
    for (uint32_t i = threadIdx.x; i < blockIdx.x; i += kThreads) mine = mine + tile_sums[i];
    warp_exclusive(mine, of_warp);
    warps_exclusive(of_warp, shared, before);
    const uint32_t first = blockIdx.x * kThreads;
    const Plan plan{all.start + first, all.context + first, all.free_base + first};
    const uint32_t used = scan_tile<1>(p, first, before, plan, shared, total);
    if (used) atomicMax(&used_after, used);
    if (first + threadIdx.x < p.requests) write_request(p, plan, first, threadIdx.x);  // what this thread planned
    __syncthreads();
    if (threadIdx.x == 0) {
        if (used_after) atomicMax(p.free_used_out, int32_t(used_after));
        if (blockIdx.x == gridDim.x - 1) p.starts[p.requests] = int32_t(total.tokens);
    }
}

// The requests of the block's tokens come into shared memory where they fit
// (a window has at least one token per request that is not empty).
template <int G>
__global__ void __launch_bounds__(kThreads) tokens_kernel(const Params p, const Plan all)
{
    __shared__ uint32_t start[kWindow], free_base[kWindow];
    __shared__ int32_t context[kWindow];
    const uint32_t first = blockIdx.x * p.tokens_per_block, last = min(first + p.tokens_per_block, p.tokens);
    wait_for_previous();
    const uint32_t end = uint32_t(p.starts[p.requests]);
    const uint32_t lo = block_count_starts(all.start, p.requests, first) - 1;  // the first starts at 0
    const uint32_t window = block_count_starts(all.start + lo, p.requests - lo, last - 1);
    Plan plan{all.start + lo, all.context + lo, all.free_base + lo};
    if (window <= kWindow) {
        for (uint32_t i = threadIdx.x; i < window; i += kThreads) {
            start[i] = plan.start[i];
            context[i] = plan.context[i];
            free_base[i] = plan.free_base[i];
        }
        plan = Plan{start, context, free_base};
        __syncthreads();
    }
    lay_out<G>(p, plan, lo, window, first, last, end);
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
    l.sums = take(ceil_div(requests, kThreads) * sizeof(Sums));
    l.start = take(requests * 4);
    l.context = take(requests * 4);
    l.free_base = take(requests * 4);
    return l;
}

lcpp_status run(void* temp, size_t temp_bytes, const lcpp_block_table_args* a, cudaStream_t s)
{
    if (!a || !a->block_size || a->max_tokens >= kMost || a->num_requests > LCPP_MAX_REQUESTS ||
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
    const Layout l = layout(n);
    if (temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;
    const Array arrays[] = {{a->context_lens, n * 4, false},
                            {a->new_lens, n * 4, false},
                            {a->free_blocks, uint64_t(a->num_free) * 4, false},
                            {a->free_used, 4, false},
                            {a->free_used_out, 4, true},
                            {a->seq_lens_out, n * 4, true},
                            {a->query_starts_out, (n + 1) * 4, true},
                            {a->slots_out, a->max_tokens * 8, true},
                            {a->positions_out, a->max_tokens * 4, true},
                            {a->token_request_out, a->max_tokens * 4, true},
                            {temp, l.bytes, true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
    for (const Array& o : arrays)  // the table is read and written
        if (overlap_rows(a->block_table, n, a->table_stride, a->table_width, 4, o.p, o.bytes)) return LCPP_ERR_INVALID_ARG;

    Params p{};
    p.context = a->context_lens;
    p.fresh = a->new_lens;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.width = a->table_width;
    p.requests = a->num_requests;
    p.block_size = a->block_size;
    p.num_free = std::min(a->num_free, kMost - 1);  // free_used counts no further
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
    // four tokens to a thread where every SM has work for a block of such threads
    // and four tokens lie in two pages at most
    const bool many = p.tokens >= uint64_t(device_sm_count()) * kThreads * 4 && p.block_size >= 4;
    p.wide = !(misaligned(p.slots, 16) || misaligned(p.positions, 16) || misaligned(p.token_request, 16));
    // tokens in equal contiguous runs over the resident blocks
    const auto grid_of = [&](const void* kernel, size_t smem) {
        const uint64_t most = uint64_t(device_sm_count()) * resident_blocks(kernel, kThreads, smem);
        p.tokens_per_block = uint32_t(align_up(std::max<uint64_t>(ceil_div(p.tokens, most), 1), kThreads * (many ? 4 : 1)));
        return unsigned(std::max<uint64_t>(1, ceil_div(p.tokens, p.tokens_per_block)));
    };
    if (n <= kFusedRequests) {
        // room in a few steps, so that few launch shapes are looked up and kept as n changes
        const uint64_t room = n <= kThreads ? kThreads : n <= 2 * kThreads ? 2 * kThreads : n <= 4 * kThreads ? 4 * kThreads : kFusedRequests;
        const size_t smem = room * 12;
        auto kernel = many ? (n <= kThreads ? fused_kernel<1, 4> : n <= 2 * kThreads ? fused_kernel<2, 4> : fused_kernel<kItems, 4>)
                           : (n <= kThreads ? fused_kernel<1, 1> : n <= 2 * kThreads ? fused_kernel<2, 1> : fused_kernel<kItems, 1>);
        if (n > 2 * kThreads)  // up to 48 KB beside the static arrays
            set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), size_t(kFusedRequests) * 12);
        const unsigned grid = grid_of(reinterpret_cast<const void*>(kernel), smem);
        kernel<<<grid, kThreads, smem, s>>>(p);
        return launched();
    }
    unsigned char* t = static_cast<unsigned char*>(temp);
    const Plan plan{reinterpret_cast<uint32_t*>(t + l.start), reinterpret_cast<int32_t*>(t + l.context),
                    reinterpret_cast<uint32_t*>(t + l.free_base)};
    Sums* sums = reinterpret_cast<Sums*>(t + l.sums);
    const unsigned tiles = unsigned(ceil_div(n, kThreads));
    totals_kernel<<<tiles, kThreads, 0, s>>>(p, sums);
    // Each launch starts while the one before it runs and waits for its end on the
    // device.  The last one waits for the second, which has itself waited.
    lcpp_status status = launch_early(starts_kernel, tiles, kThreads, 0, s, Params(p), static_cast<const Sums*>(sums), Plan(plan));
    if (status != LCPP_OK) return status;
    if (p.tokens) {
        auto kernel = many ? tokens_kernel<4> : tokens_kernel<1>;
        const unsigned grid = grid_of(reinterpret_cast<const void*>(kernel), 0);
        return launch_early(kernel, grid, kThreads, 0, s, Params(p), Plan(plan));
    }
    return LCPP_OK;
}

}  // namespace

extern "C" {

lcpp_status lcpp_block_table_temp_bytes(uint64_t num_requests, uint64_t max_tokens, size_t* temp_bytes)
{
    if (!temp_bytes || num_requests > LCPP_MAX_REQUESTS || max_tokens >= kMost) return LCPP_ERR_INVALID_ARG;
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
