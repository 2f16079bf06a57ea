// cache.cuh -- what the operators of a paged cache share: strided arrays and
// their overlaps, division by the page size, and equal shares of ragged work.
#pragma once

#include <initializer_list>
#include <vector>

#include "model.cuh"

namespace lcpp {
namespace model {

// LCPP_KERNEL_ROTARY / _PAGED_ATTENTION / _CACHE_EVICTION (include/lcpp_b200_diag.h)
constexpr int kTimerRotary = 12, kTimerAttention = 13, kTimerEviction = 14;

constexpr uint64_t kMostSlots = uint64_t(1) << 40;
constexpr uint64_t kMostStride = uint64_t(1) << 44;  // elements; products with 2^31 rows stay below 2^76, see Strided

// Elements at p + sum of index * stride, `columns` adjacent ones at each.
struct Strided {
    struct Dim {
        uint64_t n, stride;
    };
    const void* p = nullptr;
    int element = 1;
    uint64_t columns = 0;
    Dim dim[4] = {};
    int dims = 0;

    Strided(const void* base, int bytes, uint64_t cols, std::initializer_list<Dim> d) : p(base), element(bytes), columns(cols)
    {
        for (const Dim& x : d) dim[dims++] = x;
        std::sort(dim, dim + dims, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    }
    bool empty() const
    {
        for (int i = 0; i < dims; ++i)
            if (!dim[i].n) return true;
        return !columns;
    }
    // Elements from the first to the last, in 128 bits.
    unsigned __int128 extent(int of) const
    {
        unsigned __int128 e = columns;
        for (int i = 0; i < of; ++i) e += static_cast<unsigned __int128>(dim[i].n - 1) * dim[i].stride;
        return e;
    }
    bool sane() const { return empty() || extent(dims) * element < (static_cast<unsigned __int128>(1) << 62); }
    uint64_t bytes() const { return empty() ? 0 : uint64_t(extent(dims)) * element; }
    // No two of its elements share memory: each dimension steps over all that lies inside it.
    bool distinct() const
    {
        if (empty()) return true;
        for (int i = 0; i < dims; ++i)
            if (dim[i].n > 1 && extent(i) > dim[i].stride) return false;
        return true;
    }
};

// Whether the innermost dims_a and dims_b dimensions of a and b may share memory where
// b's first element lies `at` bytes behind a's.
inline bool may_meet(const Strided& a, int dims_a, const Strided& b, int dims_b, uint64_t at)
{
    if (static_cast<unsigned __int128>(at) >= a.extent(dims_a) * a.element) return false;
    while (dims_a && a.dim[dims_a - 1].n == 1) --dims_a;  // there is no second entry to step to
    while (dims_b && b.dim[dims_b - 1].n == 1) --dims_b;
    if (!dims_a && !dims_b) return true;
    const auto step = [](const Strided& x, int dims) { return dims ? x.dim[dims - 1].stride * x.element : uint64_t(0); };
    const uint64_t pitch = std::max(step(a, dims_a), step(b, dims_b)), within = pitch ? at % pitch : 0;
    if (!pitch) return true;
    if (step(a, dims_a) == pitch) --dims_a;  // else all of it is one row
    if (step(b, dims_b) == pitch) --dims_b;
    if (a.extent(dims_a) * a.element > pitch || within + b.extent(dims_b) * b.element > pitch) return true;
    return may_meet(a, dims_a, b, dims_b, within);  // one's row lies in the pitch of one row of the other's
}
// Whether a and b may share memory.  Apart, or rows of one pitch (and in these rows of
// one pitch again) of which each fits beside the other's: sure not to; everything else
// counts as shared.
inline bool may_share(const Strided& a, const Strided& b)
{
    if (!overlap(a.p, a.bytes(), b.p, b.bytes())) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x <= y ? may_meet(a, a.dims, b, b.dims, y - x) : may_meet(b, b.dims, a, a.dims, x - y);
}

// v / d for v < 2^31 through a multiplication: with l = ceil(log2 d) and
// m = floor(2^(31 + l) / d) + 1, v / d == (v * m) >> (31 + l), and m has at most 32 bits.
struct Divider {
    uint32_t d = 1, mul = 0, shift = 0;
    Divider() = default;
    explicit Divider(uint32_t by) : d(by)
    {
        uint32_t log = 0;
        while (log < 32 && (uint64_t(1) << log) < by) ++log;
        shift = 31 + log;
        mul = log >= 32 ? 0u : uint32_t((uint64_t(1) << shift) / by + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t v) const { return uint32_t((uint64_t(v) * mul) >> shift); }
};

inline bool sane_cache(const lcpp_kv_cache& c)
{
    return c.block_size && c.num_kv_heads && c.head_dim && c.head_dim <= LCPP_MAX_HEAD_DIM && c.page_stride <= kMostStride &&
           c.token_stride <= kMostStride && c.head_stride <= kMostStride &&
           uint64_t(c.num_pages) * c.block_size < kMostSlots;
}

inline Strided pages_of(const lcpp_kv_cache& c, const void* p)
{
    return Strided(p, row_dtype_bytes(c.dtype), c.head_dim,
                   {{c.num_pages, c.page_stride}, {c.block_size, c.token_stride}, {c.num_kv_heads, c.head_stride}});
}

// Keys and values that are written: no two elements share memory, k's and v's neither.
inline bool writable_cache(const lcpp_kv_cache& c)
{
    const Strided k = pages_of(c, c.k), v = pages_of(c, c.v);
    if (!k.sane() || !k.distinct()) return false;
    if (!overlap(c.k, k.bytes(), c.v, v.bytes())) return true;
    // side by side: one more dimension of two
    const int e = row_dtype_bytes(c.dtype);
    const uintptr_t a = reinterpret_cast<uintptr_t>(c.k), b = reinterpret_cast<uintptr_t>(c.v);
    const uint64_t apart = a < b ? b - a : a - b;
    return apart % e == 0 &&
           Strided(c.k, e, c.head_dim,
                   {{c.num_pages, c.page_stride}, {c.block_size, c.token_stride}, {c.num_kv_heads, c.head_stride}, {2, apart / e}})
               .distinct();
}

// Vector accesses of `bytes` bytes at multiples of as many elements from a row's start.
inline bool rows_aligned(const void* p, std::initializer_list<uint64_t> strides, int element, size_t bytes)
{
    if (misaligned(p, bytes)) return false;
    for (uint64_t s : strides)
        if (s * uint64_t(element) % bytes) return false;
    return true;
}

// Where a unit of ragged work lies: in item `item`, whose first unit is number `first`.
struct Place {
    long long first;
    uint32_t item;
    uint32_t valid;
};

// Equal shares of ragged work: items 0..n-1 have weight(i) units each; returns
// the sum of all units, and in `place` the item of unit number begin(sum).
// Every block that asks sums the weights itself (they come from L2): a thread
// takes a run of items, and the one whose run holds the unit walks it.
template <int THREADS, typename Weight, typename Begin>
__device__ __forceinline__ long long share_of(uint32_t n, Weight weight, Begin begin, Place& place)
{
    __shared__ long long warps[THREADS / kWarp];
    __shared__ Place found;
    const uint32_t run = (n + THREADS - 1) / THREADS, lo = min(n, threadIdx.x * run), hi = min(n, lo + run);
    long long mine = 0;
    for (uint32_t i = lo; i < hi; ++i) mine += weight(i);
    long long upto = mine;
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
        const long long left = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += left;
    }
    if (threadIdx.x == 0) found.valid = 0;
    if (lane == kWarp - 1) warps[warp] = upto;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kWarp; ++w) {
        if (w == warp) before = total;
        total += warps[w];
    }
    before += upto - mine;
    const long long at = begin(total);
    if (at >= before && at < before + mine) {
        uint32_t i = lo;
        long long w = weight(i);
        while (at >= before + w) {
            before += w;
            w = weight(++i);
        }
        found = Place{before, i, 1u};
    }
    __syncthreads();
    place = found;
    return total;
}

}  // namespace model
}  // namespace lcpp
