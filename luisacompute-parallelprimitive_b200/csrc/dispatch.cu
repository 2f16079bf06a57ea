// dispatch.cu -- DeviceDispatch (include/lcpp_b200_model.h): the (token,
// expert) pairs of a routed step grouped by expert, their rows moved there and
// summed back, and the gradients of both.
//
// Plan is a stable counting sort with one digit, the expert.  Every warp
// counts the experts of its own run of pairs in shared memory; sums of the
// counts over the warps before it, the blocks before it and the experts
// before it give each (warp, expert) its first row, and a second walk over the
// run ranks each 32 pairs with match.any.  Up to kSmallPairs pairs one block
// does all; beyond that one block per SM counts its tile in a first launch,
// and in a second one every block adds up all tiles' counts itself (a few
// hundred KB from L2) before it ranks its tile.
//
// The row kernels work by token: x (or its gradient) is read once and goes to,
// or comes from, the token's rows, so nothing but those rows is read or
// written top_k times.  They are bound by HBM: gather moves (1 + k) rows a
// token, combine the same, combine's gradient 1 + 2k.
#include "model.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / kWarp;
constexpr uint64_t kSmallPairs = 16384;  // one block ranks these
constexpr uint64_t kTilePairs = 4096;    // fewest pairs worth a block of their own

struct PlanParams {
    const int32_t* experts;
    int32_t* starts;
    int32_t* row_of;
    int32_t* pair_of;
    uint32_t pairs;
    uint32_t num_experts;
    uint32_t align;
    uint32_t max_rows;
    uint32_t tile;      // pairs of a block
    uint32_t per_warp;  // pairs of a warp, a multiple of 32
    uint32_t* ctrl;
    uint32_t* table;    // [tiles][num_experts]
};

// Exclusive sum over the block of one value per thread.
__device__ uint32_t block_exclusive(uint32_t v, uint32_t* warp_sums)
{
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    uint32_t inc = v;
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
        const uint32_t o = __shfl_up_sync(~0u, inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == kWarp - 1) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < kWarp; d *= 2) {
            const uint32_t o = __shfl_up_sync(~0u, w, d);
            if (lane >= d) w += o;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    const uint32_t before = warp ? warp_sums[warp - 1] : 0;
    __syncthreads();
    return before + inc - v;
}

__global__ void __launch_bounds__(kPlanThreads) count_kernel(const PlanParams p)
{
    extern __shared__ uint32_t count[];  // [num_experts]
    for (uint32_t e = threadIdx.x; e < p.num_experts; e += kPlanThreads) count[e] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * p.tile, last = min(first + p.tile, p.pairs);
    for (uint32_t i = first + threadIdx.x; i < last; i += kPlanThreads) {
        const uint32_t e = uint32_t(p.experts[i]);
        if (e < p.num_experts) atomicAdd(count + e, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.num_experts; e += kPlanThreads)
        p.table[uint64_t(blockIdx.x) * p.num_experts + e] = count[e];
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p)
{
    const uint32_t n = p.num_experts;
    extern __shared__ uint32_t dynamic[];
    uint32_t* counter = dynamic;                  // [kPlanWarps][n], then each (warp, expert)'s next row
    uint32_t* earlier = counter + kPlanWarps * n; // [n] pairs of earlier tiles
    uint32_t* total = earlier + n;                // [n] pairs of all tiles
    __shared__ uint32_t warp_sums[kPlanWarps];
    const uint32_t lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const uint32_t tile_first = blockIdx.x * p.tile, tile_last = min(tile_first + p.tile, p.pairs);
    const uint32_t first = min(tile_first + warp * p.per_warp, tile_last), last = min(first + p.per_warp, tile_last);
    uint32_t* mine = counter + warp * n;

    for (uint32_t i = threadIdx.x; i < (kPlanWarps + 2) * n; i += kPlanThreads) counter[i] = 0;
    __syncthreads();
    for (uint32_t i = first + lane; i < last; i += kWarp) {
        const uint32_t e = uint32_t(p.experts[i]);
        if (e < n) atomicAdd(mine + e, 1u);
    }
    if (gridDim.x > 1) {
        // threads in groups of one per expert, each group a share of the tiles
        const uint32_t groups = max(1u, kPlanThreads / n), group = threadIdx.x / n;
        if (group < groups) {
            for (uint32_t e = threadIdx.x - group * n; e < n; e += kPlanThreads) {
                uint32_t before = 0, all = 0;
#pragma unroll 8
                for (uint32_t b = group; b < gridDim.x; b += groups) {
                    const uint32_t c = p.table[uint64_t(b) * n + e];
                    all += c;
                    before += b < blockIdx.x ? c : 0;
                }
                if (all) atomicAdd(total + e, all);
                if (before) atomicAdd(earlier + e, before);
            }
        }
    }
    __syncthreads();
    // one thread per expert (n <= kPlanThreads): its segment, then its row for every warp
    uint32_t count = 0, segment = 0;
    if (threadIdx.x < n) {
        uint32_t in_block = 0;
        for (int w = 0; w < kPlanWarps; ++w) in_block += counter[w * n + threadIdx.x];
        count = gridDim.x > 1 ? total[threadIdx.x] : in_block;
        segment = (count + p.align - 1) / p.align * p.align;
    }
    const uint32_t start = block_exclusive(segment, warp_sums);
    if (threadIdx.x < n) {
        uint32_t row = start + earlier[threadIdx.x];
        for (int w = 0; w < kPlanWarps; ++w) {
            const uint32_t c = counter[w * n + threadIdx.x];
            counter[w * n + threadIdx.x] = row;
            row += c;
        }
        if (blockIdx.x == 0) {
            p.starts[threadIdx.x] = int32_t(start);
            if (threadIdx.x == n - 1) p.starts[n] = int32_t(start + segment);
        }
        earlier[threadIdx.x] = start + count;   // first padding row of the segment
        total[threadIdx.x] = start + segment;   // its end
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.ctrl[1] = 0;
    __syncthreads();

    for (uint32_t i0 = first; i0 < last; i0 += kWarp) {
        const uint32_t i = i0 + lane;
        const uint32_t e = i < last ? uint32_t(p.experts[i]) : ~0u;
        const bool valid = e < n;
        const uint32_t peers = __match_any_sync(~0u, valid ? e : ~0u);
        const uint32_t rank = __popc(peers & lanemask_lt());
        uint32_t row = ~0u;
        if (valid) row = mine[e] + rank;
        __syncwarp();
        if (valid && rank == 0) mine[e] += __popc(peers);
        __syncwarp();
        if (i < last) {
            p.row_of[i] = row < p.max_rows ? int32_t(row) : -1;
            if (row < p.max_rows) p.pair_of[row] = int32_t(i);
        }
    }
    // rows without a pair
    for (uint32_t e = blockIdx.x * kPlanWarps + warp; e < n; e += gridDim.x * kPlanWarps)
        for (uint32_t r = earlier[e] + lane; r < min(total[e], p.max_rows); r += kWarp) p.pair_of[r] = -1;
    for (uint64_t r = uint64_t(total[n - 1]) + blockIdx.x * kPlanThreads + threadIdx.x; r < p.max_rows;
         r += uint64_t(gridDim.x) * kPlanThreads)
        p.pair_of[r] = -1;
}

// ---------------------------------------------------------------------------
// Row kernels.  A row is `units` accesses of UB bytes; `lanes` threads (a power
// of two) share a token.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kPadRows = 64;   // rows a block looks through for padding
constexpr int kUnroll = 8;     // expert rows in flight per thread

template <int UB>
struct Unit;
template <> struct Unit<16> { using type = uint4; };
template <> struct Unit<8> { using type = uint2; };
template <> struct Unit<4> { using type = uint32_t; };
template <> struct Unit<2> { using type = uint16_t; };

struct RowParams {
    const unsigned char* x;      // token rows read
    uint64_t x_pitch;            // bytes
    const unsigned char* rows;   // expert rows read
    uint64_t rows_pitch;
    unsigned char* out;          // rows written
    uint64_t out_pitch;
    const int32_t* row_of;
    const int32_t* pair_of;
    const int32_t* starts;
    const float* weights;
    float* grad_weights;
    uint32_t tokens;
    uint32_t top_k;
    uint32_t num_experts;
    uint32_t max_rows;
    uint32_t units;
    uint32_t lanes_log2;
    uint32_t pad_blocks;
    uint32_t chunks;             // column chunks of a token
};

// Zeros in the padding rows among this block's kPadRows rows.
template <int UB>
__device__ void clear_padding(const RowParams& p, uint32_t block)
{
    using U = typename Unit<UB>::type;
    __shared__ uint32_t masks[kPadRows / kWarp];
    const uint32_t first = block * kPadRows;
    const uint32_t end = min(uint32_t(p.starts[p.num_experts]), p.max_rows);
    if (threadIdx.x < kPadRows) {
        const uint32_t r = first + threadIdx.x;
        const uint32_t m = __ballot_sync(~0u, r < end && p.pair_of[r] < 0);
        if (threadIdx.x % kWarp == 0) masks[threadIdx.x / kWarp] = m;
    }
    __syncthreads();
    for (uint32_t w = 0; w < kPadRows / kWarp; ++w) {
        for (uint32_t m = masks[w]; m; m &= m - 1) {
            U* row = reinterpret_cast<U*>(p.out + uint64_t(first + w * kWarp + __ffs(m) - 1) * p.out_pitch);
            for (uint32_t u = threadIdx.x; u < p.units; u += kRowThreads) row[u] = U{};
        }
    }
}

// Tokens' rows copied to their experts' rows.  Blocks: first the padding's.
template <int UB>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    constexpr int kUnits = 2;
    if (blockIdx.x < p.pad_blocks) {
        clear_padding<UB>(p, blockIdx.x);
        return;
    }
    const uint32_t block = blockIdx.x - p.pad_blocks;
    const uint32_t lanes = 1u << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t chunk = block % p.chunks;
    const uint32_t t = (block / p.chunks) * (kRowThreads >> p.lanes_log2) + (threadIdx.x >> p.lanes_log2);
    if (t >= p.tokens) return;
    const U* x = reinterpret_cast<const U*>(p.x + uint64_t(t) * p.x_pitch);
    const uint32_t u0 = chunk * lanes * kUnits + lane;
    U v[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
        if (u0 + i * lanes < p.units) v[i] = x[u0 + i * lanes];
    const int32_t* row_of = p.row_of + uint64_t(t) * p.top_k;
#pragma unroll 4
    for (uint32_t j = 0; j < p.top_k; ++j) {
        const uint32_t r = uint32_t(row_of[j]);
        if (r >= p.max_rows) continue;
        U* row = reinterpret_cast<U*>(p.out + uint64_t(r) * p.out_pitch);
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
            if (u0 + i * lanes < p.units) row[u0 + i * lanes] = v[i];
    }
}

template <typename T, int UB>
__device__ __forceinline__ void unpack(const typename Unit<UB>::type& raw, float (&out)[UB / sizeof(T)])
{
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < int(UB / sizeof(T)); ++i) out[i] = to_float(e[i]);
}

template <typename T, int UB>
__device__ __forceinline__ typename Unit<UB>::type pack(const float (&in)[UB / sizeof(T)])
{
    typename Unit<UB>::type raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < int(UB / sizeof(T)); ++i) e[i] = from_float<T>(in[i]);
    return raw;
}

// out[t] = sum_j w[t][j] rows[row_of[t][j]], kUnroll rows in flight per thread.
template <typename T, int UB>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    constexpr int kN = UB / int(sizeof(T));
    const uint32_t lanes = 1u << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t chunk = blockIdx.x % p.chunks;
    const uint32_t t = (blockIdx.x / p.chunks) * (kRowThreads >> p.lanes_log2) + (threadIdx.x >> p.lanes_log2);
    const uint32_t u = chunk * lanes + lane;
    if (t >= p.tokens || u >= p.units) return;
    const int32_t* row_of = p.row_of + uint64_t(t) * p.top_k;
    const float* weights = p.weights ? p.weights + uint64_t(t) * p.top_k : nullptr;
    float acc[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) acc[i] = 0.f;
    for (uint32_t j0 = 0; j0 < p.top_k; j0 += kUnroll) {
        U raw[kUnroll];
        float w[kUnroll];
        bool has[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const uint32_t r = j0 + j < p.top_k ? uint32_t(row_of[j0 + j]) : ~0u;
            has[j] = r < p.max_rows;
            w[j] = has[j] && weights ? weights[j0 + j] : 1.f;
            if (has[j]) raw[j] = reinterpret_cast<const U*>(p.rows + uint64_t(r) * p.rows_pitch)[u];
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (!has[j]) continue;
            float v[kN];
            unpack<T, UB>(raw[j], v);
#pragma unroll
            for (int i = 0; i < kN; ++i) acc[i] = fmaf(w[j], v[i], acc[i]);
        }
    }
    reinterpret_cast<U*>(p.out + uint64_t(t) * p.out_pitch)[u] = pack<T, UB>(acc);
}

// out[row] = w dy and grad_w = <rows[row], dy>, a token's lanes walking its
// columns once per kUnroll experts; the dot products are summed over a warp
// by shuffles and over a token's warps in order.
template <typename T, int UB>
__global__ void __launch_bounds__(kRowThreads) combine_backward_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    constexpr int kN = UB / int(sizeof(T));
    constexpr int kRowWarps = kRowThreads / kWarp;
    __shared__ float part[kRowWarps][kUnroll];
    if (blockIdx.x < p.pad_blocks) {
        clear_padding<UB>(p, blockIdx.x);
        return;
    }
    const uint32_t block = blockIdx.x - p.pad_blocks;
    const uint32_t lanes = 1u << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t t = block * (kRowThreads >> p.lanes_log2) + (threadIdx.x >> p.lanes_log2);
    const bool inside = t < p.tokens;
    const U* dy = reinterpret_cast<const U*>(p.x + uint64_t(inside ? t : 0) * p.x_pitch);
    const int32_t* row_of = p.row_of + uint64_t(t) * p.top_k;
    const float* weights = p.weights + uint64_t(t) * p.top_k;
    for (uint32_t j0 = 0; j0 < p.top_k; j0 += kUnroll) {
        uint32_t row[kUnroll];
        float w[kUnroll], dot[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const bool is = inside && j0 + j < p.top_k;
            row[j] = is ? uint32_t(row_of[j0 + j]) : ~0u;
            w[j] = is ? weights[j0 + j] : 0.f;
            dot[j] = 0.f;
        }
        for (uint32_t u = lane; u < p.units; u += lanes) {
            float g[kN];
            unpack<T, UB>(dy[u], g);
            U raw[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                if (row[j] < p.max_rows)
                    raw[j] = reinterpret_cast<const U*>(p.rows + uint64_t(row[j]) * p.rows_pitch)[u];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                if (row[j] >= p.max_rows) continue;
                float v[kN];
                unpack<T, UB>(raw[j], v);
#pragma unroll
                for (int i = 0; i < kN; ++i) {
                    dot[j] = fmaf(v[i], g[i], dot[j]);
                    v[i] = w[j] * g[i];
                }
                reinterpret_cast<U*>(p.out + uint64_t(row[j]) * p.out_pitch)[u] = pack<T, UB>(v);
            }
        }
        const uint32_t in_warp = min(lanes, uint32_t(kWarp));
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            for (uint32_t d = in_warp / 2; d > 0; d /= 2) dot[j] += __shfl_xor_sync(~0u, dot[j], d);
        if (lanes > kWarp) {
            const uint32_t warp = threadIdx.x / kWarp, token_warps = lanes / kWarp;
            if (threadIdx.x % kWarp == 0) {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) part[warp][j] = dot[j];
            }
            __syncthreads();
            if (inside && lane < kUnroll && j0 + lane < p.top_k) {
                float sum = 0.f;
                for (uint32_t i = 0; i < token_warps; ++i) sum += part[warp + i][lane];
                p.grad_weights[uint64_t(t) * p.top_k + j0 + lane] = sum;
            }
            __syncthreads();
        } else if (inside && lane == 0) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                if (j0 + j < p.top_k) p.grad_weights[uint64_t(t) * p.top_k + j0 + j] = dot[j];
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
uint64_t tiles_for(uint64_t pairs)
{
    if (pairs <= kSmallPairs) return 1;
    return std::min<uint64_t>(device_sm_count(), ceil_div(pairs, kTilePairs));
}

// Temp storage holds a count per (tile, expert); tiles are bounded by the SM
// count, which the query may run without: the bound is fixed instead.
constexpr uint64_t kMaxTiles = 256;

size_t plan_bytes(uint64_t pairs, uint32_t experts)
{
    if (pairs <= kSmallPairs) return kTempAlign;
    return kTempAlign + align_up(std::min(kMaxTiles, ceil_div(pairs, kTilePairs)) * experts * 4, kTempAlign);
}

bool counts_ok(uint64_t tokens, uint32_t top_k, uint32_t experts, uint64_t max_rows)
{
    return top_k >= 1 && top_k <= LCPP_MAX_TOP_K && experts >= 1 && experts <= LCPP_MAX_EXPERTS &&
           tokens < (uint64_t(1) << 31) && tokens * top_k < (uint64_t(1) << 31) && max_rows < (uint64_t(1) << 31);
}

uint64_t rows_needed(uint64_t pairs, uint32_t experts, uint32_t align)
{
    return pairs + std::min<uint64_t>(pairs, experts) * (align - 1);
}

lcpp_status plan(void* temp, size_t temp_bytes, const int32_t* experts, int32_t* starts, int32_t* row_of,
                 int32_t* pair_of, uint64_t tokens, uint32_t top_k, uint32_t num_experts, uint32_t align,
                 uint64_t max_rows, cudaStream_t s)
{
    if (!counts_ok(tokens, top_k, num_experts, max_rows) || !align) return LCPP_ERR_INVALID_ARG;
    const uint64_t pairs = tokens * top_k;
    if (rows_needed(pairs, num_experts, align) >> 31) return LCPP_ERR_INVALID_ARG;
    if (!temp || misaligned(temp, kTempAlign) || !starts || (pairs && (!experts || !row_of)) || (max_rows && !pair_of))
        return LCPP_ERR_INVALID_ARG;
    const void* words[] = {experts, starts, row_of, pair_of};
    for (const void* w : words)
        if (misaligned(w, 4)) return LCPP_ERR_INVALID_ARG;
    // the pairs are walked twice
    if (overlap(experts, pairs * 4, row_of, pairs * 4) || overlap(experts, pairs * 4, pair_of, max_rows * 4) ||
        overlap(experts, pairs * 4, starts, (uint64_t(num_experts) + 1) * 4))
        return LCPP_ERR_INVALID_ARG;
    if (temp_bytes < plan_bytes(pairs, num_experts)) return LCPP_ERR_TEMP_TOO_SMALL;
    const uint64_t tiles = std::min(kMaxTiles, tiles_for(pairs));
    PlanParams p{};
    p.experts = experts;
    p.starts = starts;
    p.row_of = row_of;
    p.pair_of = pair_of;
    p.pairs = uint32_t(pairs);
    p.num_experts = num_experts;
    p.align = align;
    p.max_rows = uint32_t(max_rows);
    p.per_warp = uint32_t(align_up(ceil_div(ceil_div(pairs, tiles), kPlanWarps), kWarp));
    p.tile = p.per_warp * kPlanWarps;
    p.ctrl = static_cast<uint32_t*>(temp);
    p.table = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(temp) + kTempAlign);
    const unsigned grid = unsigned(std::max<uint64_t>(1, pairs ? ceil_div(pairs, p.tile) : 1));
    const size_t smem = size_t(kPlanWarps + 2) * num_experts * 4;
    set_max_dynamic_smem(reinterpret_cast<const void*>(plan_kernel), size_t(kPlanWarps + 2) * LCPP_MAX_EXPERTS * 4);
    diag::KernelTimer timer(kTimerDispatch, pairs, s);
    if (grid > 1) count_kernel<<<grid, kPlanThreads, num_experts * 4, s>>>(p);
    plan_kernel<<<grid, kPlanThreads, smem, s>>>(p);
    return launched();
}

// Widest access that every row start and the row length allow.
struct Access {
    const void* base;
    uint64_t pitch;
};

template <size_t N>
int unit_bytes(const Access (&rows)[N], uint64_t row_bytes)
{
    uint64_t bits = row_bytes | 16;
    for (const Access& a : rows) bits |= reinterpret_cast<uintptr_t>(a.base) | a.pitch;
    return int(bits & (~bits + 1));  // the lowest set bit, at most 16
}

template <typename F>
lcpp_status with_unit(int bytes, F&& fn)
{
    switch (bytes) {
    case 16: return fn(std::integral_constant<int, 16>{});
    case 8: return fn(std::integral_constant<int, 8>{});
    case 4: return fn(std::integral_constant<int, 4>{});
    default: return fn(std::integral_constant<int, 2>{});
    }
}

uint32_t lanes_log2_for(uint64_t units)
{
    uint32_t log = 0;
    while (log < 8 && (uint64_t(1) << log) < units) ++log;  // at most kRowThreads
    return log;
}

bool strides_ok(uint64_t hidden, std::initializer_list<uint64_t> strides)
{
    if (hidden >> 31) return false;
    for (uint64_t s : strides)
        if (s < hidden || s >> 32) return false;
    return true;
}

lcpp_status gather(const void* x, uint64_t x_stride, const int32_t* row_of, const int32_t* pair_of,
                   const int32_t* starts, void* rows, uint64_t rows_stride, uint64_t tokens, uint32_t top_k,
                   uint32_t num_experts, uint64_t max_rows, uint64_t hidden, lcpp_dtype dtype, cudaStream_t s)
{
    const int size = row_dtype_bytes(dtype);
    if (!size) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!counts_ok(tokens, top_k, num_experts, max_rows) || !strides_ok(hidden, {x_stride, rows_stride}))
        return LCPP_ERR_INVALID_ARG;
    if (!hidden || !max_rows) return LCPP_OK;
    if (!pair_of || !starts || !rows || (tokens && (!x || !row_of))) return LCPP_ERR_INVALID_ARG;
    if (misaligned(x, size) || misaligned(rows, size) || misaligned(row_of, 4) || misaligned(pair_of, 4) ||
        misaligned(starts, 4))
        return LCPP_ERR_INVALID_ARG;
    if (overlap(x, span_bytes(tokens, x_stride, hidden, size), rows, span_bytes(max_rows, rows_stride, hidden, size)))
        return LCPP_ERR_INVALID_ARG;
    RowParams p{};
    p.x = static_cast<const unsigned char*>(x);
    p.x_pitch = x_stride * size;
    p.out = static_cast<unsigned char*>(rows);
    p.out_pitch = rows_stride * size;
    p.row_of = row_of;
    p.pair_of = pair_of;
    p.starts = starts;
    p.tokens = uint32_t(tokens);
    p.top_k = top_k;
    p.num_experts = num_experts;
    p.max_rows = uint32_t(max_rows);
    const Access accesses[] = {{x, p.x_pitch}, {rows, p.out_pitch}};
    const int ub = unit_bytes(accesses, hidden * size);
    p.units = uint32_t(hidden * size / ub);
    p.lanes_log2 = lanes_log2_for(ceil_div(p.units, 2));
    p.chunks = uint32_t(ceil_div(p.units, uint64_t(2) << p.lanes_log2));
    p.pad_blocks = uint32_t(ceil_div(max_rows, kPadRows));
    const uint64_t grid = p.pad_blocks + ceil_div(tokens, kRowThreads >> p.lanes_log2) * p.chunks;
    if (grid >> 31) return LCPP_ERR_INVALID_ARG;
    diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
    return with_unit(ub, [&](auto unit) {
        gather_kernel<decltype(unit)::value><<<unsigned(grid), kRowThreads, 0, s>>>(p);
        return launched();
    });
}

lcpp_status combine(const void* rows, uint64_t rows_stride, const int32_t* row_of, const float* weights, void* out,
                    uint64_t out_stride, uint64_t tokens, uint32_t top_k, uint64_t max_rows, uint64_t hidden,
                    lcpp_dtype dtype, cudaStream_t s)
{
    const int size = row_dtype_bytes(dtype);
    if (!size) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!counts_ok(tokens, top_k, 1, max_rows) || !strides_ok(hidden, {rows_stride, out_stride}))
        return LCPP_ERR_INVALID_ARG;
    if (!hidden || !tokens) return LCPP_OK;
    if (!row_of || !out || (max_rows && !rows)) return LCPP_ERR_INVALID_ARG;
    if (misaligned(rows, size) || misaligned(out, size) || misaligned(row_of, 4) || misaligned(weights, 4))
        return LCPP_ERR_INVALID_ARG;
    if (overlap(out, span_bytes(tokens, out_stride, hidden, size), rows, span_bytes(max_rows, rows_stride, hidden, size)))
        return LCPP_ERR_INVALID_ARG;
    RowParams p{};
    p.rows = static_cast<const unsigned char*>(rows);
    p.rows_pitch = rows_stride * size;
    p.out = static_cast<unsigned char*>(out);
    p.out_pitch = out_stride * size;
    p.row_of = row_of;
    p.weights = weights;
    p.tokens = uint32_t(tokens);
    p.top_k = top_k;
    p.max_rows = uint32_t(max_rows);
    const Access accesses[] = {{rows, p.rows_pitch}, {out, p.out_pitch}};
    const int ub = unit_bytes(accesses, hidden * size);
    p.units = uint32_t(hidden * size / ub);
    p.lanes_log2 = lanes_log2_for(p.units);
    p.chunks = uint32_t(ceil_div(p.units, uint64_t(1) << p.lanes_log2));
    const uint64_t grid = ceil_div(tokens, kRowThreads >> p.lanes_log2) * p.chunks;
    if (grid >> 31) return LCPP_ERR_INVALID_ARG;
    diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
    return with_row_type(dtype, [&](auto t) {
        using T = decltype(t);
        return with_unit(ub, [&](auto unit) {
            constexpr int kUb = decltype(unit)::value;
            if constexpr (kUb >= int(sizeof(T)))
                combine_kernel<T, kUb><<<unsigned(grid), kRowThreads, 0, s>>>(p);
            return launched();
        });
    });
}

lcpp_status combine_backward(const void* grad_out, uint64_t grad_out_stride, const void* rows, uint64_t rows_stride,
                             const int32_t* row_of, const int32_t* pair_of, const int32_t* starts,
                             const float* weights, void* grad_rows, uint64_t grad_rows_stride, float* grad_weights,
                             uint64_t tokens, uint32_t top_k, uint32_t num_experts, uint64_t max_rows,
                             uint64_t hidden, lcpp_dtype dtype, cudaStream_t s)
{
    const int size = row_dtype_bytes(dtype);
    if (!size) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!counts_ok(tokens, top_k, num_experts, max_rows) ||
        !strides_ok(hidden, {grad_out_stride, rows_stride, grad_rows_stride}))
        return LCPP_ERR_INVALID_ARG;
    if (tokens && (!row_of || !weights || !grad_weights || (hidden && !grad_out))) return LCPP_ERR_INVALID_ARG;
    if (max_rows && (!pair_of || !starts || (hidden && (!rows || !grad_rows)))) return LCPP_ERR_INVALID_ARG;
    if (misaligned(grad_out, size) || misaligned(rows, size) || misaligned(grad_rows, size) ||
        misaligned(row_of, 4) || misaligned(pair_of, 4) || misaligned(starts, 4) || misaligned(weights, 4) ||
        misaligned(grad_weights, 4))
        return LCPP_ERR_INVALID_ARG;
    const uint64_t rows_span = span_bytes(max_rows, rows_stride, hidden, size),
                   grad_rows_span = span_bytes(max_rows, grad_rows_stride, hidden, size);
    // in place: a row is read and written by the same thread, unit by unit
    if (!(rows == grad_rows && rows_stride == grad_rows_stride) && overlap(rows, rows_span, grad_rows, grad_rows_span))
        return LCPP_ERR_INVALID_ARG;
    if (overlap(grad_out, span_bytes(tokens, grad_out_stride, hidden, size), grad_rows, grad_rows_span))
        return LCPP_ERR_INVALID_ARG;
    RowParams p{};
    p.x = static_cast<const unsigned char*>(grad_out);
    p.x_pitch = grad_out_stride * size;
    p.rows = static_cast<const unsigned char*>(rows);
    p.rows_pitch = rows_stride * size;
    p.out = static_cast<unsigned char*>(grad_rows);
    p.out_pitch = grad_rows_stride * size;
    p.row_of = row_of;
    p.pair_of = pair_of;
    p.starts = starts;
    p.weights = weights;
    p.grad_weights = grad_weights;
    p.tokens = uint32_t(tokens);
    p.top_k = top_k;
    p.num_experts = num_experts;
    p.max_rows = uint32_t(max_rows);
    const Access accesses[] = {{grad_out, p.x_pitch}, {rows, p.rows_pitch}, {grad_rows, p.out_pitch}};
    const int ub = unit_bytes(accesses, hidden * size);
    p.units = uint32_t(hidden * size / ub);
    p.lanes_log2 = lanes_log2_for(p.units);
    p.pad_blocks = uint32_t(ceil_div(max_rows, kPadRows));
    const uint64_t grid = p.pad_blocks + ceil_div(tokens, kRowThreads >> p.lanes_log2);
    if (!grid) return LCPP_OK;
    if (grid >> 31) return LCPP_ERR_INVALID_ARG;
    diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
    return with_row_type(dtype, [&](auto t) {
        using T = decltype(t);
        return with_unit(ub, [&](auto unit) {
            constexpr int kUb = decltype(unit)::value;
            if constexpr (kUb >= int(sizeof(T)))
                combine_backward_kernel<T, kUb><<<unsigned(grid), kRowThreads, 0, s>>>(p);
            return launched();
        });
    });
}

}  // namespace

extern "C" {

lcpp_status lcpp_dispatch_temp_bytes(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, size_t* temp_bytes)
{
    if (!temp_bytes || !counts_ok(num_tokens, top_k, num_experts, 0)) return LCPP_ERR_INVALID_ARG;
    *temp_bytes = plan_bytes(num_tokens * top_k, num_experts);
    return LCPP_OK;
}

lcpp_status lcpp_dispatch_max_rows(uint64_t num_tokens, uint32_t top_k, uint32_t num_experts, uint32_t row_align,
                                   uint64_t* max_rows)
{
    if (!max_rows || !row_align || !counts_ok(num_tokens, top_k, num_experts, 0)) return LCPP_ERR_INVALID_ARG;
    *max_rows = rows_needed(num_tokens * top_k, num_experts, row_align);
    return LCPP_OK;
}

lcpp_status lcpp_dispatch_plan(void* temp, size_t temp_bytes, const int32_t* d_experts, int32_t* d_expert_starts_out,
                               int32_t* d_row_of_out, int32_t* d_pair_of_out, uint64_t num_tokens, uint32_t top_k,
                               uint32_t num_experts, uint32_t row_align, uint64_t max_rows, lcpp_stream_t stream)
{
    return guarded("lcpp_dispatch_plan", [&] {
        return plan(temp, temp_bytes, d_experts, d_expert_starts_out, d_row_of_out, d_pair_of_out, num_tokens, top_k,
                    num_experts, row_align, max_rows, reinterpret_cast<cudaStream_t>(stream));
    });
}

lcpp_status lcpp_dispatch_gather(const void* d_x, uint64_t x_stride, const int32_t* d_row_of,
                                 const int32_t* d_pair_of, const int32_t* d_expert_starts, void* d_rows_out,
                                 uint64_t rows_stride, uint64_t num_tokens, uint32_t top_k, uint32_t num_experts,
                                 uint64_t max_rows, uint64_t hidden, lcpp_dtype dtype, lcpp_stream_t stream)
{
    return guarded("lcpp_dispatch_gather", [&] {
        return gather(d_x, x_stride, d_row_of, d_pair_of, d_expert_starts, d_rows_out, rows_stride, num_tokens, top_k,
                      num_experts, max_rows, hidden, dtype, reinterpret_cast<cudaStream_t>(stream));
    });
}

lcpp_status lcpp_dispatch_combine(const void* d_rows, uint64_t rows_stride, const int32_t* d_row_of,
                                  const float* d_weights, void* d_out, uint64_t out_stride, uint64_t num_tokens,
                                  uint32_t top_k, uint64_t max_rows, uint64_t hidden, lcpp_dtype dtype,
                                  lcpp_stream_t stream)
{
    return guarded("lcpp_dispatch_combine", [&] {
        return combine(d_rows, rows_stride, d_row_of, d_weights, d_out, out_stride, num_tokens, top_k, max_rows,
                       hidden, dtype, reinterpret_cast<cudaStream_t>(stream));
    });
}

lcpp_status lcpp_dispatch_combine_backward(const void* d_grad_out, uint64_t grad_out_stride, const void* d_rows,
                                           uint64_t rows_stride, const int32_t* d_row_of, const int32_t* d_pair_of,
                                           const int32_t* d_expert_starts, const float* d_weights,
                                           void* d_grad_rows_out, uint64_t grad_rows_stride,
                                           float* d_grad_weights_out, uint64_t num_tokens, uint32_t top_k,
                                           uint32_t num_experts, uint64_t max_rows, uint64_t hidden,
                                           lcpp_dtype dtype, lcpp_stream_t stream)
{
    return guarded("lcpp_dispatch_combine_backward", [&] {
        return combine_backward(d_grad_out, grad_out_stride, d_rows, rows_stride, d_row_of, d_pair_of, d_expert_starts,
                                d_weights, d_grad_rows_out, grad_rows_stride, d_grad_weights_out, num_tokens, top_k,
                                num_experts, max_rows, hidden, dtype, reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
