// dispatch.cu -- DeviceDispatch (include/lcpp_b200_model.h): the (token,
// expert) pairs of a routed step grouped by expert, their rows moved there and
// summed back, and the gradients of both.
//
// Plan is a stable counting sort with one digit, the expert.  Every warp
// counts the experts of its own run of pairs in shared memory; sums of the
// counts over the warps before it, the blocks before it and the experts
// before it give each (warp, expert) its first row, and a second walk over the
// run ranks each 32 pairs by ballots.  Up to kSmallPairs pairs one block
// does all; beyond that up to one block per SM counts its tile in a first
// launch, and in a second one every block adds up all tiles' counts itself (a
// few hundred KB from L2) before it ranks its tile.
//
// 131072 pairs of 256 experts take 9.1 us in two launches, 128 pairs of 128
// experts 3.4 us in one of 256 threads: both are latency (the second launch waits
// 2.3 us for the tiles' counts and as long for the walks).
//
// The row kernels work by token: x (or its gradient) is read once and goes to,
// or comes from, the token's rows, so nothing but those rows is read or
// written top_k times.  They are bound by HBM: gather moves (1 + k) rows a
// token, combine the same, combine's gradient 1 + 2k.  Measured with 4096
// bfloat16 columns, 16384 tokens, 8 of 256 experts, segments of 128: gather
// 212 us (1.21 GB and 134 MB of zeros in padding rows, 6.3 TB/s), combine 175 us
// (1.21 GB, 6.9 TB/s: above the copy rate of 6.4, half of which is writes; eight of
// combine's nine rows are reads, which reach 7.0 alone), its gradient 373 us
// (2.28 GB and the padding, 6.5 TB/s).
#include "model.cuh"

using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kFewThreads = 256;
// These, of at most kFewThreads experts, take a block of kFewThreads: 256 pairs of
// 8, 64, 128 and 256 experts 2.5, 3.0, 3.5 and 4.4 us against 3.2, 3.4, 3.7 and 4.3
// with kPlanThreads, but 512 pairs 3.0, 3.6, 4.0 and 5.0 against 3.2, 3.5, 3.7 and 4.3.
constexpr uint64_t kFewPairs = 256;
// These take one block: 2048 pairs of 64, 256 and 1024 experts 5.0, 5.9 and 9.9 us
// against 6.2, 6.9 and 10.0 in two launches, 4096 pairs 6.5, 7.4 and 11.6 against
// 6.3, 6.8 and 9.5.
constexpr uint64_t kSmallPairs = 2048;
// Fewest pairs of a block among several: 16384 pairs of 256 experts 7.1 us, the
// same with 256 or 512, 7.9 with 2048.
constexpr uint64_t kTilePairs = 1024;

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
    uint32_t* table;    // [tiles][table_pitch]
    uint32_t table_pitch;  // num_experts, rounded up to 4
};

// Exclusive sum over the block of one value per thread.
template <int THREADS>
__device__ uint32_t block_exclusive(uint32_t v, uint32_t* warp_sums)
{
    constexpr int kWarps = THREADS / kWarp;
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
        uint32_t w = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
        for (int d = 1; d < kWarps; d *= 2) {
            const uint32_t o = __shfl_up_sync(~0u, w, d);
            if (lane >= d) w += o;
        }
        if (lane < kWarps) warp_sums[lane] = w;
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
    for (uint32_t e = threadIdx.x; e < p.table_pitch; e += kPlanThreads)
        p.table[blockIdx.x * p.table_pitch + e] = e < p.num_experts ? count[e] : 0;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) plan_kernel(const PlanParams p)
{
    constexpr int kWarps = THREADS / kWarp;
    const uint32_t n = p.num_experts;
    extern __shared__ uint32_t dynamic[];
    uint32_t* counter = dynamic;                  // [kWarps][n], then each (warp, expert)'s next row
    uint32_t* earlier = counter + kWarps * n; // [n] pairs of earlier tiles
    uint32_t* total = earlier + n;                // [n] pairs of all tiles
    __shared__ uint32_t warp_sums[kWarps];
    const uint32_t lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const uint32_t tile_first = blockIdx.x * p.tile, tile_last = min(tile_first + p.tile, p.pairs);
    const uint32_t first = min(tile_first + warp * p.per_warp, tile_last), last = min(first + p.per_warp, tile_last);
    uint32_t* mine = counter + warp * n;

    for (uint32_t i = threadIdx.x; i < (kWarps + 2) * n; i += THREADS) counter[i] = 0;
    __syncthreads();
    for (uint32_t i = first + lane; i < last; i += kWarp) {
        const uint32_t e = uint32_t(p.experts[i]);
        if (e < n) atomicAdd(mine + e, 1u);
    }
    if (gridDim.x > 1) {
        // Threads in groups of one per four experts, each group a share of the
        // tiles (at most kMaxTiles): a thread's loads are all in flight at once.
        const uint32_t quads = p.table_pitch / 4, groups = THREADS / quads, group = threadIdx.x / quads;
        const uint32_t quad = threadIdx.x - group * quads;
        if (group < groups) {
            uint4 before{0, 0, 0, 0}, all{0, 0, 0, 0};
#pragma unroll 8
            for (uint32_t b = group; b < gridDim.x; b += groups) {
                const uint4 c = reinterpret_cast<const uint4*>(p.table + b * p.table_pitch)[quad];
                const bool is = b < blockIdx.x;
                all = uint4{all.x + c.x, all.y + c.y, all.z + c.z, all.w + c.w};
                before = uint4{before.x + (is ? c.x : 0), before.y + (is ? c.y : 0), before.z + (is ? c.z : 0),
                               before.w + (is ? c.w : 0)};
            }
            const uint32_t alls[4] = {all.x, all.y, all.z, all.w}, befores[4] = {before.x, before.y, before.z, before.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t e = quad * 4 + i;
                if (e < n && alls[i]) atomicAdd(total + e, alls[i]);
                if (e < n && befores[i]) atomicAdd(earlier + e, befores[i]);
            }
        }
    }
    __syncthreads();
    // one thread per expert (n <= THREADS): its segment, then its row for every warp
    uint32_t count = 0, segment = 0;
    if (threadIdx.x < n) {
        uint32_t in_block = 0;
        for (int w = 0; w < kWarps; ++w) in_block += counter[w * n + threadIdx.x];
        count = gridDim.x > 1 ? total[threadIdx.x] : in_block;
        segment = (count + p.align - 1) / p.align * p.align;
    }
    const uint32_t start = block_exclusive<THREADS>(segment, warp_sums);
    if (threadIdx.x < n) {
        uint32_t row = start + earlier[threadIdx.x];
        for (int w = 0; w < kWarps; ++w) {
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
        // lanes with the same expert, by its bits
        uint32_t peers = __ballot_sync(~0u, valid);
        for (uint32_t b = 1; b < n; b *= 2) {
            const uint32_t ones = __ballot_sync(~0u, e & b);
            peers &= e & b ? ones : ~ones;
        }
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
    for (uint32_t e = blockIdx.x * kWarps + warp; e < n; e += gridDim.x * kWarps)
        for (uint32_t r = earlier[e] + lane; r < min(total[e], p.max_rows); r += kWarp) p.pair_of[r] = -1;
    for (uint64_t r = uint64_t(total[n - 1]) + blockIdx.x * THREADS + threadIdx.x; r < p.max_rows;
         r += uint64_t(gridDim.x) * THREADS)
        p.pair_of[r] = -1;
}

// ---------------------------------------------------------------------------
// Row kernels.  A row is `units` accesses of UB bytes; `lanes` threads (a power
// of two) share a token.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kPadRows = 64;   // most rows a block looks through for padding

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
    uint32_t pad_rows;           // rows of a padding block
    uint32_t chunks;             // column chunks of a token
    uint32_t rows_per_pass;      // expert rows of a token taken together
};

// Zeros in the padding rows among this block's pad_rows rows.
template <int UB>
__device__ void clear_padding(const RowParams& p, uint32_t block)
{
    using U = typename Unit<UB>::type;
    __shared__ uint32_t masks[kPadRows / kWarp];
    const uint32_t first = block * p.pad_rows;
    const uint32_t end = min(min(uint32_t(p.starts[p.num_experts]), p.max_rows), first + p.pad_rows);
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

// Tokens' rows copied to their experts' rows, N accesses per thread.  Blocks:
// first the padding's.  16 bytes per thread: 222 us with the plan at the sizes
// above, 32 and 64 bytes 227, and no faster with streaming stores.
template <int UB, int N>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    if (blockIdx.x < p.pad_blocks) {
        clear_padding<UB>(p, blockIdx.x);
        return;
    }
    const uint32_t block = blockIdx.x - p.pad_blocks;
    const uint32_t lanes = 1u << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t t = (block / p.chunks) * (kRowThreads >> p.lanes_log2) + (threadIdx.x >> p.lanes_log2);
    if (t >= p.tokens) return;
    const U* x = reinterpret_cast<const U*>(p.x + uint64_t(t) * p.x_pitch);
    const uint32_t u0 = (block % p.chunks) * lanes * N + lane;
    U v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (u0 + i * lanes < p.units) v[i] = x[u0 + i * lanes];
    const int32_t* row_of = p.row_of + uint64_t(t) * p.top_k;
#pragma unroll 4
    for (uint32_t j = 0; j < p.top_k; ++j) {
        const uint32_t r = uint32_t(row_of[j]);
        if (r >= p.max_rows) continue;
        U* row = reinterpret_cast<U*>(p.out + uint64_t(r) * p.out_pitch);
#pragma unroll
        for (int i = 0; i < N; ++i)
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

// out[t] = sum_j w[t][j] rows[row_of[t][j]]: N accesses per thread of R rows at
// a time, all in flight before the first is used.  R x N of 16-byte accesses at
// 16384 x 4096, 8 rows: 4 x 2 175 us, 8 x 1 203, 6 x 1 210; of 2-byte ones
// (2881 columns, which allow no wider access) at 8191 tokens, 6 rows: 2 x 16
// 130 us, 4 x 8 162, 4 x 16 360.
template <typename T, int UB, int R, int N>
__global__ void __launch_bounds__(kRowThreads, 4) combine_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    constexpr int kN = UB / int(sizeof(T));
    const uint32_t lanes = 1u << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t t = (blockIdx.x / p.chunks) * (kRowThreads >> p.lanes_log2) + (threadIdx.x >> p.lanes_log2);
    const uint32_t u0 = (blockIdx.x % p.chunks) * lanes * N + lane;
    if (t >= p.tokens || u0 >= p.units) return;
    const int32_t* row_of = p.row_of + uint64_t(t) * p.top_k;
    const float* weights = p.weights ? p.weights + uint64_t(t) * p.top_k : nullptr;
    float acc[N][kN];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < kN; ++e) acc[i][e] = 0.f;
    for (uint32_t j0 = 0; j0 < p.top_k; j0 += p.rows_per_pass) {
        const uint32_t j1 = min(j0 + p.rows_per_pass, p.top_k);
        U raw[R][N];
        float w[R];
        bool has[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const uint32_t r = j0 + j < j1 ? uint32_t(row_of[j0 + j]) : ~0u;
            has[j] = r < p.max_rows;
            w[j] = has[j] && weights ? weights[j0 + j] : 1.f;
            const U* row = reinterpret_cast<const U*>(p.rows + uint64_t(has[j] ? r : 0) * p.rows_pitch);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (has[j] && u0 + i * lanes < p.units) raw[j][i] = row[u0 + i * lanes];
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!has[j]) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float v[kN];
                unpack<T, UB>(raw[j][i], v);
#pragma unroll
                for (int e = 0; e < kN; ++e) acc[i][e] = fmaf(w[j], v[e], acc[i][e]);
            }
        }
    }
    U* out = reinterpret_cast<U*>(p.out + uint64_t(t) * p.out_pitch);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (u0 + i * lanes < p.units) out[u0 + i * lanes] = pack<T, UB>(acc[i]);
}

// out[row] = w dy and grad_w = <rows[row], dy>, a token's lanes walking its
// columns once per pass of up to R experts; the dot products are summed over a
// warp by shuffles and over a token's warps in order.  R x N of 16-byte accesses:
// 4 x 2 and 8 x 1 take 373 and 366 us at 8 rows of 4096 (16384 tokens), 122 and
// 133 at 10 rows of 2048, 65 and 100 at 2 rows, where 2 x 4 takes 57.
template <typename T, int UB, int R, int N>
__global__ void __launch_bounds__(kRowThreads, 3) combine_backward_kernel(const RowParams p)
{
    using U = typename Unit<UB>::type;
    constexpr int kN = UB / int(sizeof(T));
    constexpr int kRowWarps = kRowThreads / kWarp;
    __shared__ float part[kRowWarps][R];
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
    for (uint32_t j0 = 0; j0 < p.top_k; j0 += p.rows_per_pass) {
        const uint32_t j1 = min(j0 + p.rows_per_pass, p.top_k);
        uint32_t row[R];
        float w[R], dot[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool is = inside && j0 + j < j1;
            row[j] = is ? uint32_t(row_of[j0 + j]) : ~0u;
            w[j] = is ? weights[j0 + j] : 0.f;
            dot[j] = 0.f;
        }
        for (uint32_t u0 = lane; u0 < p.units; u0 += lanes * N) {
            U own[N], raw[R][N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (u0 + i * lanes < p.units) own[i] = dy[u0 + i * lanes];
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (row[j] >= p.max_rows) continue;
                const U* from = reinterpret_cast<const U*>(p.rows + uint64_t(row[j]) * p.rows_pitch);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (u0 + i * lanes < p.units) raw[j][i] = from[u0 + i * lanes];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (u0 + i * lanes >= p.units) continue;
                float g[kN];
                unpack<T, UB>(own[i], g);
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    if (row[j] >= p.max_rows) continue;
                    float v[kN];
                    unpack<T, UB>(raw[j][i], v);
#pragma unroll
                    for (int e = 0; e < kN; ++e) {
                        dot[j] = fmaf(v[e], g[e], dot[j]);
                        v[e] = w[j] * g[e];
                    }
                    reinterpret_cast<U*>(p.out + uint64_t(row[j]) * p.out_pitch)[u0 + i * lanes] = pack<T, UB>(v);
                }
            }
        }
        const uint32_t in_warp = min(lanes, uint32_t(kWarp));
#pragma unroll
        for (int j = 0; j < R; ++j)
            for (uint32_t d = in_warp / 2; d > 0; d /= 2) dot[j] += __shfl_xor_sync(~0u, dot[j], d);
        if (lanes > kWarp) {
            const uint32_t warp = threadIdx.x / kWarp, token_warps = lanes / kWarp;
            if (threadIdx.x % kWarp == 0) {
#pragma unroll
                for (int j = 0; j < R; ++j) part[warp][j] = dot[j];
            }
            __syncthreads();
            if (inside && lane < R && j0 + lane < j1) {
                float sum = 0.f;
                for (uint32_t i = 0; i < token_warps; ++i) sum += part[warp + i][lane];
                p.grad_weights[uint64_t(t) * p.top_k + j0 + lane] = sum;
            }
            __syncthreads();
        } else if (inside && lane == 0) {
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (j0 + j < j1) p.grad_weights[uint64_t(t) * p.top_k + j0 + j] = dot[j];
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
    return kTempAlign + align_up(std::min(kMaxTiles, ceil_div(pairs, kTilePairs)) * align_up(experts, 4) * 4, kTempAlign);
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
    if (temp_bytes < plan_bytes(pairs, num_experts)) return LCPP_ERR_TEMP_TOO_SMALL;
    const Array arrays[] = {{experts, pairs * 4, false},
                            {starts, (uint64_t(num_experts) + 1) * 4, true},
                            {row_of, pairs * 4, true},
                            {pair_of, max_rows * 4, true},
                            {temp, plan_bytes(pairs, num_experts), true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
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
    const bool few = pairs <= kFewPairs && num_experts <= uint32_t(kFewThreads);
    const int threads = few ? kFewThreads : kPlanThreads, warps = threads / kWarp;
    p.per_warp = uint32_t(align_up(ceil_div(ceil_div(pairs, tiles), warps), kWarp));
    p.tile = p.per_warp * warps;
    p.ctrl = static_cast<uint32_t*>(temp);
    p.table = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(temp) + kTempAlign);
    p.table_pitch = uint32_t(align_up(num_experts, 4));
    const unsigned grid = unsigned(std::max<uint64_t>(1, pairs ? ceil_div(pairs, p.tile) : 1));
    const size_t smem = size_t(warps + 2) * num_experts * 4;
    diag::KernelTimer timer(kTimerDispatch, pairs, s);
    if (few) {
        plan_kernel<kFewThreads><<<1, threads, smem, s>>>(p);
        return launched();
    }
    set_max_dynamic_smem(reinterpret_cast<const void*>(plan_kernel<kPlanThreads>),
                         size_t(kPlanThreads / kWarp + 2) * LCPP_MAX_EXPERTS * 4);
    if (grid > 1) count_kernel<<<grid, kPlanThreads, num_experts * 4, s>>>(p);
    plan_kernel<kPlanThreads><<<grid, threads, smem, s>>>(p);
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

// Padding is looked for by up to four blocks per SM.
void set_padding(RowParams& p)
{
    p.pad_rows = uint32_t(std::min<uint64_t>(kPadRows, std::max<uint64_t>(1, ceil_div(p.max_rows, uint64_t(device_sm_count()) * 4))));
    p.pad_blocks = uint32_t(ceil_div(p.max_rows, p.pad_rows));
}

// Threads per token: of 32 to kRowThreads the power of two that leaves the
// fewest idle in the last chunk (the larger of equals), fewer for short rows.
uint32_t lanes_log2_for(uint64_t units, int per_thread)
{
    uint32_t best = 0;
    while (best < 5 && (uint64_t(per_thread) << best) < units) ++best;
    if (best < 5) return best;
    uint64_t best_slots = ~0ull;
    for (uint32_t log = 5; (1 << log) <= kRowThreads; ++log) {
        const uint64_t slots = align_up(units, uint64_t(per_thread) << log);
        if (slots <= best_slots) {
            best = log;
            best_slots = slots;
        }
    }
    return best;
}

// top_k rows in equal passes of at most `most`.
uint32_t rows_per_pass_for(uint32_t top_k, int most) { return uint32_t(ceil_div(top_k, ceil_div(top_k, most))); }

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
    const Array inputs[] = {{row_of, tokens * top_k * 4, false}, {pair_of, max_rows * 4, false},
                            {starts, (uint64_t(num_experts) + 1) * 4, false}};
    for (const Array& i : inputs)
        if (overlap_rows(rows, max_rows, rows_stride, hidden, size, i.p, i.bytes)) return LCPP_ERR_INVALID_ARG;
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
    return with_unit(ub, [&](auto unit) {
        constexpr int kUb = decltype(unit)::value, kN = std::min(8, 16 / kUb);
        p.lanes_log2 = lanes_log2_for(p.units, kN);
        p.chunks = uint32_t(ceil_div(p.units, uint64_t(kN) << p.lanes_log2));
        set_padding(p);
        const uint64_t grid = p.pad_blocks + ceil_div(tokens, kRowThreads >> p.lanes_log2) * p.chunks;
        if (grid >> 31) return LCPP_ERR_INVALID_ARG;
        diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
        gather_kernel<kUb, kN><<<unsigned(grid), kRowThreads, 0, s>>>(p);
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
    for (const void* i : {static_cast<const void*>(row_of), static_cast<const void*>(weights)})
        if (overlap_rows(out, tokens, out_stride, hidden, size, i, tokens * top_k * 4)) return LCPP_ERR_INVALID_ARG;
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
    return with_row_type(dtype, [&](auto t) {
        using T = decltype(t);
        return with_unit(ub, [&](auto unit) {
            constexpr int kUb = decltype(unit)::value;
            const auto go = [&](auto kernel, int rows_most, int per_thread) -> lcpp_status {
                p.rows_per_pass = rows_per_pass_for(top_k, rows_most);
                p.lanes_log2 = lanes_log2_for(p.units, per_thread);
                p.chunks = uint32_t(ceil_div(p.units, uint64_t(per_thread) << p.lanes_log2));
                const uint64_t grid = ceil_div(tokens, kRowThreads >> p.lanes_log2) * p.chunks;
                if (grid >> 31) return LCPP_ERR_INVALID_ARG;
                diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
                kernel<<<unsigned(grid), kRowThreads, 0, s>>>(p);
                return launched();
            };
            if constexpr (kUb < int(sizeof(T))) return LCPP_ERR_INTERNAL;  // rows are aligned to their elements
            else if constexpr (kUb < 16) return go(combine_kernel<T, kUb, 2, 32 / kUb>, 2, 32 / kUb);
            else return go(combine_kernel<T, kUb, 4, 2>, 4, 2);
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
    const uint64_t pairs = tokens * top_k;
    // a token's threads read a weight before they write its gradient, so the two may share their place
    const Array arrays[] = {{row_of, pairs * 4, false},
                            {pair_of, max_rows * 4, false},
                            {starts, (uint64_t(num_experts) + 1) * 4, false},
                            {weights == grad_weights ? nullptr : weights, pairs * 4, false},
                            {grad_weights, pairs * 4, true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
    for (const Array& a : arrays) {
        if (overlap_rows(grad_rows, max_rows, grad_rows_stride, hidden, size, a.p, a.bytes) ||
            (a.written && (overlap_rows(grad_out, tokens, grad_out_stride, hidden, size, a.p, a.bytes) ||
                           overlap_rows(rows, max_rows, rows_stride, hidden, size, a.p, a.bytes))))
            return LCPP_ERR_INVALID_ARG;
    }
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
    return with_row_type(dtype, [&](auto t) {
        using T = decltype(t);
        return with_unit(ub, [&](auto unit) {
            constexpr int kUb = decltype(unit)::value;
            const auto go = [&](auto kernel, int rows_most, int per_thread) -> lcpp_status {
                p.rows_per_pass = rows_per_pass_for(top_k, rows_most);
                // Twice a thread's accesses or more, to share the cost of the sums
                // over a token's lanes, where that still fills the SMs twice.
                const uint64_t wide = uint64_t(per_thread) * kRowThreads * device_sm_count() * 4;
                p.lanes_log2 = lanes_log2_for(p.units, tokens * p.units >= wide ? 2 * per_thread : per_thread);
                set_padding(p);
                const uint64_t grid = p.pad_blocks + ceil_div(tokens, kRowThreads >> p.lanes_log2);
                if (!grid) return LCPP_OK;
                if (grid >> 31) return LCPP_ERR_INVALID_ARG;
                diag::KernelTimer timer(kTimerDispatch, tokens * top_k, s);
                kernel<<<unsigned(grid), kRowThreads, 0, s>>>(p);
                return launched();
            };
            if constexpr (kUb < int(sizeof(T))) return LCPP_ERR_INTERNAL;  // rows are aligned to their elements
            else if constexpr (kUb < 16) return go(combine_backward_kernel<T, kUb, 2, std::min(8, 32 / kUb)>, 2, std::min(8, 32 / kUb));
            else if (top_k <= 2) return go(combine_backward_kernel<T, kUb, 2, 4>, 2, 4);
            else return go(combine_backward_kernel<T, kUb, 4, 2>, 4, 2);
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
