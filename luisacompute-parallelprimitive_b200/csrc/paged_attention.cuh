// paged_attention.cuh -- DevicePagedAttention (include/lcpp_b200_model.h): one
// new query of each request over the pages of its keys and values.
//
// With x_t = scale q . k_t (base 2 from here on), one pass over the tokens keeps
// a reference m, the sum l of 2^(x_t - m) and the vector o of 2^(x_t - m) v_t;
// parts of the tokens join as o = sum_i 2^(m_i - M) o_i, l alike, out = o / l.
// m follows the maximum only when a logit passes it by 2^8: between, a tile costs
// a vote instead of reductions and rescaling, and no term leaves its range.
//
// Work.  A unit is a request's tokens under one kv head, with up to 4 to 32 query
// heads on it (see choose), cut into tiles of 16 tokens.  All tiles of the call are
// numbered and every block takes an equal run of them, so a few long requests
// fill the GPU as well as many short ones.  The lengths are on the device: each
// block sums them itself.  A unit that a run covers whole is written out by its
// block, the parts of the others by join_kernel, which starts early and waits.
//
// A warp works on its own: of a block's four (two for 256 columns of 32 bits) it takes
// every fourth (second) tile of the run, copies the tile's 16 keys, then its 16 values, into slots of a ring of its own with
// cp.async, some slots ahead and across the borders of units, and needs the
// block's other warps only where a unit ends.  Page ids are read four tiles before
// the copies that need them.
//
// Bound by memory where contexts are long: every key and value is read once.  64
// requests of 16384 tokens and fewer, 32 heads on 8 of 128 in bfloat16: 382 to 405 us by
// machine, 6.4 to 6.8 TB/s (a copy reaches 6.5); 2 requests of 131072, 16 on 2 of 256 in
// float16: 78 us, 5.5 TB/s.  301 of 1500 under a window of 1000, 7 of 80 in float32, reach
// 5.3 TB/s (198 us): their slots hold 128 columns, so less is under way.
// Short ones are a chain of latencies (lengths, page ids, keys, values, a part's end,
// the join's launch): 1 request of 700 tokens takes 9.7 us.  Finer runs than equal
// ones, and blocks that the hardware hands out in waves, measured slower.
// The matrix products take 15 % of the tensor cores' time: mma.sync on tiles of 16
// tokens, whose few heads would leave most of a larger instruction's columns empty.
#pragma once

#include "cache.cuh"

namespace lcpp {
namespace model {
namespace attention {

constexpr int kTile = 16;              // tokens of a tile
constexpr uint32_t kMostBlocks = 800;  // the partial results' room
constexpr int32_t kLost = 1 << 30;     // beside a request in `split`: the run wrote a row that is to be computed again
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
    const void* q;
    void* out;
    const void* k;
    const void* v;
    uint64_t q_request, q_head, out_request, out_head;
    uint64_t page_stride, token_stride, head_stride;
    const int32_t* table;
    uint64_t table_stride;
    const int32_t* lens;
    Divider page;         // by the page size
    bool page_tiles;      // a tile lies in one page
    bool wide_q;          // queries start on 16-byte boundaries
    bool wide_out;        // rows of the output on boundaries of four elements
    uint32_t longest;     // tokens that a row of the table holds
    uint32_t num_pages;
    uint32_t requests, heads, kv_heads, group;
    uint32_t chunks;      // units that a kv head's queries are divided into
    uint32_t per_unit;    // query heads of a unit, at most
    uint32_t dim;
    uint32_t window;
    float scale;          // with log2 e, or with 1 / softcap
    float softcap;        // with log2 e; 0: none
    float* lse;
    float* part;          // [block][2][heads of a unit][columns] and, behind them, [block][2][heads of a unit][2]
    int32_t* split;       // [block][4]: request (and kLost), unit, first block and further blocks of the unit that its run ends in
    uint32_t warps;       // of a block of the decode kernel
    Divider by_group, by_unit;  // by `group` and `per_unit`, for the scores
    float* logits;        // [tile][per_unit][16] in base 2, or NULL
    long long logit_tiles;
    float* lse2;          // [request][head] in base 2 for the scores
    long long* first;     // [request] number of its first tile, for the scores
    const float* scores;
    float* scores_out;
    float decay;
};

// A request's tokens that are looked at, [first, end), in tiles that start at
// multiples of 16.
struct Tokens {
    uint32_t first, end;
    __device__ __forceinline__ uint32_t base() const { return first / kTile * kTile; }
    __device__ __forceinline__ uint32_t tiles() const { return (end - base() + kTile - 1) / kTile; }
};
__device__ __forceinline__ Tokens tokens_of_length(const Params& p, int32_t length)
{
    const uint32_t n = min(uint32_t(max(length, 0)), p.longest);
    return Tokens{p.window && n > p.window ? n - p.window : 0u, n};
}
__device__ __forceinline__ Tokens tokens_of(const Params& p, uint32_t r) { return tokens_of_length(p, p.lens[r]); }

// Tiles of a block's run: equal ones, of not less than a tile for each warp unless
// units have fewer (a part's end costs a block a microsecond or two).
__device__ __forceinline__ long long run_of(long long all, uint64_t units, uint32_t blocks, int warps)
{
    const long long equal = (all + blocks - 1) / blocks;
    return equal >= warps ? equal : max(equal, min((long long)warps, (all + (long long)units - 1) / (long long)units));
}

// The block's run of tiles, and the walk over the parts of units in it.
struct Walk {
    uint32_t r, unit, tiles, t, t_end;
    Tokens tokens;
    int32_t next_length;  // of request r + 1, read ahead
    long long left;       // tiles of the run behind this part

    __device__ __forceinline__ void part()
    {
        const long long room = left;
        t_end = uint32_t(min((long long)tiles, t + room));
        left = room - (t_end - t);
    }
    __device__ __forceinline__ void read_ahead(const Params& p) { next_length = r + 1 < p.requests ? p.lens[r + 1] : 0; }
    // At tile `begin` of all, which lies in request `place`, for a run up to `end`.
    __device__ __forceinline__ void start(const Params& p, const Place& place, long long begin, long long end)
    {
        r = place.item;
        tokens = tokens_of(p, r);
        read_ahead(p);
        tiles = tokens.tiles();
        unit = uint32_t((begin - place.first) / tiles);
        t = uint32_t((begin - place.first) - (long long)unit * tiles);
        left = end - begin;
        part();
    }
    // To the part after this one; false: the run has ended.
    __device__ __forceinline__ bool next(const Params& p)
    {
        if (left == 0) return false;
        t = 0;
        if (++unit == p.kv_heads * p.chunks) {
            unit = 0;
            do {  // the run has tiles left, so there is such a request
                tokens = tokens_of_length(p, next_length);
                tiles = tokens.tiles();
                ++r;
                read_ahead(p);
            } while (tiles == 0);
        }
        part();
        return true;
    }
};

__device__ __forceinline__ uint32_t smem_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
// L2 is asked for 64 bytes of a line: rows that begin in the middle of one would
// bring in their neighbours' halves, which other blocks read at other times
// (301 x 1500 tokens of 7 x 80 bfloat16 columns: 150 us with whole lines, 130).
__device__ __forceinline__ void copy_16b(uint32_t to, const void* from, bool valid)
{
    asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_16b(uint32_t to, const void* from)
{
    asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_4b(uint32_t to, const void* from)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float logit(const Params& p, float dot)
{
    const float x = dot * p.scale;
    return p.softcap > 0.f ? p.softcap * tanhf(x) : x;
}
// Factor of what was summed under reference `from` when it becomes `to`.
__device__ __forceinline__ float rebase(float from, float to) { return from == -INFINITY ? 0.f : exp2_fast(from - to); }

// The same for a part that is joined; one whose logits were all NaN has no
// reference, but a sum that says so.
__device__ __forceinline__ float share(float from, float sum, float to)
{
    return from == -INFINITY ? (sum == 0.f ? 0.f : sum) : exp2_fast(from - to);
}
__device__ __forceinline__ void put_lse(const Params& p, uint64_t at, float reference, float sum)
{
    const float value = sum == 0.f ? -INFINITY : reference + log2f(sum);
    if (p.lse) p.lse[at] = value * kLn2;
    if (p.lse2) p.lse2[at] = value;
}

// ---------------------------------------------------------------------------
// A warp's tile in 16 bits: tensor cores, tokens as rows and heads as columns
// of the first product, the head's columns as rows of the second one.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void multiply<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void multiply<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ void multiply_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void multiply_first<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void multiply_first<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Two floats as 16-bit numbers in a word, and what their rounding left out in another.
template <typename T>
__device__ __forceinline__ void split_pair(float low, float high, uint32_t& word, uint32_t& rest);
template <>
__device__ __forceinline__ void split_pair<__nv_bfloat16>(float low, float high, uint32_t& word, uint32_t& rest)
{
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(word) : "f"(high), "f"(low));
    low -= __uint_as_float(word << 16);
    high -= __uint_as_float(word & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(rest) : "f"(high), "f"(low));
}
template <>
__device__ __forceinline__ void split_pair<__half>(float low, float high, uint32_t& word, uint32_t& rest)
{
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(word) : "f"(high), "f"(low));
    low -= __half2float(__ushort_as_half(static_cast<unsigned short>(word)));
    high -= __half2float(__ushort_as_half(static_cast<unsigned short>(word >> 16)));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(rest) : "f"(high), "f"(low));
}

// Swizzle of the 16-byte chunks of rows of CHUNKS: 8 rows of one chunk, or 8 chunks
// of one row, lie in different banks.  Rows of an odd number of 64 bytes alternate
// between the banks' halves by themselves.
template <int CHUNKS>
__device__ __forceinline__ int swizzled(int row, int chunk)
{
    static_assert(CHUNKS % 4 == 0, "");
    return CHUNKS % 8 ? chunk ^ (row >> 1 & 3) : chunk ^ (row & 7);
}
// The address `even` chunks on from a swizzled one of chunk 0 or 1: an exclusive or,
// and a constant.
template <int CHUNKS>
__device__ __forceinline__ uint32_t chunks_on(uint32_t address, int even)
{
    constexpr int kLow = CHUNKS % 8 ? 3 : 7;
    return (address ^ ((even & kLow) * 16)) + (even & ~kLow) * 16;
}

template <typename T, int D, int H>
struct Tile;

// H is a multiple of 8: H / 8 tiles of 8 heads.
template <typename T, int D, int H>
struct Tile16 {
    static constexpr int kN = H / 8;
    static constexpr int kWarpBytes = 0;
    // float16's range: terms are kept at up to 2^8 of the reference, whose own is
    // set 2^7 up, so that they end at 2^15 and small ones keep their digits.
    static constexpr float kShift = std::is_same<T, __half>::value ? 7.f : 0.f;

    float o[D / 16][kN][4];  // column lane / 4 (+ 8), heads lane % 4 * 2 (+ 1)
    float m[kN][2], l[kN][2];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][n][c] = 0.f;
        }
    }

    // The tile's logits from its keys, and its terms: the second product's second
    // operand, as two 16-bit numbers each, high part and rest: 16 digits of bfloat16
    // and 22 of float16, against 8 and 11 that one would leave.  The products with
    // the rest cost tensor-core time that the copies leave free.
    uint32_t high[kN][2], rest[kN][2];

    __device__ __forceinline__ void keys(const Params& p, const unsigned char* rows, const void* queries, void*,
                                         uint32_t valid, float* logits, uint32_t heads)
    {
        // the sum over the columns in several chains: a product waits for the one before it in its chain
        constexpr int kChains = kN == 1 ? 4 : 2;
        const int lane = threadIdx.x % kWarp;
        float c[kChains][kN][4];
        const int row = lane % 16, head = lane % 8;
        const uint32_t at = smem_address(rows) + row * (D * 2) + swizzled<D / 8>(row, lane / 16) * 16;
        // lane / 8 is a chunk of four: two pairs of even ones
        const uint32_t q = smem_address(queries) + head * (D * 2) + chunks_on<D / 8>(swizzled<D / 8>(head, lane / 8 % 2) * 16, lane / 16 * 2);
#pragma unroll
        for (int step = 0; step < D / 16; step += 2) {
            uint32_t a[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) load_matrices(a[i], chunks_on<D / 8>(at, (step + i) * 2));
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                uint32_t b[4];  // the heads' next 32 columns
                load_matrices(b, chunks_on<D / 8>(q, step * 2) + n * 8 * (D * 2));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (step + i < kChains) multiply_first<T>(c[(step + i) % kChains][n], a[i], b[2 * i], b[2 * i + 1]);
                    else multiply<T>(c[(step + i) % kChains][n], a[i], b[2 * i], b[2 * i + 1]);
                }
            }
        }
        float s[kN][4];
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float dot = c[0][n][j] + c[1][n][j];
                if (kChains == 4) dot += c[kChains - 2][n][j] + c[kChains - 1][n][j];
                s[n][j] = dot * p.scale;
            }
        if (p.softcap > 0.f) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = p.softcap * tanhf(s[n][j]);
        }
        if (valid != 0xffffu) {
            const bool valid0 = valid >> (lane / 4) & 1, valid1 = valid >> (lane / 4 + 8) & 1;
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(j < 2 ? valid0 : valid1)) s[n][j] = -INFINITY;
        }
        if (logits) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t of = n * 8 + lane % 4 * 2 + (j & 1);
                    if (of < heads) logits[of * kTile + lane / 4 + (j < 2 ? 0 : 8)] = s[n][j];
                }
        }
        bool past = false;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) past |= s[n][j] > m[n][j & 1] + (8.f + kShift);
        if (__any_sync(~0u, past)) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float top = fmaxf(s[n][h], s[n][h + 2]);
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                    const float to = fmaxf(m[n][h], top - kShift), factor = rebase(m[n][h], to);
                    m[n][h] = to;
                    l[n][h] *= factor;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[i][n][h] *= factor;
                        o[i][n][h + 2] *= factor;
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const float reference[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = exp2_fast(s[n][j] - reference[j & 1]);
            l[n][0] += e[0] + e[2];
            l[n][1] += e[1] + e[3];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                uint32_t word, left;
                split_pair<T>(e[w * 2], e[w * 2 + 1], word, left);
                high[n][w] = transposed(word);
                rest[n][w] = transposed(left);
            }
        }
    }

    __device__ __forceinline__ void values(const unsigned char* rows, const void*)
    {
        const int lane = threadIdx.x % kWarp, row = lane % 8 + lane / 16 * 8;
        const uint32_t at = smem_address(rows) + row * (D * 2) + swizzled<D / 8>(row, lane / 8 % 2) * 16;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            uint32_t a[4];
            load_matrices_transposed(a, chunks_on<D / 8>(at, i * 2));
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                multiply<T>(o[i][n], a, high[n][0], high[n][1]);
                multiply<T>(o[i][n], a, rest[n][0], rest[n][1]);
            }
        }
    }

    // The warp's references and sums, [head].
    __device__ __forceinline__ void put_sums(float* m_out, float* l_out)
    {
        const int lane = threadIdx.x % kWarp;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) l[n][h] += __shfl_xor_sync(~0u, l[n][h], d);
                if (lane < 4) {
                    m_out[n * 8 + lane * 2 + h] = m[n][h];
                    l_out[n * 8 + lane * 2 + h] = l[n][h];
                }
            }
    }
    // The vectors relative to the largest of the warps' references, [warp][head].
    template <int WARPS>
    __device__ __forceinline__ void rescale(const float* m_all)
    {
        const int lane = threadIdx.x % kWarp;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, m_all[w * H + n * 8 + lane % 4 * 2 + h]);
                const float f = share(m[n][h], l[n][h], top);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    o[i][n][h] *= f;
                    o[i][n][h + 2] *= f;
                }
            }
    }
    // Puts the vectors of the pass-th kPass heads to to[head][D], 8 columns swapped
    // with 8 so that the lanes' heads lie in different banks.
    static constexpr int kPass = 8;
    static __device__ __forceinline__ int place(int head, int column) { return head * D + (column ^ (head / 2 % 4 * 8)); }
    __device__ __forceinline__ void put(float* to, int pass)
    {
        const int lane = threadIdx.x % kWarp;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            if (n != pass) continue;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) to[place(lane % 4 * 2 + j % 2, i * 16 + j / 2 * 8 + lane / 4)] = o[i][n][j];
        }
    }
};

template <int D, int H>
struct Tile<__nv_bfloat16, D, H> : Tile16<__nv_bfloat16, D, H> {};
template <int D, int H>
struct Tile<__half, D, H> : Tile16<__half, D, H> {};

// ---------------------------------------------------------------------------
// A warp's tile in 32 bits: multiply-adds.  A lane takes a token and half of the
// columns for the logits, then 4 columns (or 8, or 4 of every second token) of
// all tokens for the vectors; the terms pass through shared memory.
// ---------------------------------------------------------------------------
template <int D, int H>
struct Tile<float, D, H> {
    static constexpr int kWarpBytes = kTile * H * 4;
    static constexpr int kChunks = D / 4;
    static constexpr int kLanes = kChunks < kWarp ? kChunks : kWarp;  // lanes of a row
    static constexpr int kPer = kChunks / kLanes;                    // chunks of a lane
    static constexpr int kTokenStep = kWarp / kLanes;
    static constexpr float kShift = 0.f;
    static_assert(kChunks % kLanes == 0 && kWarp % kLanes == 0, "");

    float4 o[H][kPer];
    float m[H], l[H];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }

    __device__ __forceinline__ void keys(const Params& p, const unsigned char* rows, const void* queries, void* own,
                                         uint32_t valid, float* logits, uint32_t heads)
    {
        const int lane = threadIdx.x % kWarp, token = lane % 16, part = lane / 16;
        const float4* k = reinterpret_cast<const float4*>(rows) + token * kChunks;
        const float4* q = static_cast<const float4*>(queries);
        float s[H];
#pragma unroll
        for (int h = 0; h < H; ++h) s[h] = 0.f;
        const int half = int(p.dim + 7) / 8;  // the chunks that hold columns, in two halves
#pragma unroll 4
        for (int i = 0; i < half; ++i) {
            const int chunk = part * half + i;
            const float4 a = k[swizzled<kChunks>(token, chunk)];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const float4 b = q[h * kChunks + swizzled<kChunks>(h, chunk)];
                s[h] = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s[h]))));
            }
        }
        bool past = false;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            s[h] += __shfl_xor_sync(~0u, s[h], 16);
            s[h] = valid >> token & 1 ? logit(p, s[h]) : -INFINITY;
            past |= s[h] > m[h] + 8.f;
            if (logits && part == 0 && h < int(heads)) logits[h * kTile + token] = s[h];
        }
        if (__any_sync(~0u, past)) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                float top = s[h];
#pragma unroll
                for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                const float to = fmaxf(m[h], top), factor = rebase(m[h], to);
                m[h] = to;
                l[h] *= factor;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    o[h][i].x *= factor, o[h][i].y *= factor, o[h][i].z *= factor, o[h][i].w *= factor;
                }
            }
        }
        float* term = static_cast<float*>(own);
        __syncwarp();  // the tile before has been read
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const float e = exp2_fast(s[h] - (m[h] == -INFINITY ? 0.f : m[h]));
            if (part == 0) {
                l[h] += e;
                term[token * H + h] = e;
            }
        }
        __syncwarp();
    }

    __device__ __forceinline__ void values(const unsigned char* rows, const void* own)
    {
        const int lane = threadIdx.x % kWarp, column = lane % kLanes;
        const float* term = static_cast<const float*>(own);
        const float4* v = reinterpret_cast<const float4*>(rows);
#pragma unroll 4
        for (int t = lane / kLanes; t < kTile; t += kTokenStep) {
            float e[H];
            if constexpr (H % 4 == 0) {
#pragma unroll
                for (int h = 0; h < H; h += 4)
                    *reinterpret_cast<float4*>(e + h) = *reinterpret_cast<const float4*>(term + t * H + h);
            } else {
#pragma unroll
                for (int h = 0; h < H; ++h) e[h] = term[t * H + h];
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float4 x = v[t * kChunks + swizzled<kChunks>(t, column + i * kLanes)];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    o[h][i].x = fmaf(e[h], x.x, o[h][i].x);
                    o[h][i].y = fmaf(e[h], x.y, o[h][i].y);
                    o[h][i].z = fmaf(e[h], x.z, o[h][i].z);
                    o[h][i].w = fmaf(e[h], x.w, o[h][i].w);
                }
            }
        }
    }

    __device__ __forceinline__ void put_sums(float* m_out, float* l_out)
    {
        const int lane = threadIdx.x % kWarp;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int d = 1; d < 32; d *= 2) l[h] += __shfl_xor_sync(~0u, l[h], d);
            if (lane == 0) {
                m_out[h] = m[h];
                l_out[h] = l[h];
            }
        }
    }
    template <int WARPS>
    __device__ __forceinline__ void rescale(const float* m_all)
    {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, m_all[w * H + h]);
            const float f = share(m[h], l[h], top);
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[h][i].x *= f, o[h][i].y *= f, o[h][i].z *= f, o[h][i].w *= f;
        }
    }
    static constexpr int kPass = H;
    static __device__ __forceinline__ int place(int head, int column) { return head * D + column; }
    __device__ __forceinline__ void put(float* to, int)
    {
        const int lane = threadIdx.x % kWarp;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                float4 x = o[h][i];
#pragma unroll
                for (int d = kLanes; d < kWarp; d *= 2) {  // the lanes of the other tokens
                    x.x += __shfl_xor_sync(~0u, x.x, d);
                    x.y += __shfl_xor_sync(~0u, x.y, d);
                    x.z += __shfl_xor_sync(~0u, x.z, d);
                    x.w += __shfl_xor_sync(~0u, x.w, d);
                }
                if (lane < kLanes) *reinterpret_cast<float4*>(to + place(h, (lane + i * kLanes) * 4)) = x;
            }
    }
};

// A tile that a warp will copy: what its rows' places are worked out from.
struct alignas(16) Note {
    uint64_t head;   // the kv head's offset, with that of the tile in its page where it lies in one
    uint32_t token;  // the first one
    uint32_t mask;   // rows of the request and its window
};

// Shared memory of a block.
template <typename T, int D, int H, int SLOTS, int WARPS>
struct Room {
    using Work = Tile<T, D, H>;
    static constexpr int kRowBytes = D * int(sizeof(T));
    static constexpr int kSlotBytes = kTile * kRowBytes;  // a tile's keys, or its values
    static constexpr int kRing = SLOTS * kSlotBytes;      // of a warp
    static constexpr int kMasks = SLOTS / 2 + 2;          // tiles between the copies and the products
    static constexpr int kNotes = 4;                      // tiles whose page ids come ahead of the copies
    static constexpr int kNoteBytes = 16 + kTile * 4;
    static constexpr int kQueries = WARPS * kRing;        // this part's, the next one's
    static constexpr int kQueryBytes = H * kRowBytes;
    static constexpr int kAhead = kQueries + 2 * kQueryBytes;
    static constexpr int kOwn = kAhead + WARPS * kNotes * kNoteBytes;
    static constexpr int kStats = kOwn + WARPS * Work::kWarpBytes;  // m, l [warp][head], then of the unit [head]
    static constexpr int kValid = kStats + (2 * WARPS + 2) * H * 4;
    static constexpr int kFree = kValid + WARPS * kMasks * 4;
    static constexpr int kLostRows = kFree + WARPS * 4;   // whether the run has any
    static constexpr int kBytes = kLostRows + 4;
    static_assert(Work::kPass * D * 4 <= kSlotBytes, "a warp's vectors fit its free slot");
    static_assert(SLOTS <= 2 * kNotes, "page ids have come when they are needed");
};

__device__ __forceinline__ bool finite(float x) { return x - x == 0.f; }
// Terms of up to 2^8 (float16: 2^15) times a value may pass what 32 bits hold where the
// mean does not, and two parts of a term make NaN of an infinite value.  Neither comes
// back to a finite number on its way, so a row with weights whose vector has ended as
// one is right; the others are computed again (mend_row).
__device__ __forceinline__ bool lost(float weights, float4 x)
{
    return weights != 0.f && finite(weights) && !(finite(x.x) && finite(x.y) && finite(x.z) && finite(x.w));
}

// Zeros for the requests without tokens, divided among the blocks.
template <typename T>
__device__ __forceinline__ void clear_empty(const Params& p)
{
    for (uint32_t r = blockIdx.x; r < p.requests; r += gridDim.x) {
        if (tokens_of(p, r).tiles()) continue;
        for (uint32_t i = threadIdx.x; i < p.heads * p.dim; i += blockDim.x) {
            const uint32_t h = i / p.dim;
            static_cast<T*>(p.out)[r * p.out_request + h * p.out_head + (i - h * p.dim)] = from_float<T>(0.f);
        }
        for (uint32_t h = threadIdx.x; h < p.heads; h += blockDim.x) {
            if (p.lse) p.lse[uint64_t(r) * p.heads + h] = -INFINITY;
            if (p.lse2) p.lse2[uint64_t(r) * p.heads + h] = -INFINITY;
        }
    }
}

// Four adjacent elements, as far as the row goes.
template <typename T>
__device__ __forceinline__ void store_4(T* to, float4 x, bool wide, uint32_t columns)
{
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(to) = x;
        } else {
            const T e[4] = {from_float<T>(x.x), from_float<T>(x.y), from_float<T>(x.z), from_float<T>(x.w)};
            const auto word = [&](int i) {
                return uint32_t(*reinterpret_cast<const uint16_t*>(&e[i])) |
                       uint32_t(*reinterpret_cast<const uint16_t*>(&e[i + 1])) << 16;
            };
            *reinterpret_cast<uint2*>(to) = make_uint2(word(0), word(2));
        }
    } else {
        to[0] = from_float<T>(x.x);
        if (columns > 1) to[1] = from_float<T>(x.y);
        if (columns > 2) to[2] = from_float<T>(x.z);
        if (columns > 3) to[3] = from_float<T>(x.w);
    }
}

// kWide: 16-byte copies; else element by element, for rows that start anywhere.
template <typename T, int D, int H, int SLOTS, int WARPS, int BLOCKS, bool kWide>
__global__ void __launch_bounds__(WARPS * kWarp, BLOCKS) decode_kernel(const Params p)
{
    using Work = Tile<T, D, H>;
    using R = Room<T, D, H, SLOTS, WARPS>;
    constexpr int kWarps = WARPS, kThreads = kWarps * kWarp;
    constexpr int kRowBytes = R::kRowBytes, kChunks = kRowBytes / 16, kIn = 16 / int(sizeof(T));
    static_assert((kWarps & (kWarps - 1)) == 0, "");
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    let_next_start();

    unsigned char* ring = smem + warp * R::kRing;
    if (p.dim < D)  // columns past the head's are zeros throughout
        for (int i = lane; i < R::kRing / 16; i += kWarp) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);

    const uint32_t units = p.kv_heads * p.chunks;
    long long begin = -1, end = -1;
    Place place;
    const long long total = share_of<kThreads>(
        p.requests, [&](uint32_t r) { return (long long)(tokens_of(p, r).tiles()) * units; },
        [&](long long all) {
            const long long per = run_of(all, uint64_t(units) * p.requests, gridDim.x, kWarps);
            begin = blockIdx.x * per;
            end = min(all, begin + per);
            return begin < all ? begin : -1;
        },
        place);
    int4* split = reinterpret_cast<int4*>(p.split) + blockIdx.x;
    if (begin >= total) {
        if (threadIdx.x == 0) *split = make_int4(0, 0, 0, 0);
        clear_empty<T>(p);
        return;
    }

    Walk now;
    now.start(p, place, begin, end);

    // A part's queries, [head] rows swizzled like the keys'.
    const auto load_queries = [&](const Walk& w, int buffer) {
        const uint32_t kv_head = w.unit / p.chunks, head0 = (w.unit - kv_head * p.chunks) * p.per_unit;
        const uint32_t heads = min(p.per_unit, p.group - head0);
        const T* q = static_cast<const T*>(p.q) + w.r * p.q_request + (kv_head * p.group + head0) * p.q_head;
        unsigned char* to = smem + R::kQueries + buffer * R::kQueryBytes;
        for (int at = threadIdx.x; at < H * kChunks; at += kThreads) {
            const uint32_t head = at / kChunks, chunk = at % kChunks, column = chunk * kIn;
            unsigned char* into = to + head * kRowBytes + swizzled<kChunks>(head, chunk) * 16;
            const bool live = head < heads && column < p.dim;
            const T* from = live ? q + head * p.q_head + column : q;
            if (p.wide_q) {
                copy_16b(smem_address(into), from, live);
            } else {
                for (int c = 0; c < kIn; ++c)
                    reinterpret_cast<T*>(into)[c] = live && column + c < p.dim ? from[c] : from_float<T>(0.f);
            }
        }
    };

    // Three walks over the run: its tiles go to the warps in turn, also across its
    // parts.  `ahead` notes a warp's tiles and sends for their page ids, kNotes tiles
    // before the copies of their rows, for a load waits a microsecond and more behind
    // the copies of the whole GPU.
    Walk ahead = now;
    uint32_t ahead_t = ahead.t + warp;
    bool more = true;
    const auto settle = [&] {
        while (ahead_t >= ahead.t_end) {
            const uint32_t turn = ahead_t - ahead.t_end;  // tiles of the next part before the warp's
            if (!ahead.next(p)) {
                more = false;
                return;
            }
            ahead_t = turn;
        }
    };
    unsigned char* notes = smem + R::kAhead + warp * R::kNotes * R::kNoteBytes;
    int note_in = 0, note_out = 0, noted = 0;
    const auto note_next = [&] {
        if (!more) return;
        unsigned char* at = notes + note_in * R::kNoteBytes;
        const uint32_t token = ahead.tokens.base() + ahead_t * kTile, row = p.page_tiles ? 0 : lane;
        if (row < kTile && token + row < ahead.tokens.end && (lane == 0 || !p.page_tiles))
            copy_4b(smem_address(at + 16 + row * 4), p.table + ahead.r * p.table_stride + p.page.quotient(token + row));
        const uint32_t skip = ahead.tokens.first > token ? ahead.tokens.first - token : 0;
        if (lane == 0) {
            Note& n = *reinterpret_cast<Note*>(at);
            n.head = uint64_t(ahead.unit / p.chunks) * p.head_stride;
            if (p.page_tiles) n.head += (token - p.page.quotient(token) * p.page.d) * p.token_stride;
            n.token = token;
            n.mask = (0xffffu << skip) & (0xffffu >> (kTile - min(ahead.tokens.end - token, uint32_t(kTile))));
        }
        note_in = note_in + 1 == R::kNotes ? 0 : note_in + 1;
        ++noted;
        ahead_t += kWarps;
        settle();
    };
    settle();

    // The copies: a noted tile's keys, and at the next call its values.
    uint32_t* masks = reinterpret_cast<uint32_t*>(smem + R::kValid) + warp * R::kMasks;
    int slot_in = 0, mask_in = 0;
    uint64_t row_offset = 0;  // of the lane's row, or of the first of all
    uint32_t mask = 0;
    bool values_next = false;
    const auto copy_rows = [&](const T* from) {
        unsigned char* to = ring + slot_in * R::kSlotBytes;
        if (kWide) {
            const uint32_t address = smem_address(to);
            constexpr int kCopies = kTile * kChunks / kWarp;
            if (p.page_tiles && kWarp % kChunks == 0) {
                // a lane's rows are so many apart, their chunks an exclusive or
                constexpr int kApart = kWarp % kChunks == 0 ? kWarp / kChunks : 1;
                const int row0 = lane / kChunks, chunk = lane % kChunks;
                const T* at = from + row_offset + row0 * p.token_stride + chunk * kIn;
                const uint32_t into = address + row0 * kRowBytes + swizzled<kChunks>(row0, chunk) * 16;
                const auto to_row = [&](int i) { return (into ^ (i * kApart % 8 * 16)) + i * kApart * kRowBytes; };
                if (chunk * kIn >= p.dim) {
                } else if (mask == 0xffffu) {
#pragma unroll
                    for (int i = 0; i < kCopies; ++i, at += kApart * p.token_stride) copy_16b(to_row(i), at);
                } else {
#pragma unroll
                    for (int i = 0; i < kCopies; ++i, at += kApart * p.token_stride)
                        copy_16b(to_row(i), at, mask >> (row0 + i * kApart) & 1);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const int at = i * kWarp + lane, row = at / kChunks, chunk = at % kChunks;
                    const uint64_t offset = p.page_tiles ? row_offset + row * p.token_stride : __shfl_sync(~0u, row_offset, row);
                    if (chunk * kIn < p.dim)
                        copy_16b(address + row * kRowBytes + swizzled<kChunks>(row, chunk) * 16, from + offset + chunk * kIn, mask >> row & 1);
                }
            }
        } else {
            for (int row = 0; row < kTile; ++row) {
                const uint64_t offset = p.page_tiles ? row_offset + row * p.token_stride : __shfl_sync(~0u, row_offset, row);
                const bool live = mask >> row & 1;
                for (uint32_t c = lane; c < p.dim; c += kWarp) {
                    T* into = reinterpret_cast<T*>(to + row * kRowBytes + swizzled<kChunks>(row, c / kIn) * 16) + c % kIn;
                    *into = live ? from[offset + c] : from_float<T>(0.f);
                }
            }
        }
    };
    const auto copy_next = [&] {
        if (noted) {
            if (!values_next) {
                const unsigned char* at = notes + note_out * R::kNoteBytes;
                const Note n = *reinterpret_cast<const Note*>(at);
                const uint32_t row = p.page_tiles ? 0 : lane % kTile, token = n.token + row;
                const uint32_t id = reinterpret_cast<const uint32_t*>(at + 16)[row];
                const bool live = id < p.num_pages && (p.page_tiles || (n.mask >> row & 1));
                mask = n.mask & __ballot_sync(~0u, live);
                if (lane == 0) masks[mask_in] = mask;
                mask_in = mask_in + 1 == R::kMasks ? 0 : mask_in + 1;
                row_offset = id * p.page_stride + n.head;
                if (!p.page_tiles) row_offset += (token - p.page.quotient(token) * p.page.d) * p.token_stride;
                if (!live) row_offset = 0;
                copy_rows(static_cast<const T*>(p.k));
            } else {
                copy_rows(static_cast<const T*>(p.v));
                note_out = note_out + 1 == R::kNotes ? 0 : note_out + 1;
                --noted;
                note_next();
            }
            values_next = !values_next;
        }
        commit_copies();
        slot_in = slot_in + 1 == SLOTS ? 0 : slot_in + 1;
    };

    int* any_lost = reinterpret_cast<int*>(smem + R::kLostRows);
    if (threadIdx.x == 0) *any_lost = 0;
    load_queries(now, 0);
#pragma unroll
    for (int i = 0; i < R::kNotes; ++i) note_next();
    commit_copies();
    wait_copies<0>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < SLOTS - 1; ++i) copy_next();
    clear_empty<T>(p);
    __syncthreads();

    float* m_all = reinterpret_cast<float*>(smem + R::kStats);
    float* l_all = m_all + kWarps * H;
    float* unit_m = l_all + kWarps * H;
    float* unit_l = unit_m + H;
    int* free_slot = reinterpret_cast<int*>(smem + R::kFree);
    int slot = 0, mask_out = 0, buffer = 0;
    long long first_tile = begin;  // number of the part's first tile
    Work work;
    // The oldest slot, once its copies have come; the newest is filled meanwhile.
    const auto next_slot = [&] {
        wait_copies<SLOTS - 2>();
        __syncwarp();
        copy_next();
        const unsigned char* rows = ring + slot * R::kSlotBytes;
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
        return rows;
    };
    while (true) {
        const uint32_t kv_head = now.unit / p.chunks, head0 = (now.unit - kv_head * p.chunks) * p.per_unit;
        const uint32_t heads = min(p.per_unit, p.group - head0), head = kv_head * p.group + head0;
        Walk then = now;
        const bool again = then.next(p);
        if (again) load_queries(then, buffer ^ 1);
        work.clear();
        uint32_t own_tiles = 0;
        for (uint32_t t = now.t + ((warp - uint32_t(first_tile - begin)) & (kWarps - 1)); t < now.t_end; t += kWarps) {
            const long long number = first_tile + (t - now.t);
            float* logits = p.logits && number < p.logit_tiles ? p.logits + number * p.per_unit * kTile : nullptr;
            void* own = smem + R::kOwn + warp * Work::kWarpBytes;
            const unsigned char* keys = next_slot();
            work.keys(p, keys, smem + R::kQueries + buffer * R::kQueryBytes, own, masks[mask_out], logits, heads);
            mask_out = mask_out + 1 == R::kMasks ? 0 : mask_out + 1;
            work.values(next_slot(), own);
            ++own_tiles;
        }
        if (own_tiles * 2 < SLOTS) {  // else the next queries' copies have been waited for
            commit_copies();
            wait_copies<0>();
        }

        // The warps' parts add up in their order.  Each puts its vectors into its slot
        // that is filled next, relative to the largest of the warps' references.
        work.put_sums(m_all + warp * H, l_all + warp * H);
        if (lane == 0) free_slot[warp] = slot_in;
        __syncthreads();
        work.template rescale<kWarps>(m_all);
        if (threadIdx.x < H) {
            float top = -INFINITY, all = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_all[w * H + threadIdx.x]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float l = l_all[w * H + threadIdx.x];
                all += share(m_all[w * H + threadIdx.x], l, top) * l;
            }
            unit_m[threadIdx.x] = top;
            unit_l[threadIdx.x] = all;
        }
        const bool whole = now.t == 0 && now.t_end == now.tiles;
        const uint32_t part_of = blockIdx.x * 2 + (now.t ? 0 : 1);
#pragma unroll
        for (int pass = 0; pass < H / Work::kPass; ++pass) {
            work.put(reinterpret_cast<float*>(ring + slot_in * R::kSlotBytes), pass);
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < Work::kPass * D / 4; i += kThreads) {
                const uint32_t in_pass = i / (D / 4), h = pass * Work::kPass + in_pass, column = i % (D / 4) * 4;
                if (h >= heads) break;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* from = reinterpret_cast<const float*>(smem + w * R::kRing + free_slot[w] * R::kSlotBytes);
                    const float4 y = *reinterpret_cast<const float4*>(from + Work::place(in_pass, column));
                    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                }
                if (!whole) {
                    *reinterpret_cast<float4*>(p.part + (uint64_t(part_of) * H + h) * D + column) = x;
                } else if (column < p.dim) {
                    const float all = unit_l[h], by = 1.f / all;
                    float4 y = make_float4(x.x * by, x.y * by, x.z * by, x.w * by);
                    if (all == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);  // whatever the values were
                    if (lost(all, y)) *any_lost = 1;
                    store_4(static_cast<T*>(p.out) + now.r * p.out_request + (head + h) * p.out_head + column, y, p.wide_out,
                            p.dim - column);
                }
            }
            if (pass == 0 && threadIdx.x < heads) {
                if (whole) {
                    put_lse(p, uint64_t(now.r) * p.heads + head + threadIdx.x, unit_m[threadIdx.x], unit_l[threadIdx.x]);
                } else {
                    float2* stats = reinterpret_cast<float2*>(p.part + uint64_t(gridDim.x) * 2 * H * D);
                    stats[uint64_t(part_of) * H + threadIdx.x] = make_float2(unit_m[threadIdx.x], unit_l[threadIdx.x]);
                }
            }
            __syncthreads();
        }
        if (p.dim < D) {  // and the slot's last columns are zeros again
            uint4* to = reinterpret_cast<uint4*>(ring + slot_in * R::kSlotBytes);
            for (int i = lane; i < R::kSlotBytes / 16; i += kWarp) to[i] = make_uint4(0, 0, 0, 0);
        }
        if (threadIdx.x == 0) {
            if (p.first && now.unit == 0 && now.t == 0) p.first[now.r] = first_tile;
            if (!again) {
                const long long per = run_of(total, uint64_t(units) * p.requests, gridDim.x, kWarps), unit_begin = first_tile - now.t;
                const int32_t from = int32_t(unit_begin / per), to = int32_t((unit_begin + now.tiles - 1) / per);
                *split = make_int4(int32_t(now.r) | (*any_lost ? kLost : 0), int32_t(now.unit), from, now.t_end < now.tiles ? to - from : 0);
            }
        }
        if (!again) break;
        first_tile += now.t_end - now.t;
        now = then;
        buffer ^= 1;
    }
    wait_copies<0>();
}

constexpr int kJoinWarps = 8, kJoinThreads = kJoinWarps * kWarp;

// 2^x for x <= 0 in the range of 64 bits, with the digits of 32.
__device__ __forceinline__ double exp2_wide(float x)
{
    if (x < -1000.f) return 0.0;
    const float whole = rintf(x);
    return double(exp2_fast(x - whole)) * __hiloint2double((1023 + int(whole)) << 20, 0);
}

// One row of the output by one block, its sums in 64 bits, where none of 32-bit values
// ends, and its terms one number each: sum_t p_t v_t as it stands, infinities and NaN
// among the values.  Slow (every eighth token a warp's, one after the other): no
// ordinary call has such a row.  room: [4][D].
template <typename T, int D>
__device__ __forceinline__ void mend_row(const Params& p, uint32_t r, uint32_t head, float* room, double2* stats)
{
    constexpr int kPer = D / kWarp;
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const Tokens seen = tokens_of(p, r);
    const uint64_t kv_offset = head / p.group * p.head_stride;
    double* sums = reinterpret_cast<double*>(room);  // [D]
    float* q = room + 2 * D;
    __syncthreads();  // the room is free
    for (uint32_t column = threadIdx.x; column < D; column += kJoinThreads)
        q[column] = column < p.dim ? to_float((static_cast<const T*>(p.q) + r * p.q_request + head * p.q_head)[column]) : 0.f;
    __syncthreads();
    double o[kPer], l = 0.0;
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < kPer; ++c) o[c] = 0.0;
#pragma unroll 1
    for (uint32_t t = seen.first + warp; t < seen.end; t += kJoinWarps) {
        const uint32_t page = p.page.quotient(t), id = uint32_t(p.table[r * p.table_stride + page]);
        if (id >= p.num_pages) continue;
        const uint64_t at = id * p.page_stride + (t - page * p.page.d) * p.token_stride + kv_offset + lane;
        const T* k_row = static_cast<const T*>(p.k) + at;
        const T* v_row = static_cast<const T*>(p.v) + at;
        float v[kPer], x = 0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
            const bool in = c * kWarp + lane < p.dim;
            v[c] = in ? to_float(v_row[c * kWarp]) : 0.f;
            x = fmaf(q[c * kWarp + lane], in ? to_float(k_row[c * kWarp]) : 0.f, x);
        }
#pragma unroll
        for (int d = 1; d < kWarp; d *= 2) x += __shfl_xor_sync(~0u, x, d);
        x = logit(p, x);
        if (x > m) {
            const double f = m == -INFINITY ? 1.0 : exp2_wide(m - x);  // before the first one there is nothing but zeros and NaN
            l *= f;
#pragma unroll
            for (int c = 0; c < kPer; ++c) o[c] *= f;
            m = x;
        }
        const double e = x == -INFINITY ? 0.0 : exp2_wide(x - m);
        l += e;
#pragma unroll
        for (int c = 0; c < kPer; ++c) o[c] += e * v[c];
    }
    // the warps' parts, in their order
    if (lane == 0) stats[warp] = make_double2(m, l);
    __syncthreads();
    double all = 0.0;
    float top = -INFINITY;
#pragma unroll 1
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, float(stats[w].x));
    const auto factor = [&](float from) { return from == -INFINITY ? 1.0 : exp2_wide(from - top); };
#pragma unroll 1
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
        all += factor(float(stats[w].x)) * stats[w].y;
        if (warp == w) {
#pragma unroll
            for (int c = 0; c < kPer; ++c) {
                double& sum = sums[c * kWarp + lane];
                sum = factor(m) * o[c] + (w ? sum : 0.0);
            }
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(p.out) + r * p.out_request + head * p.out_head;
    for (uint32_t column = threadIdx.x; column < p.dim; column += kJoinThreads)
        out[column] = from_float<T>(float(all == 0.0 ? 0.0 : sums[column] / all));
}

// A unit whose tiles lie in the runs of `count` + 1 blocks: the last part of the
// first of them and the first parts of the others join, in order.  The first `count`
// blocks here share its heads; a block's warps take a head each, or where it has
// fewer, every so-many-th part of one.  Few numbers, so latency: one block of 1024
// threads for a unit measured slower.
template <typename T, int D, int H>
__global__ void __launch_bounds__(kJoinThreads, 4) join_kernel(const __grid_constant__ Params p)
{
    __shared__ __align__(16) float sums[kJoinWarps / 2][D];
    __shared__ float2 stats_of[kJoinWarps];
    __shared__ double2 mend_stats[kJoinWarps];
    __shared__ uint32_t lost_heads;  // of the unit that is joined here
    let_next_start();
    if (threadIdx.x == 0) lost_heads = 0;
    __syncthreads();
    wait_for_previous();
    const int4 split = reinterpret_cast<const int4*>(p.split)[blockIdx.x];
    const uint32_t r = uint32_t(split.x & ~kLost), unit = uint32_t(split.y), block = uint32_t(split.z), count = uint32_t(split.w);
    const uint32_t kv_head = unit / p.chunks, head0 = unit % p.chunks * p.per_unit;
    const uint32_t heads = min(p.per_unit, p.group - head0), turn = blockIdx.x - block;
    const bool joins = count != 0 && turn < heads;
    if (!joins && !(split.x & kLost)) return;
    const uint32_t mine = joins ? (heads - turn + count - 1) / count : 0;  // the heads turn, turn + count, ...
    uint32_t at_once = 1;
    while (at_once < mine && at_once < kJoinWarps) at_once *= 2;
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const uint32_t groups = kJoinWarps / at_once, place_in = warp % at_once, group = warp / at_once;
    const float2* stats = reinterpret_cast<const float2*>(p.part + uint64_t(gridDim.x) * 2 * H * D);

    constexpr int kPer = D / kWarp, kAhead = 4;
    for (uint32_t i0 = 0; i0 < mine; i0 += at_once) {
        const bool live = i0 + place_in < mine;
        const uint32_t h = turn + (i0 + place_in) * count;
        float o[kPer], top = -INFINITY, all = 0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) o[c] = 0.f;
        for (uint32_t i = live ? group : count + 1; i <= count; i += groups * kAhead) {
            float2 s[kAhead];
            float x[kAhead][kPer];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint32_t at = i + u * groups;
                s[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < kPer; ++c) x[u][c] = 0.f;
                if (at > count) continue;
                const uint64_t slot = uint64_t(block + at) * 2 + (at ? 0 : 1);
                s[u] = stats[slot * H + h];
                const float* part = p.part + (slot * H + h) * D + lane;
#pragma unroll
                for (int c = 0; c < kPer; ++c) x[u][c] = part[c * kWarp];
            }
            float to = top;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) to = fmaxf(to, s[u].x);
            const float keep = share(top, all, to);
            all *= keep;
#pragma unroll
            for (int c = 0; c < kPer; ++c) o[c] *= keep;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float f = share(s[u].x, s[u].y, to);
                all += f * s[u].y;
#pragma unroll
                for (int c = 0; c < kPer; ++c) o[c] += f * x[u][c];
            }
            top = to;
        }
        if (groups > 1) {
            if (lane == 0) stats_of[warp] = make_float2(top, all);
            __syncthreads();
            const float own = all;
            float to = -INFINITY;
            all = 0.f;
            for (uint32_t g = 0; g < groups; ++g) to = fmaxf(to, stats_of[g * at_once + place_in].x);
            for (uint32_t g = 0; g < groups; ++g) {
                const float2 of = stats_of[g * at_once + place_in];
                all += share(of.x, of.y, to) * of.y;
            }
            const float factor = share(top, own, to);
            top = to;
            for (uint32_t g = 0; g < groups; ++g) {
                if (group == g) {
#pragma unroll
                    for (int c = 0; c < kPer; ++c) {
                        float& sum = sums[place_in][c * kWarp + lane];
                        o[c] = factor * o[c] + (g ? sum : 0.f);
                        sum = o[c];
                    }
                }
                __syncthreads();
            }
        }
        if (live && group == groups - 1) {
            const uint32_t head = kv_head * p.group + head0 + h;
            T* out = static_cast<T*>(p.out) + r * p.out_request + head * p.out_head;
            const float by = 1.f / all;
            bool none = false;
#pragma unroll
            for (int c = 0; c < kPer; ++c) {
                const float y = all == 0.f ? 0.f : o[c] * by;  // without weights zeros, whatever the values were
                none |= lost(all, make_float4(y, 0.f, 0.f, 0.f));
                if (c * kWarp + lane < p.dim) out[c * kWarp + lane] = from_float<T>(y);
            }
            if (__any_sync(~0u, none) && lane == 0) atomicOr(&lost_heads, 1u << h);
            if (lane == 0) put_lse(p, uint64_t(r) * p.heads + head, top, all);
        }
    }
    __syncthreads();
    if (!lost_heads && !(split.x & kLost)) return;

    // rows that are computed again: of this unit, then of the units that lie whole in the block's run of tiles
    uint32_t again = lost_heads, row_r = r, first_head = kv_head * p.group + head0;
    Walk now;
    bool more = split.x & kLost, started = false;
    while (true) {
        while (!again && more) {
            if (!started) {
                const uint32_t units = p.kv_heads * p.chunks;
                long long begin = -1, end = -1;
                Place place;
                share_of<kJoinThreads>(
                    p.requests, [&](uint32_t i) { return (long long)(tokens_of(p, i).tiles()) * units; },
                    [&](long long all) {
                        const long long per = run_of(all, uint64_t(units) * p.requests, gridDim.x, int(p.warps));
                        begin = blockIdx.x * per;
                        end = min(all, begin + per);
                        return begin < all ? begin : -1;
                    },
                    place);
                now.start(p, place, begin, end);
                started = true;
            } else if (!now.next(p)) {
                more = false;
                break;
            }
            if (now.t || now.t_end != now.tiles) continue;
            const uint32_t kv = now.unit / p.chunks, h0 = (now.unit - kv * p.chunks) * p.per_unit;
            row_r = now.r;
            first_head = kv * p.group + h0;
            for (uint32_t h = 0; h < min(p.per_unit, p.group - h0); ++h) {
                const T* row = static_cast<const T*>(p.out) + row_r * p.out_request + (first_head + h) * p.out_head;
                bool none = false;
                for (uint32_t column = threadIdx.x; column < p.dim; column += kJoinThreads) none |= !finite(to_float(row[column]));
                if (__syncthreads_or(none)) again |= 1u << h;
            }
        }
        if (!again) return;
        mend_row<T, D>(p, row_r, first_head + __ffs(again) - 1, &sums[0][0], mend_stats);
        again &= again - 1;
    }
}

// SLOTS of the warps' rings, WARPS of a block, BLOCKS on an SM.
template <typename T, int D, int H, int SLOTS, int WARPS, int BLOCKS>
lcpp_status launch(const Params& base, bool wide, size_t part_bytes_at_most, cudaStream_t s)
{
    Params p = base;
    using R = Room<T, D, H, SLOTS, WARPS>;
    constexpr int kThreads = WARPS * kWarp;
    static_assert(BLOCKS * (R::kBytes + 1024) <= 228 * 1024, "shared memory of an SM");
    auto kernel = wide ? decode_kernel<T, D, H, SLOTS, WARPS, BLOCKS, true> : decode_kernel<T, D, H, SLOTS, WARPS, BLOCKS, false>;
    set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), R::kBytes);
    const unsigned blocks = std::min<unsigned>(
        kMostBlocks, unsigned(device_sm_count()) * resident_blocks(reinterpret_cast<const void*>(kernel), kThreads, R::kBytes));
    if (uint64_t(blocks) * 2 * H * (D + 2) * 4 > part_bytes_at_most) return LCPP_ERR_INTERNAL;
    p.warps = WARPS;
    kernel<<<blocks, kThreads, R::kBytes, s>>>(p);
    const lcpp_status status = launched();
    if (status != LCPP_OK) return status;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.stream = s;
    config.attrs = &early;
    config.numAttrs = 1;
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(kJoinThreads);
    LCPP_CUDA_TRY(cudaLaunchKernelEx(&config, join_kernel<T, D, H>, p));
    return LCPP_OK;
}

// Heads of a unit and padded columns for a group of `group` query heads and
// heads of `dim` columns; the temp query and the launch go by the same choice.
struct Choice {
    uint32_t columns, heads, chunks, per_unit;
};
inline Choice choose(uint32_t group, uint32_t dim, bool f32)
{
    Choice c{};
    c.columns = dim <= 64 ? 64 : !f32 && dim <= 96 ? 96 : dim <= 128 ? 128 : (f32 || dim > 192) ? 256 : 192;
    // what a warp's accumulators hold: up to 128 registers of them in 16 bits, 32 in 32, where
    // a lane's loads of its token's queries bound the time (larger groups read the cache once
    // for each chunk of theirs)
    const uint32_t most = f32 ? (c.columns == 256 ? 4 : 8) : (c.columns <= 128 ? 32 : 16);
    c.chunks = (group + most - 1) / most;
    c.per_unit = (group + c.chunks - 1) / c.chunks;
    c.chunks = (group + c.per_unit - 1) / c.per_unit;
    c.heads = f32 ? 1 : 8;
    while (c.heads < c.per_unit) c.heads *= 2;
    return c;
}

lcpp_status run_f32(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s);
lcpp_status run_f16(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s);
lcpp_status run_bf16(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s);

// Slots and blocks: as many copies under way as an SM's shared memory holds, divided
// so that the accumulators fit the registers.  Measured, long contexts in bfloat16:
// 64 columns, 8 heads: 4 slots and 5 blocks 69 us, 2 slots 84; 128, 8 heads: 2 slots
// and 4 blocks 390 us, 3 slots and 3 blocks 404; 128, 16 heads: 3 and 3 114 us, 2 and
// 3 126; 256, 8 heads: 2 slots and 3 blocks 203 us, 3 and 2 209.  float32, 256
// columns: 2 and 3 543 us, 3 and 1 691.
template <typename T>
lcpp_status run_16bit(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s)
{
    switch (c.columns) {
    case 64:
        return c.heads == 8    ? launch<T, 64, 8, 4, 4, 5>(p, wide, part_bytes, s)
               : c.heads == 16 ? launch<T, 64, 16, 4, 4, 4>(p, wide, part_bytes, s)
                               : launch<T, 64, 32, 4, 4, 2>(p, wide, part_bytes, s);
    case 96:
        return c.heads == 8    ? launch<T, 96, 8, 3, 4, 4>(p, wide, part_bytes, s)
               : c.heads == 16 ? launch<T, 96, 16, 3, 4, 3>(p, wide, part_bytes, s)
                               : launch<T, 96, 32, 4, 4, 2>(p, wide, part_bytes, s);
    case 128:
        return c.heads == 8    ? launch<T, 128, 8, 2, 4, 4>(p, wide, part_bytes, s)
               : c.heads == 16 ? launch<T, 128, 16, 3, 4, 3>(p, wide, part_bytes, s)
                               : launch<T, 128, 32, 4, 4, 2>(p, wide, part_bytes, s);
    case 192:
        return c.heads == 8 ? launch<T, 192, 8, 3, 4, 2>(p, wide, part_bytes, s) : launch<T, 192, 16, 3, 4, 2>(p, wide, part_bytes, s);
    default:
        return c.heads == 8 ? launch<T, 256, 8, 2, 4, 3>(p, wide, part_bytes, s) : launch<T, 256, 16, 2, 4, 2>(p, wide, part_bytes, s);
    }
}

}  // namespace attention
}  // namespace model
}  // namespace lcpp
