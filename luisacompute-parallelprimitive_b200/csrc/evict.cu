// evict.cu -- DeviceCacheEviction (include/lcpp_b200_model.h): requests cut down
// to the tokens with the most attention weight.
//
// A request's tokens get 32-bit keys that order like (protected, score).  The
// budget-th largest comes out of up to three passes over 11, 11 and 10 of their
// bits, each a histogram of the keys that share the bits found so far; they end
// when all keys that share them are kept.  Tokens above it are kept, and of those
// equal to it the first ones.  A kept token past the first `budget` places fills a
// place whose token is not kept: numbers within two counts over the tokens pair
// them off, no other token moves, and moves do not touch one another's slots.
//
// A cluster of 1 to 8 blocks works on a request, each on a run of its tokens
// whose keys stay in shared memory; the blocks read one another's histograms and
// counts there.  A histogram has four copies, for every fourth lane one: equal
// scores would serialise on a single one.
//
// Bound by latency: of 2100 tokens a pass over the keys costs about 1.4 us of barriers and
// dependent steps, beside the start, the keys' loads and the sorting out.  64 requests of
// 2100 tokens and fewer cut to 2048, with the pages' release: 14.4 us; 16 of 131072 to
// 8192: 33.7 us (39.4 with page ids read token by token from L2 and every bin of the other
// blocks read by all), of which the release, a block a request, takes 4.
#include <cooperative_groups.h>

#include "cache.cuh"

namespace cg = cooperative_groups;
using namespace lcpp;
using namespace lcpp::model;

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / kWarp;
constexpr int kMostCluster = 8;
constexpr int kAhead = 4;              // tokens whose loads a thread has under way
constexpr uint32_t kPages = 2048;      // page ids of a block's run that come into shared memory; others are read where needed
constexpr uint32_t kKeys = 38 * 1024;  // keys of a block that stay in shared memory; others are read again
constexpr uint32_t kProtected = 0xffffffffu, kNaN = 0xfffffffeu;

struct Params {
    const int32_t* lens;
    const int32_t* table;
    uint64_t table_stride;
    const float* scores;
    const int32_t* positions;
    const int32_t* evicted;
    Divider page;
    uint32_t longest, num_pages, requests;
    uint32_t budget, trigger, first, recent, max_moves;
    int32_t* lens_out;
    int32_t* evicted_out;
    int32_t* counts;
    longlong2* moves;
    uint64_t moves_stride;
};

// What the blocks of a cluster read of one another.
constexpr int kBins = 2048, kCopies = 4;
struct alignas(16) Shared {
    uint32_t histogram[2][kBins];  // from the largest digit down
    uint32_t groups[2][kWarps];    // sums of so many bins each
    uint32_t broken;            // a page id out of range
    uint32_t holes, fillers;    // of the block's tokens
};

__device__ __forceinline__ uint32_t key_of(float score)
{
    if (score != score) return kNaN;
    const uint32_t bits = __float_as_uint(score + 0.f);  // + 0: both zeros alike
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ uint32_t length_of(const int32_t* lens, uint32_t r, uint32_t longest)
{
    return min(uint32_t(max(lens[r], 0)), longest);
}

// Exclusive sum over the lanes of a warp, and the sum of all.
__device__ __forceinline__ uint32_t lanes_before(uint32_t mine, uint32_t& total)
{
    const int lane = threadIdx.x % kWarp;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
        const uint32_t left = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += left;
    }
    total = __shfl_sync(~0u, upto, kWarp - 1);
    return upto - mine;
}
// Sum over the warps before, and over all; nobody may be reading `warps` any more.
__device__ __forceinline__ uint32_t warps_before(uint32_t of_warp, uint32_t* warps, uint32_t& total)
{
    static_assert(kWarps == kWarp, "a lane for each warp");
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    if (lane == 0) warps[warp] = of_warp;
    __syncthreads();
    return __shfl_sync(~0u, lanes_before(warps[lane], total), warp);
}

// The key of one token, read again: for those that have no room in shared memory.
__device__ __noinline__ uint32_t key_again(const Params& p, const int32_t* row, uint32_t token, int64_t recent)
{
    const uint32_t page = p.page.quotient(token), id = uint32_t(row[page]);  // looked up before: in range
    const uint64_t slot = uint64_t(id) * p.page.d + (token - page * p.page.d);
    const int64_t at = p.positions ? int64_t(p.positions[slot]) : int64_t(token);
    return at < p.first || at >= recent ? kProtected : key_of(p.scores[slot]);
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const __grid_constant__ Params p)
{
    extern __shared__ uint32_t dynamic[];
    uint32_t* copies = dynamic;  // [kBins][kCopies], from the largest digit down
    uint32_t* pages = dynamic + kBins * kCopies;
    uint32_t* keys = pages + kPages;
    __shared__ Shared shared;
    __shared__ uint32_t warps[3][kWarps];
    __shared__ uint32_t found[5];  // digit, keys above it, keys of it in the blocks before and in all; a broken page
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t r = blockIdx.x / blocks;
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    let_next_start();

    const uint32_t n = length_of(p.lens, r, p.longest);
    const int32_t before = p.evicted ? p.evicted[r] : 0;
    const auto leave = [&] {  // as it is
        if (rank == 0 && threadIdx.x == 0) {
            p.lens_out[r] = int32_t(n);
            p.counts[r] = 0;
            if (p.evicted_out) p.evicted_out[r] = before;
        }
    };
    if (n <= p.trigger) {
        leave();
        return;
    }
    // the block's run of tokens
    const uint32_t run = (n + blocks - 1) / blocks, lo = min(n, rank * run), count = min(n - lo, run);
    const int32_t* row = p.table + r * p.table_stride;
    const int64_t recent = int64_t(n) + (p.positions ? before : 0) - p.recent;
    // four tokens' keys; 0, which no token has, past the last one
    const auto keys_at = [&](uint32_t i) {
        if (i + 3 < kKeys) return *reinterpret_cast<const uint4*>(keys + i);
        const auto one = [&](uint32_t at) { return at >= count ? 0u : at < kKeys ? keys[at] : key_again(p, row, lo + at, recent); };
        return make_uint4(one(i), one(i + 1), one(i + 2), one(i + 3));
    };

    // the pages of the run
    const uint32_t first_page = p.page.quotient(lo), end_page = count ? p.page.quotient(lo + count - 1) + 1 : first_page;
    const bool staged = end_page - first_page <= kPages;
    if (staged)
        for (uint32_t i = threadIdx.x; i < end_page - first_page; i += kThreads) pages[i] = uint32_t(row[first_page + i]);
    const auto page_id = [&](uint32_t page) { return staged ? pages[page - first_page] : uint32_t(row[page]); };

    if (threadIdx.x == 0) shared.broken = 0;
    // keys are read by fours: the last ones are filled up, which the room, a multiple of four, allows
    if (threadIdx.x < (4 - count % 4) % 4 && count < kKeys) keys[count + threadIdx.x] = 0;
    for (int i = threadIdx.x; i < kBins * kCopies; i += kThreads) copies[i] = 0;
    __syncthreads();
    bool broken = false;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads * kAhead) {  // whose loads are under way together
        float score[kAhead];
        int32_t position[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t at = i + u * kThreads, token = lo + at, page = p.page.quotient(token);
            const uint32_t id = at < count ? page_id(page) : 0;
            const bool in = at < count && id < p.num_pages;
            broken |= at < count && !in;
            const uint64_t slot = uint64_t(id) * p.page.d + (token - page * p.page.d);
            score[u] = in ? p.scores[slot] : 0.f;
            position[u] = in && p.positions ? p.positions[slot] : int32_t(token);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t at = i + u * kThreads;
            if (at >= count) continue;
            const int64_t place = position[u];
            const uint32_t key = place < p.first || place >= recent ? kProtected : key_of(score[u]);
            if (at < kKeys) keys[at] = key;
            atomicAdd(&copies[(kBins - 1 - (key >> 21)) * kCopies + lane % kCopies], 1u);
        }
    }
    if (broken) shared.broken = 1;

    uint32_t top = 0, need = p.budget;  // bits found; tokens to keep among the keys that share them
    uint32_t equal_before = 0;          // keys equal to the last one in the blocks before this one
    const auto meet = [&] {
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    };
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        if (pass) {
            for (uint32_t i = threadIdx.x * 4; i < count; i += kThreads * 4) {
                const uint4 k = keys_at(i);
                const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (key[u] == 0 || (key[u] ^ top) >> (shift + bits)) continue;
                    const uint32_t digit = key[u] >> shift & ((1u << bits) - 1);
                    atomicAdd(&copies[(kBins - 1 - digit) * kCopies + lane % kCopies], 1u);
                }
            }
        }
        __syncthreads();
        // a thread's two bins
        static_assert(kBins == 2 * kThreads && kCopies == 4, "");
        uint4* bin = reinterpret_cast<uint4*>(copies) + threadIdx.x * 2;
        const uint4 x = bin[0], y = bin[1];
        bin[0] = bin[1] = make_uint4(0, 0, 0, 0);  // for the next pass
        const uint2 mine = make_uint2(x.x + x.y + x.z + x.w, y.x + y.y + y.z + y.w);
        // The bin of the last kept key: there are at least `need` such keys.
        const auto look_in = [&](uint32_t above, uint2 in_bin, uint2 earlier, uint32_t bin_pair) {
            if (above >= need || above + in_bin.x + in_bin.y < need) return;
            const bool second = above + in_bin.x < need;
            found[0] = kBins - 1 - 2 * bin_pair - second;
            found[1] = above + (second ? in_bin.x : 0);
            found[2] = second ? earlier.y : earlier.x;
            found[3] = second ? in_bin.y : in_bin.x;
        };
        uint32_t of_warp, all;
        if (blocks == 1) {
            uint32_t above = lanes_before(mine.x + mine.y, of_warp);
            above += warps_before(of_warp, warps[0], all);
            look_in(above, mine, make_uint2(0, 0), threadIdx.x);
            if (threadIdx.x == 0) found[4] = shared.broken;
        } else {
            reinterpret_cast<uint2*>(shared.histogram[pass & 1])[threadIdx.x] = mine;
            of_warp = __reduce_add_sync(~0u, mine.x + mine.y);
            if (lane == 0) shared.groups[pass & 1][warp] = of_warp;
            cluster.sync();  // the other buffer is free again, too
            if (warp == 0) {
                // first the group of 64 bins over all blocks, then the bin: little is read from the others
                uint32_t sum = 0, any = 0;
#pragma unroll
                for (uint32_t b = 0; b < kMostCluster; ++b) {
                    const Shared* other = cluster.map_shared_rank(&shared, b < blocks ? b : 0);
                    sum += b < blocks ? other->groups[pass & 1][lane] : 0;
                    any |= other->broken;
                }
                const uint32_t above = lanes_before(sum, all);
                const int at = __ffs(__ballot_sync(~0u, above < need && above + sum >= need)) - 1;
                uint2 in_bin = make_uint2(0, 0), earlier = make_uint2(0, 0);
#pragma unroll
                for (uint32_t b = 0; b < kMostCluster; ++b) {
                    const Shared* other = cluster.map_shared_rank(&shared, b < blocks ? b : 0);
                    const uint2 c = b < blocks ? reinterpret_cast<const uint2*>(other->histogram[pass & 1])[at * kWarp + lane]
                                               : make_uint2(0, 0);
                    in_bin.x += c.x, in_bin.y += c.y;
                    if (b < rank) earlier.x += c.x, earlier.y += c.y;
                }
                look_in(__shfl_sync(~0u, above, at) + lanes_before(in_bin.x + in_bin.y, all), in_bin, earlier, at * kWarp + lane);
                if (lane == 0) found[4] = any;
            }
        }
        __syncthreads();
        if (pass == 0 && found[4]) {
            leave();
            meet();  // nobody leaves while others read
            return;
        }
        top |= found[0] << shift;
        need -= found[1];
        equal_before = found[2];
        if (found[3] == need) {  // so the keys above top - 1 are; top is not 0, for some key is not kept
            top -= 1;
            need = 0;
            break;
        }
    }

    // Each warp takes a run of the block's tokens, 128 at a time and a lane four.
    // Equal keys are numbered first (where not all or none of them are kept), then
    // holes and fillers counted, then numbered.
    const uint32_t part = uint32_t(align_up(ceil_div(count, kWarps), 4 * kWarp));
    const uint32_t from = min(count, warp * part), to = min(count, from + part);
    uint32_t total, equal_base = 0;
    if (need) {
        uint32_t equals = 0;
        for (uint32_t i = from + lane * 4; i < to; i += 4 * kWarp) {
            const uint4 k = keys_at(i);
            equals += (k.x == top) + (k.y == top) + (k.z == top) + (k.w == top);
        }
        equal_base = equal_before + warps_before(__reduce_add_sync(~0u, equals), warps[1], total);
    }
    const auto sort_out = [&](auto take) {  // take(lane's first token in the block, masks of its holes and fillers)
        uint32_t number = equal_base;
        for (uint32_t i0 = from; i0 < to; i0 += 4 * kWarp) {
            const uint32_t i = i0 + lane * 4;
            const uint4 k = i < to ? keys_at(i) : make_uint4(0, 0, 0, 0);
            const uint32_t key[4] = {k.x, k.y, k.z, k.w};
            uint32_t same = 0, before_me = 0;
            if (need) {
                uint32_t in_warp;
#pragma unroll
                for (int u = 0; u < 4; ++u) same += key[u] == top;
                before_me = number + lanes_before(same, in_warp);
                number += in_warp;
            }
            uint32_t hole = 0, filler = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool kept = key[u] > top || (key[u] == top && before_me++ < need);
                const bool front = lo + i + u < p.budget;
                hole |= uint32_t(key[u] && front && !kept) << u;
                filler |= uint32_t(!front && kept) << u;
            }
            take(i, hole, filler);
        }
    };
    uint32_t holes = 0, fillers = 0;
    sort_out([&](uint32_t, uint32_t hole, uint32_t filler) {
        holes += __popc(hole);
        fillers += __popc(filler);
    });
    holes = __reduce_add_sync(~0u, holes);
    fillers = __reduce_add_sync(~0u, fillers);
    if (lane == 0) {
        warps[0][warp] = holes;
        warps[2][warp] = fillers;
    }
    __syncthreads();
    uint32_t hole = __shfl_sync(~0u, lanes_before(warps[0][lane], total), warp);
    if (threadIdx.x == 0) shared.holes = total;
    uint32_t filler = __shfl_sync(~0u, lanes_before(warps[2][lane], total), warp);
    if (threadIdx.x == 0) shared.fillers = total;
    meet();
    const Shared* other = cluster.map_shared_rank(&shared, lane < blocks ? lane : 0);
    const uint32_t others_holes = lane < blocks ? other->holes : 0, others_fillers = lane < blocks ? other->fillers : 0;
    hole += __reduce_add_sync(~0u, lane < rank ? others_holes : 0);
    filler += __reduce_add_sync(~0u, lane < rank ? others_fillers : 0);
    const uint32_t moves = __reduce_add_sync(~0u, others_fillers);
    meet();  // nobody leaves while others read
    if (moves > p.max_moves) {
        leave();
        return;
    }
    longlong2* out = p.moves + r * p.moves_stride;
    sort_out([&](uint32_t i, uint32_t hole_mask, uint32_t filler_mask) {
        uint32_t in_warp;
        if (!__any_sync(~0u, hole_mask | filler_mask)) return;
        uint32_t to_hole = hole + lanes_before(__popc(hole_mask), in_warp);
        hole += in_warp;
        uint32_t to_filler = filler + lanes_before(__popc(filler_mask), in_warp);
        filler += in_warp;
        int64_t slot[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t token = lo + i + u, page = p.page.quotient(token);
            const uint32_t id = (hole_mask | filler_mask) >> u & 1 ? page_id(page) : 0;
            slot[u] = int64_t(uint64_t(id) * p.page.d + (token - page * p.page.d));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (filler_mask >> u & 1) out[to_filler++].x = slot[u];
            else if (hole_mask >> u & 1) out[to_hole++].y = slot[u];
        }
    });
    if (rank == 0 && threadIdx.x == 0) {
        p.lens_out[r] = int32_t(p.budget);
        p.counts[r] = int32_t(moves);
        if (p.evicted_out) p.evicted_out[r] = int32_t(before + int64_t(n) - p.budget);
    }
}

// The pages that no token needs any more, back on the free list: a launch of its own,
// because a request's pages lie behind those of all requests before it.
constexpr int kReleaseThreads = 256;
__global__ void __launch_bounds__(kReleaseThreads) release_kernel(const Params p, int32_t* free_blocks, const int32_t* free_used,
                                                           int32_t* free_used_out, uint32_t num_free)
{
    wait_for_previous();
    const auto pages = [&](uint32_t tokens) { return tokens ? p.page.quotient(tokens - 1) + 1 : 0u; };
    const auto kept = [&](uint32_t r) { return pages(uint32_t(p.lens_out[r])); };
    const auto freed = [&](uint32_t r) { return (long long)(pages(length_of(p.lens, r, p.longest)) - kept(r)); };
    long long begin = -1, end = -1;
    Place place;
    const long long total = share_of<kReleaseThreads>(
        p.requests, freed,
        [&](long long all) {
            const long long per = (all + gridDim.x - 1) / gridDim.x;
            begin = blockIdx.x * per;
            end = min(all, begin + per);
            return begin < all ? begin : -1;
        },
        place);
    const long long used = min((long long)max(*free_used, 0), (long long)num_free);
    if (blockIdx.x == 0 && threadIdx.x == 0) *free_used_out = int32_t(max(used - total, 0ll));
    if (begin >= total) return;
    uint32_t r = place.item;
    long long first = place.first;
    for (long long i = begin + threadIdx.x; i < end; i += kReleaseThreads) {
        while (i >= first + freed(r)) first += freed(r++);
        const long long at = used - total + i;
        if (at >= 0) free_blocks[at] = p.table[r * p.table_stride + kept(r) + uint32_t(i - first)];
    }
}

struct Moves {
    unsigned char* k;
    unsigned char* v;
    uint64_t page, token, head;  // strides in bytes
    Divider vectors;             // accesses of a head
    Divider block;               // slots of a page
    bool small;                  // slots are counted in 31 bits
    uint32_t heads;
    uint64_t num_slots;
    const longlong2* moves;
    uint64_t moves_stride;
    const int32_t* counts;
    uint32_t max_moves, requests;
    float* scores;
    int32_t* positions;
};

// Accesses are V bytes of a key and of a value, four of each under way in a thread.
// kByWarp: a warp takes a move.  Else threads take all accesses in their order,
// moves that have few for a warp side by side (256 bytes a token, 225 x 732 moves:
// 61 us by warps, 29 us in order; 2048 bytes, 16 x 7600 moves: 151 and 202 us, for
// every access finds its move anew).
constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / kWarp, kMoveAhead = 4;
template <typename V, bool kByWarp>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const Moves p)
{
    const auto moves_of = [&](uint32_t r) { return (long long)min(uint32_t(max(p.counts[r], 0)), p.max_moves); };
    long long begin = -1, end = -1;
    Place place;
    const long long total = share_of<kMoveThreads>(
        p.requests, moves_of,
        [&](long long all) {
            const long long per = (all + gridDim.x - 1) / gridDim.x;
            begin = blockIdx.x * per;
            end = min(all, begin + per);
            return begin < all ? begin : -1;
        },
        place);
    if (begin >= total) return;
    const uint32_t each = p.heads * p.vectors.d;
    // the place of a slot
    const auto place_of = [&](uint64_t slot) {
        const uint64_t page = p.small ? p.block.quotient(uint32_t(slot)) : slot / p.block.d;
        return page * p.page + (slot - page * p.block.d) * p.token;
    };
    uint32_t r = place.item;
    if (kByWarp) {
        const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
        long long first = place.first;
        for (long long i = begin + warp; i < end; i += kMoveWarps) {
            while (i >= first + moves_of(r)) first += moves_of(r++);
            const longlong2 move = p.moves[r * p.moves_stride + uint64_t(i - first)];
            if (uint64_t(move.x) >= p.num_slots || uint64_t(move.y) >= p.num_slots) continue;
            const uint64_t from = place_of(uint64_t(move.x)), to = place_of(uint64_t(move.y));
            for (uint32_t at = lane; at < each; at += kWarp * kMoveAhead) {
                V k[kMoveAhead], v[kMoveAhead];
                uint64_t offset[kMoveAhead];
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u) {
                    const uint32_t x = at + u * kWarp;
                    if (x >= each) continue;
                    const uint32_t head = p.vectors.quotient(x);
                    offset[u] = head * p.head + (x - head * p.vectors.d) * sizeof(V);
                    k[u] = *reinterpret_cast<const V*>(p.k + from + offset[u]);
                    v[u] = *reinterpret_cast<const V*>(p.v + from + offset[u]);
                }
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u) {
                    if (at + u * kWarp >= each) continue;
                    *reinterpret_cast<V*>(p.k + to + offset[u]) = k[u];
                    *reinterpret_cast<V*>(p.v + to + offset[u]) = v[u];
                }
            }
            if (lane == 0) {
                if (p.scores) p.scores[move.y] = p.scores[move.x];
                if (p.positions) p.positions[move.y] = p.positions[move.x];
            }
        }
        return;
    }
    long long first = place.first, i = begin;  // the access's move, and the first one of its request
    uint32_t at = threadIdx.x;                 // the access in its move
    while (true) {
        V k[kMoveAhead], v[kMoveAhead];
        uint64_t to[kMoveAhead];
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u) {
            to[u] = ~0ull;
            while (at >= each) {
                at -= each;
                ++i;
            }
            if (i < end) {
                while (i >= first + moves_of(r)) first += moves_of(r++);
                const longlong2 move = p.moves[r * p.moves_stride + uint64_t(i - first)];
                if (uint64_t(move.x) < p.num_slots && uint64_t(move.y) < p.num_slots) {
                    const uint32_t head = p.vectors.quotient(at);
                    const uint64_t offset = head * p.head + (at - head * p.vectors.d) * sizeof(V);
                    const uint64_t from = place_of(uint64_t(move.x)) + offset;
                    to[u] = place_of(uint64_t(move.y)) + offset;
                    k[u] = *reinterpret_cast<const V*>(p.k + from);
                    v[u] = *reinterpret_cast<const V*>(p.v + from);
                    if (at == 0) {
                        if (p.scores) p.scores[move.y] = p.scores[move.x];
                        if (p.positions) p.positions[move.y] = p.positions[move.x];
                    }
                }
            }
            at += kMoveThreads;
        }
#pragma unroll
        for (int u = 0; u < kMoveAhead; ++u) {
            if (to[u] == ~0ull) continue;
            *reinterpret_cast<V*>(p.k + to[u]) = k[u];
            *reinterpret_cast<V*>(p.v + to[u]) = v[u];
        }
        if (i >= end) return;
    }
}

lcpp_status plan(const lcpp_cache_evict_args* a, cudaStream_t s)
{
    if (!a || !a->block_size || !a->budget || a->budget >= uint32_t(1) << 31 || a->trigger < a->budget ||
        uint64_t(a->keep_first) + a->keep_recent > a->budget || a->num_requests > LCPP_MAX_REQUESTS ||
        a->table_stride < a->table_width || a->table_stride > kMostStride || a->moves_stride < a->max_moves ||
        a->moves_stride > kMostStride / 16 || uint64_t(a->num_pages) * a->block_size >= kMostSlots)
        return LCPP_ERR_INVALID_ARG;
    const uint64_t n = a->num_requests, slots = uint64_t(a->num_pages) * a->block_size;
    const bool release = a->free_blocks || a->free_used || a->free_used_out;
    if (release && (!a->free_used || !a->free_used_out || (a->num_free && !a->free_blocks))) return LCPP_ERR_INVALID_ARG;
    if (n && (!a->seq_lens || !a->seq_lens_out || !a->move_counts_out || (a->max_moves && !a->moves_out) ||
              (a->table_width && !a->block_table) || (slots && !a->slot_scores)))
        return LCPP_ERR_INVALID_ARG;
    const void* words[] = {a->seq_lens,        a->block_table,  a->slot_scores,     a->slot_positions, a->evicted,
                           a->seq_lens_out,    a->evicted_out,  a->move_counts_out, a->free_blocks,    a->free_used,
                           a->free_used_out};
    for (const void* w : words)
        if (misaligned(w, 4)) return LCPP_ERR_INVALID_ARG;
    if (misaligned(a->moves_out, 16)) return LCPP_ERR_INVALID_ARG;
    const bool in_place = a->evicted == a->evicted_out;
    const Array arrays[] = {{a->seq_lens, n * 4, false},
                            {a->slot_scores, slots * 4, false},
                            {a->slot_positions, a->slot_positions ? slots * 4 : 0, false},
                            {in_place ? nullptr : a->evicted, n * 4, false},
                            {a->seq_lens_out, n * 4, true},
                            {a->evicted_out, n * 4, true},
                            {a->move_counts_out, n * 4, true},
                            {a->moves_out, span_bytes(n, a->moves_stride, a->max_moves, 16), true},
                            {a->free_blocks, uint64_t(a->num_free) * 4, true},
                            {a->free_used, 4, false},
                            {a->free_used_out, 4, true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
    for (const Array& o : arrays)
        if (o.written && overlap_rows(a->block_table, n, a->table_stride, a->table_width, 4, o.p, o.bytes))
            return LCPP_ERR_INVALID_ARG;

    Params p{};
    p.lens = a->seq_lens;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.scores = a->slot_scores;
    p.positions = a->slot_positions;
    p.evicted = a->evicted;
    p.page = Divider(a->block_size);
    p.longest = uint32_t(std::min<uint64_t>(uint64_t(a->table_width) * a->block_size, 0x7fffffffu));
    p.num_pages = a->num_pages;
    p.requests = a->num_requests;
    p.budget = a->budget;
    p.trigger = a->trigger;
    p.first = a->keep_first;
    p.recent = a->keep_recent;
    p.max_moves = a->max_moves;
    p.lens_out = a->seq_lens_out;
    p.evicted_out = a->evicted_out;
    p.counts = a->move_counts_out;
    p.moves = reinterpret_cast<longlong2*>(a->moves_out);
    p.moves_stride = a->moves_stride;

    diag::KernelTimer timer(kTimerEviction, n, s);
    if (n) {
        // Blocks for 2048 tokens and more of what a row of the table holds (the lengths are on
        // the device; 64 requests of 2100 tokens with their release 11.5 us under a table as
        // wide, 23.7 under one for 131072), as long as the requests leave SMs for them; and of
        // no more than have room for their keys.  Clusters of 1 / 2 / 4 / 8: 16 requests
        // of 4096 tokens 13.5 / 14.0 / 13.7 / 14.9 us, of 16384 25.8 / 20.3 / 16.9 / 17.3,
        // 64 of 16384 28.6 / 23.4 / 29.9 / 54.7, 100 of 131072 468 / 235 / 137 / 176.
        uint32_t cluster = 1;
        while (cluster < kMostCluster && ((p.longest / cluster > 4096 && n * cluster * 2 <= uint64_t(device_sm_count())) ||
                                          ceil_div(p.longest, cluster) > kKeys))
            cluster *= 2;
        const uint32_t run = uint32_t(ceil_div(p.longest, cluster));
        // room in a few steps, so that few launch shapes are set up
        uint32_t room = 4096;
        while (room < kKeys && room < run) room *= 2;
        const size_t smem = (kBins * kCopies + kPages + std::min(room, kKeys)) * 4;
        set_max_dynamic_smem(reinterpret_cast<const void*>(plan_kernel), (kBins * kCopies + kPages + kKeys) * 4);
        cudaLaunchAttribute shape{};
        shape.id = cudaLaunchAttributeClusterDimension;
        shape.val.clusterDim.x = cluster;
        shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(unsigned(n * cluster));
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = smem;
        config.stream = s;
        config.attrs = &shape;
        config.numAttrs = 1;
        LCPP_CUDA_TRY(cudaLaunchKernelEx(&config, plan_kernel, p));
    }
    if (!release) return LCPP_OK;
    if (n == 0) {
        release_kernel<<<1, kReleaseThreads, 0, s>>>(p, a->free_blocks, a->free_used, a->free_used_out, a->num_free);
        return launched();
    }
    return launch_early(release_kernel, unsigned(std::min<uint64_t>(n, device_sm_count())), kReleaseThreads, 0, s, Params(p),
                        static_cast<int32_t*>(a->free_blocks), static_cast<const int32_t*>(a->free_used),
                        static_cast<int32_t*>(a->free_used_out), uint32_t(a->num_free));
}

lcpp_status move(const lcpp_kv_cache* c, const int64_t* moves, uint64_t moves_stride, uint32_t max_moves,
                 const int32_t* counts, uint32_t num_requests, float* scores, int32_t* positions, cudaStream_t s)
{
    if (!c || !sane_cache(*c) || num_requests > LCPP_MAX_REQUESTS || moves_stride < max_moves ||
        moves_stride > kMostStride / 16)
        return LCPP_ERR_INVALID_ARG;
    const int e = row_dtype_bytes(c->dtype);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    const uint64_t n = num_requests, slots = uint64_t(c->num_pages) * c->block_size;
    if (!n || !max_moves || !slots) return LCPP_OK;
    if (!moves || !counts || !c->k || !c->v || misaligned(moves, 16) || misaligned(counts, 4) || misaligned(c->k, e) ||
        misaligned(c->v, e) || misaligned(scores, 4) || misaligned(positions, 4) || !writable_cache(*c))
        return LCPP_ERR_INVALID_ARG;
    const Strided k = pages_of(*c, c->k), v = pages_of(*c, c->v);
    const Array arrays[] = {{moves, span_bytes(n, moves_stride, max_moves, 16), false},
                            {counts, n * 4, false},
                            {scores, slots * 4, true},
                            {positions, slots * 4, true}};
    if (clash(arrays)) return LCPP_ERR_INVALID_ARG;
    for (const Array& x : arrays)
        if (overlap(k.p, k.bytes(), x.p, x.bytes) || overlap(v.p, v.bytes(), x.p, x.bytes)) return LCPP_ERR_INVALID_ARG;
    if (uint64_t(c->num_kv_heads) * c->head_dim >= uint64_t(1) << 31) return LCPP_ERR_INVALID_ARG;

    const bool wide = c->head_dim * e % 16 == 0 && rows_aligned(c->k, {c->page_stride, c->token_stride, c->head_stride}, e, 16) &&
                      !misaligned(c->v, 16);
    const uint32_t access = wide ? 16 : e;
    Moves p{};
    p.k = static_cast<unsigned char*>(c->k);
    p.v = static_cast<unsigned char*>(c->v);
    p.page = c->page_stride * e;
    p.token = c->token_stride * e;
    p.head = c->head_stride * e;
    p.vectors = Divider(c->head_dim * e / access);
    p.heads = c->num_kv_heads;
    p.block = Divider(c->block_size);
    p.small = slots < uint64_t(1) << 31;
    p.num_slots = slots;
    p.moves = reinterpret_cast<const longlong2*>(moves);
    p.moves_stride = moves_stride;
    p.counts = counts;
    p.max_moves = max_moves;
    p.requests = num_requests;
    p.scores = scores;
    p.positions = positions;
    const auto launch = [&](auto kernel) {
        const uint64_t most = uint64_t(device_sm_count()) * resident_blocks(reinterpret_cast<const void*>(kernel), kMoveThreads, 0);
        const uint64_t accesses = std::min<uint64_t>(n * max_moves, uint64_t(1) << 32) * (p.heads * p.vectors.d);
        const unsigned blocks = unsigned(std::min<uint64_t>(most, ceil_div(accesses, kMoveThreads)));
        kernel<<<blocks, kMoveThreads, 0, s>>>(p);
        return launched();
    };
    diag::KernelTimer timer(kTimerEviction, n, s);
    if (p.heads * p.vectors.d >= 2 * kWarp)
        return wide ? launch(move_kernel<uint4, true>) : e == 4 ? launch(move_kernel<uint32_t, true>) : launch(move_kernel<unsigned short, true>);
    return wide ? launch(move_kernel<uint4, false>) : e == 4 ? launch(move_kernel<uint32_t, false>) : launch(move_kernel<unsigned short, false>);
}

}  // namespace

extern "C" {

lcpp_status lcpp_cache_evict_plan(const lcpp_cache_evict_args* args, lcpp_stream_t stream)
{
    return guarded("lcpp_cache_evict_plan", [&] { return plan(args, reinterpret_cast<cudaStream_t>(stream)); });
}

lcpp_status lcpp_cache_evict_move(const lcpp_kv_cache* cache, const int64_t* moves, uint64_t moves_stride,
                                  uint32_t max_moves, const int32_t* move_counts, uint32_t num_requests,
                                  float* slot_scores, int32_t* slot_positions, lcpp_stream_t stream)
{
    return guarded("lcpp_cache_evict_move", [&] {
        return move(cache, moves, moves_stride, max_moves, move_counts, num_requests, slot_scores, slot_positions,
                    reinterpret_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
