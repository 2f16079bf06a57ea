// paged_attention.cu -- DevicePagedAttention's entry points, and the scores of
// the cache's tokens (include/lcpp_b200_model.h, paged_attention.cuh).
//
// The share that a token gets of a head's attention is 2^(x - lse), which is
// known when all of the head's tokens are: where scores are wanted the decode
// kernel leaves its logits, 4 bytes for each token and head against the 4 D / g
// (16 bits, g query heads to a kv head) that it reads for them, and scores_kernel
// sums them for each token in the order of the heads.  The logits stay in L2; their
// writes, the third launch and its dependent loads are what scores cost (48 requests of
// 4096 tokens and fewer, 40 heads: 97 us with them, 86 without).
#include "paged_attention.cuh"

using namespace lcpp;
using namespace lcpp::model;
using namespace lcpp::model::attention;

namespace {

constexpr int kScoreThreads = 256, kScoreWarps = kScoreThreads / kWarp;

// A warp takes 16 tokens: a lane four of them under every eighth head.  Bound by the
// latency of page id, score, log-sum and logits, of which the first two are loaded
// before the wait and the others together (102.6 -> 97.9 us for the call above).
__global__ void __launch_bounds__(kScoreThreads) scores_kernel(const Params p)
{
    const auto weight = [&](uint32_t r) {  // tiles before the window, then those of the logits
        const Tokens t = tokens_of(p, r);
        return (long long)(t.base() / kTile + t.tiles());
    };
    long long begin = -1, end = -1;
    Place place;
    const long long total = share_of<kScoreThreads>(
        p.requests, weight,
        [&](long long all) {
            const long long per = max((all + gridDim.x - 1) / gridDim.x, (long long)kScoreWarps);
            begin = blockIdx.x * per;
            end = min(all, begin + per);
            return begin < all ? begin : -1;
        },
        place);
    if (begin >= total) {
        if (blockIdx.x == 0) wait_for_previous();  // this launch ends after the ones before
        return;
    }
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp, quad = lane % 4, part = lane / 4;
    const uint32_t units = p.kv_heads * p.chunks;
    uint32_t r = place.item;
    long long first = place.first;
    bool waited = false;
    for (long long at = begin + warp; at < end || !waited; at += kScoreWarps) {
        const bool live = at < end;
        float before_score = 0.f;  // of the token that the lane writes: 4 quad + part of the tile
        int64_t slot = -1;
        Tokens seen{};
        if (live) {
            while (at >= first + weight(r)) first += weight(r++);
            seen = tokens_of(p, r);
            const uint32_t token = uint32_t(at - first) * kTile + quad * 4 + part;
            if (part < 4 && token < seen.end) {
                const uint32_t page = p.page.quotient(token), id = uint32_t(p.table[r * p.table_stride + page]);
                if (id < p.num_pages) {
                    slot = int64_t(uint64_t(id) * p.page.d + (token - page * p.page.d));
                    if (p.scores) before_score = p.scores[slot];
                }
            }
        }
        // up to here nothing is read that the launches before this one write
        if (!waited) wait_for_previous();
        waited = true;
        if (!live) break;
        const uint32_t before = seen.base() / kTile, tiles = seen.tiles();
        const long long number = p.first[r];
        if (number + (long long)tiles * units > p.logit_tiles) continue;
        float mass[4] = {0.f, 0.f, 0.f, 0.f};
        if (at - first >= before) {
            const uint32_t t = uint32_t(at - first) - before;
            const float* lse = p.lse2 + uint64_t(r) * p.heads;
            const float4* x = reinterpret_cast<const float4*>(p.logits) + (number + t) * p.per_unit * (kTile / 4) + quad;
            const long long pitch = (long long)tiles * p.per_unit * (kTile / 4);
            constexpr int kAhead = 5;  // heads of a lane under way
            for (uint32_t h0 = part; h0 < p.heads; h0 += kAhead * (kWarp / 4)) {
                float of[kAhead];
                float4 logits[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const uint32_t head = h0 + u * (kWarp / 4);
                    of[u] = -INFINITY;
                    if (head >= p.heads) continue;
                    // the head's unit, and its place in it
                    const uint32_t kv_head = p.by_group.quotient(head), in_group = head - kv_head * p.group;
                    const uint32_t chunk = p.by_unit.quotient(in_group), h = in_group - chunk * p.per_unit;
                    of[u] = lse[head];
                    logits[u] = x[(kv_head * p.chunks + chunk) * pitch + h * (kTile / 4)];
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (of[u] == -INFINITY) continue;
                    mass[0] += exp2_fast(logits[u].x - of[u]);
                    mass[1] += exp2_fast(logits[u].y - of[u]);
                    mass[2] += exp2_fast(logits[u].z - of[u]);
                    mass[3] += exp2_fast(logits[u].w - of[u]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 4; d < kWarp; d *= 2) mass[i] += __shfl_xor_sync(~0u, mass[i], d);
        const float own = part == 0 ? mass[0] : part == 1 ? mass[1] : part == 2 ? mass[2] : mass[3];
        if (slot >= 0) p.scores_out[slot] = p.decay * before_score + own;
    }
}

constexpr uint32_t kMostHeads = 1u << 16;

struct Layout {
    size_t part, split, lse2, first, logits, part_bytes, bytes;
    uint64_t tiles;
};

Layout layout(uint64_t requests, uint32_t heads, uint32_t kv_heads, const Choice& c, uint64_t score_slots)
{
    Layout l{};
    const auto take = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += align_up(bytes, kTempAlign);
        return at;
    };
    l.part_bytes = size_t(kMostBlocks) * 2 * c.heads * (c.columns + 2) * 4;
    l.part = take(l.part_bytes);
    l.split = take(kMostBlocks * 16);
    if (!score_slots) return l;
    l.lse2 = take(requests * heads * 4);
    l.first = take(requests * 8);
    // every request's tokens in tiles of 16, a partial one at either end, no slot twice
    l.tiles = (score_slots + 2 * (kTile - 1) * requests) / kTile * kv_heads * c.chunks;
    l.logits = take(l.tiles * c.per_unit * kTile * 4);
    return l;
}

bool sane_heads(uint32_t requests, uint32_t heads, uint32_t kv_heads, uint32_t dim)
{
    return requests <= LCPP_MAX_REQUESTS && heads && heads <= kMostHeads && kv_heads && heads % kv_heads == 0 && dim &&
           dim <= LCPP_MAX_HEAD_DIM;
}

lcpp_status run(void* temp, size_t temp_bytes, const lcpp_paged_attention_args* a, cudaStream_t s)
{
    if (!a || !sane_heads(a->num_requests, a->num_heads, a->cache.num_kv_heads, a->cache.head_dim) ||
        !sane_cache(a->cache) || a->table_stride < a->table_width || a->table_stride > kMostStride ||
        a->q_request_stride > kMostStride || a->q_head_stride > kMostStride || a->out_request_stride > kMostStride ||
        a->out_head_stride > kMostStride || !(a->softcap >= 0.f) || !std::isfinite(a->softcap) ||
        !std::isfinite(a->scale) || !std::isfinite(a->score_decay))
        return LCPP_ERR_INVALID_ARG;
    const lcpp_kv_cache& cache = a->cache;
    const int e = row_dtype_bytes(cache.dtype);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    const uint64_t n = a->num_requests, slots = uint64_t(cache.num_pages) * cache.block_size;
    if (!temp || misaligned(temp, kTempAlign)) return LCPP_ERR_INVALID_ARG;
    if (a->slot_scores && !a->slot_scores_out) return LCPP_ERR_INVALID_ARG;
    if (n == 0) return LCPP_OK;
    if (!a->q || !a->out || !a->seq_lens || (a->table_width && !a->block_table) || (slots && (!cache.k || !cache.v)))
        return LCPP_ERR_INVALID_ARG;
    for (const void* x : {a->q, static_cast<const void*>(a->out), static_cast<const void*>(cache.k), static_cast<const void*>(cache.v)})
        if (misaligned(x, e)) return LCPP_ERR_INVALID_ARG;
    for (const void* x : {static_cast<const void*>(a->block_table), static_cast<const void*>(a->seq_lens),
                          static_cast<const void*>(a->lse_out), static_cast<const void*>(a->slot_scores),
                          static_cast<const void*>(a->slot_scores_out)})
        if (misaligned(x, 4)) return LCPP_ERR_INVALID_ARG;

    const Strided k = pages_of(cache, cache.k), v = pages_of(cache, cache.v);
    const Strided q(a->q, e, cache.head_dim, {{n, a->q_request_stride}, {a->num_heads, a->q_head_stride}});
    const Strided out(a->out, e, cache.head_dim, {{n, a->out_request_stride}, {a->num_heads, a->out_head_stride}});
    if (!k.sane() || !q.sane() || !out.sane() || !out.distinct()) return LCPP_ERR_INVALID_ARG;
    const uint64_t score_slots = a->slot_scores_out ? slots : 0;
    const Choice c = choose(a->num_heads / cache.num_kv_heads, cache.head_dim, cache.dtype == LCPP_F32);
    const Layout l = layout(n, a->num_heads, cache.num_kv_heads, c, score_slots);
    if (temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;

    const Strided written[] = {out, Strided(a->lse_out, 4, a->lse_out ? n * a->num_heads : 0, {}),
                               Strided(a->slot_scores_out, 4, score_slots, {}), Strided(temp, 1, l.bytes, {})};
    const Strided read[] = {k, v, q, Strided(a->block_table, 4, a->table_width, {{n, a->table_stride}}),
                            Strided(a->seq_lens, 4, n, {}),
                            Strided(a->slot_scores, 4, a->slot_scores && a->slot_scores != a->slot_scores_out ? slots : 0, {})};
    for (size_t i = 0; i < sizeof(written) / sizeof(written[0]); ++i) {
        for (const Strided& x : read)
            if (!x.sane() || may_share(written[i], x)) return LCPP_ERR_INVALID_ARG;
        for (size_t j = 0; j < i; ++j)
            if (may_share(written[i], written[j])) return LCPP_ERR_INVALID_ARG;
    }

    unsigned char* t = static_cast<unsigned char*>(temp);
    Params p{};
    p.q = a->q;
    p.out = a->out;
    p.k = cache.k;
    p.v = cache.v;
    p.q_request = a->q_request_stride;
    p.q_head = a->q_head_stride;
    p.out_request = a->out_request_stride;
    p.out_head = a->out_head_stride;
    p.page_stride = cache.page_stride;
    p.token_stride = cache.token_stride;
    p.head_stride = cache.head_stride;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.lens = a->seq_lens;
    p.page = Divider(cache.block_size);
    // without pages every row is empty: nothing asks for an address in them
    p.longest = slots ? uint32_t(std::min<uint64_t>(uint64_t(a->table_width) * cache.block_size, 0x7fffffffu)) : 0u;
    p.page_tiles = cache.block_size % kTile == 0;
    p.wide_q = rows_aligned(a->q, {a->q_request_stride, a->q_head_stride}, e, 16) && cache.head_dim * e % 16 == 0;
    p.wide_out = rows_aligned(a->out, {a->out_request_stride, a->out_head_stride}, e, 4 * e) && cache.head_dim % 4 == 0;
    p.num_pages = cache.num_pages;
    p.requests = a->num_requests;
    p.heads = a->num_heads;
    p.kv_heads = cache.num_kv_heads;
    p.group = a->num_heads / cache.num_kv_heads;
    p.chunks = c.chunks;
    p.per_unit = c.per_unit;
    p.dim = cache.head_dim;
    p.window = a->window;
    p.scale = a->softcap > 0.f ? a->scale / a->softcap : a->scale * kLog2e;
    p.softcap = a->softcap * kLog2e;
    // products of factors that are numbers and may be none: 0 * inf would make NaN of logits of 0
    if (!std::isfinite(p.scale) || !std::isfinite(p.softcap)) return LCPP_ERR_INVALID_ARG;
    p.lse = a->lse_out;
    p.part = reinterpret_cast<float*>(t + l.part);
    p.split = reinterpret_cast<int32_t*>(t + l.split);
    if (score_slots) {
        p.by_group = Divider(p.group);
        p.by_unit = Divider(p.per_unit);
        p.lse2 = reinterpret_cast<float*>(t + l.lse2);
        p.first = reinterpret_cast<long long*>(t + l.first);
        p.logits = reinterpret_cast<float*>(t + l.logits);
        p.logit_tiles = (long long)l.tiles;
        p.scores = a->slot_scores;
        p.scores_out = a->slot_scores_out;
        p.decay = a->score_decay;
    }
    const bool wide = cache.head_dim * e % 16 == 0 &&
                      rows_aligned(cache.k, {cache.page_stride, cache.token_stride, cache.head_stride}, e, 16) &&
                      !misaligned(cache.v, 16);
    diag::KernelTimer timer(kTimerAttention, n, s);
    const lcpp_status status = cache.dtype == LCPP_F32   ? run_f32(p, c, wide, l.part_bytes, s)
                               : cache.dtype == LCPP_F16 ? run_f16(p, c, wide, l.part_bytes, s)
                                                         : run_bf16(p, c, wide, l.part_bytes, s);
    if (status != LCPP_OK || !score_slots) return status;
    const unsigned blocks =
        unsigned(device_sm_count() * resident_blocks(reinterpret_cast<const void*>(scores_kernel), kScoreThreads, 0));
    return launch_early(scores_kernel, blocks, kScoreThreads, 0, s, Params(p));
}

}  // namespace

extern "C" {

lcpp_status lcpp_paged_attention_temp_bytes(uint32_t num_requests, uint32_t num_heads, uint32_t num_kv_heads,
                                            uint32_t head_dim, uint64_t score_slots, size_t* temp_bytes)
{
    if (!temp_bytes || !sane_heads(num_requests, num_heads, num_kv_heads, head_dim) || score_slots >= kMostSlots)
        return LCPP_ERR_INVALID_ARG;
    // enough for either kind of type
    size_t most = 0;
    for (const bool f32 : {false, true})
        most = std::max(most, layout(num_requests, num_heads, num_kv_heads,
                                     choose(num_heads / num_kv_heads, head_dim, f32), score_slots)
                                  .bytes);
    *temp_bytes = most;
    return LCPP_OK;
}

lcpp_status lcpp_paged_attention_decode(void* temp, size_t temp_bytes, const lcpp_paged_attention_args* args,
                                        lcpp_stream_t stream)
{
    return guarded("lcpp_paged_attention_decode",
                   [&] { return run(temp, temp_bytes, args, reinterpret_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
