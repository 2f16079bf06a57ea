// paged_attention_f32.cu -- DevicePagedAttention for caches of this type (paged_attention.cuh).
#include "paged_attention.cuh"

namespace lcpp {
namespace model {
namespace attention {

lcpp_status run_f32(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s)
{
    switch (c.columns) {
    case 64:
        return c.heads == 1   ? launch<float, 64, 1, 4, 4, 3>(p, wide, part_bytes, s)
               : c.heads == 2 ? launch<float, 64, 2, 4, 4, 3>(p, wide, part_bytes, s)
               : c.heads == 4 ? launch<float, 64, 4, 4, 4, 3>(p, wide, part_bytes, s)
                              : launch<float, 64, 8, 4, 4, 3>(p, wide, part_bytes, s);
    case 128:
        return c.heads == 1   ? launch<float, 128, 1, 3, 4, 2>(p, wide, part_bytes, s)
               : c.heads == 2 ? launch<float, 128, 2, 3, 4, 2>(p, wide, part_bytes, s)
               : c.heads == 4 ? launch<float, 128, 4, 3, 4, 2>(p, wide, part_bytes, s)
                              : launch<float, 128, 8, 3, 4, 2>(p, wide, part_bytes, s);
    default:
        return c.heads == 1   ? launch<float, 256, 1, 2, 2, 3>(p, wide, part_bytes, s)
               : c.heads == 2 ? launch<float, 256, 2, 2, 2, 3>(p, wide, part_bytes, s)
                              : launch<float, 256, 4, 2, 2, 3>(p, wide, part_bytes, s);
    }
}

}  // namespace attention
}  // namespace model
}  // namespace lcpp
