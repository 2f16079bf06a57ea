// paged_attention_bf16.cu -- DevicePagedAttention for caches of this type (paged_attention.cuh).
#include "paged_attention.cuh"

namespace lcpp {
namespace model {
namespace attention {

lcpp_status run_bf16(const Params& p, const Choice& c, bool wide, size_t part_bytes, cudaStream_t s)
{
    return run_16bit<__nv_bfloat16>(p, c, wide, part_bytes, s);
}

}  // namespace attention
}  // namespace model
}  // namespace lcpp
