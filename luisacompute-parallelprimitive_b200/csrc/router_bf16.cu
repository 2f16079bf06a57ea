// router_bf16.cu -- DeviceRouter's kernels for bf16 logits.
#include "router.cuh"

namespace lcpp {
namespace router {

lcpp_status forward_bf16(const Params& p, bool sigmoid, cudaStream_t s)
{
    return forward_rows<__nv_bfloat16>(p, sigmoid, s);
}

lcpp_status backward_bf16(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    return backward_rows<__nv_bfloat16>(p, sigmoid, s);
}

}  // namespace router
}  // namespace lcpp
