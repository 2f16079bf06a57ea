// router_f32.cu -- DeviceRouter's kernels for f32 logits.
#include "router.cuh"

namespace lcpp {
namespace router {

lcpp_status forward_f32(const Params& p, bool sigmoid, cudaStream_t s)
{
    return forward_rows<float>(p, sigmoid, s);
}

lcpp_status backward_f32(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    return backward_rows<float>(p, sigmoid, s);
}

}  // namespace router
}  // namespace lcpp
