// router_f16.cu -- DeviceRouter's kernels for f16 logits.
#include "router.cuh"

namespace lcpp {
namespace router {

lcpp_status forward_f16(const Params& p, bool sigmoid, cudaStream_t s)
{
    return forward_rows<__half>(p, sigmoid, s);
}

lcpp_status backward_f16(const BackParams& p, bool sigmoid, cudaStream_t s)
{
    return backward_rows<__half>(p, sigmoid, s);
}

}  // namespace router
}  // namespace lcpp
