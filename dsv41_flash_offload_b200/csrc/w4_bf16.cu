// 4-bit products with bf16 inputs.
#include "w4_kernel.cuh"

namespace dsv41 {

cudaError_t launch_w4_bf16(const W4Params& p, int group, bool gated, cudaStream_t st)
{
    return launch_w4_typed<__nv_bfloat16>(p, group, gated, st);
}

}  // namespace dsv41
