// Attention of drafted tokens over a bf16 cache.
#include "tree_attn_kernel.cuh"

namespace dsv41 {

cudaError_t launch_tree_attn_bf16(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return launch_tree_attn_typed<__nv_bfloat16>(p, max_rows, st);
}

}  // namespace dsv41
