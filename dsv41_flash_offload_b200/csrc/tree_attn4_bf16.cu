// Attention of drafted tokens over a cache in 4 bits, bf16 queries and outputs.
#include "tree_attn_kernel.cuh"

namespace dsv41 {

cudaError_t launch_tree_attn4_bf16(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return p.window < kNoWindow || !p.tree_mask ? launch_tree_attn4_typed<__nv_bfloat16, true>(p, max_rows, st) : launch_tree_attn4_typed<__nv_bfloat16, false>(p, max_rows, st);
}

}  // namespace dsv41
