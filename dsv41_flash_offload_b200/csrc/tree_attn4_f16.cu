// Attention of drafted tokens over a cache in 4 bits, fp16 queries and outputs.
#include "tree_attn_kernel.cuh"

namespace dsv41 {

cudaError_t launch_tree_attn4_f16(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return p.window < kNoWindow || !p.tree_mask ? launch_tree_attn4_typed<__half, true>(p, max_rows, st) : launch_tree_attn4_typed<__half, false>(p, max_rows, st);
}

}  // namespace dsv41
