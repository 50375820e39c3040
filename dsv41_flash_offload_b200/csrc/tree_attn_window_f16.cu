// Attention of drafted tokens through a window over an fp16 cache.
#include "tree_attn_kernel.cuh"

namespace dsv41 {

cudaError_t launch_tree_attn_window_f16(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return launch_tree_attn_typed<__half, true>(p, max_rows, st);
}

}  // namespace dsv41
