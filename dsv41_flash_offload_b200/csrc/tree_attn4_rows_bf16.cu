// Attention of few rows over a cache in 4 bits, bf16 queries and outputs.
#include "tree_attn4_rows.cuh"

namespace dsv41 {

cudaError_t launch_tree_attn4_rows_bf16(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return launch_tree_attn4_rows<__nv_bfloat16>(p, max_rows, st);
}

}  // namespace dsv41
