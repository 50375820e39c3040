// Attention of drafted tokens over a paged cache (dsv41_tree_attention): the mathematics, the choice of type
// and the workspace (tree_attn_kernel.cuh has the kernel).
//
// For request b with s_b keys in the cache, the last n_b of them its new tokens, token i and query head
// hq = h * G + g:
//     out[i, hq] = sum_j p_ij v[j, h] / sum_j p_ij,   p_ij = exp(scale * q[i, hq] . k[j, h] - m_i)
// over the keys j that i sees: all of the context, and among the new tokens its ancestors and itself (a bit
// mask per token), or the tokens before it and itself (no mask). A row that sees nothing is zero.
//
// All G query heads of a KV head and all new tokens of a request share its keys, so they are the rows
// (r = i * G + g) of one product: each key and value is read once per tile of rows, and the softmax runs over
// the keys in one pass (running maximum m and sum l in fp32, the accumulator rescaled when m grows).
//
// Split: the (request, KV head, row tile, key tile) units of the call are cut into equal runs, one per
// CTA and SM, whatever the lengths are; the cut is computed in the kernel from the lengths (the host does
// not know them). A segment (the units of one row tile) that crosses CTAs leaves (m, l, O) per part in the
// workspace and the CTA that arrives last joins the parts in order: one launch, results independent of timing.
#include "internal.h"
#include "paged.h"

namespace dsv41 {

cudaError_t launch_tree_attn(const TreeAttnParams& p, int dtype, int max_rows, cudaStream_t st)
{
    return dtype == 0 ? launch_tree_attn_f16(p, max_rows, st) : launch_tree_attn_bf16(p, max_rows, st);
}

// Most parts a call can leave: two per CTA (one CTA per SM), of a row tile of the padded head size.
AttnWorkspace tree_attn_workspace(int head_dim)
{
    const int64_t dt = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    const int64_t ctas = num_sms(), rows = 2 * ctas * (dt == 256 ? 128 : 256);
    AttnWorkspace w;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    w.counters = 256;
    w.part_ml = w.counters + up(2 * ctas * sizeof(int));
    w.part_o = w.part_ml + up(rows * sizeof(float2));
    w.total = w.part_o + up(rows * dt * sizeof(float));
    return w;
}

}  // namespace dsv41
