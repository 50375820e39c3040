// Attention of drafted tokens over a paged cache (dsv41_tree_attention): the mathematics, the choice of type
// and the workspace (tree_attn_kernel.cuh has the kernel).
//
// For request b with s_b keys in the cache, the last n_b of them its new tokens, token i and query head
// hq = h * G + g:
//     out[i, hq] = sum_j p_ij v[j, h] / sum_j p_ij,   p_ij = exp(scale * q[i, hq] . k[j, h] - m_i)
// over the keys j that i sees: all of the context, and among the new tokens its ancestors and itself (a bit
// mask per token), or the tokens before it and itself (no mask). A row that sees nothing is zero. With a window it sees the last
// `window` of these and those at the first `sinks` positions; tiles of keys that no row of a row tile sees are not read.
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
    if (p.window < kNoWindow) return dtype == 0 ? launch_tree_attn_window_f16(p, max_rows, st) : launch_tree_attn_window_bf16(p, max_rows, st);
    return dtype == 0 ? launch_tree_attn_f16(p, max_rows, st) : launch_tree_attn_bf16(p, max_rows, st);
}

// Over a cache in 4 bits, up to 16 rows codes are decoded straight into the fragments of warp-level matrix instructions
// (tree_attn4_rows.cuh), more go through shared memory to the fifth-generation tensor cores. 4 requests of 32-64k keys, 8 KV heads of
// 128: 8 rows 80 us (141 the other way), 16 rows 100 (140), 24 rows, for which the first reads the keys twice, 169 and 142. Heads of 64:
// 60 (109), 72 (107), 118 and 107; of 256: 141 (377), 180 (380), 311 and 385 (there the first would still be the faster one).
constexpr int kFewRows = 16;

cudaError_t launch_tree_attn4(const TreeAttnParams& p, int dtype, int max_rows, cudaStream_t st)
{
    if (max_rows <= kFewRows) return dtype == 0 ? launch_tree_attn4_rows_f16(p, max_rows, st) : launch_tree_attn4_rows_bf16(p, max_rows, st);
    return dtype == 0 ? launch_tree_attn4_f16(p, max_rows, st) : launch_tree_attn4_bf16(p, max_rows, st);
}

// Most parts a call can leave: two per CTA, of a row tile of the padded head size; CTAs that share an SM (up to kAttnCtas) have
// smaller row tiles.
AttnWorkspace tree_attn_workspace(int head_dim)
{
    const int64_t dt = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    const int64_t ctas = num_sms(), rows = 2 * ctas * (dt == 256 ? 128 : 256);
    AttnWorkspace w;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    w.counters = 256;
    w.part_ml = w.counters + up(kAttnCtas * ctas * sizeof(int));
    w.part_o = w.part_ml + up(rows * sizeof(float2));
    w.total = w.part_o + up(rows * dt * sizeof(float));
    return w;
}

}  // namespace dsv41
