// Launch interface of the paged-cache kernels (paged.cu, tree_attn.cu) for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv41 {

constexpr int kMaxRequests = 2048;   // requests per step
constexpr int kMaxMaskWords = 4;     // 64-bit words of a drafted token's ancestor mask
// status bits of a request
constexpr int kTabNoPages = 1, kTabTooWide = 2, kTabBadParent = 4, kTabBigTree = 8, kTabNoRoom = 16, kTabPastTokens = 32;

struct StepTablesParams {
    const int *context_lens, *new_lens, *held_pages;   // [batch]
    int* block_table;                                  // [batch][table_stride], width columns
    int64_t table_stride;
    int* free_pages;                                   // stack of free_capacity entries
    const int* free_count;
    int batch, width, free_capacity, page_size, num_tokens, mask_words;
    const int* parents;                                // [num_tokens] or NULL
    int *cu_lens, *seq_lens;                           // [batch + 1], [batch]
    int64_t* slots;                                    // [num_tokens]
    int *positions, *requests;                         // [num_tokens]
    int *held_out, *free_count_out, *status;           // [batch], [1], [batch]
    int64_t* tree_mask;                                // [num_tokens][mask_words] (with parents)
};

struct StoreKvParams {
    const void *k, *v;                                 // [num_tokens][kv_heads][head_dim], 16-bit elements
    int64_t k_stride_token, k_stride_head, v_stride_token, v_stride_head;
    const int64_t* slots;
    void *k_cache, *v_cache;                           // [num_pages][page_size][kv_heads][head_dim]
    int64_t stride_page, stride_slot, stride_head;
    int num_tokens, kv_heads, head_dim, num_pages, page_size;
};

// unsigned division by a constant of the call: n / d for 0 <= n < 2^31 as a multiply and a shift.
// With l = ceil(log2 d) and m = ceil(2^(31 + l) / d): m d - 2^(31 + l) < d <= 2^l, so the error n (m d - 2^(31+l))
// stays below 2^(31 + l) and the quotient is exact.
struct FastDiv {
    uint32_t mul;
    int shift;   // l - 1; -1: d is 1
    static FastDiv make(int d)
    {
        int l = 0;
        while ((1ll << l) < d) ++l;
        FastDiv f{0, l - 1};
        if (l) f.mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
        return f;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int div(int n) const { return shift < 0 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
#endif
};

struct TreeAttnParams {
    const void* q;                                     // [num_tokens][q_heads][head_dim]
    int64_t q_stride_token, q_stride_head;
    const void *k_cache, *v_cache;                     // same strides (elements)
    int64_t stride_page, stride_slot, stride_head;
    const int* block_table;
    int64_t table_stride;
    const int *seq_lens, *cu_lens;
    const int64_t* tree_mask;                          // [num_tokens][mask_words] or NULL (causal)
    void* out;
    int64_t out_stride_token, out_stride_head;
    float* lse;                                        // [num_tokens][q_heads] or NULL
    float2* part_ml;
    float* part_o;
    int* counters;                                     // zero between calls
    int* status;
    int batch, num_tokens, q_heads, kv_heads, group, head_dim, page_size, num_pages, max_keys, mask_words;
    FastDiv page_div, group_div;
    int box, slot_first;                               // tensor copies: tokens, and whether slots lie within heads (set by the launch)
    float scale_log2;                                  // |scale| * log2(e), not 0 (inf * 0 is NaN)
    int flip;                                          // the scale is negative
};

struct AttnWorkspace {   // the status word lies at 0
    size_t counters, part_ml, part_o, total;
};
AttnWorkspace tree_attn_workspace(int head_dim);

// dtype 0 fp16, 1 bf16; max_rows: upper bound on a request's new tokens times the group (picks the row tile)
cudaError_t launch_tree_attn(const TreeAttnParams& p, int dtype, int max_rows, cudaStream_t st);
cudaError_t launch_tree_attn_f16(const TreeAttnParams& p, int max_rows, cudaStream_t st);
cudaError_t launch_tree_attn_bf16(const TreeAttnParams& p, int max_rows, cudaStream_t st);
cudaError_t launch_step_tables(const StepTablesParams& p, cudaStream_t st);
cudaError_t launch_store_kv(const StoreKvParams& p, cudaStream_t st);

}  // namespace dsv41
