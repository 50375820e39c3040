/*
 * dsv41_b200 -- C ABI of the B200 (sm_100a) routed-expert MoE FFN over EXL3 mul1 K=3 weights.
 *
 * Plain pointers and sizes only (no torch types). Every compute entry point is asynchronous on
 * the caller's CUDA stream (`stream` is a cudaStream_t passed as void*; NULL = legacy default
 * stream), allocates nothing, returns 0 on success or a negative DSV41_E* code, and leaves a
 * message for dsv41_last_error(). Kernels never trap: a device-side wait that runs out writes a
 * nonzero status word into the workspace, read back with dsv41_read_status().
 *
 * Reference interfaces replaced (paths inside the reference project 0xSero/dsv41-flash-offload):
 *   dsv41_moe_forward       apply_exl3_fused_moe(x2d, ids, weights, layer, inners, expert_map,
 *                           limit) -> out fp32 [T, H]: the routing prep
 *                           (patches/vllm-exl3-host-dma.patch:203-312) plus the
 *                           exllamav3_ext.exl3_moe launch contract (patch:315-449), and the
 *                           busy-expert path apply_exl3_batched_fat (patch:182-201) for experts
 *                           over fat_threshold rows; wrapped in the reference by
 *                           ct/ct_vllm.py:181-225 (_fused)
 *   dsv41_permute           the routing prep alone (patch:204-226, :300-312) and the split
 *                           kernel's histogram/compaction (ct/ft_tier_cu_v.cu:16-101, ft_split)
 *   dsv41_combine           the weighted accumulate of routed expert outputs into the fp32
 *                           layer output (ct/ft_tier_cu_v.cu:103-127 ft_combine;
 *                           kernels/cpu_avx2/ft_core.h:911-931)
 *   dsv41_decode_dense      the reconstruct step of the fat path / LinearEXL3.get_weight_tensor
 *                           (patch:182-201, pack/prepare_pack.py:64-65), restated from
 *                           kernels/cpu_avx2/ft_core.h:977-992 (dense_weights)
 *   dsv41_expert_gemm       runtime/dma_gemm.py:5-26 run_batch -> apply_exl3_batched_fat:
 *                           busy experts' reconstruct + GEMM, accumulated into out
 */
#ifndef DSV41_B200_H
#define DSV41_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DSV41_ABI_VERSION 2

enum {
    DSV41_OK = 0,
    DSV41_E_INVALID = -1,  /* bad argument / shape */
    DSV41_E_CUDA = -2,     /* CUDA runtime error (launch or attribute) */
    DSV41_E_WORKSPACE = -3 /* workspace too small */
};

enum { DSV41_DTYPE_F16 = 0, DSV41_DTYPE_BF16 = 1, DSV41_DTYPE_F32 = 2 };

/* One MoE layer's expert weights, all device pointers (vllm_exl3 Exl3MoEMethod layout,
 * patches/vllm-exl3-host-dma.patch:633-684 and its per-expert pointer tables, patch:66-69):
 *   gate_ptrs/up_ptrs [E]  int64 addresses of int16 trellis [H/16][I/16][16*bits] (48 at 3 bits)
 *   down_ptrs [E]          int64 addresses of int16 trellis [I/16][H/16][16*bits]
 *   w13_suh [E][2][H], w13_svh [E][2][I], w2_suh [E][I], w2_svh [E][H]  fp16
 * Every trellis address must be 16-byte aligned. H and I are multiples of 256. */
typedef struct dsv41_moe_layer {
    int32_t num_experts;
    int32_t hidden;
    int32_t intermediate;
    int32_t bits;       /* bits per weight K of every trellis tile: 2, 3 or 4 (0 = 3, the reference's build) */
    const int64_t* gate_ptrs;
    const int64_t* up_ptrs;
    const int64_t* down_ptrs;
    const void* w13_suh;
    const void* w13_svh;
    const void* w2_suh;
    const void* w2_svh;
} dsv41_moe_layer;

/* Options of one forward call.
 *   fat_threshold: experts with more than this many rows use the tensor-core grouped GEMM
 *                  (VLLM_EXL3_FAT_THRESHOLD, patch:146; 32 deployed); < 0 routes everything
 *                  through the decode GEMV.
 *   limit:         SwiGLU clamp (SWIGLU_LIMIT_DEFAULT 10.0, patch:5); 0 disables it.
 *   expert_map:    optional device int32 [map_len] global -> local expert id (-1 = not local),
 *                  as vLLM's expert_map; NULL = identity. */
typedef struct dsv41_moe_options {
    int32_t fat_threshold;
    float limit;
    const int32_t* expert_map;
    int32_t map_len;
    int32_t split_k;    /* 0 = automatic */
    int32_t max_routes; /* upper bound on routes with a valid local expert; row buffers are sized by it
                           (0 = T*topk). A call with more valid routes drops them all, writes zeros and
                           sets status 3 (see dsv41_read_status). Used by expert-parallel callers whose
                           rows carry mostly non-local route slots. */
} dsv41_moe_options;

/* Last error message of the calling thread ("" if none). */
const char* dsv41_last_error(void);
/* ABI version (DSV41_ABI_VERSION) and a build string. */
int dsv41_abi_version(void);
const char* dsv41_build_info(void);

/* Workspace bytes that dsv41_moe_forward needs for T tokens x topk routes. */
int dsv41_moe_workspace_size(int32_t T, int32_t topk, int32_t num_experts, int32_t hidden,
                             int32_t intermediate, const dsv41_moe_options* opt, size_t* bytes);

/* out[T][H] (fp32, overwritten) = sum over valid routes (t, j) of weights[t][j] * expert(x[t]).
 *   x [T][H] of x_dtype (cast to fp16 first, as the reference does), ids [T][topk] int64
 *   (negative or >= E = skipped), weights [T][topk] fp32. x and out must be 16-byte aligned and
 *   the workspace 256-byte aligned (DSV41_E_INVALID otherwise; device allocations are). */
int dsv41_moe_forward(const dsv41_moe_layer* layer, const void* x, int32_t x_dtype, int32_t T,
                      const int64_t* ids, const float* weights, int32_t topk,
                      const dsv41_moe_options* opt, float* out, void* workspace,
                      size_t workspace_bytes, void* stream);

/* dsv41_moe_forward for callers that cannot allocate device memory (no counterpart in the
 * reference). Same arguments and results as dsv41_moe_forward, minus the workspace: the scratch
 * is a fixed 32 MiB device array inside this library, held by every GPU that uses it until the
 * process exits. Requests needing more scratch than that fail with DSV41_E_WORKSPACE and a
 * message (at E=384 H=4096 I=2048 top-8 it covers decode batches up to 64 tokens). The first
 * call on a device looks the array up (make it before any stream capture); calls share the array,
 * so calls that overlap on the GPU race. Every argument is checked before anything is queued.
 * Allocates nothing. The status word of these calls lives in the array: read it with
 * dsv41_moe_noalloc_read_status, not dsv41_read_status. */
int dsv41_moe_forward_noalloc(const dsv41_moe_layer* layer, const void* x, int32_t x_dtype, int32_t T,
                              const int64_t* ids, const float* weights, int32_t topk,
                              const dsv41_moe_options* opt, float* out, void* stream);
/* dsv41_read_status for dsv41_moe_forward_noalloc on the current device (no counterpart in the
 * reference): synchronise `stream`, return the status word of the library's static scratch (0 = ok,
 * 1 = a bounded device wait ran out, 3 = more valid routes than options.max_routes) and clear it.
 * The next dsv41_moe_forward_noalloc call also clears it, so read it after each call you check. */
int dsv41_moe_noalloc_read_status(void* stream, int32_t* status);

/* Routing permutation (bit-exact, stable by (local expert, flat route index)):
 *   counts/offsets [E+1] int64 (index E = invalid-route sentinel), token_sorted/route_sorted
 *   [T*topk] int32, weight_sorted [T*topk] fp32, route_pos [T*topk] int32 (sorted position of
 *   each flat route, -1 when skipped). Any output pointer may be NULL. */
size_t dsv41_permute_workspace_size(int32_t T, int32_t topk, int32_t num_experts);
int dsv41_permute(const int64_t* ids, const float* weights, int32_t T, int32_t topk,
                  int32_t num_experts, const int32_t* expert_map, int32_t map_len,
                  int64_t* counts, int64_t* offsets, int32_t* token_sorted, float* weight_sorted,
                  int32_t* route_sorted, int32_t* route_pos, void* workspace,
                  size_t workspace_bytes, void* stream);

/* out[T][H] fp32 = sum_j weights[t][j] * y[route_pos[t*topk+j]][:] over route_pos >= 0;
 * y [rows][H] fp16. accumulate != 0 adds into out instead of overwriting it. */
int dsv41_combine(const void* y, const int32_t* route_pos, const float* weights, int32_t T,
                  int32_t topk, int32_t hidden, int32_t accumulate, float* out, void* stream);

/* Decode one trellis matrix [k/16][n/16][48] int16 into dense fp16 W [k][n] (bit-exact). */
int dsv41_decode_dense(const void* trellis, int32_t k, int32_t n, void* w_out, void* stream);
/* Same for K = bits per weight (2, 3 or 4): trellis [k/16][n/16][16*bits] int16 (the 2-bit packs
 * and 4-bit layers the reference's checkpoints also carry, patch:519-528, pack/prepare_pack.py:47). */
int dsv41_decode_dense_bits(const void* trellis, int32_t k, int32_t n, int32_t bits, void* w_out, void* stream);

/* Busy-expert GEMM path on pre-permuted rows (run_batch semantics): for each listed expert e
 * with counts[e] rows starting at offsets[e] of token_sorted/weight_sorted, out[token] +=
 * weight * expert_e(x[token]). experts [n_experts] int32 (device). */
int dsv41_expert_gemm(const dsv41_moe_layer* layer, const void* x, int32_t x_dtype, int32_t T,
                      const int32_t* experts, int32_t n_experts, const int64_t* counts,
                      const int64_t* offsets, const int32_t* token_sorted,
                      const float* weight_sorted, int32_t total_rows, float limit, float* out,
                      void* workspace, size_t workspace_bytes, void* stream);
int dsv41_expert_gemm_workspace_size(int32_t total_rows, int32_t n_experts, int32_t hidden,
                                     int32_t intermediate, size_t* bytes);

/* Synchronise `stream` and return the device status word of a workspace (0 = ok,
 * 1 = a bounded device wait ran out, 3 = more valid routes than options.max_routes), then clear it. */
int dsv41_read_status(const void* workspace, void* stream, int32_t* status);

/* Failure-detection self test (no counterpart entry in the reference; its combine kernel
 * ct/ft_tier_cu_v.cu:103-127 bounds its device spin the same way, by %globaltimer, and counts a
 * timeout in a stats word instead of trapping): launches one warp that waits
 * on a device barrier nothing ever completes, through the bounded wait every pipeline kernel uses;
 * after limit_us (1..2,000,000) it writes status 1 into the workspace's status word and returns.
 * Read it with dsv41_read_status; the stream and context stay usable. */
int dsv41_wait_selftest(void* workspace, uint32_t limit_us, void* stream);

/* Router top-k (no counterpart in the reference: vLLM's FusedMoE router produces topk_ids/weights before
 * apply_exl3_experts, patches/vllm-exl3-host-dma.patch:496-505). vLLM's two published rules:
 * scores = softmax(logits) over all experts, or sigmoid(logits); selection = scores (+ correction_bias
 * when given); with num_expert_group > 1 only the topk_group best groups compete (group score: sum
 * of its two best selection values with a bias, else its best); ids = top-k selection (ties: lower
 * id); weights = scores at ids, renormalised to sum 1 if `renormalize`, times routed_scaling_factor.
 * E <= 1024, topk <= 32. dsv41_moe_forward_logits = router + dsv41_moe_forward in one call (ids and
 * weights stay in the workspace unless ids_out/weights_out are given). */
enum { DSV41_ROUTER_SOFTMAX = 0, DSV41_ROUTER_SIGMOID = 1 };
typedef struct dsv41_router_options {
    int32_t scoring;                /* DSV41_ROUTER_SOFTMAX or DSV41_ROUTER_SIGMOID */
    int32_t renormalize;            /* nonzero: weights / sum(weights) over the k chosen */
    int32_t num_expert_group;       /* 0 or 1 = no grouping */
    int32_t topk_group;
    const float* correction_bias;   /* device [E] fp32 or NULL */
    float routed_scaling_factor;    /* 1.0 = none */
} dsv41_router_options;

int dsv41_router_topk(const void* logits, int32_t logits_dtype, int32_t T, int32_t num_experts, int32_t topk,
                      const dsv41_router_options* router, int64_t* ids, float* weights, void* stream);
int dsv41_moe_forward_logits(const dsv41_moe_layer* layer, const void* x, int32_t x_dtype, int32_t T,
                             const void* logits, int32_t logits_dtype, const dsv41_router_options* router, int32_t topk,
                             const dsv41_moe_options* opt, float* out, int64_t* ids_out, float* weights_out,
                             void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------
 * Expert parallelism over NVLink peer memory (no counterpart in the reference, which runs one GPU
 * with experts in host RAM, docker/entrypoint.sh:135-140). Experts are sharded: global expert e
 * lives on rank e / (num_global_experts / world). Each rank allocates one shared buffer
 * (dsv41_ep_peer_alloc: cudaMalloc + cudaIpcGetMemHandle), exchanges the 64-byte handles with its
 * peers over the host, opens theirs (dsv41_ep_peer_open) and fills bases[] (own buffer at
 * bases[rank]). dsv41_ep_peer_forward then runs one step of the layer for this rank's T <=
 * tokens_cap tokens with no collective library: the row transform reads each routed token row
 * from its rank (plain peer loads) and the down pass stores each expert output row into the
 * receive slot of its token's rank (plain peer stores), whose combine then sums its own slots;
 * step stamps in the shared buffers order the ranks (bounded waits, status 1 on expiry ->
 * dsv41_ep_peer_read_status). Every rank must call it once per step with the same
 * `step` sequence (0, 1, 2, ...), topk and tokens_cap. The buffers alternate by step parity, so a
 * CUDA graph of one step replays only for steps of the same parity. Hidden size up to 8192.
 * ------------------------------------------------------------------------------------------ */
#define DSV41_MAX_PEERS 8
#define DSV41_IPC_HANDLE_BYTES 64
typedef struct dsv41_ep_peer_group {
    int32_t rank, world;            /* world <= DSV41_MAX_PEERS */
    int32_t num_global_experts;     /* divisible by world */
    int32_t tokens_cap;             /* max tokens per rank and step (same on every rank) */
    void* bases[DSV41_MAX_PEERS];   /* device address of each rank's shared buffer in this process */
    int32_t wait_limit_us;          /* limit of each wait for the peers' step stamps, 1..2,000,000 us
                                       (0 = 2 s, the reference combine wait's bound); on expiry the
                                       step's exchange gives up with status 1 */
} dsv41_ep_peer_group;

int dsv41_ep_peer_buffer_size(const dsv41_ep_peer_group* group, const dsv41_moe_layer* local_layer, int32_t topk,
                              int32_t fat_threshold, size_t* bytes);
int dsv41_ep_peer_alloc(size_t bytes, void** base, void* ipc_handle);
int dsv41_ep_peer_open(const void* ipc_handle, void** peer_base);
int dsv41_ep_peer_close(void* peer_base);
int dsv41_ep_peer_free(void* base);
int dsv41_ep_peer_forward(const dsv41_moe_layer* local_layer, const dsv41_ep_peer_group* group, uint32_t step,
                          const void* x, int32_t x_dtype, int32_t T, const int64_t* ids, const float* weights,
                          int32_t topk, float limit, int32_t fat_threshold, float* out, void* stream);
int dsv41_ep_peer_read_status(const dsv41_ep_peer_group* group, const dsv41_moe_layer* local_layer, int32_t topk,
                              int32_t fat_threshold, void* stream, int32_t* status);

/* ------------------------------------------------------------------------------------------
 * A decode step with drafted tokens around the routed experts (no counterpart in the reference,
 * whose serving engine brings its own cache and attention): the page tables and slot maps of the
 * step, the store of the new keys and values, attention of the drafted tokens over the paged cache,
 * and products with 4-bit weights (projections, shared expert, head).
 *
 * A paged cache is [num_pages][page_size][kv_heads][head_dim] for keys and the same for values; slot
 * s is token s % page_size of page s / page_size. block_table[b][c] is the page of tokens
 * c * page_size .. of request b.
 * ------------------------------------------------------------------------------------------ */
#define DSV41_MAX_REQUESTS 2048
#define DSV41_MAX_MASK_WORDS 4

/* Status bits of one request after dsv41_step_tables. A refused request (NO_PAGES, TOO_WIDE) keeps the
 * pages it holds, gets seq_lens 0 and slots -1. */
enum {
    DSV41_TABLES_NO_PAGES = 1,   /* the free pages do not reach to it (requests are served in order) */
    DSV41_TABLES_TOO_WIDE = 2,   /* its pages exceed the table's width */
    DSV41_TABLES_BAD_PARENT = 4, /* a parent is not an earlier token of the request (taken as -1) */
    DSV41_TABLES_BIG_TREE = 8,   /* tokens past 64 * mask_words: they are in no mask */
    DSV41_TABLES_NO_ROOM = 16,   /* the stack has no room for the pages it would return: it keeps them, and is served */
    DSV41_TABLES_PAST_TOKENS = 32 /* its new tokens pass num_tokens: seq_lens 0, slots -1; its pages are exchanged */
};

/* Bring the pages of every request in line with its length. Request b has context_lens[b] tokens in the
 * cache, new_lens[b] new ones in this step and holds held_pages[b] pages, listed in its row of block_table.
 * It needs ceil((context + new) / page_size): surplus pages go back on the stack of free pages (in request
 * order; where the call would leave more on it than free_capacity, which a stack for every page of the pool never
 * meets, the first request whose pages do not fit and those behind it keep theirs), missing ones then come off its
 * top (in request order) into the row. Entries of a row past its
 * pages are stale. All pointers are device memory; num_tokens >= sum of new_lens (the caller knows it as
 * the length of the step's token batch; later entries get slot -1, position 0, request -1; a request whose tokens
 * pass it gets a status bit).
 * Outputs: cu_lens [batch + 1] running sums of new_lens; seq_lens [batch] = context + new; held_out [batch];
 * free_count_out [1]; status [batch]; per token: slots (int64), positions, requests (its b). Without
 * parents a token's position is context + its index; with parents ([num_tokens], index of the parent
 * within the request, -1 = the context) it is context + its depth, and tree_mask [num_tokens][mask_words]
 * holds a bit for each ancestor and itself. The outputs may not overlap the inputs. */
typedef struct dsv41_step_tables_args {
    int32_t batch, width, page_size, num_tokens;
    const int32_t* context_lens;
    const int32_t* new_lens;
    const int32_t* held_pages;
    int32_t* block_table;         /* [batch][table_stride], updated */
    int64_t table_stride;
    int32_t* free_pages;          /* [free_capacity], updated */
    const int32_t* free_count;    /* [1] */
    int32_t free_capacity;
    int32_t mask_words;           /* 1..DSV41_MAX_MASK_WORDS (with parents) */
    const int32_t* parents;       /* or NULL */
    int32_t* cu_lens;
    int32_t* seq_lens;
    int64_t* slots;
    int32_t* positions;
    int32_t* requests;
    int32_t* held_out;
    int32_t* free_count_out;
    int32_t* status;
    int64_t* tree_mask;           /* or NULL (without parents) */
} dsv41_step_tables_args;
int dsv41_step_tables(const dsv41_step_tables_args* args, void* stream);

/* cache[slots[t]] = k[t], v[t]; a slot outside the cache (-1) stores nothing. 16-bit elements; head_dim a
 * multiple of 8, addresses 16-byte aligned, strides (in elements) multiples of 8, the caches' not 0 (but for
 * dimensions of one). Slots that repeat within a call
 * leave one of their tokens, whichever. */
typedef struct dsv41_store_kv_args {
    int32_t num_tokens, kv_heads, head_dim, num_pages, page_size;
    const void* k;
    const void* v;
    int64_t k_stride_token, k_stride_head, v_stride_token, v_stride_head;
    const int64_t* slots;
    void* k_cache;
    void* v_cache;
    int64_t stride_page, stride_slot, stride_head;   /* of both caches */
} dsv41_store_kv_args;
int dsv41_store_kv(const dsv41_store_kv_args* args, void* stream);

/* out[t][hq] = softmax(scale * q . k) v over the keys that token t of its request sees. Request b owns rows
 * cu_lens[b] .. cu_lens[b + 1] - 1 of q, its keys are the first seq_lens[b] of its pages, the last of them its
 * new tokens. Token i sees the whole context and, with tree_mask, the new tokens of its bits; without, the
 * new tokens up to itself. Keys and values that a row does not see never reach it, whatever they hold. Infinite and NaN
 * values that it sees reach it as the definition has it: a weight is zero only where the score is -inf (0 * inf is
 * NaN). A row that sees nothing, or only scores of -inf, is 0 (lse -inf); so are the rows of a request with
 * seq_lens[b] < its new tokens or >
 * max_keys. Query head hq reads KV head hq / (q_heads / kv_heads). head_dim a multiple of 8 up to 256. dtype of q,
 * caches and out: fp16 or bf16. max_new: upper bound on a request's new tokens (a hint that picks the row
 * tile); num_tokens * q_heads up to 2^31 - 256. Addresses 16-byte aligned, strides (in elements) multiples of 8, those of
 * out not 0. lse [num_tokens][q_heads] (natural
 * logarithm of the sums) or NULL. The workspace is zeroed once after allocation; every call leaves its counters
 * zero. One workspace serves one call at a time (replays of a graph use the one it was captured with); its status
 * word is read with dsv41_read_status (1 = a bounded device wait ran out: zero the workspace before the next call). */
typedef struct dsv41_tree_attention_args {
    int32_t dtype, batch, num_tokens, max_new;
    int32_t q_heads, kv_heads, head_dim, page_size, num_pages, max_keys;
    const void* q;
    int64_t q_stride_token, q_stride_head;
    const void* k_cache;
    const void* v_cache;
    int64_t stride_page, stride_slot, stride_head;
    const int32_t* block_table;
    int64_t table_stride;
    const int32_t* seq_lens;
    const int32_t* cu_lens;
    const int64_t* tree_mask;     /* [num_tokens][mask_words] or NULL */
    int32_t mask_words;
    float scale;
    void* out;
    int64_t out_stride_token, out_stride_head;
    float* lse;
} dsv41_tree_attention_args;
int dsv41_tree_attention_workspace_size(int32_t head_dim, size_t* bytes);
int dsv41_tree_attention(const dsv41_tree_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);
/* The same through a window: of what a token sees without it, it sees the last `window` keys (itself counted, in the order
 * of the cache) and those at the first `sinks` positions of its request. window 0: all of them (sinks 0 then). With a window
 * seq_lens go up to 2^30. */
int dsv41_tree_attention_window(const dsv41_tree_attention_args* args, int32_t window, int32_t sinks, void* workspace,
                                size_t workspace_bytes, void* stream);

/* A cache in 4 bits: keys and values of num_pages pages of page_size tokens (a multiple of 8), kv_heads heads of head_dim
 * (a multiple of 32 up to 256). Columns come in groups of 32: with lo and hi the smallest and largest value of a token's group, T the type (fp16 or
 * bf16), s = T((hi - lo) / 15) (the next smaller number where T(lo + 15 s) would not be finite), code = round((x - lo) / s) in
 * 0..15, halves to even, 0 where s is 0, a code stands for T(lo + s code), rounded once. A group stands for NaN if one of its
 * values is not finite, or if hi - lo is not in fp32 (bf16 only: 3.4e38 or more from end to end, whatever lies between).
 * 20 bytes a group. Up to 2^31 - 1 records of 8 tokens of a head, page_size * kv_heads up to 2^24. data:
 * dsv41_kv4_cache_size bytes, 16-byte aligned, its layout the library's own ([page][head][keys, values], pages contiguous).
 * One cache holds one type: that of the calls that store into it. */
typedef struct dsv41_kv4_cache {
    int32_t num_pages, page_size, kv_heads, head_dim;
    void* data;
} dsv41_kv4_cache;
/* k, v: [num_tokens][kv_heads][head_dim], 16-byte aligned, strides (in elements) multiples of 8; slots as dsv41_store_kv's. */
typedef struct dsv41_kv4_tokens {
    int32_t dtype, num_tokens;
    void* k;
    void* v;
    int64_t k_stride_token, k_stride_head, v_stride_token, v_stride_head;
    const int64_t* slots;
} dsv41_kv4_tokens;
int dsv41_kv4_cache_size(int32_t num_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, size_t* bytes);
/* store: k and v into the tokens' slots; a slot outside the cache stores nothing. A slot may not come twice in a call (its
 * codes and scales could be of different tokens). load: what the slots stand for into k and v (strides not 0), zeros for a slot
 * outside. move: the codes of from[t] to to[t] as they are, all read before any is written (a slot may be in both; none twice
 * in `to`); nothing where either lies outside. room: num_tokens * kv_heads * head_dim / 32 * 40 bytes, 16-byte aligned. */
int dsv41_kv4_store(const dsv41_kv4_cache* cache, const dsv41_kv4_tokens* tokens, void* stream);
int dsv41_kv4_load(const dsv41_kv4_cache* cache, const dsv41_kv4_tokens* tokens, void* stream);
int dsv41_kv4_move(const dsv41_kv4_cache* cache, const int64_t* from, const int64_t* to, int32_t num_tokens, void* room, size_t room_bytes,
                   void* stream);
/* dsv41_tree_attention_window over a cache in 4 bits: k_cache, v_cache and their strides are not read, kv_heads, head_dim,
 * page_size and num_pages are the cache's, dtype is that of q, out and the cache. The same workspaces. seq_lens go up to 2^30. */
int dsv41_tree_attention4(const dsv41_tree_attention_args* args, const dsv41_kv4_cache* cache, int32_t window, int32_t sinks, void* workspace,
                          size_t workspace_bytes, void* stream);

/* 4-bit weights: w[n][k] = scale[n][k / group] * (code - zero[n][k / group]), codes 0..15, zero points
 * 0..15 (8 where there are none), groups of 32, 64 or 128 inputs, k a multiple of the group, any n.
 * dsv41_w4_pack lays a matrix out once: codes [n][k / 2] uint8 (even k in the low nibble), scales
 * [n][k / group] fp16 or bf16, zeros [n][k / group] uint8 or NULL -> data, dsv41_w4_layout_size bytes. */
typedef struct dsv41_w4_weight {
    int32_t n, k, group;
    int32_t has_zeros;
    int32_t scale_dtype;          /* DSV41_DTYPE_F16 or DSV41_DTYPE_BF16 */
    const void* data;
} dsv41_w4_weight;
int dsv41_w4_layout_size(int32_t n, int32_t k, int32_t group, int32_t has_zeros, size_t* bytes);
int dsv41_w4_pack(const void* codes, const void* scales, const void* zeros, int32_t n, int32_t k, int32_t group,
                  void* data, size_t data_bytes, void* stream);
/* out[t][n] = sum_k w[n][k] x[t][k], fp32 sums, x fp16 or bf16 [tokens][x_stride] (16-byte aligned, x_stride a
 * multiple of 8), out fp32, fp16 or bf16 [tokens][out_stride]; accumulate (fp32 out only) adds into out. */
int dsv41_w4_linear(const dsv41_w4_weight* w, const void* x, int32_t x_dtype, int64_t x_stride, int32_t tokens,
                    void* out, int32_t out_dtype, int64_t out_stride, int32_t accumulate, void* stream);
/* out[t][n] = min(silu(g), limit) * clamp(u, -limit, limit) with g, u the products with gate and up (same n,
 * k, group, scale type, both or neither with zero points); limit 0 = no clamp (the routed experts' SwiGLU).
 * NaN products give NaN, and so does a gate of -inf (its silu is -inf / inf). */
int dsv41_w4_gated(const dsv41_w4_weight* gate, const dsv41_w4_weight* up, const void* x, int32_t x_dtype,
                   int64_t x_stride, int32_t tokens, float limit, void* out, int32_t out_dtype, int64_t out_stride,
                   void* stream);

/* Scores of rows of logits [rows][row_stride] (fp16, bf16 or fp32; any stride in elements, rows need no alignment beyond
 * their type's). Per row, with p the softmax of its vocab logits: logprobs[given] = log p of the given tokens (-inf for
 * one outside 0..vocab - 1), entropy = -sum p log p, lse = log of the sum of exponentials, and the `top` tokens
 * with the largest logits in descending order, equal ones by the lowest index, with their log p. Tokens with a logit
 * of -inf are no alternatives: places that find none hold id -1 and -inf. A row of -inf alone: -inf, entropy 0, lse
 * -inf. A row that holds NaN or +inf has no distribution: NaN throughout, ids -1. */
enum { DSV41_MAX_TOP = 32, DSV41_MAX_GIVEN = 1024 };
typedef struct dsv41_token_logprobs_args {
    int32_t dtype, rows, vocab, given, top;
    const void* logits;
    int64_t row_stride;
    const int64_t* tokens;        /* [rows][given] */
    float* logprobs;              /* [rows][given] */
    float* entropy;               /* [rows] */
    float* lse;                   /* [rows] */
    int64_t* top_ids;             /* [rows][top] */
    float* top_logprobs;          /* [rows][top] */
} dsv41_token_logprobs_args;
int dsv41_token_logprobs(const dsv41_token_logprobs_args* args, void* stream);

/* Profiling (no counterpart in the reference; used by bench.py to time each kernel on the stream
 * it runs on). While enabled, dsv41_moe_forward records CUDA events at its stage boundaries for up
 * to DSV41_TIMING_MAX_CALLS calls (not under stream capture). dsv41_read_stage_times synchronises
 * them and writes DSV41_N_STAGES times in ms per recorded call, in the order permute, row prep,
 * decode-GEMV (both passes, one launch, when split_k is 1), gate/up GEMM, down decode-GEMV (its own
 * launch when split_k > 1, else empty), down GEMM, combine; then it forgets them. */
#define DSV41_N_STAGES 7
#define DSV41_TIMING_MAX_CALLS 256
int dsv41_set_stage_timing(int32_t enable);
int dsv41_read_stage_times(float* ms, int32_t max_calls, int32_t* n_calls);

#ifdef __cplusplus
}
#endif
#endif /* DSV41_B200_H */
