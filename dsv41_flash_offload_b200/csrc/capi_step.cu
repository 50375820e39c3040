// C ABI of the operators of a drafted decode step around the routed experts (declared in
// include/dsv41_b200.h): argument checks, then one launch each on the caller's stream.
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/dsv41_b200.h"
#include "internal.h"
#include "paged.h"
#include "w4.h"

namespace dsv41 {

static_assert(kMaxRequests == DSV41_MAX_REQUESTS && kMaxMaskWords == DSV41_MAX_MASK_WORDS, "header limits");
static_assert(kTabNoPages == DSV41_TABLES_NO_PAGES && kTabTooWide == DSV41_TABLES_TOO_WIDE &&
                  kTabBadParent == DSV41_TABLES_BAD_PARENT && kTabBigTree == DSV41_TABLES_BIG_TREE &&
                  kTabNoRoom == DSV41_TABLES_NO_ROOM && kTabPastTokens == DSV41_TABLES_PAST_TOKENS, "header status bits");

static bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// a dimension whose entries are all one place
static bool repeats(int64_t stride, int extent) { return stride == 0 && extent > 1; }

static int launched(cudaError_t err, const char* what)
{
    if (err == cudaSuccess) return DSV41_OK;
    return set_error(DSV41_E_CUDA, "%s: %s (%s)", what, cudaGetErrorString(err), cudaGetErrorName(err));
}

static int check_weight(const dsv41_w4_weight* w, const char* name)
{
    if (!w) return set_error(DSV41_E_INVALID, "%s weight is NULL", name);
    if (w->n <= 0 || w->k <= 0) return set_error(DSV41_E_INVALID, "%s weight n=%d k=%d", name, w->n, w->k);
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return set_error(DSV41_E_INVALID, "%s weight group %d (32, 64 or 128)", name, w->group);
    if ((int64_t)(w->n / 16 + 1) * (w->k / 128 + 1) > 0x7fffffffll) return set_error(DSV41_E_INVALID, "%s weight n=%d k=%d is too large", name, w->n, w->k);
    if (w->k % w->group) return set_error(DSV41_E_INVALID, "%s weight k=%d is not a multiple of its group %d", name, w->k, w->group);
    if (w->scale_dtype != DSV41_DTYPE_F16 && w->scale_dtype != DSV41_DTYPE_BF16)
        return set_error(DSV41_E_INVALID, "%s weight scales must be fp16 or bf16", name);
    if (!w->data || !aligned(w->data, 256)) return set_error(DSV41_E_INVALID, "%s weight data must be 256-byte aligned", name);
    return DSV41_OK;
}

static W4Mat w4_mat(const dsv41_w4_weight& w)
{
    const W4Layout l = W4Layout::make(w.n, w.k, w.group, w.has_zeros != 0);
    const unsigned char* d = static_cast<const unsigned char*>(w.data);
    W4Mat m;
    m.codes = reinterpret_cast<const uint4*>(d);
    m.scales = reinterpret_cast<const uint32_t*>(d + l.scales_off);
    m.zeros = w.has_zeros ? reinterpret_cast<const uint16_t*>(d + l.zeros_off) : nullptr;
    return m;
}

static int w4_run(const dsv41_w4_weight* a, const dsv41_w4_weight* b, const void* x, int x_dtype, int64_t x_stride,
                  int tokens, float limit, void* out, int out_dtype, int64_t out_stride, int accumulate, void* stream)
{
    int rc = check_weight(a, b ? "gate" : "4-bit");
    if (rc) return rc;
    if (b) {
        if ((rc = check_weight(b, "up"))) return rc;
        if (b->n != a->n || b->k != a->k || b->group != a->group || b->scale_dtype != a->scale_dtype ||
            !b->has_zeros != !a->has_zeros)
            return set_error(DSV41_E_INVALID, "gate and up differ in size, group, zero points or scale type");
    }
    if (x_dtype != DSV41_DTYPE_F16 && x_dtype != DSV41_DTYPE_BF16)
        return set_error(DSV41_E_INVALID, "x dtype %d (fp16 or bf16)", x_dtype);
    if (out_dtype < DSV41_DTYPE_F16 || out_dtype > DSV41_DTYPE_F32) return set_error(DSV41_E_INVALID, "out dtype %d", out_dtype);
    if (accumulate && out_dtype != DSV41_DTYPE_F32) return set_error(DSV41_E_INVALID, "accumulate needs an fp32 out");
    if (tokens < 0 || tokens > 65535 * 8) return set_error(DSV41_E_INVALID, "tokens=%d (0..%d)", tokens, 65535 * 8);
    if (tokens == 0) return DSV41_OK;
    if (!x || !out) return set_error(DSV41_E_INVALID, "NULL pointer");
    if (x_stride < a->k || x_stride % 8 || out_stride < a->n)
        return set_error(DSV41_E_INVALID, "x_stride %lld (>= k, a multiple of 8), out_stride %lld (>= n)", (long long)x_stride, (long long)out_stride);
    if (!aligned(x, 16)) return set_error(DSV41_E_INVALID, "x must be 16-byte aligned");
    if (!aligned(out, out_dtype == DSV41_DTYPE_F32 ? 4 : 2)) return set_error(DSV41_E_INVALID, "out is misaligned");
    if (!std::isfinite(limit) || limit < 0.0f) return set_error(DSV41_E_INVALID, "limit %g", limit);
    const W4Layout l = W4Layout::make(a->n, a->k, a->group, false);
    W4Params p{};
    p.a = w4_mat(*a);
    if (b) p.b = w4_mat(*b);
    p.x = x;
    p.out = out;
    p.x_stride = x_stride;
    p.out_stride = out_stride;
    p.tokens = tokens;
    p.n = a->n;
    p.k = a->k;
    p.n16 = l.n16;
    p.k128 = l.k128;
    p.scale_bf16 = a->scale_dtype == DSV41_DTYPE_BF16;
    p.out_dtype = out_dtype;
    p.accumulate = accumulate;
    p.limit = limit;
    return launched(launch_w4(p, x_dtype, a->group, b != nullptr, static_cast<cudaStream_t>(stream)), "4-bit product");
}

}  // namespace dsv41

using namespace dsv41;

extern "C" {

int dsv41_step_tables(const dsv41_step_tables_args* a, void* stream)
{
    if (!a) return set_error(DSV41_E_INVALID, "args is NULL");
    if (a->batch < 1 || a->batch > kMaxRequests) return set_error(DSV41_E_INVALID, "batch=%d (1..%d)", a->batch, kMaxRequests);
    if (a->width < 1 || a->table_stride < a->width || (int64_t)a->batch * a->width > 0x7fffffffll)
        return set_error(DSV41_E_INVALID, "block table of %d columns, stride %lld", a->width, (long long)a->table_stride);
    if (a->page_size < 1) return set_error(DSV41_E_INVALID, "page_size=%d", a->page_size);
    if (a->num_tokens < 0) return set_error(DSV41_E_INVALID, "num_tokens=%d", a->num_tokens);
    if (a->free_capacity < 0) return set_error(DSV41_E_INVALID, "free_capacity=%d", a->free_capacity);
    if (!a->context_lens || !a->new_lens || !a->held_pages || !a->block_table || !a->free_count || !a->cu_lens ||
        !a->seq_lens || !a->held_out || !a->free_count_out || !a->status || (a->free_capacity && !a->free_pages) ||
        (a->num_tokens && (!a->slots || !a->positions || !a->requests)))
        return set_error(DSV41_E_INVALID, "NULL pointer");
    if (a->held_out == a->held_pages || a->free_count_out == a->free_count)
        return set_error(DSV41_E_INVALID, "an output overlaps its input");
    if (!aligned(a->slots, 8) || !aligned(a->positions, 4) || !aligned(a->requests, 4))
        return set_error(DSV41_E_INVALID, "slots, positions or requests are misaligned");
    if (a->parents) {
        if (a->mask_words < 1 || a->mask_words > kMaxMaskWords)
            return set_error(DSV41_E_INVALID, "mask_words=%d (1..%d)", a->mask_words, kMaxMaskWords);
        if (a->num_tokens && !a->tree_mask) return set_error(DSV41_E_INVALID, "parents without tree_mask");
    }
    StepTablesParams p{};
    p.context_lens = a->context_lens;
    p.new_lens = a->new_lens;
    p.held_pages = a->held_pages;
    p.block_table = a->block_table;
    p.table_stride = a->table_stride;
    p.free_pages = a->free_pages;
    p.free_count = a->free_count;
    p.batch = a->batch;
    p.width = a->width;
    p.free_capacity = a->free_capacity;
    p.page_size = a->page_size;
    p.num_tokens = a->num_tokens;
    p.mask_words = a->mask_words;
    p.parents = a->parents;
    p.cu_lens = a->cu_lens;
    p.seq_lens = a->seq_lens;
    p.slots = a->slots;
    p.positions = a->positions;
    p.requests = a->requests;
    p.held_out = a->held_out;
    p.free_count_out = a->free_count_out;
    p.status = a->status;
    p.tree_mask = a->tree_mask;
    return launched(launch_step_tables(p, static_cast<cudaStream_t>(stream)), "step tables");
}

int dsv41_store_kv(const dsv41_store_kv_args* a, void* stream)
{
    if (!a) return set_error(DSV41_E_INVALID, "args is NULL");
    if (a->num_tokens < 0 || a->kv_heads < 1 || a->head_dim < 8 || a->head_dim % 8)
        return set_error(DSV41_E_INVALID, "num_tokens=%d kv_heads=%d head_dim=%d (a multiple of 8)", a->num_tokens, a->kv_heads, a->head_dim);
    if (a->num_pages < 0 || a->page_size < 1) return set_error(DSV41_E_INVALID, "num_pages=%d page_size=%d", a->num_pages, a->page_size);
    if (a->num_tokens == 0) return DSV41_OK;
    if (!a->k || !a->v || !a->slots || !a->k_cache || !a->v_cache) return set_error(DSV41_E_INVALID, "NULL pointer");
    if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16))
        return set_error(DSV41_E_INVALID, "k, v and the caches must be 16-byte aligned");
    const int64_t strides[] = {a->k_stride_token, a->k_stride_head, a->v_stride_token, a->v_stride_head,
                               a->stride_page, a->stride_slot, a->stride_head};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(DSV41_E_INVALID, "stride %lld is not a multiple of 8 elements", (long long)s);
    if (repeats(a->stride_page, a->num_pages) || repeats(a->stride_slot, a->page_size) || repeats(a->stride_head, a->kv_heads))
        return set_error(DSV41_E_INVALID, "the caches repeat in memory: a stride of 0 cannot be stored through");
    StoreKvParams p{};
    p.k = a->k;
    p.v = a->v;
    p.k_stride_token = a->k_stride_token;
    p.k_stride_head = a->k_stride_head;
    p.v_stride_token = a->v_stride_token;
    p.v_stride_head = a->v_stride_head;
    p.slots = a->slots;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.stride_page = a->stride_page;
    p.stride_slot = a->stride_slot;
    p.stride_head = a->stride_head;
    p.num_tokens = a->num_tokens;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.num_pages = a->num_pages;
    p.page_size = a->page_size;
    return launched(launch_store_kv(p, static_cast<cudaStream_t>(stream)), "store of keys and values");
}

int dsv41_tree_attention_workspace_size(int32_t head_dim, size_t* bytes)
{
    if (!bytes) return set_error(DSV41_E_INVALID, "bytes is NULL");
    if (head_dim < 8 || head_dim > 256 || head_dim % 8)
        return set_error(DSV41_E_INVALID, "head_dim=%d (a multiple of 8 up to 256)", head_dim);
    *bytes = tree_attn_workspace(head_dim).total;
    return DSV41_OK;
}

int dsv41_tree_attention(const dsv41_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!a) return set_error(DSV41_E_INVALID, "args is NULL");
    size_t need = 0;
    int rc = dsv41_tree_attention_workspace_size(a->head_dim, &need);
    if (rc) return rc;
    if (a->dtype != DSV41_DTYPE_F16 && a->dtype != DSV41_DTYPE_BF16)
        return set_error(DSV41_E_INVALID, "dtype %d (fp16 or bf16)", a->dtype);
    if (a->batch < 1 || a->batch > kMaxRequests) return set_error(DSV41_E_INVALID, "batch=%d (1..%d)", a->batch, kMaxRequests);
    if (a->num_tokens < 0 || a->max_new < 0) return set_error(DSV41_E_INVALID, "num_tokens=%d max_new=%d", a->num_tokens, a->max_new);
    if (a->kv_heads < 1 || a->q_heads < a->kv_heads || a->q_heads % a->kv_heads)
        return set_error(DSV41_E_INVALID, "q_heads=%d is not a multiple of kv_heads=%d", a->q_heads, a->kv_heads);
    // the kernel counts a request's rows and rounds them up to whole tiles in 32 bits
    if ((int64_t)a->num_tokens * a->q_heads > 0x7fffffffll - 255)
        return set_error(DSV41_E_INVALID, "num_tokens * q_heads over 2^31 - 256");
    if (a->page_size < 1 || a->num_pages < 0 || a->max_keys < 0)
        return set_error(DSV41_E_INVALID, "page_size=%d num_pages=%d max_keys=%d", a->page_size, a->num_pages, a->max_keys);
    if (a->max_keys > 0x7fffff00) return set_error(DSV41_E_INVALID, "max_keys=%d", a->max_keys);
    if (a->num_tokens == 0) return DSV41_OK;
    if (!a->q || !a->k_cache || !a->v_cache || !a->block_table || !a->seq_lens || !a->cu_lens || !a->out || !workspace)
        return set_error(DSV41_E_INVALID, "NULL pointer");
    if (a->tree_mask && (a->mask_words < 1 || a->mask_words > kMaxMaskWords))
        return set_error(DSV41_E_INVALID, "mask_words=%d (1..%d)", a->mask_words, kMaxMaskWords);
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16))
        return set_error(DSV41_E_INVALID, "q, out and the caches must be 16-byte aligned");
    if (!aligned(workspace, 256)) return set_error(DSV41_E_INVALID, "the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return set_error(DSV41_E_WORKSPACE, "workspace %zu bytes < required %zu", workspace_bytes, need);
    const int64_t strides[] = {a->q_stride_token, a->q_stride_head, a->out_stride_token, a->out_stride_head,
                               a->stride_page, a->stride_slot, a->stride_head};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(DSV41_E_INVALID, "stride %lld is not a multiple of 8 elements", (long long)s);
    if (repeats(a->out_stride_token, a->num_tokens) || repeats(a->out_stride_head, a->q_heads))
        return set_error(DSV41_E_INVALID, "out repeats in memory: a stride of 0 cannot be written through");
    if (!std::isfinite(a->scale)) return set_error(DSV41_E_INVALID, "scale %g", a->scale);
    TreeAttnParams p{};
    p.q = a->q;
    p.q_stride_token = a->q_stride_token;
    p.q_stride_head = a->q_stride_head;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.stride_page = a->stride_page;
    p.stride_slot = a->stride_slot;
    p.stride_head = a->stride_head;
    p.block_table = a->block_table;
    p.table_stride = a->table_stride;
    p.seq_lens = a->seq_lens;
    p.cu_lens = a->cu_lens;
    p.tree_mask = a->tree_mask;
    p.out = a->out;
    p.out_stride_token = a->out_stride_token;
    p.out_stride_head = a->out_stride_head;
    p.lse = a->lse;
    const AttnWorkspace w = tree_attn_workspace(a->head_dim);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    p.status = reinterpret_cast<int*>(ws);
    p.counters = reinterpret_cast<int*>(ws + w.counters);
    p.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
    p.part_o = reinterpret_cast<float*>(ws + w.part_o);
    p.batch = a->batch;
    p.num_tokens = a->num_tokens;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.group = a->q_heads / a->kv_heads;
    p.head_dim = a->head_dim;
    p.page_size = a->page_size;
    p.num_pages = a->num_pages;
    p.max_keys = a->max_keys;
    p.mask_words = a->mask_words;
    p.page_div = FastDiv::make(a->page_size);
    p.group_div = FastDiv::make(p.group);
    // a scale of 0 (every key counts alike) becomes one that no score survives
    p.scale_log2 = std::fmax(std::fabs(a->scale) * 1.4426950408889634f, 1e-37f);
    p.flip = a->scale < 0.0f;
    const int64_t rows = (int64_t)(a->max_new ? a->max_new : 1) * p.group;
    return launched(launch_tree_attn(p, a->dtype, (int)(rows > 1024 ? 1024 : rows), static_cast<cudaStream_t>(stream)),
                    "tree attention");
}

int dsv41_w4_layout_size(int32_t n, int32_t k, int32_t group, int32_t has_zeros, size_t* bytes)
{
    if (!bytes) return set_error(DSV41_E_INVALID, "bytes is NULL");
    if (n <= 0 || k <= 0 || (group != 32 && group != 64 && group != 128) || k % group)
        return set_error(DSV41_E_INVALID, "n=%d k=%d group=%d (k a multiple of a group of 32, 64 or 128)", n, k, group);
    *bytes = W4Layout::make(n, k, group, has_zeros != 0).total;
    return DSV41_OK;
}

int dsv41_w4_pack(const void* codes, const void* scales, const void* zeros, int32_t n, int32_t k, int32_t group,
                  void* data, size_t data_bytes, void* stream)
{
    size_t need = 0;
    int rc = dsv41_w4_layout_size(n, k, group, zeros != nullptr, &need);
    if (rc) return rc;
    if (!codes || !scales || !data) return set_error(DSV41_E_INVALID, "NULL pointer");
    if (!aligned(scales, 2) || !aligned(data, 256)) return set_error(DSV41_E_INVALID, "scales or data is misaligned");
    if (data_bytes < need) return set_error(DSV41_E_WORKSPACE, "data %zu bytes < required %zu", data_bytes, need);
    return launched(launch_w4_pack(static_cast<const uint8_t*>(codes), static_cast<const uint16_t*>(scales),
                                   static_cast<const uint8_t*>(zeros), n, k, group, data, static_cast<cudaStream_t>(stream)),
                    "4-bit layout");
}

int dsv41_w4_linear(const dsv41_w4_weight* w, const void* x, int32_t x_dtype, int64_t x_stride, int32_t tokens,
                    void* out, int32_t out_dtype, int64_t out_stride, int32_t accumulate, void* stream)
{
    return w4_run(w, nullptr, x, x_dtype, x_stride, tokens, 0.0f, out, out_dtype, out_stride, accumulate, stream);
}

int dsv41_w4_gated(const dsv41_w4_weight* gate, const dsv41_w4_weight* up, const void* x, int32_t x_dtype,
                   int64_t x_stride, int32_t tokens, float limit, void* out, int32_t out_dtype, int64_t out_stride,
                   void* stream)
{
    if (!up) return set_error(DSV41_E_INVALID, "up weight is NULL");
    return w4_run(gate, up, x, x_dtype, x_stride, tokens, limit, out, out_dtype, out_stride, 0, stream);
}

}  // extern "C"
