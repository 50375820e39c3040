// C ABI of the operators of a drafted decode step around the routed experts (declared in
// include/dsv41_b200.h): argument checks, then one launch each on the caller's stream.
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/dsv41_b200.h"
#include "internal.h"
#include "kv4.cuh"
#include "logprobs.h"
#include "paged.h"
#include "w4.h"

namespace dsv41 {

static_assert(kMaxRequests == DSV41_MAX_REQUESTS && kMaxMaskWords == DSV41_MAX_MASK_WORDS, "header limits");
static_assert(kTabNoPages == DSV41_TABLES_NO_PAGES && kTabTooWide == DSV41_TABLES_TOO_WIDE &&
                  kTabBadParent == DSV41_TABLES_BAD_PARENT && kTabBigTree == DSV41_TABLES_BIG_TREE &&
                  kTabNoRoom == DSV41_TABLES_NO_ROOM && kTabPastTokens == DSV41_TABLES_PAST_TOKENS, "header status bits");
static_assert(kMaxTop == DSV41_MAX_TOP && kMaxGiven == DSV41_MAX_GIVEN, "header limits");

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

static int check_window(int window, int sinks)
{
    if (window < 0 || sinks < 0) return set_error(DSV41_E_INVALID, "window=%d (0: none) sinks=%d", window, sinks);
    if (sinks && !window) return set_error(DSV41_E_INVALID, "sinks=%d without a window", sinks);
    return DSV41_OK;
}
static void set_window(TreeAttnParams& p, int window, int sinks)
{
    p.window = window > 0 && window < kNoWindow ? window : kNoWindow;
    p.sinks = p.window < kNoWindow ? sinks : 0;
    // (positions are taken against the window: no request is longer than "none" reaches)
    if ((window || p.packed) && p.max_keys > kNoWindow) p.max_keys = kNoWindow;
}

// checks of an attention call and the kernel's parameters; cache: in 4 bits, instead of k_cache and v_cache
static int attn_params(TreeAttnParams& p, const dsv41_tree_attention_args* a, const dsv41_kv4_cache* cache, int window, int sinks, void* workspace,
                       size_t workspace_bytes, bool* run)
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
    if ((rc = check_window(window, sinks))) return rc;
    if (a->max_keys > 0x7fffff00) return set_error(DSV41_E_INVALID, "max_keys=%d", a->max_keys);
    *run = a->num_tokens > 0;
    if (!*run) return DSV41_OK;
    if (!a->q || (!cache && (!a->k_cache || !a->v_cache)) || !a->block_table || !a->seq_lens || !a->cu_lens || !a->out || !workspace)
        return set_error(DSV41_E_INVALID, "NULL pointer");
    if (a->tree_mask && (a->mask_words < 1 || a->mask_words > kMaxMaskWords))
        return set_error(DSV41_E_INVALID, "mask_words=%d (1..%d)", a->mask_words, kMaxMaskWords);
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || (!cache && (!aligned(a->k_cache, 16) || !aligned(a->v_cache, 16))))
        return set_error(DSV41_E_INVALID, "q, out and the caches must be 16-byte aligned");
    if (!aligned(workspace, 256)) return set_error(DSV41_E_INVALID, "the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return set_error(DSV41_E_WORKSPACE, "workspace %zu bytes < required %zu", workspace_bytes, need);
    const int64_t strides[] = {a->q_stride_token, a->q_stride_head, a->out_stride_token, a->out_stride_head,
                               cache ? 0 : a->stride_page, cache ? 0 : a->stride_slot, cache ? 0 : a->stride_head};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(DSV41_E_INVALID, "stride %lld is not a multiple of 8 elements", (long long)s);
    if (repeats(a->out_stride_token, a->num_tokens) || repeats(a->out_stride_head, a->q_heads))
        return set_error(DSV41_E_INVALID, "out repeats in memory: a stride of 0 cannot be written through");
    if (!std::isfinite(a->scale)) return set_error(DSV41_E_INVALID, "scale %g", a->scale);
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
    // (a cache without pages: what its keys are read from and thrown away has to exist)
    p.packed = !cache ? nullptr : cache->num_pages ? static_cast<const unsigned char*>(cache->data) : ws;
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
    set_window(p, window, sinks);
    return DSV41_OK;
}
// upper bound on a request's rows (picks the row tile)
static int attn_rows(const dsv41_tree_attention_args* a)
{
    const int64_t rows = (int64_t)(a->max_new ? a->max_new : 1) * (a->q_heads / a->kv_heads);
    return (int)(rows > 1024 ? 1024 : rows);
}

static int check_kv4(const dsv41_kv4_cache* c, bool data)
{
    if (!c) return set_error(DSV41_E_INVALID, "cache is NULL");
    if (c->num_pages < 0 || c->kv_heads < 1) return set_error(DSV41_E_INVALID, "num_pages=%d kv_heads=%d", c->num_pages, c->kv_heads);
    if (c->page_size < kKv4Tokens || c->page_size % kKv4Tokens)
        return set_error(DSV41_E_INVALID, "page_size=%d (a multiple of %d for a cache in 4 bits)", c->page_size, kKv4Tokens);
    if (c->head_dim < kKv4Chunk || c->head_dim > 256 || c->head_dim % kKv4Chunk)
        return set_error(DSV41_E_INVALID, "head_dim=%d (a multiple of %d up to 256 for a cache in 4 bits)", c->head_dim, kKv4Chunk);
    if ((int64_t)c->page_size * c->kv_heads > (1 << 24)) return set_error(DSV41_E_INVALID, "pages of %d tokens and %d heads", c->page_size, c->kv_heads);
    if ((int64_t)c->num_pages * c->kv_heads * 2 * (c->page_size / kKv4Tokens) > 0x7fffffffll)
        return set_error(DSV41_E_INVALID, "num_pages=%d: over 2^31 - 1 records of %d tokens", c->num_pages, kKv4Tokens);
    if (data && c->num_pages && (!c->data || !aligned(c->data, 16))) return set_error(DSV41_E_INVALID, "the cache's data must be 16-byte aligned");
    return DSV41_OK;
}
static void kv4_cache(Kv4Params& p, const dsv41_kv4_cache* c)
{
    p.data = static_cast<unsigned char*>(c->data);
    p.num_pages = c->num_pages;
    p.page_size = c->page_size;
    p.kv_heads = c->kv_heads;
    p.chunks = c->head_dim / kKv4Chunk;
    p.page_div = FastDiv::make(c->page_size);
    p.few_slots = (int64_t)c->num_pages * c->page_size <= 0x7fffffffll;
}
static int kv4_params(Kv4Params& p, const dsv41_kv4_cache* c, const dsv41_kv4_tokens* a)
{
    const int rc = check_kv4(c, true);
    if (rc) return rc;
    if (!a) return set_error(DSV41_E_INVALID, "tokens is NULL");
    if (a->dtype != DSV41_DTYPE_F16 && a->dtype != DSV41_DTYPE_BF16) return set_error(DSV41_E_INVALID, "dtype %d (fp16 or bf16)", a->dtype);
    if (a->num_tokens < 0) return set_error(DSV41_E_INVALID, "num_tokens=%d", a->num_tokens);
    if (a->num_tokens == 0) return DSV41_OK;
    if (!a->k || !a->v || !a->slots) return set_error(DSV41_E_INVALID, "NULL pointer");
    if (!aligned(a->k, 16) || !aligned(a->v, 16)) return set_error(DSV41_E_INVALID, "k and v must be 16-byte aligned");
    const int64_t strides[] = {a->k_stride_token, a->k_stride_head, a->v_stride_token, a->v_stride_head};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(DSV41_E_INVALID, "stride %lld is not a multiple of 8 elements", (long long)s);
    kv4_cache(p, c);
    p.k = a->k;
    p.v = a->v;
    p.k_stride_token = a->k_stride_token;
    p.k_stride_head = a->k_stride_head;
    p.v_stride_token = a->v_stride_token;
    p.v_stride_head = a->v_stride_head;
    p.slots = a->slots;
    p.num_tokens = a->num_tokens;
    return DSV41_OK;
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
    return dsv41_tree_attention_window(a, 0, 0, workspace, workspace_bytes, stream);
}

int dsv41_tree_attention_window(const dsv41_tree_attention_args* a, int32_t window, int32_t sinks, void* workspace, size_t workspace_bytes,
                                void* stream)
{
    TreeAttnParams p{};
    bool run = false;
    const int rc = attn_params(p, a, nullptr, window, sinks, workspace, workspace_bytes, &run);
    if (rc || !run) return rc;
    return launched(launch_tree_attn(p, a->dtype, attn_rows(a), static_cast<cudaStream_t>(stream)), "tree attention");
}

int dsv41_kv4_cache_size(int32_t num_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, size_t* bytes)
{
    if (!bytes) return set_error(DSV41_E_INVALID, "bytes is NULL");
    const dsv41_kv4_cache c{num_pages, page_size, kv_heads, head_dim, nullptr};
    const int rc = check_kv4(&c, false);
    if (rc) return rc;
    *bytes = (size_t)num_pages * kv_heads * 2 * kv4_block(page_size, head_dim / kKv4Chunk);
    return DSV41_OK;
}

int dsv41_kv4_store(const dsv41_kv4_cache* cache, const dsv41_kv4_tokens* a, void* stream)
{
    Kv4Params p{};
    const int rc = kv4_params(p, cache, a);
    if (rc || p.num_tokens == 0) return rc;
    return launched(launch_kv4_store(p, a->dtype, static_cast<cudaStream_t>(stream)), "store in 4 bits");
}

int dsv41_kv4_load(const dsv41_kv4_cache* cache, const dsv41_kv4_tokens* a, void* stream)
{
    Kv4Params p{};
    const int rc = kv4_params(p, cache, a);
    if (rc || p.num_tokens == 0) return rc;
    if (repeats(a->k_stride_token, a->num_tokens) || repeats(a->v_stride_token, a->num_tokens) || repeats(a->k_stride_head, cache->kv_heads) ||
        repeats(a->v_stride_head, cache->kv_heads))
        return set_error(DSV41_E_INVALID, "k or v repeats in memory: a stride of 0 cannot be written through");
    return launched(launch_kv4_load(p, a->dtype, static_cast<cudaStream_t>(stream)), "load from 4 bits");
}

int dsv41_kv4_move(const dsv41_kv4_cache* cache, const int64_t* from, const int64_t* to, int32_t num_tokens, void* room, size_t room_bytes,
                   void* stream)
{
    const int rc = check_kv4(cache, true);
    if (rc) return rc;
    if (num_tokens < 0) return set_error(DSV41_E_INVALID, "num_tokens=%d", num_tokens);
    if (num_tokens == 0) return DSV41_OK;
    if (!from || !to || !room) return set_error(DSV41_E_INVALID, "NULL pointer");
    if (!aligned(room, 16)) return set_error(DSV41_E_INVALID, "room must be 16-byte aligned");
    Kv4Params p{};
    kv4_cache(p, cache);
    const size_t need = (size_t)num_tokens * p.kv_heads * 2 * p.chunks * 20;
    if (room_bytes < need) return set_error(DSV41_E_WORKSPACE, "room %zu bytes < required %zu", room_bytes, need);
    p.slots = from;
    p.moved = static_cast<unsigned char*>(room);
    p.num_tokens = num_tokens;
    return launched(launch_kv4_move(p, to, static_cast<cudaStream_t>(stream)), "move within a cache in 4 bits");
}

int dsv41_tree_attention4(const dsv41_tree_attention_args* a, const dsv41_kv4_cache* cache, int32_t window, int32_t sinks, void* workspace,
                          size_t workspace_bytes, void* stream)
{
    if (!a) return set_error(DSV41_E_INVALID, "args is NULL");
    int rc = check_kv4(cache, true);
    if (rc) return rc;
    if (a->kv_heads != cache->kv_heads || a->head_dim != cache->head_dim || a->page_size != cache->page_size || a->num_pages != cache->num_pages)
        return set_error(DSV41_E_INVALID, "the arguments' heads, head_dim, page_size or num_pages are not the cache's");
    TreeAttnParams p{};
    bool run = false;
    rc = attn_params(p, a, cache, window, sinks, workspace, workspace_bytes, &run);
    if (rc || !run) return rc;
    return launched(launch_tree_attn4(p, a->dtype, attn_rows(a), static_cast<cudaStream_t>(stream)), "tree attention over 4 bits");
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

int dsv41_token_logprobs(const dsv41_token_logprobs_args* a, void* stream)
{
    if (!a) return set_error(DSV41_E_INVALID, "args is NULL");
    if (a->dtype < DSV41_DTYPE_F16 || a->dtype > DSV41_DTYPE_F32) return set_error(DSV41_E_INVALID, "dtype %d (fp16, bf16 or fp32)", a->dtype);
    if (a->rows < 0 || a->rows > (1 << 27)) return set_error(DSV41_E_INVALID, "rows=%d (0..2^27)", a->rows);
    if (a->vocab < 1 || a->vocab > 0x7fffff00) return set_error(DSV41_E_INVALID, "vocab=%d", a->vocab);
    if (a->given < 0 || a->given > kMaxGiven) return set_error(DSV41_E_INVALID, "given=%d (0..%d tokens a row)", a->given, kMaxGiven);
    if (a->top < 0 || a->top > kMaxTop) return set_error(DSV41_E_INVALID, "top=%d (0..%d)", a->top, kMaxTop);
    if (a->row_stride < 0) return set_error(DSV41_E_INVALID, "row_stride %lld", (long long)a->row_stride);
    if (a->rows == 0) return DSV41_OK;
    if (!a->logits || !a->entropy || !a->lse || (a->given && (!a->tokens || !a->logprobs)) || (a->top && (!a->top_ids || !a->top_logprobs)))
        return set_error(DSV41_E_INVALID, "NULL pointer");
    if (!aligned(a->logits, a->dtype == DSV41_DTYPE_F32 ? 4 : 2) || !aligned(a->tokens, 8) || !aligned(a->top_ids, 8))
        return set_error(DSV41_E_INVALID, "logits, tokens or top_ids is misaligned");
    LogprobParams p{};
    p.logits = a->logits;
    p.row_stride = a->row_stride;
    p.tokens = a->tokens;
    p.rows = a->rows;
    p.vocab = a->vocab;
    p.given = a->given;
    p.top = a->top;
    p.logprobs = a->logprobs;
    p.entropy = a->entropy;
    p.lse = a->lse;
    p.top_ids = a->top_ids;
    p.top_logprobs = a->top_logprobs;
    return launched(launch_logprobs(p, a->dtype, static_cast<cudaStream_t>(stream)), "log probabilities");
}

}  // extern "C"
