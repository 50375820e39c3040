// Block tables, slot maps and the store of new keys and values for a paged cache (dsv41_step_tables,
// dsv41_store_kv).
//
// Tables. A cache is a pool of pages of P token slots. For request b with c_b tokens in the cache, n_b new
// ones this step, h_b pages held and W table columns:
//     need_b = ceil((c_b + n_b) / P)        give_b = max(h_b - need_b, 0)     take_b = max(need_b - h_b, 0)
// (need_b > W: the request is refused and keeps what it holds). Returned pages are pushed on the stack of
// free pages in request order, then pages are popped in request order:
//     the j-th popped page is entry F + G - 1 - j of the stack, F its height before, G = sum give_b
// (where more would be left on the stack than it holds: over the requests before the first whose pages pass its end;
// from there on all keep theirs)
// and request b is admitted iff the running sum of takes through b fits F + G. Every quantity is a prefix
// sum over requests, so each CTA computes the sums itself (batch <= 2048: three values per request, one
// block scan) and then fills its own share of the outputs. A popped page that was returned in the same call
// is read from its giver's table row (which this call never writes) rather than from the stack, so CTAs
// need not wait for one another and one launch does it all.
//
// Bound: a decode step is latency (launch, lengths, scan, outputs): 48 requests with trees 12 us on the GPU; a
// prefill writes 16 bytes per token: 512 requests, half a million tokens in 19 us, most of it that latency too. One launch
// instead of a scan and a fill saves a launch and a trip of the sums through memory.
//
// Store. cache[slot[t]] = kv[t] in 16-byte pieces; bound by HBM (every byte read once and written once): 16384 tokens of
// 8 heads of 128, 134 MB in 26 us, 5.1 TB/s; 100 tokens 8 us, a launch.
#include "common.cuh"
#include "internal.h"
#include "paged.h"

namespace dsv41 {

constexpr int kTabThreads = 256;
constexpr int kTabPerThread = kMaxRequests / kTabThreads;
constexpr int kTabTokens = 4;   // consecutive tokens per thread: full 16-byte stores of positions and requests

// sums saturate at 2^31 - 1 (all terms are >= 0, so the saturating sum is associative)
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

struct TabReq {
    int ctx, fresh, held;   // tokens in the cache, new tokens, pages held (all clamped to >= 0)
    int want;               // pages after the call if the request is admitted
    bool fits;
};

__device__ __forceinline__ TabReq tab_req(const StepTablesParams& p, int b)
{
    TabReq r;
    r.ctx = max(p.context_lens[b], 0);
    r.fresh = max(p.new_lens[b], 0);
    r.held = min(max(p.held_pages[b], 0), p.width);
    const int64_t need = ((int64_t)r.ctx + r.fresh + p.page_size - 1) / p.page_size;
    r.fits = need <= p.width;
    r.want = r.fits ? (int)need : r.held;
    return r;
}

// largest b in [0, n) with start[b] <= v (start ascending, start[0] = 0)
__device__ __forceinline__ int last_le(const uint32_t* start, int n, uint32_t v)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kTabThreads) step_tables_kernel(const StepTablesParams p)
{
    extern __shared__ uint32_t sm[];   // exclusive prefix sums [B + 1] of new tokens, takes, gives
    __shared__ uint32_t warp_tot[3][kTabThreads / 32];
    const int B = p.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t* cu = sm;
    uint32_t* tk = sm + B + 1;
    uint32_t* gv = sm + 2 * (B + 1);

    // block scan: thread t owns requests [t * per, (t + 1) * per)
    const int per = (B + kTabThreads - 1) / kTabThreads;
    uint32_t v[3][kTabPerThread], tot[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kTabPerThread; ++i) {
        if (i >= per) break;
        const int b = tid * per + i;
        v[0][i] = tot[0], v[1][i] = tot[1], v[2][i] = tot[2];
        if (b >= B) continue;
        const TabReq r = tab_req(p, b);
        tot[0] = sat_add(tot[0], r.fresh);
        tot[1] = sat_add(tot[1], max(r.want - r.held, 0));
        tot[2] = sat_add(tot[2], max(r.held - r.want, 0));
    }
    uint32_t inc[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        uint32_t x = tot[s];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = sat_add(x, y);
        }
        inc[s] = x;
        if (lane == 31) warp_tot[s][warp] = x;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        uint32_t before = 0;
        for (int w = 0; w < warp; ++w) before = sat_add(before, warp_tot[s][w]);
        uint32_t up = __shfl_up_sync(0xffffffffu, inc[s], 1);
        const uint32_t base = sat_add(before, lane ? up : 0u);
        uint32_t* dst = sm + s * (B + 1);
#pragma unroll
        for (int i = 0; i < kTabPerThread; ++i) {
            if (i >= per) break;
            const int b = tid * per + i;
            if (b < B) dst[b] = sat_add(base, v[s][i]);
        }
        if (tid == kTabThreads - 1) dst[B] = sat_add(base, tot[s]);
    }
    __syncthreads();

    const uint32_t height = (uint32_t)min(max(*p.free_count, 0), p.free_capacity);
    const uint32_t room = p.free_capacity - height, tokens = p.num_tokens;
    uint32_t given = gv[B], served = cu[B];        // pages that go back; tokens of the requests that end within the token arrays
    const bool odd = given > room || served > tokens;
    if (__builtin_expect(odd, 0)) {
        const uint32_t all = sat_add(height, given), popped = tk[last_le(tk, B + 1, all)];
        if (all - popped > (uint32_t)p.free_capacity) given = gv[last_le(gv, B + 1, room)];
        if (served > tokens) served = cu[last_le(cu, B, tokens)];
    }
    const uint32_t top = height + given;           // stack height after the returns
    auto admitted = [&](const TabReq& r, int b) { return r.fits && (r.want <= r.held || tk[b + 1] <= top); };
    auto keeps = [&](const TabReq& r, int b) { return odd && r.want < r.held && gv[b + 1] > given; };
    // new tokens that the token arrays have no entry for: not served, for attention would take them for context
    auto past = [&](const TabReq& r, int b) { return odd && r.fresh > 0 && cu[b + 1] > tokens; };
    auto flags_of = [&](const TabReq& r, int b, bool ok) {
        return (ok ? 0 : r.fits ? kTabNoPages : kTabTooWide) | (keeps(r, b) ? kTabNoRoom : 0) | (past(r, b) ? kTabPastTokens : 0);
    };
    // entry i of the stack after the returns (i < top)
    auto stack_page = [&](uint32_t i) {
        if (i < height) return p.free_pages[i];
        const uint32_t e = i - height;
        const int b = last_le(gv, B, e);   // gives of 0 share a start with their successor: the last one gives
        return p.block_table[(int64_t)b * p.table_stride + tab_req(p, b).want + (int)(e - gv[b])];
    };

    const int stride = gridDim.x * kTabThreads, first = blockIdx.x * kTabThreads + tid;
    // pages taken: into the tables
    for (uint32_t j = first; j < tk[B] && j < top; j += stride) {
        const int b = last_le(tk, B, j);
        const TabReq r = tab_req(p, b);
        if (admitted(r, b))
            p.block_table[(int64_t)b * p.table_stride + r.held + (int)(j - tk[b])] = stack_page(top - 1 - j);
    }
    // pages returned: onto the stack
    for (uint32_t e = first; e < given; e += stride)
        if (height + e < (uint32_t)p.free_capacity) p.free_pages[height + e] = stack_page(height + e);   // (the others are taken)

    // per-request outputs
    uint32_t used = 0;   // pages popped: the largest admitted running sum of takes
    if (blockIdx.x == 0) {
        for (int b = tid; b < B; b += kTabThreads) {
            const TabReq r = tab_req(p, b);
            const bool ok = admitted(r, b);
            p.cu_lens[b] = (int)cu[b];
            p.seq_lens[b] = ok && !past(r, b) ? (int)min((int64_t)r.ctx + r.fresh, (int64_t)0x7fffffff) : 0;
            p.held_out[b] = ok && !keeps(r, b) ? r.want : r.held;
            if (!p.parents) p.status[b] = flags_of(r, b, ok);
            if (ok) used = max(used, tk[b + 1] <= top ? tk[b + 1] : 0u);
        }
        used = __reduce_max_sync(0xffffffffu, used);
        __syncthreads();
        if (lane == 0) warp_tot[0][warp] = used;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kTabThreads / 32; ++w) used = max(used, warp_tot[0][w]);
            p.cu_lens[B] = (int)cu[B];
            *p.free_count_out = (int)(top - used);
        }
    }

    // slot of position pos of request b: a page taken in this call is looked up where it comes from
    auto slot_of = [&](const TabReq& r, int b, bool ok, int64_t pos) -> int64_t {
        if (!ok) return -1;
        const int page = (int)(pos / p.page_size), in_page = (int)(pos - (int64_t)page * p.page_size);
        const int id = page < r.held ? p.block_table[(int64_t)b * p.table_stride + page]
                                     : stack_page(top - 1 - (tk[b] + (uint32_t)(page - r.held)));
        return (int64_t)id * p.page_size + in_page;
    };

    if (!p.parents) {
        // token-parallel, kTabTokens consecutive tokens per thread; 16-byte stores where the arrays allow them
        const bool vector = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.requests) |
                              reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
        for (int64_t t0 = (int64_t)first * kTabTokens; t0 < p.num_tokens; t0 += (int64_t)stride * kTabTokens) {
            int64_t slot[kTabTokens];
            int pos[kTabTokens], req[kTabTokens];
            int b = last_le(cu, B, (uint32_t)t0);
            TabReq r = tab_req(p, b);
            bool ok = admitted(r, b);
#pragma unroll
            for (int i = 0; i < kTabTokens; ++i) {
                const uint32_t t = (uint32_t)t0 + i;
                if (t >= cu[B]) {   // past the last request's tokens
                    slot[i] = -1, pos[i] = 0, req[i] = -1;
                    continue;
                }
                if (t >= cu[b + 1]) {
                    b = last_le(cu, B, t);
                    r = tab_req(p, b);
                    ok = admitted(r, b);
                }
                const int64_t at = (int64_t)r.ctx + (t - cu[b]);
                slot[i] = slot_of(r, b, ok && t < served, at);
                pos[i] = (int)at;
                req[i] = b;
            }
            if (vector && t0 + kTabTokens <= p.num_tokens) {
                *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                *reinterpret_cast<int4*>(p.requests + t0) = make_int4(req[0], req[1], req[2], req[3]);
                *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
                *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
            } else {
                for (int i = 0; i < kTabTokens && t0 + i < p.num_tokens; ++i) {
                    p.positions[t0 + i] = pos[i];
                    p.requests[t0 + i] = req[i];
                    p.slots[t0 + i] = slot[i];
                }
            }
        }
        return;
    }
    // drafted trees: one warp per request, one lane per token; ancestors by walking the parents, which
    // lie before their children, so every walk ends
    const int warps = gridDim.x * (kTabThreads / 32);
    for (int b = blockIdx.x * (kTabThreads / 32) + warp; b < B; b += warps) {
        const TabReq r = tab_req(p, b);
        const bool ok = admitted(r, b);
        int flags = flags_of(r, b, ok);
        for (int at = lane; at < r.fresh; at += 32) {
            const int64_t t = (int64_t)cu[b] + at;
            if (t >= p.num_tokens) break;
            uint64_t bits[kMaxMaskWords] = {0, 0, 0, 0};
            int depth = 0, cur = at;
            while (true) {
#pragma unroll
                for (int w = 0; w < kMaxMaskWords; ++w)
                    if (cur >> 6 == w) bits[w] |= 1ull << (cur & 63);
                ++depth;
                const int up = p.parents[cu[b] + cur];
                if (up < -1 || up >= cur) {
                    if (cur == at) flags |= kTabBadParent;
                    break;
                }
                if (up < 0) break;
                cur = up;
            }
            if (at >= 64 * p.mask_words) flags |= kTabBigTree;
#pragma unroll
            for (int w = 0; w < kMaxMaskWords; ++w)
                if (w < p.mask_words) p.tree_mask[t * p.mask_words + w] = (int64_t)bits[w];
            p.slots[t] = slot_of(r, b, ok && t < served, (int64_t)r.ctx + at);
            p.positions[t] = (int)min((int64_t)r.ctx + depth - 1, (int64_t)0x7fffffff);
            p.requests[t] = b;
        }
        flags = __reduce_or_sync(0xffffffffu, flags);
        if (lane == 0) p.status[b] = flags;
    }
    // padding past the last request's tokens
    for (int64_t t = (int64_t)cu[B] + first; t < p.num_tokens; t += stride) {
        p.slots[t] = -1;
        p.positions[t] = 0;
        p.requests[t] = -1;
        for (int w = 0; w < p.mask_words; ++w) p.tree_mask[t * p.mask_words + w] = 0;
    }
}

cudaError_t launch_step_tables(const StepTablesParams& p, cudaStream_t st)
{
    // one thread per kTabTokens tokens (or one warp per request with trees), at most 2 CTAs per SM: more
    // would only repeat the scan
    const int64_t work = p.parents ? ((int64_t)p.batch * 32) : (p.num_tokens + kTabTokens - 1) / kTabTokens;
    const int64_t ctas = (work + kTabThreads - 1) / kTabThreads;
    const int64_t cap = 2 * num_sms();
    const int grid = (int)(ctas < 1 ? 1 : (ctas > cap ? cap : ctas));
    step_tables_kernel<<<grid, kTabThreads, 3 * (p.batch + 1) * sizeof(uint32_t), st>>>(p);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------
// store of new keys and values
// ---------------------------------------------------------------------------------------------
constexpr int kStoreThreads = 256;
constexpr int kStoreUnroll = 4;

// One warp copies kStoreUnroll x 32 16-byte pieces of one token's K or V row (all loads before the stores).
__global__ void __launch_bounds__(kStoreThreads) store_kv_kernel(const StoreKvParams p)
{
    const int lane = threadIdx.x & 31;
    const int per_head = p.head_dim / 8, pieces = p.kv_heads * per_head;
    const int parts = (pieces + 32 * kStoreUnroll - 1) / (32 * kStoreUnroll);
    const int64_t units = (int64_t)p.num_tokens * 2 * parts;
    const int64_t nwarps = (int64_t)gridDim.x * (kStoreThreads / 32);
    const int64_t slots = (int64_t)p.num_pages * p.page_size;
    for (int64_t u = (int64_t)blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5); u < units; u += nwarps) {
        const int64_t t = u / (2 * parts);
        const int rest = (int)(u - t * 2 * parts), which = rest / parts, c0 = (rest - which * parts) * 32 * kStoreUnroll;
        const int64_t slot = p.slots[t];
        if (slot < 0 || slot >= slots) continue;   // no slot: not stored
        const int64_t page = slot / p.page_size, in_page = slot - page * p.page_size;
        const uint16_t* src = static_cast<const uint16_t*>(which ? p.v : p.k) + t * (which ? p.v_stride_token : p.k_stride_token);
        const int64_t src_head = which ? p.v_stride_head : p.k_stride_head;
        uint16_t* dst = static_cast<uint16_t*>(which ? p.v_cache : p.k_cache) + page * p.stride_page + in_page * p.stride_slot;
        uint4 v[kStoreUnroll];
        int64_t to[kStoreUnroll];
#pragma unroll
        for (int i = 0; i < kStoreUnroll; ++i) {
            const int c = c0 + 32 * i + lane;
            if (c < pieces) {
                const int head = c / per_head, d = (c - head * per_head) * 8;
                v[i] = __ldcs(reinterpret_cast<const uint4*>(src + head * src_head + d));
                to[i] = head * p.stride_head + d;
            }
        }
#pragma unroll
        for (int i = 0; i < kStoreUnroll; ++i)
            if (c0 + 32 * i + lane < pieces) *reinterpret_cast<uint4*>(dst + to[i]) = v[i];
    }
}

cudaError_t launch_store_kv(const StoreKvParams& p, cudaStream_t st)
{
    const int pieces = p.kv_heads * (p.head_dim / 8), parts = (pieces + 32 * kStoreUnroll - 1) / (32 * kStoreUnroll);
    const int64_t ctas = ((int64_t)p.num_tokens * 2 * parts + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
    const int64_t cap = 8 * num_sms();
    store_kv_kernel<<<(int)(ctas > cap ? cap : ctas), kStoreThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace dsv41
