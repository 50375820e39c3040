// Device helpers of the attention kernels: 16-bit pairs, asynchronous copies, a kernel's view of a request, key tiles and
// positions in the list of units, mask windows, the cut of the work, and the join of what was cut.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.h"

namespace dsv41 {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v)
{
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <typename T>
__device__ constexpr uint32_t exp_bits()
{
    return std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
}
// the pair with infinities and NaN replaced by zero
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t v)
{
    constexpr uint32_t e = exp_bits<T>();
    if ((v & e) == e) v &= 0xffff0000u;
    if ((v & (e << 16)) == (e << 16)) v &= 0x0000ffffu;
    return v;
}
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint4 v)
{
    constexpr uint32_t e = exp_bits<T>();
    auto bad = [](uint32_t w) { return (w & e) == e || (w & (e << 16)) == (e << 16); };
    return bad(v.x) || bad(v.y) || bad(v.z) || bad(v.w);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live)
{
    const int n = live ? 16 : 0;   // 0: sixteen zero bytes
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One request as the kernel sees it: n new tokens from row q0 of the batch, seq keys (0 when the lengths do
// not hold the new tokens: a refused request, whose rows see nothing), clamped to what the arrays hold.
struct AttnReq {
    int q0, n, seq;
};
__device__ __forceinline__ AttnReq attn_req(const TreeAttnParams& p, int b)
{
    AttnReq r;
    r.q0 = min(max(p.cu_lens[b], 0), p.num_tokens);
    r.n = max(min(p.cu_lens[b + 1], p.num_tokens) - r.q0, 0);
    r.seq = p.seq_lens[b];
    if (r.seq < r.n || r.seq > p.max_keys) r.seq = 0;
    return r;
}

// The key tiles of a row tile, in order. Without a window: all of the request's. With one (WIN): those of the first
// `sinks` positions, then those from the first key that the window of one of its rows reaches; without a mask also only up to the last
// token of the row tile, so that a prompt's row tiles have lists of their own (a list that is the same for all, long enough for the
// longest, cost 1330 us for 900 on 2 x 6000-8192 tokens through a window of 2048: the tiles too many are masked, the
// slowest kind).
template <int RT, int KT, bool WIN>
struct KeyTiles {
    __device__ __forceinline__ int tile(int x) const { return x; }
    // of row tile rt; how many there are
    __device__ __forceinline__ int place(const TreeAttnParams&, const AttnReq& r, int) { return max((r.seq + KT - 1) / KT, 1); }
};
template <int RT, int KT>
struct KeyTiles<RT, KT, true> {
    int sinks, skip;   // tile x of the list is tile x (x < sinks) or x + skip of the request
    __device__ __forceinline__ int tile(int x) const { return x < sinks ? x : x + skip; }
    __device__ __forceinline__ int place(const TreeAttnParams& p, const AttnReq& r, int rt)
    {
        sinks = skip = 0;
        if (r.seq <= 0) return 1;
        const int ctx = r.seq - r.n;
        int before = 0, last = r.seq - 1;   // the row tile's first token (and itself), if it says where the window begins; its last key
        if (!p.tree_mask) {
            before = p.group_div.div(rt * RT) + 1;
            last = ctx + p.group_div.div(min(rt * RT + RT, r.n * p.group) - 1);
        }
        const int end = last / KT + 1, first = max(ctx + before - p.window, 0) / KT;
        sinks = min((min(p.sinks, r.seq) + KT - 1) / KT, end);
        skip = max(first - sinks, 0);
        return end - skip;
    }
};

// Position in the list of units: request, KV head, row tile, key tile.
template <int RT, int KT, bool WIN>
struct UnitCursor {
    int b, h, rt, kt, nrt, nkt;
    AttnReq r;
    KeyTiles<RT, KT, WIN> keys;
    __device__ __forceinline__ void enter(const TreeAttnParams& p)
    {
        r = attn_req(p, b);
        nrt = (r.n * p.group + RT - 1) / RT;
        if (!WIN) nkt = keys.place(p, r, 0);
    }
    __device__ __forceinline__ void place(const TreeAttnParams& p)
    {
        if (WIN) nkt = keys.place(p, r, rt);
    }
    __device__ __forceinline__ int tile() const { return keys.tile(kt); }
    __device__ __forceinline__ void next(const TreeAttnParams& p)
    {
        if (++kt < nkt) return;
        kt = 0;
        if (++rt < nrt) return place(p);
        rt = 0;
        if (++h < p.kv_heads) return place(p);
        h = 0;
        while (++b < p.batch) {
            enter(p);
            if (r.n > 0) return place(p);
        }
    }
};

// bits j0 .. j0 + 63 of what new token i sees, bit x for new token j0 + x; a negative j is context: seen
__device__ __forceinline__ uint64_t seen_window(const TreeAttnParams& p, const AttnReq& r, int i, int j0)
{
    auto word = [&](int w) -> uint64_t {
        if (w < 0) return ~0ull;
        if (p.tree_mask) return w < p.mask_words ? (uint64_t)p.tree_mask[(int64_t)(r.q0 + i) * p.mask_words + w] : 0ull;
        return w < (i >> 6) ? ~0ull : w > (i >> 6) ? 0ull : (~0ull >> (63 - (i & 63)));
    };
    const int w = j0 >> 6, sh = j0 & 63;
    uint64_t v = word(w) >> sh;
    if (sh) v |= word(w + 1) << (64 - sh);
    const int left = r.n - j0;   // new tokens from j0 on
    return left >= 64 ? v : left <= 0 ? 0ull : v & (~0ull >> (64 - left));
}

// position of the first key in the window of new token i: the last `window` keys of those that it sees (negative: all of them are)
__device__ __forceinline__ int window_start(const TreeAttnParams& p, const AttnReq& r, int i)
{
    const int ctx = r.seq - r.n;
    if (!p.tree_mask) return ctx + i + 1 - p.window;
    int seen = 0;
    for (int j = 0; j < r.n && j < 64 * p.mask_words; j += 64) seen += __popcll(seen_window(p, r, i, j));
    if (seen <= p.window) return ctx + seen - p.window;
    int over = seen - p.window;   // ancestors in front of it
    for (int j = 0;; j += 64) {
        uint64_t v = seen_window(p, r, i, j);
        const int here = __popcll(v);
        if (over >= here) {
            over -= here;
            continue;
        }
        for (; over > 0; --over) v &= v - 1;
        return ctx + j + __ffsll((long long)v) - 1;
    }
}
// bits of positions pos0 .. pos0 + 63 that are among the first `sinks`, or from `start` on
__device__ __forceinline__ uint64_t window_bits(const TreeAttnParams& p, int start, int pos0)
{
    const int cut = start - pos0, first = p.sinks - pos0;
    const uint64_t in = cut <= 0 ? ~0ull : cut >= 64 ? 0ull : ~0ull << cut;
    return in | (first <= 0 ? 0ull : first >= 64 ? ~0ull : (1ull << first) - 1);
}
// what new token i sees of positions pos0 .. pos0 + 63
template <bool WIN>
__device__ __forceinline__ uint64_t seen_keys(const TreeAttnParams& p, const AttnReq& r, int i, int pos0)
{
    const uint64_t seen = seen_window(p, r, i, pos0 - (r.seq - r.n));
    return WIN ? seen & window_bits(p, window_start(p, r, i), pos0) : seen;
}
// Where the rows of a row tile (tokens first .. last) may differ in what they see: keys from `from` on are new tokens that not
// all of them see, keys before `edge` lie in front of the window of one of them (the first p.sinks do not).
template <bool WIN>
struct MaskedKeys {
    int from, edge;
    __device__ __forceinline__ MaskedKeys() {}
    __device__ __forceinline__ MaskedKeys(const TreeAttnParams& p, const AttnReq& r, int first, int last)
    {
        const int ctx = r.seq - r.n;
        from = p.tree_mask ? ctx : ctx + first + 1;
        edge = ctx + (p.tree_mask ? r.n : last + 1) - p.window;
    }
    template <int KT>
    __device__ __forceinline__ bool tile(const TreeAttnParams& p, int pos0) const
    {
        return pos0 + KT > from || (WIN && pos0 < edge && pos0 + KT > p.sinks);
    }
};
template <int RT, bool WIN, typename Cursor>
__device__ __forceinline__ MaskedKeys<WIN> masked_keys(const TreeAttnParams& p, const Cursor& c)
{
    return MaskedKeys<WIN>(p, c.r, p.group_div.div(c.rt * RT), p.group_div.div(min(c.rt * RT + RT, c.r.n * p.group) - 1));
}

// ---- the cut of a call's units into runs, one per CTA ----
// Calls whose segments can each have CTAs of their own: segments of up to 2 * R tiles stay whole, longer ones are cut into
// equal parts of R at most (R = SMALL, or 2 * SMALL where there is no room for that; a place on the line is a CTA).
// Others: a segment of nkt tiles costs what nkt + extra tiles do (its rows' loads, its end), so the runs are cut from a
// line on which each segment begins with `extra` empty places.
// Every thread sums its requests' places and tiles; the one whose request holds the run's first place, and the
// one that holds its end, tell the others.
__device__ __forceinline__ int cut_parts(int tiles, int r) { return tiles <= 2 * r ? 1 : (tiles + r - 1) / r; }
template <int WARPS>
struct CutShared {
    int64_t warp_sum[WARPS][4];
    int64_t first[3], end, tiles0;
};
// sums of the threads before this one and of all (those that hold requests are the first `threads`)
template <int WARPS>
__device__ __forceinline__ void scan_sums(CutShared<WARPS>& sm, const int64_t (&sum)[4], int64_t (&before)[4], int64_t (&all)[4], int threads)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, holders = (threads + 31) / 32;
    int64_t inc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        inc[k] = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, inc[k], o);
            if (lane >= o) inc[k] += y;
        }
        if (lane == 31) sm.warp_sum[warp][k] = inc[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        before[k] = inc[k] - sum[k], all[k] = 0;
#pragma unroll 1
        for (int w = 0; w < holders; ++w) {
            if (w < warp) before[k] += sm.warp_sum[w][k];
            all[k] += sm.warp_sum[w][k];
        }
    }
}
// Sums over the row tiles of one head of a request, each with its own number of key tiles (WIN, no mask): places, tiles, parts for
// R = SMALL and 2 * SMALL. By a whole warp, a request a lane: those with many row tiles are summed by all lanes together.
template <int RT, int KT, int EXTRA, int SMALL>
__device__ __noinline__ void head_sums(const TreeAttnParams& p, int n, int seq, int64_t* s)
{
    const int lane = threadIdx.x & 31, nrt = n > 0 ? (n * p.group + RT - 1) / RT : 0;
    auto add = [&](const AttnReq& r, int rt, int64_t* to) {
        const int nt = KeyTiles<RT, KT, true>().place(p, r, rt);
        to[0] += nt + EXTRA, to[1] += nt, to[2] += cut_parts(nt, SMALL), to[3] += cut_parts(nt, 2 * SMALL);
    };
    s[0] = s[1] = s[2] = s[3] = 0;
    if (nrt <= 4)
        for (int rt = 0; rt < nrt; ++rt) add(AttnReq{0, n, seq}, rt, s);
    for (uint32_t many = __ballot_sync(0xffffffffu, nrt > 4); many; many &= many - 1) {
        const int l = __ffs(many) - 1, tiles = __shfl_sync(0xffffffffu, nrt, l);
        const AttnReq r{0, __shfl_sync(0xffffffffu, n, l), __shfl_sync(0xffffffffu, seq, l)};
        int64_t v[4] = {0, 0, 0, 0};
        for (int rt = lane; rt < tiles; rt += 32) add(r, rt, v);
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
            if (lane == l) s[k] = v[k];
        }
        __syncwarp();
    }
}

// The cut where row tiles of a request may differ in their number of key tiles.
template <int RT, int KT, int EXTRA, int SMALL, int WARPS>
__device__ __forceinline__ void cut_lists(const TreeAttnParams& p, CutShared<WARPS>& sm, int64_t& run, int64_t& v0, int& part_tiles)
{
    constexpr int kThreads = WARPS * 32, kSums = 4;   // places on the line, tiles, parts for R = SMALL and 2 * SMALL
    const int tid = threadIdx.x;
    const int per = (p.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    const bool own_lists = !p.tree_mask;   // row tiles of a request differ in their number of key tiles
    auto row_tiles = [&](const AttnReq& r) { return r.n > 0 ? (r.n * p.group + RT - 1) / RT : 0; };
    auto tiles = [&](const AttnReq& r) { return KeyTiles<RT, KT, true>().place(p, r, 0); };
    // sums over one head of request b (of this thread's; all threads go round together)
    auto sums = [&](const AttnReq& r, int64_t* s) {
        if (own_lists && __any_sync(0xffffffffu, row_tiles(r) > 1)) return head_sums<RT, KT, EXTRA, SMALL>(p, r.n, r.seq, s);
        const int64_t n = row_tiles(r);
        const int nt = tiles(r);
        s[0] = n * (nt + EXTRA), s[1] = n * nt, s[2] = n * cut_parts(nt, SMALL), s[3] = n * cut_parts(nt, 2 * SMALL);
    };
    int64_t sum[kSums] = {}, head[kSums];
    AttnReq mine{0, 0, 0};
    for (int i = 0; i < per; ++i) {
        mine = b0 + i < b1 ? attn_req(p, b0 + i) : AttnReq{0, 0, 0};
        sums(mine, head);
#pragma unroll
        for (int k = 0; k < kSums; ++k) sum[k] += head[k] * p.kv_heads;
    }
    int64_t before[kSums], all[kSums];
    scan_sums(sm, sum, before, all, (p.batch + per - 1) / per);
    part_tiles = all[2] <= gridDim.x ? SMALL : all[3] <= gridDim.x ? 2 * SMALL : 0;
    auto places_in = [&](const int64_t* s) { return part_tiles == SMALL ? s[2] : part_tiles ? s[3] : s[0]; };
    const int64_t total = places_in(all);
    run = part_tiles ? 1 : (total + gridDim.x - 1) / gridDim.x;
    v0 = run * blockIdx.x;
    const int64_t v1 = min(v0 + run, total);
    if (tid == 0) {
        if (v0 >= total) sm.tiles0 = sm.end = 0;
        else if (!part_tiles && v1 >= total) sm.end = all[1];
    }
    int64_t at = places_in(before), tiles0 = before[1];
    for (int i = 0; i < per; ++i) {
        if (per > 1) {
            mine = b0 + i < b1 ? attn_req(p, b0 + i) : AttnReq{0, 0, 0};
            sums(mine, head);
        }
        const int64_t per_head = places_in(head), places = per_head * p.kv_heads;
        // place v of this request: its segment, the place within that, and the tiles before it
        struct Found {
            int64_t segment, in, tiles;
            int nt;
        };
        auto find = [&](int64_t v) {
            Found f;
            const int64_t h = v / per_head;
            f.in = v - h * per_head;
            auto places_of = [&](int nt) { return part_tiles ? cut_parts(nt, part_tiles) : nt + EXTRA; };
            int64_t rt = 0, passed = 0;
            if (own_lists) {
                for (;; ++rt) {
                    f.nt = KeyTiles<RT, KT, true>().place(p, mine, (int)rt);
                    if (f.in < places_of(f.nt)) break;
                    f.in -= places_of(f.nt);
                    passed += f.nt;
                }
            } else {
                f.nt = tiles(mine);
                rt = f.in / places_of(f.nt);
                f.in -= rt * places_of(f.nt);
                passed = rt * f.nt;
            }
            f.segment = h * row_tiles(mine) + rt;
            f.tiles = tiles0 + h * head[1] + passed + max(f.in - EXTRA, (int64_t)0);
            return f;
        };
        if (v0 >= at && v0 < at + places) {
            const Found f = find(v0 - at);
            sm.first[0] = b0 + i;
            sm.first[1] = f.segment;
            sm.first[2] = f.in;
            if (part_tiles) {
                const int len = cut_parts(f.nt, part_tiles), tpp = (f.nt + len - 1) / len;
                sm.tiles0 = f.in * tpp;
                sm.end = min((f.in + 1) * tpp, (int64_t)f.nt);
            } else {
                sm.tiles0 = f.tiles;
            }
        }
        if (!part_tiles && v1 < total && v1 >= at && v1 < at + places) sm.end = find(v1 - at).tiles;
        at += places;
        tiles0 += head[1] * p.kv_heads;
    }
}

// The cut where all row tiles of a request have the same key tiles (no window). A part's place is found in 32 bits (there are no more
// of them than CTAs), a run's ends with a division of 64 bits each: found as in cut_lists, one token over 2048 keys took 18.5 us
// a call for 16.9, 16 trees over 0.1-4k keys 44.4 for 43.6.
template <int RT, int KT, int EXTRA, int SMALL, int WARPS>
__device__ __forceinline__ void cut_even(const TreeAttnParams& p, CutShared<WARPS>& sm, int64_t& run, int64_t& v0, int& part_tiles)
{
    constexpr int kThreads = WARPS * 32;
    const int tid = threadIdx.x;
    const int per = (p.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    auto segments = [&](const AttnReq& r) { return r.n > 0 ? (int64_t)((r.n * p.group + RT - 1) / RT) * p.kv_heads : 0; };
    auto tiles = [&](const AttnReq& r) { return KeyTiles<RT, KT, false>().place(p, r, 0); };
    int64_t sum[4] = {};
    AttnReq mine;
    for (int b = b0; b < b1; ++b) {
        mine = attn_req(p, b);
        const int64_t n = segments(mine);
        const int nt = tiles(mine);
        sum[0] += n * (nt + EXTRA);
        sum[1] += n * nt;
        sum[2] += n * cut_parts(nt, SMALL);
        sum[3] += n * cut_parts(nt, 2 * SMALL);
    }
    int64_t before[4], all[4];
    scan_sums(sm, sum, before, all, (p.batch + per - 1) / per);
    part_tiles = all[2] <= gridDim.x ? SMALL : all[3] <= gridDim.x ? 2 * SMALL : 0;
    if (part_tiles) {
        int64_t at = part_tiles == SMALL ? before[2] : before[3];
        run = 1;
        v0 = blockIdx.x;
        if (tid == 0 && v0 >= (part_tiles == SMALL ? all[2] : all[3])) sm.tiles0 = sm.end = 0;
        for (int b = b0; b < b1; ++b) {
            if (per > 1) mine = attn_req(p, b);
            const int nt = tiles(mine), len = cut_parts(nt, part_tiles);
            const int64_t places = segments(mine) * len;
            if (v0 >= at && v0 < at + places) {
                const int in = (int)(v0 - at), part = in % len, each = (nt + len - 1) / len;
                sm.first[0] = b;
                sm.first[1] = in / len;
                sm.first[2] = part;
                sm.tiles0 = part * each;
                sm.end = min((part + 1) * each, nt);
            }
            at += places;
        }
        return;
    }
    run = (all[0] + gridDim.x - 1) / gridDim.x;
    v0 = run * blockIdx.x;
    const int64_t v1 = min(v0 + run, all[0]);
    if (tid == 0) {
        if (v0 >= all[0]) sm.tiles0 = sm.end = 0;
        else if (v1 >= all[0]) sm.end = all[1];
    }
    int64_t at = before[0], tiles0 = before[1];
    for (int b = b0; b < b1; ++b) {
        if (per > 1) mine = attn_req(p, b);
        const int64_t n = segments(mine), nt = tiles(mine), len = nt + EXTRA, places = n * len;
        auto tiles_before = [&](int64_t segment, int64_t in) { return tiles0 + segment * nt + max(in - EXTRA, (int64_t)0); };
        if (v0 >= at && v0 < at + places) {
            const int64_t segment = (v0 - at) / len, in = v0 - at - segment * len;
            sm.first[0] = b;
            sm.first[1] = segment;
            sm.first[2] = in;
            sm.tiles0 = tiles_before(segment, in);
        }
        if (v1 < all[0] && v1 >= at && v1 < at + places) {
            const int64_t segment = (v1 - at) / len;
            sm.end = tiles_before(segment, v1 - at - segment * len);
        }
        at += places;
        tiles0 += n * nt;
    }
}

template <int RT, int KT, bool WIN, int EXTRA, int SMALL, int WARPS>
__device__ __forceinline__ void cut_runs(const TreeAttnParams& p, CutShared<WARPS>& sm, int64_t& run, int64_t& v0, int& part_tiles)
{
    if constexpr (WIN) cut_lists<RT, KT, EXTRA, SMALL>(p, sm, run, v0, part_tiles);
    else cut_even<RT, KT, EXTRA, SMALL>(p, sm, run, v0, part_tiles);
}

// Join of a segment's parts (runs fc .. lc): a thread takes 16 columns of a row, a batch of parts at a time with all its
// loads in flight (one trip to L2 a batch), and rescales what it has as the softmax does. Rows r0 .. r0 + rows - 1 of
// the row tile, by `threads` threads. A part is [column / 4][row][4]: neighbours in a warp are neighbouring rows
// here and where it is written. All by value: what a function reads through a reference (the kernel's parameters, the
// cursor) costs a trip to L2 a field and row (50 rows of 4 parts: 13000 cycles).
struct JoinArgs {
    const float2* ml;
    const float4* o;
    void* out;            // the request's first row, the KV head's first query head
    float* lse;           // the same, or null
    int64_t stride_token, stride_head;
    FastDiv group_div;
    int group, q_heads, head_dim, row0;   // row0: first row of the row tile
};
template <typename T, int DT, int RT>
__device__ __noinline__ void join_parts(const JoinArgs a, int fc, int lc, int r0, int rows, int thread, int threads)
{
    constexpr int kBatch = 4;
    const int blocks = (a.head_dim + 15) / 16;
    for (int e = thread; e < rows * blocks; e += threads) {
        const int block = e / rows, r = r0 + e - block * rows;
        float mm = -INFINITY, ll = 0.0f, acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
#pragma unroll 1
        for (int q0 = fc; q0 <= lc; q0 += kBatch) {
            float2 v[kBatch];
            float4 po[kBatch][4];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int q = q0 + i;
                const int64_t slot = 2 * q + (q == fc ? 1 : 0);
                const float4* src = a.o + slot * (RT * DT / 4) + block * 4 * RT + r;
                v[i] = q <= lc ? __ldcg(a.ml + slot * RT + r) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int k = 0; k < 4; ++k) po[i][k] = q <= lc ? __ldcg(src + k * RT) : make_float4(0, 0, 0, 0);
            }
            float top = mm;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) top = fmaxf(top, v[i].x);
            const float safe = top == -INFINITY ? 0.0f : top, keep = exp2_fast(mm - safe);
            ll *= keep;
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] *= keep;
            mm = top;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const float w = exp2_fast(v[i].x - safe);
                ll += v[i].y * w;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    acc[4 * k] += po[i][k].x * w, acc[4 * k + 1] += po[i][k].y * w, acc[4 * k + 2] += po[i][k].z * w,
                        acc[4 * k + 3] += po[i][k].w * w;
            }
        }
        // 0 * inf is NaN where a part's weight vanishes in 32 bits: what the parts hold of infinities and NaN itself instead
        float test = 0.0f;   // NaN if a sum is not finite (columns past the head size hold anything)
#pragma unroll
        for (int j = 0; j < 16; j += 8)
            if (block * 16 + j < a.head_dim)
#pragma unroll
                for (int c = 0; c < 8; ++c) test = fmaf(acc[j + c], 0.0f, test);
        if (__builtin_expect(test != 0.0f, 0)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float4 bad = make_float4(0, 0, 0, 0);
#pragma unroll 1
                for (int q = fc; q <= lc; ++q) {
                    const float4 v = __ldcg(a.o + (int64_t)(2 * q + (q == fc ? 1 : 0)) * (RT * DT / 4) + (block * 4 + k) * RT + r);
                    if (!(fabsf(v.x) < INFINITY)) bad.x += v.x;
                    if (!(fabsf(v.y) < INFINITY)) bad.y += v.y;
                    if (!(fabsf(v.z) < INFINITY)) bad.z += v.z;
                    if (!(fabsf(v.w) < INFINITY)) bad.w += v.w;
                }
                if (bad.x != 0.0f) acc[4 * k] = bad.x;
                if (bad.y != 0.0f) acc[4 * k + 1] = bad.y;
                if (bad.z != 0.0f) acc[4 * k + 2] = bad.z;
                if (bad.w != 0.0f) acc[4 * k + 3] = bad.w;
            }
        }
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        const int row = a.row0 + r, i = a.group_div.div(row), g = row - i * a.group;
        T* out = static_cast<T*>(a.out) + i * a.stride_token + g * a.stride_head + block * 16;
#pragma unroll
        for (int j = 0; j < 16; j += 8)
            if (block * 16 + j < a.head_dim)
                *reinterpret_cast<uint4*>(out + j) =
                    make_uint4(pack2<T>(acc[j] * inv, acc[j + 1] * inv), pack2<T>(acc[j + 2] * inv, acc[j + 3] * inv),
                               pack2<T>(acc[j + 4] * inv, acc[j + 5] * inv), pack2<T>(acc[j + 6] * inv, acc[j + 7] * inv));
        if (a.lse && block == 0)
            a.lse[(int64_t)i * a.q_heads + g] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
    }
}

}  // namespace dsv41
