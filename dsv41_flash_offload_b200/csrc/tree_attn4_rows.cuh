// Attention of few rows over a cache in 4 bits (tree_attn.cu has the mathematics, kv4.cuh the cache): warp-level matrix
// instructions on codes decoded in registers.
//
// Both products take the cache's side as their A operand, so that what a lane loads and decodes is its fragment and nothing
// goes through shared memory: S^T = K Q^T (16 keys by 8 rows an instruction), O^T += V^T P^T (16 columns by 8 rows).
// A warp takes 16 keys at a time, two records of 8 tokens:
//   K   lane (g, t) holds words of key g of each record (g permuted: see below); a word of 8 columns is one register of two
//       instructions' A, whose columns are matched by the order in which Q lies in shared memory
//   V   lane (g, t) holds words of keys t and t + 4 of each record; the keys of a pair are merged by byte permutes before they are
//       decoded, so a pair is one column of two keys
//   P   leaves the first product with keys down and rows across, and is turned by movmatrix into the B operand of the second
// The k-th pair of keys in V's and P's order is (t, t + 4); row x of the first product is key (x >> 1) + 4 (x & 1) of its record.
// Each lane's loads then are constant offsets from two addresses per operand: a record's address is the warp's.
//
// Every warp has its own running maximum, sum and O (RT = 8 or 16 rows); nothing is exchanged before the end of a segment, where the
// four warps of a CTA join through shared memory. The deferred rescale, P's rounding and the exponentials are those of the
// other kernel (tree_attn_kernel.cuh).
//
// Values of NaN. A chunk that stands for NaN does so in all of its columns. In tiles that all rows see it reaches every row by itself. In
// others (new tokens, a window's edge, keys behind the last) such chunks enter as zeros, and the rows that see the key
// note the chunk; their columns are NaN at the end of the segment. Keys need no such care: their scores are masked.
#pragma once
#include "internal.h"
#include "kv4.cuh"
#include "tree_attn.cuh"

namespace dsv41 {

template <int NC, int NT>
struct RowsCfg {
    static constexpr int warps = 4, threads = warps * 32;
    static constexpr int rt = 8 * NT, kt = 16 * warps;    // rows and keys of a tile
    static constexpr int dim = NC * kKv4Chunk;
    // K: `nc` 32-bit words a lane, key and record. V: slices of `vcols` columns, `vw` words a lane, key and slice
    static constexpr bool wide = NC % 4 == 0;
    static constexpr int vw = wide ? 2 : 1, vslices = wide ? NC / 4 : (NC + 1) / 2, vcols = 64 * vw;
    static constexpr int q_pitch = (NC | 1) * 64;         // bytes of a row of Q: two neighbours lie in different banks
    static constexpr int o_pitch = dim + 4;               // floats
    static constexpr int q_b = rt * q_pitch, o_b = warps * rt * o_pitch * 4;
    static constexpr int smem = q_b + o_b;
    static constexpr int extra = 4;                       // what a segment costs beside its tiles, in tiles
    static constexpr int small = 8;                       // tiles of a part where segments have CTAs of their own
    // registers: O takes 8 NC NT, the codes and scales under way 12 to 40
    static constexpr int ctas = NC * NT <= 4 ? 4 : NC * NT <= 8 ? 3 : 2;
    // column of a lane's word x of a slice (V), and the chunk of word x (K)
    __host__ __device__ static constexpr int k_chunk(int x, int t) { return wide ? t + 4 * (x / 4) : NC == 2 ? t >> 1 : x; }
    __host__ __device__ static constexpr int k_word(int x, int t) { return wide ? x % 4 : NC == 2 ? 2 * (t & 1) + x : t; }
};

template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <int N>
__device__ __forceinline__ void load_words(const unsigned char* from, uint32_t* w)
{
    if constexpr (N == 4) {
        const uint4 v = load_early16(from);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = load_early8(from);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = load_early4(from);
    }
}

// chunks (bits) of NaN among the values that each row sees of the 16 keys from pos0 on: lane r answers for row r
template <typename T, int NC, int NT>
__device__ __noinline__ uint32_t nan_chunks(const TreeAttnParams& p, const UnitCursor<8 * NT, 64, true>* cursor, int pos0)
{
    const UnitCursor<8 * NT, 64, true> c = *cursor;
    const int lane = threadIdx.x & 31, at = c.rt * 8 * NT + lane;
    if (lane >= 8 * NT || at >= c.r.n * p.group) return 0;
    const uint64_t seen = seen_keys<true>(p, c.r, p.group_div.div(at), pos0);
    uint32_t chunks = 0;
#pragma unroll 1
    for (int k = 0; k < 16; ++k) {
        const int pos = pos0 + k;
        if (pos >= c.r.seq || !((seen >> k) & 1)) continue;
        const int pg = p.page_div.div(pos), id = p.block_table[(int64_t)c.b * p.table_stride + pg], in_page = pos - pg * p.page_size;
        if ((unsigned)id >= (unsigned)p.num_pages) continue;
        const unsigned char* rec = p.packed + (((int64_t)id * p.kv_heads + c.h) * 2 + 1) * kv4_block(p.page_size, NC) +
                                   (in_page / kKv4Tokens) * kv4_record(NC);
        for (int x = 0; x < NC; ++x)
            chunks |= (uint32_t)kv4_nan<T>(*reinterpret_cast<const uint32_t*>(rec + NC * kKv4Codes + x * kKv4Scales + (in_page % kKv4Tokens) * 4)) << x;
    }
    return chunks;
}

template <typename T, int NC, int NT>
__global__ void __launch_bounds__(RowsCfg<NC, NT>::threads, RowsCfg<NC, NT>::ctas) tree_attn4_rows_kernel(const __grid_constant__ TreeAttnParams p)
{
    using Cfg = RowsCfg<NC, NT>;
    constexpr int RT = Cfg::rt, KT = Cfg::kt, VW = Cfg::vw, VS = Cfg::vslices, DIM = Cfg::dim;
    using Cursor = UnitCursor<RT, KT, true>;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char* sq = smem;
    float* so = reinterpret_cast<float*>(smem + Cfg::q_b);       // [warp][row][column]
    __shared__ float2 s_ml[Cfg::warps][RT];
    __shared__ uint32_t s_nan[Cfg::warps][RT];                   // chunks of NaN that a row saw in masked tiles
    __shared__ CutShared<Cfg::warps> cut;
    __shared__ int s_last;
    __shared__ Cursor s_seg;                                     // the segment under way
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    int64_t run, v0;
    int part_tiles;
    cut_runs<RT, KT, true, Cfg::extra, Cfg::small>(p, cut, run, v0, part_tiles);
    __syncthreads();
    const int count = (int)(cut.end - cut.tiles0);
    if (count <= 0) return;
    Cursor ahead;   // of the tile that is looked up
    ahead.b = (int)cut.first[0];
    ahead.enter(p);
    ahead.h = (int)cut.first[1] / ahead.nrt;
    ahead.rt = (int)cut.first[1] - ahead.h * ahead.nrt;
    ahead.kt = part_tiles ? (int)cut.tiles0 : max((int)cut.first[2] - Cfg::extra, 0);
    ahead.place(p);
    if (tid == 0) s_seg = ahead;
    if (tid < Cfg::warps * RT) s_nan[tid / RT][tid % RT] = 0;
    __syncthreads();
    int64_t v_seg = v0 - cut.first[2];

    // ---- keys and values on their way ----
    constexpr int kRecord = kv4_record(NC);
    const int ps8 = p.page_size / kKv4Tokens;
    // this warp's record x of a tile, x = 0, 1 by lane parity: a page number that is on its way, and where in the page
    int id = -1, in_page = 0, head = 0;
    auto look_up = [&](const Cursor& c) {
        const int pos = c.tile() * KT + warp * 16 + (lane & 1) * kKv4Tokens, pg = p.page_div.div(pos);
        id = pos < c.r.seq ? __ldg(p.block_table + (int64_t)c.b * p.table_stride + pg) : -1;
        in_page = pos - pg * p.page_size;
        head = c.h;
    };
    uint32_t kc[2][NC], ks[2][Cfg::wide ? NC / 4 : NC == 2 ? 1 : NC];         // keys: [record][word]
    uint32_t vc[2][2][VS][VW], vs[2][2][VS];                                  // values: [record][key t, t + 4][slice][word]
    constexpr int KS = sizeof(ks[0]) / 4, W = NC / KS;
    const int kx = (g >> 1) + 4 * (g & 1);                                    // this lane's key of a record
    // a lane's codes and scales within a record of keys, of values
    const unsigned char* const k_codes = p.packed + Cfg::k_chunk(0, t) * kKv4Codes + kx * 16 + Cfg::k_word(0, t) * 4;
    const unsigned char* const k_scales = p.packed + NC * kKv4Codes + Cfg::k_chunk(0, t) * kKv4Scales + kx * 4;
    const int v_chunk = VW == 2 ? g >> 1 : g >> 2, v_word = VW == 2 ? 2 * (g & 1) : g & 3;   // of a slice
    const unsigned char* const v_codes = p.packed + v_chunk * kKv4Codes + t * 16 + v_word * 4;
    const unsigned char* const v_scales = p.packed + NC * kKv4Codes + v_chunk * kKv4Scales + t * 4;
    // The records of a tile, by number; 0 where there is none (past the end, or not a page of this cache): what is read there becomes
    // zeros before it is used.
    int rec[2];
    bool none[2] = {false, false}, none_next[2];
    auto resolve = [&]() {
        const int at = (unsigned)id < (unsigned)p.num_pages ? (id * p.kv_heads + head) * 2 * ps8 + in_page / kKv4Tokens : -1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            rec[x] = __shfl_sync(0xffffffffu, at, x);
            none_next[x] = rec[x] < 0;
            rec[x] = max(rec[x], 0);
        }
    };
    auto load_keys = [&]() {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* codes = k_codes + (int64_t)rec[x] * kRecord;
            const unsigned char* scales = k_scales + (int64_t)rec[x] * kRecord;
#pragma unroll
            for (int i = 0; i < NC; i += W) {   // (a lane's chunks: 4 apart, or neighbours, or one)
                load_words<W>(codes + (W == 4 ? i : i / W) * kKv4Codes, kc[x] + i);
                load_words<1>(scales + (W == 4 ? i : i / W) * kKv4Scales, ks[x] + i / W);
            }
        }
    };
    auto load_values = [&]() {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = none_next[x] ? 0 : rec[x] + ps8;
            const unsigned char* codes = v_codes + (int64_t)at * kRecord;
            const unsigned char* scales = v_scales + (int64_t)at * kRecord;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int s = 0; s < VS; ++s) {
                    constexpr int kChunks = 2 * VW;
                    if ((NC % kChunks) && s == VS - 1 && v_chunk >= NC % kChunks) {   // (an odd number of chunks: half of the last slice)
                        vc[x][j][s][0] = vs[x][j][s] = 0;
                        continue;
                    }
                    load_words<VW>(codes + s * kChunks * kKv4Codes + j * 64, vc[x][j][s]);
                    load_words<1>(scales + s * kChunks * kKv4Scales + j * 16, vs[x][j] + s);
                }
        }
    };

    float o[VS][VW][4][NT][4];   // [slice][word][pair of columns][8 rows][column, row]
    float m[NT][2], l[NT][2];    // of rows 2 t and 2 t + 1 of each 8
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < VS * VW * 4 * NT * 4; ++i) (&o[0][0][0][0][0])[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < NT; ++i) m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.0f;
    };
    // the segment's rows, each as [word x of a lane][t][16 bytes]: what lane t multiplies with its word x
    auto load_rows = [&]() {
        const Cursor& c = s_seg;
        const int rows = min(RT, c.r.n * p.group - c.rt * RT);
        for (int i = tid; i < RT * NC * 4; i += Cfg::threads) {
            const int row = i / (NC * 4), x = i / 4 % NC, tt = i & 3;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < rows) {
                const int at = c.rt * RT + row, n = p.group_div.div(at), hq = c.h * p.group + at - n * p.group;
                const T* q = static_cast<const T*>(p.q) + (int64_t)(c.r.q0 + n) * p.q_stride_token + (int64_t)hq * p.q_stride_head;
                v = *reinterpret_cast<const uint4*>(q + Cfg::k_chunk(x, tt) * kKv4Chunk + Cfg::k_word(x, tt) * 8);
            }
            *reinterpret_cast<uint4*>(sq + row * Cfg::q_pitch + x * 64 + tt * 16) = v;
        }
    };

    look_up(ahead);
    resolve();
    load_keys();
    load_values();
    auto look_ahead = [&](int tile) {   // tile: the one that `ahead` goes to
        id = -1;
        if (tile >= count) return;
        ahead.next(p);
        look_up(ahead);
    };
    look_ahead(1);
    load_rows();
    clear();
    __syncthreads();

    const float f = p.flip ? -p.scale_log2 : p.scale_log2;
    int kt = s_seg.kt, nkt = s_seg.nkt, kt_first = kt;
    int sinks, skip;            // of the segment: its list of tiles
    MaskedKeys<true> mask;
    auto enter = [&]() {
        const Cursor& c = s_seg;
        sinks = c.keys.sinks, skip = c.keys.skip;
        mask = masked_keys<RT, true>(p, c);
    };
    enter();
    for (int it = 0; it < count; ++it) {
        none[0] = none_next[0], none[1] = none_next[1];
        if (__builtin_expect(none[0] || none[1], 0)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (!none[x]) continue;
#pragma unroll
                for (int i = 0; i < KS; ++i) ks[x][i] = 0;
#pragma unroll
                for (int i = 0; i < 2 * VS; ++i) (&vs[x][0][0])[i] = 0;
            }
        }
        // ---- scores ----
        float s[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
        for (int x = 0; x < NC; ++x) {
            const uint32_t sa = ks[0][x / W], sb = ks[1][x / W];
            const uint32_t sa2 = prmt(sa, sa, 0x1010), la2 = prmt(sa, sa, 0x3232), sb2 = prmt(sb, sb, 0x1010), lb2 = prmt(sb, sb, 0x3232);
            const uint32_t a0[4] = {kv4_pair<T, 0>(kc[0][x], sa2, la2), kv4_pair<T, 0>(kc[1][x], sb2, lb2),
                                    kv4_pair<T, 1>(kc[0][x], sa2, la2), kv4_pair<T, 1>(kc[1][x], sb2, lb2)};
            const uint32_t a1[4] = {kv4_pair<T, 2>(kc[0][x], sa2, la2), kv4_pair<T, 2>(kc[1][x], sb2, lb2),
                                    kv4_pair<T, 3>(kc[0][x], sa2, la2), kv4_pair<T, 3>(kc[1][x], sb2, lb2)};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint4 b = *reinterpret_cast<const uint4*>(sq + (i * 8 + g) * Cfg::q_pitch + x * 64 + t * 16);
                mma16816<T>(s[i], a0, b.x, b.y);
                mma16816<T>(s[i], a1, b.z, b.w);
            }
        }
        // ---- the next tile's keys ----
        resolve();
        load_keys();
        look_ahead(it + 2);

        // ---- softmax ----
        const int pos0 = (kt < sinks ? kt : kt + skip) * KT;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] *= f;
        if (__builtin_expect(mask.template tile<KT>(p, pos0), 0)) {   // rows differ in what they see
            const AttnReq r = s_seg.r;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = min(s_seg.rt * RT + i * 8 + 2 * t + j, r.n * p.group - 1);
                    const uint64_t seen = r.seq > 0 ? seen_keys<true>(p, r, p.group_div.div(at), pos0) >> (warp * 16 + kx) : 0ull;
                    if (!(seen & 1)) s[i][j] = -INFINITY;
                    if (!((seen >> 8) & 1)) s[i][2 + j] = -INFINITY;
                }
            // values: past the last key anything may lie
            const int first = pos0 + warp * 16;
            bool odd = false;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int a = 0; a < VS; ++a) {
                        if (first + x * kKv4Tokens + t + 4 * j >= r.seq) vs[x][j][a] = 0;
                        odd |= kv4_nan<T>(vs[x][j][a]);
                    }
            if (__builtin_expect(__any_sync(0xffffffffu, odd), 0)) {
                const uint32_t chunks = nan_chunks<T, NC, NT>(p, &s_seg, first);
                if (lane < RT) s_nan[warp][lane] |= chunks;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2 * 2 * VS; ++i)
                    if (kv4_nan<T>((&vs[0][0][0])[i])) (&vs[0][0][0])[i] = 0;
            }
        }
        bool grow = false;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) grow |= fmaxf(s[i][j], s[i][2 + j]) > m[i][j] + 8.0f;   // (from -inf: any score)
        if (__builtin_expect(__any_sync(0xffffffffu, grow), 0)) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float keep[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(s[i][j], s[i][2 + j]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const bool up = top > m[i][j] + 8.0f;   // (all lanes of the row agree)
                    keep[j] = up ? exp2_fast(m[i][j] - top) : 1.0f;
                    if (up) m[i][j] = top;
                    l[i][j] *= keep[j];
                }
#pragma unroll
                for (int a = 0; a < VS; ++a)
#pragma unroll
                    for (int w = 0; w < VW; ++w)
#pragma unroll
                        for (int b = 0; b < 4; ++b)
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[a][w][b][i][j] *= keep[j & 1];
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const float b0 = m[i][0] == -INFINITY ? 0.0f : m[i][0], b1 = m[i][1] == -INFINITY ? 0.0f : m[i][1];
            const float e0 = exp2_fast(s[i][0] - b0), e1 = exp2_fast(s[i][1] - b1), e2 = exp2_fast(s[i][2] - b0), e3 = exp2_fast(s[i][3] - b1);
            l[i][0] += e0 + e2;
            l[i][1] += e1 + e3;
            pb[i][0] = turn8x8(pack2<T>(e0, e1));
            pb[i][1] = turn8x8(pack2<T>(e2, e3));
        }
        // ---- values ----
#pragma unroll
        for (int a = 0; a < VS; ++a) {
            const uint32_t s0 = prmt(vs[0][0][a], vs[0][1][a], 0x5410), l0 = prmt(vs[0][0][a], vs[0][1][a], 0x7632);
            const uint32_t s1 = prmt(vs[1][0][a], vs[1][1][a], 0x5410), l1 = prmt(vs[1][0][a], vs[1][1][a], 0x7632);
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                // even and odd columns of both keys of a pair
                const uint32_t x0 = prmt(vc[0][0][a][w], vc[0][1][a][w], 0x5410), y0 = prmt(vc[0][0][a][w], vc[0][1][a][w], 0x7632);
                const uint32_t x1 = prmt(vc[1][0][a][w], vc[1][1][a][w], 0x5410), y1 = prmt(vc[1][0][a][w], vc[1][1][a][w], 0x7632);
                auto product = [&](auto which) {
                    constexpr int b = decltype(which)::value;
                    const uint32_t v[4] = {kv4_pair<T, b>(x0, s0, l0), kv4_pair<T, b>(y0, s0, l0), kv4_pair<T, b>(x1, s1, l1), kv4_pair<T, b>(y1, s1, l1)};
#pragma unroll
                    for (int i = 0; i < NT; ++i) mma16816<T>(o[a][w][b][i], v, pb[i][0], pb[i][1]);
                };
                product(std::integral_constant<int, 0>());
                product(std::integral_constant<int, 1>());
                product(std::integral_constant<int, 2>());
                product(std::integral_constant<int, 3>());
            }
        }
        load_values();
        if (__builtin_expect(++kt < nkt && it < count - 1, 1)) continue;

        // ---- end of the segment, or of this CTA's run ----
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], d);
                if (g == 0) s_ml[warp][i * 8 + 2 * t + j] = make_float2(m[i][j], l[i][j]);
#pragma unroll
                for (int a = 0; a < VS; ++a)
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const int col = a * Cfg::vcols + g * 8 * VW + w * 8;
                        if (col >= DIM) continue;
                        float4* to = reinterpret_cast<float4*>(so + (warp * RT + i * 8 + 2 * t + j) * Cfg::o_pitch + col);
                        to[0] = make_float4(o[a][w][0][i][j], o[a][w][0][i][2 + j], o[a][w][1][i][j], o[a][w][1][i][2 + j]);
                        to[1] = make_float4(o[a][w][2][i][j], o[a][w][2][i][2 + j], o[a][w][3][i][j], o[a][w][3][i][2 + j]);
                    }
            }
        __syncthreads();
        const Cursor c = s_seg;
        const int rows = min(RT, c.r.n * p.group - c.rt * RT);
        const bool whole = kt_first == 0 && kt == nkt;
        const int slot = 2 * blockIdx.x + (kt_first > 0 ? 0 : 1);   // a part: its segment began in an earlier run, or not
        float4* part = reinterpret_cast<float4*>(p.part_o + (int64_t)slot * RT * DIM);   // [column / 4][row]
        for (int i = tid; i < rows * (DIM / 8); i += Cfg::threads) {
            const int row = i % rows, d = i / rows * 8;
            float top = -INFINITY, sum = 0.0f, v[8];
#pragma unroll
            for (int w = 0; w < Cfg::warps; ++w) top = fmaxf(top, s_ml[w][row].x);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
            bool nan = false;
#pragma unroll
            for (int w = 0; w < Cfg::warps; ++w) {
                const float2 ml = s_ml[w][row];
                const float e = exp2_fast(ml.x - base);
                sum += ml.y * e;
                const float4* from = reinterpret_cast<const float4*>(so + (w * RT + row) * Cfg::o_pitch + d);
                const float4 a = from[0], b = from[1];
                v[0] = fmaf(a.x, e, v[0]), v[1] = fmaf(a.y, e, v[1]), v[2] = fmaf(a.z, e, v[2]), v[3] = fmaf(a.w, e, v[3]);
                v[4] = fmaf(b.x, e, v[4]), v[5] = fmaf(b.y, e, v[5]), v[6] = fmaf(b.z, e, v[6]), v[7] = fmaf(b.w, e, v[7]);
                nan |= (s_nan[w][row] >> (d / kKv4Chunk)) & 1;
            }
            const float scale = nan ? NAN : !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= scale;
            if (whole) {
                const int at = c.rt * RT + row, n = p.group_div.div(at), hq = c.h * p.group + at - n * p.group;
                T* out = static_cast<T*>(p.out) + (int64_t)(c.r.q0 + n) * p.out_stride_token + (int64_t)hq * p.out_stride_head + d;
                *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
                if (d == 0 && p.lse)
                    p.lse[(int64_t)(c.r.q0 + n) * p.q_heads + hq] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
            } else {
                part[d / 4 * RT + row] = make_float4(v[0], v[1], v[2], v[3]);
                part[(d / 4 + 1) * RT + row] = make_float4(v[4], v[5], v[6], v[7]);
                if (d == 0) p.part_ml[(int64_t)slot * RT + row] = make_float2(top, sum);
            }
        }
        if (!whole) {
            const int fc = part_tiles ? (int)v_seg : (int)((v_seg + Cfg::extra) / run);   // runs with tiles of it
            const int lc = part_tiles ? fc + cut_parts(nkt, part_tiles) - 1 : (int)((v_seg + nkt + Cfg::extra - 1) / run);
            int* counter = p.counters + fc;
            __syncthreads();
            if (tid == 0) {
                __threadfence();   // the CTA's stores, ordered before this thread by the barrier
                const bool all_in = atomicAdd(counter, 1) == lc - fc;
                if (all_in) __threadfence();
                s_last = all_in;
            }
            __syncthreads();
            if (s_last) {
                JoinArgs a;
                a.ml = p.part_ml;
                a.o = reinterpret_cast<const float4*>(p.part_o);
                a.out = static_cast<T*>(p.out) + c.r.q0 * p.out_stride_token + (int64_t)c.h * p.group * p.out_stride_head;
                a.lse = p.lse ? p.lse + (int64_t)c.r.q0 * p.q_heads + c.h * p.group : nullptr;
                a.stride_token = p.out_stride_token, a.stride_head = p.out_stride_head;
                a.group_div = p.group_div;
                a.group = p.group, a.q_heads = p.q_heads, a.head_dim = DIM, a.row0 = c.rt * RT;
                join_parts<T, DIM, RT>(a, fc, lc, 0, rows, tid, Cfg::threads);
                if (tid == 0) *counter = 0;   // ready for the next call
            }
        }
        if (it == count - 1) break;
        __syncthreads();   // all have read the segment's place, rows and sums
        if (tid == 0) {
            Cursor n = c;
            n.kt = nkt - 1;
            n.next(p);
            s_seg = n;
        }
        if (tid < Cfg::warps * RT) s_nan[tid / RT][tid % RT] = 0;
        v_seg += nkt + Cfg::extra;
        __syncthreads();
        kt = kt_first = 0;
        nkt = s_seg.nkt;
        enter();
        load_rows();
        clear();
        __syncthreads();
    }
}

template <typename T, int NC, int NT>
static cudaError_t launch_rows(const TreeAttnParams& p, cudaStream_t st)
{
    using Cfg = RowsCfg<NC, NT>;
    auto kernel = tree_attn4_rows_kernel<T, NC, NT>;
    static bool ready[64] = {};   // the attribute is per device and kernel, and stays
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    static_assert(Cfg::ctas <= kAttnCtas && Cfg::ctas * Cfg::rt <= 128, "workspace: parts and counters");
    kernel<<<num_sms() * Cfg::ctas, Cfg::threads, Cfg::smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int NC>
static cudaError_t launch_rows_tile(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    return max_rows <= 8 ? launch_rows<T, NC, 1>(p, st) : launch_rows<T, NC, 2>(p, st);
}

template <typename T>
static cudaError_t launch_tree_attn4_rows(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    switch (p.head_dim / kKv4Chunk) {
        case 1: return launch_rows_tile<T, 1>(p, max_rows, st);
        case 2: return launch_rows_tile<T, 2>(p, max_rows, st);
        case 3: return launch_rows_tile<T, 3>(p, max_rows, st);
        case 4: return launch_rows_tile<T, 4>(p, max_rows, st);
        case 5: return launch_rows_tile<T, 5>(p, max_rows, st);
        case 6: return launch_rows_tile<T, 6>(p, max_rows, st);
        case 7: return launch_rows_tile<T, 7>(p, max_rows, st);
        default: return launch_rows_tile<T, 8>(p, max_rows, st);
    }
}

}  // namespace dsv41
