// Attention of few rows over a cache in 4 bits (tree_attn.cu has the mathematics, kv4.cuh the cache): warp-level matrix
// instructions on codes decoded in registers.
//
// Both products take the cache's side as their A operand, so that what a lane decodes is its fragment:
// S^T = K Q^T (16 keys by 8 rows an instruction), O^T += V^T P^T (16 columns by 8 rows).
// A tile of keys is 32 for each warp, which takes 16 at a time, two records of 8 tokens:
//   K   lane (g, t) holds words of key g of each record (g permuted: see below); a word of 8 columns is one register of two
//       instructions' A, whose columns are matched by the order in which Q lies in shared memory
//   V   lane (g, t) holds words of keys t and t + 4 of each record; the keys of a pair are merged by byte permutes before they are
//       decoded, so a pair is one column of two keys
//   P   leaves the first product with keys down and rows across, and is turned by movmatrix into the B operand of the second
// The k-th pair of keys in V's and P's order is (t, t + 4); row x of the first product is key (x >> 1) + 4 (x & 1) of its record.
// A warp's records are copied to a ring of its own in shared memory (cp.async; 2 to 4 steps of 16 keys), where a
// lane's words are constant offsets from a stage's address. Registers had no room for words on their way: what was spilled for them waited for
// the loads. The products of a step's values and of the next step's keys are one stretch of code, two chains
// that hide each other's latencies.
//
// Every warp has its own running maximum, sum and O (RT = 8 or 16 rows); nothing is exchanged before the end of a segment, where the
// four warps of a CTA join through shared memory. The deferred rescale, P's rounding and the exponentials are those of the
// other kernel (tree_attn_kernel.cuh).
//
// Measured: one token of 8 rows a KV head (8 heads of 128, bf16) over 4 requests of 65-131k keys 141 us, 3.5 TB/s of codes (floor 75 us);
// one request of 131k keys 68 us (26); 4 of 32-64k keys 80 us, with 16 rows 100 us. Bound by instructions: 420 a step of 16 keys, 256 of
// them the decoding (a shift or mask, two 16-bit operations for two values), at 0.6 a cycle and scheduler: ALU 41%, fp16 and
// integer products 43% of their pipes, matrix instructions 16%, loads hardly waited for. A fifth or more of a call this size is start (lengths,
// pages, first records: 8 us) and join. More CTAs an SM, loads to registers, bulk copies measured the same or slower.
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
    static constexpr int rt = 8 * NT, kt = 32 * warps;    // rows and keys of a tile
    static constexpr int dim = NC * kKv4Chunk;
    // K: NC 32-bit words a lane, key and record, k_width at a time. V: slices of `vcols` columns, `vw` words a lane, key and slice
    static constexpr bool wide = NC % 4 == 0;
    static constexpr int k_width = wide ? 4 : NC == 2 ? 2 : 1, k_scales = NC / k_width;
    static constexpr int vw = wide ? 2 : 1, vslices = wide ? NC / 4 : (NC + 1) / 2, vcols = 64 * vw;
    static constexpr int record_b = kv4_record(NC), stage_b = 4 * record_b;   // 16 keys: two records of keys, two of values
    static constexpr int q_pitch = (NC | 1) * 64;         // bytes of a row of Q: two neighbours lie in different banks
    static constexpr int o_regs = vslices * vw * 4 * NT * 4;
    static constexpr int q_b = rt * q_pitch, o_b = 2 * o_regs * 128;
    static constexpr int extra = 2;                       // what a segment costs beside its tiles, in tiles
    static constexpr int small = 2;                       // tiles of a part where segments have CTAs of their own
    static constexpr int ctas = o_regs <= 16 ? 4 : o_regs <= 64 ? 3 : 2;   // (registers; 4 of 32: a tenth spilled, no faster)
    static constexpr int fit = (232448 / ctas - 4096 - q_b - o_b) / (warps * stage_b), stages = fit < 4 ? fit : 4;
    static_assert(stages >= 2, "keys of two steps");
    static constexpr int smem = q_b + o_b + warps * stages * stage_b;
    // chunk of a lane's word x of keys, and the word within that
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
// f(0), ..., f(N - 1), each as a constant
template <typename F, int... I>
__device__ __forceinline__ void for_each_of(F f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F f)
{
    for_each_of(f, std::make_integer_sequence<int, N>());
}

__device__ __forceinline__ void send16(uint32_t to, const unsigned char* from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
template <int N>
__device__ __forceinline__ void get_words(uint32_t from, uint32_t* w)
{
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(from) : "memory");
}
__device__ __forceinline__ void put_word(uint32_t to, uint32_t w) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(w) : "memory"); }

// chunks (bits) of NaN among the values that each row sees of the 16 keys from pos0 on: lane r answers for row r
template <typename T, int NC, int NT>
__device__ __noinline__ uint32_t nan_chunks(const TreeAttnParams& p, const UnitCursor<8 * NT, RowsCfg<NC, NT>::kt, true>* cursor, int pos0)
{
    const UnitCursor<8 * NT, RowsCfg<NC, NT>::kt, true> c = *cursor;
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

// Join of a segment's parts (runs fc .. lc) by the CTA that arrived last: the parts' weights first, in shared memory, then each thread sums 4 columns of
// a row over all parts, in order, with many loads in flight. (16 columns a thread and a batch of 4 parts at a time, each
// rescaled as it came, took 12 to 16 us for 24 parts and 30 us for 74: a trip to L2 a batch.)
template <typename T, int NC, int NT>
__device__ __noinline__ void join_rows(const TreeAttnParams& p, const UnitCursor<8 * NT, RowsCfg<NC, NT>::kt, true>& c, int rows, int fc, int lc, float* room)
{
    using Cfg = RowsCfg<NC, NT>;
    constexpr int RT = Cfg::rt, DIM = Cfg::dim, kStep = Cfg::threads / RT, kItems = RT * DIM / 4, kPer = (kItems + Cfg::threads - 1) / Cfg::threads;
    constexpr int kMost = Cfg::o_b / 4 / RT - 2 * kStep;    // parts whose weights there is room for at a time
    const int tid = threadIdx.x, r = tid % RT, k = tid / RT, parts = lc - fc + 1;
    float *red = room, *sums = room + kStep * RT, *weight = room + 2 * kStep * RT;
    auto slot = [&](int q) { return (int64_t)2 * (fc + q) + (q == 0 ? 1 : 0); };
    float top = -INFINITY, sum = 0.0f;
    for (int q = k; q < parts; q += kStep) top = fmaxf(top, __ldcg(p.part_ml + slot(q) * RT + r).x);
    red[k * RT + r] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kStep; ++i) top = fmaxf(top, red[i * RT + r]);
    const float base = top == -INFINITY ? 0.0f : top;
    float4 acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = make_float4(0, 0, 0, 0);
    for (int q0 = 0; q0 < parts; q0 += kMost) {
        const int n = min(kMost, parts - q0);
        for (int q = k; q < n; q += kStep) {
            const float2 v = __ldcg(p.part_ml + slot(q0 + q) * RT + r);
            const float w = exp2_fast(v.x - base);
            sum = fmaf(v.y, w, sum);
            weight[q * RT + r] = w;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int item = tid + i * Cfg::threads, row = item % RT;
            if (item >= kItems) break;
            const float4* from = reinterpret_cast<const float4*>(p.part_o) + item;   // [column / 4][row]
            constexpr int kBatch = 12;
#pragma unroll 1
            for (int q = 0; q < n; q += kBatch) {
                float4 v[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) v[j] = q + j < n ? __ldcg(from + slot(q0 + q + j) * kItems) : make_float4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const float w = q + j < n ? weight[(q + j) * RT + row] : 0.0f;
                    acc[i].x = fmaf(v[j].x, w, acc[i].x), acc[i].y = fmaf(v[j].y, w, acc[i].y);
                    acc[i].z = fmaf(v[j].z, w, acc[i].z), acc[i].w = fmaf(v[j].w, w, acc[i].w);
                }
            }
        }
        __syncthreads();
    }
    sums[k * RT + r] = sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int item = tid + i * Cfg::threads, row = item % RT, col = item / RT * 4;
        if (item >= kItems || row >= rows) continue;
        float l = 0.0f, m = -INFINITY;
        for (int j = 0; j < kStep; ++j) l += sums[j * RT + row], m = fmaxf(m, red[j * RT + row]);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int at = c.rt * RT + row, t = p.group_div.div(at), hq = c.h * p.group + at - t * p.group;
        T* out = static_cast<T*>(p.out) + (int64_t)(c.r.q0 + t) * p.out_stride_token + (int64_t)hq * p.out_stride_head + col;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(acc[i].x * inv, acc[i].y * inv), pack2<T>(acc[i].z * inv, acc[i].w * inv));
        if (col == 0 && p.lse) p.lse[(int64_t)(c.r.q0 + t) * p.q_heads + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
}

template <typename T, int NC, int NT>
__global__ void __launch_bounds__(RowsCfg<NC, NT>::threads, RowsCfg<NC, NT>::ctas) tree_attn4_rows_kernel(const __grid_constant__ TreeAttnParams p)
{
    using Cfg = RowsCfg<NC, NT>;
    constexpr int RT = Cfg::rt, KT = Cfg::kt, VW = Cfg::vw, VS = Cfg::vslices, DIM = Cfg::dim, KS = Cfg::k_scales, W = Cfg::k_width;
    using Cursor = UnitCursor<RT, KT, true>;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char* sq = smem;
    float* so = reinterpret_cast<float*>(smem + Cfg::q_b);       // [warp & 1][register of O][lane]
    __shared__ float2 s_ml[Cfg::warps][RT];
    __shared__ uint32_t s_nan[Cfg::warps][RT];                   // chunks of NaN that a row saw in masked tiles
    __shared__ CutShared<Cfg::warps> cut;
    __shared__ int s_last;
    __shared__ Cursor s_seg, s_ahead[Cfg::warps];                // the segment under way, and that of the tile each warp looks up
    __shared__ int64_t s_place;                                  // place on the line where the segment begins
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    int64_t run, v0;
    int part_tiles;
    cut_runs<RT, KT, true, Cfg::extra, Cfg::small>(p, cut, run, v0, part_tiles);
    __syncthreads();
    const int count = (int)(cut.end - cut.tiles0);
    if (count <= 0) return;
    if (tid < Cfg::warps) {
        Cursor c;
        c.b = (int)cut.first[0];
        c.enter(p);
        c.h = (int)cut.first[1] / c.nrt;
        c.rt = (int)cut.first[1] - c.h * c.nrt;
        c.kt = part_tiles ? (int)cut.tiles0 : max((int)cut.first[2] - Cfg::extra, 0);
        c.place(p);
        s_ahead[tid] = c;
        if (tid == 0) s_seg = c, s_place = v0 - cut.first[2];
    }
    if (tid < Cfg::warps * RT) s_nan[tid / RT][tid % RT] = 0;
    __syncthreads();

    // ---- keys and values on their way ----
    const int blocks = 2 * count;   // steps of 16 keys a warp
    constexpr int kRecord = Cfg::record_b;
    const int ps8 = p.page_size / kKv4Tokens;
    // The tile that is looked up: what changes only with the row tile lies in shared memory.
    int a_kt, a_nkt, a_sinks, a_skip, a_seq, a_head;
    const int* a_pages;
    auto enter_ahead = [&]() {
        const Cursor& c = s_ahead[warp];
        a_kt = c.kt, a_nkt = c.nkt, a_sinks = c.keys.sinks, a_skip = c.keys.skip, a_seq = c.r.seq, a_head = c.h;
        a_pages = p.block_table + (int64_t)c.b * p.table_stride;
    };
    // this warp's record x of it, x = 0 .. 3 by lane: a page number that is on its way, and where in the page
    int id = -1, in_page = 0;
    auto look_up = [&]() {
        const int pos = (a_kt < a_sinks ? a_kt : a_kt + a_skip) * KT + warp * 32 + (lane & 3) * kKv4Tokens, pg = p.page_div.div(pos);
        id = pos < a_seq ? __ldg(a_pages + pg) : -1;
        in_page = pos - pg * p.page_size;
    };
    // The records of a tile, a lane each, by number; -1 where there is none (past the end, or not a page of this cache): its scales
    // become zeros in shared memory.
    int rec;
    auto resolve = [&]() {
        rec = (unsigned)id < (unsigned)p.num_pages ? (id * p.kv_heads + a_head) * 2 * ps8 + in_page / kKv4Tokens : -1;
    };
    auto look_ahead = [&](int tile) {   // to the next one, which is tile `tile` of the run
        id = -1;
        if (tile >= count) return;
        if (__builtin_expect(++a_kt == a_nkt, 0)) {
            Cursor c = s_ahead[warp];
            c.kt = a_nkt - 1;
            c.next(p);
            __syncwarp();
            if (lane == 0) s_ahead[warp] = c;
            __syncwarp();
            enter_ahead();
        }
        look_up();
    };
    // The warp's ring: 16 keys a stage, [keys: record 0, 1][values: record 0, 1].
    constexpr int S = Cfg::stages;
    const uint32_t ring = smem_addr(smem) + Cfg::q_b + Cfg::o_b + warp * S * Cfg::stage_b;
    uint32_t none = 0;        // two bits for each 16 keys that have been sent for, from the ones under way on: records that there are not
    int sent = 0, to_stage = 0;
    const unsigned char* const from_lane = p.packed + lane * 16;
    auto send = [&]() {       // for the next 16 keys, as one line of 16-byte pieces, a lane every 32nd
        if (sent < blocks) {
            const int block = sent & 1;
            if (block == 0) {
                resolve();
                look_ahead(sent / 2 + 1);
            }
            const uint32_t to = ring + to_stage * Cfg::stage_b + lane * 16;
            const uint32_t live = __ballot_sync(0xffffffffu, rec >= 0) >> (2 * block);
            none |= (~live & 3) << (2 * min(sent, S - 1));
            constexpr int kPieces = kRecord / 16;
#pragma unroll
            for (int i = 0; i < 4 * kPieces; i += 32) {
                // record of the line: keys 0, 1, values 0, 1
                int r = i / kPieces;
#pragma unroll
                for (int next = (i / kPieces + 1) * kPieces; next < i + 32; next += kPieces) r += lane >= next - i;
                const int at = __shfl_sync(0xffffffffu, rec, 2 * block + (r & 1));
                if (at >= 0 && r < 4) send16(to + i * 16, from_lane + (int64_t)(at - r + (r >= 2 ? ps8 : 0)) * kRecord + i * 16);
            }
            if (++to_stage == S) to_stage = 0;
        }
        ++sent;
        cp_async_commit();
    };

    float o[VS][VW][4][NT][4];   // [slice][word][pair of columns][8 rows][column, row]
    float m[NT][2], l[NT][2];    // of rows 2 t and 2 t + 1 of each 8
    constexpr int kO = VS * VW * 4 * NT * 4;
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < kO; ++i) (&o[0][0][0][0][0])[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < NT; ++i) m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.0f;
    };
    // the segment's rows, each as [word x of a lane][t][16 bytes]: what lane t multiplies with its word x
    auto load_rows = [&]() {
        const Cursor& c = s_seg;
        const int rows = min(RT, c.r.n * p.group - c.rt * RT);
        for (int i = tid; i < RT * NC * 4; i += Cfg::threads) {
            const int row = i / (NC * 4), x = i / 4 % NC, tt = i & 3;
            const int at = min(c.rt * RT + row, c.r.n * p.group - 1), n = p.group_div.div(at), hq = c.h * p.group + at - n * p.group;
            const T* q = static_cast<const T*>(p.q) + (int64_t)(c.r.q0 + n) * p.q_stride_token + (int64_t)hq * p.q_stride_head;
            cp_async16(smem_addr(sq) + row * Cfg::q_pitch + x * 64 + tt * 16, q + Cfg::k_chunk(x, tt) * kKv4Chunk + Cfg::k_word(x, tt) * 8, row < rows);
        }
        cp_async_commit();
    };

    enter_ahead();
    look_up();
    load_rows();
    for (int i = 0; i < S; ++i) send();
    clear();
    cp_async_wait<S>();   // the rows
    __syncthreads();

    const float f = p.flip ? -p.scale_log2 : p.scale_log2;
    int kt, nkt, kt_first, sinks, skip;   // of the segment: tile and tiles, its list of tiles
    MaskedKeys<true> mask;
    auto enter = [&]() {
        const Cursor& c = s_seg;
        kt = kt_first = c.kt, nkt = c.nkt, sinks = c.keys.sinks, skip = c.keys.skip;
        mask = masked_keys<RT, true>(p, c);
    };
    enter();
    int stage = 0;
    // the keys after those under way (and before the ones sent for last) have landed in a stage; where there are no such records,
    // their scales become zeros
    auto landed = [&](int at, uint32_t missing) {
        cp_async_wait<S - 2>();
        __syncwarp();
        if (__builtin_expect(missing != 0, 0)) {
            const uint32_t to = ring + at * Cfg::stage_b + NC * kKv4Codes + lane * 4;
            for (int x = 0; x < 4; ++x)
                if ((missing >> (x & 1)) & 1)
                    for (int i = 0; i < NC * kKv4Scales; i += 128)
                        if (i + lane * 4 < NC * kKv4Scales) put_word(to + x * kRecord + i, 0);
            __syncwarp();
        }
    };
    // this lane's key of a record of keys, its words of a slice of values, and its places in a stage
    const int kx = (g >> 1) + 4 * (g & 1), v_chunk = VW == 2 ? g >> 1 : g >> 2, v_word = VW == 2 ? 2 * (g & 1) : g & 3;
    const uint32_t k_at = Cfg::k_chunk(0, t) * kKv4Codes + kv4_place(Cfg::k_chunk(0, t), kx) * 16 + Cfg::k_word(0, t) * 4;
    const uint32_t ks_at = NC * kKv4Codes + Cfg::k_chunk(0, t) * kKv4Scales + kx * 4;
    uint32_t v_at[2];               // (of keys t and t + 4)
#pragma unroll
    for (int j = 0; j < 2; ++j) v_at[j] = 2 * kRecord + v_chunk * kKv4Codes + kv4_place(v_chunk, t + 4 * j) * 16 + v_word * 4;
    const uint32_t vs_at = 2 * kRecord + NC * kKv4Codes + v_chunk * kKv4Scales + t * 4;
    float s[NT][4], s_odd[NT][4];   // scores, in two sums: shorter chains
    uint32_t pb[NT][2];             // their weights, as the second product's operand
    uint32_t vs[2][2][VS];          // scales of values: [record][key t, t + 4][slice]
    // word group x0 of the keys of a stage
    auto add_scores = [&](uint32_t from, auto group) {
        constexpr int x0 = decltype(group)::value * W;
        constexpr int kStep = W == 4 ? x0 : x0 / W;   // a lane's chunks: 4 apart, or neighbours, or one
        uint32_t c[2][W], sc[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            // (chunks that are not a multiple of 4 apart have other places)
            const uint32_t at = W == 1 ? x0 * kKv4Codes + kv4_place(x0, kx) * 16 + t * 4 : k_at + kStep * kKv4Codes;
            get_words<W>(from + x * kRecord + at, c[x]);
            get_words<1>(from + x * kRecord + ks_at + kStep * kKv4Scales, sc + x);
        }
        const Scale2<T> sa(sc[0]), sb(sc[1]);
#pragma unroll
        for (int x = 0; x < W; ++x) {
            const uint32_t a0[4] = {kv4_pair<T, 0>(c[0][x], sa), kv4_pair<T, 0>(c[1][x], sb), kv4_pair<T, 1>(c[0][x], sa), kv4_pair<T, 1>(c[1][x], sb)};
            const uint32_t a1[4] = {kv4_pair<T, 2>(c[0][x], sa), kv4_pair<T, 2>(c[1][x], sb), kv4_pair<T, 3>(c[0][x], sa), kv4_pair<T, 3>(c[1][x], sb)};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint4 b = *reinterpret_cast<const uint4*>(sq + (i * 8 + g) * Cfg::q_pitch + (x0 + x) * 64 + t * 16);
                mma16816<T>(s[i], a0, b.x, b.y);
                mma16816<T>(s_odd[i], a1, b.z, b.w);
            }
        }
    };
    auto get_value_scales = [&](uint32_t from) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int a = 0; a < VS; ++a) {
                    constexpr int kChunks = 2 * VW;
                    vs[x][j][a] = 0;
                    if (!((NC % kChunks) && a == VS - 1 && v_chunk >= NC % kChunks))   // (an odd number of chunks: half of the last slice)
                        get_words<1>(from + x * kRecord + vs_at + a * kChunks * kKv4Scales + j * 16, &vs[x][j][a]);
                }
    };
    // slice a of the values of a stage, weighted
    auto add_values = [&](uint32_t from, auto slice) {
        constexpr int a = decltype(slice)::value, kChunks = 2 * VW;
        uint32_t c[2][2][VW];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // (slices of two chunks: places differ; a chunk that there is not has scales of 0, whatever is read for it)
                const uint32_t at = VW == 2 || a % 2 == 0 ? v_at[j] : v_at[j] + (kv4_place(2 + v_chunk, t + 4 * j) - kv4_place(v_chunk, t + 4 * j)) * 16;
                get_words<VW>(from + x * kRecord + a * kChunks * kKv4Codes + at, c[x][j]);
            }
        const Scale2<T> s0(vs[0][0][a], vs[0][1][a]), s1(vs[1][0][a], vs[1][1][a]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            // even and odd columns of both keys of a pair
            const uint32_t x0 = prmt(c[0][0][w], c[0][1][w], 0x5410), y0 = prmt(c[0][0][w], c[0][1][w], 0x7632);
            const uint32_t x1 = prmt(c[1][0][w], c[1][1][w], 0x5410), y1 = prmt(c[1][0][w], c[1][1][w], 0x7632);
            auto product = [&](auto which) {
                constexpr int b = decltype(which)::value;
                const uint32_t v[4] = {kv4_pair<T, b>(x0, s0), kv4_pair<T, b>(y0, s0), kv4_pair<T, b>(x1, s1), kv4_pair<T, b>(y1, s1)};
#pragma unroll
                for (int i = 0; i < NT; ++i) mma16816<T>(o[a][w][b][i], v, pb[i][0], pb[i][1]);
            };
            product(std::integral_constant<int, 0>());
            product(std::integral_constant<int, 1>());
            product(std::integral_constant<int, 2>());
            product(std::integral_constant<int, 3>());
        }
    };
    auto clear_scores = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = s_odd[i][j] = 0.0f;
    };
    auto scores = [&](int at) {
        const uint32_t from = ring + at * Cfg::stage_b;
        clear_scores();
        for_each<KS>([&](auto x) { add_scores(from, x); });
    };
    // scores to weights: key x of the record, first + 8 record + key
    auto softmax = [&](int first, bool masked) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = (s[i][j] + s_odd[i][j]) * f;
        if (__builtin_expect(masked, 0)) {   // rows differ in what they see
            const AttnReq r = s_seg.r;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = min(s_seg.rt * RT + i * 8 + 2 * t + j, r.n * p.group - 1);
                    const uint64_t seen = r.seq > 0 ? seen_keys<true>(p, r, p.group_div.div(at), first) >> kx : 0ull;
                    if (!(seen & 1)) s[i][j] = -INFINITY;
                    if (!((seen >> 8) & 1)) s[i][2 + j] = -INFINITY;
                }
            bool odd = false;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int a = 0; a < VS; ++a) {
                        if (first + x * kKv4Tokens + t + 4 * j >= r.seq) vs[x][j][a] = 0;   // (anything may lie there)
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
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const float b0 = m[i][0] == -INFINITY ? 0.0f : m[i][0], b1 = m[i][1] == -INFINITY ? 0.0f : m[i][1];
            const float e0 = exp2_fast(s[i][0] - b0), e1 = exp2_fast(s[i][1] - b1), e2 = exp2_fast(s[i][2] - b0), e3 = exp2_fast(s[i][3] - b1);
            l[i][0] += e0 + e2;
            l[i][1] += e1 + e3;
            pb[i][0] = turn8x8(pack2<T>(e0, e1));
            pb[i][1] = turn8x8(pack2<T>(e2, e3));
        }
    };
    landed(0, none & 3);
    scores(0);
    for (int it = 0; it < count; ++it) {
        const int pos0 = (kt < sinks ? kt : kt + skip) * KT;
        const bool masked = mask.template tile<KT>(p, pos0);
#pragma unroll 1
        for (int block = 0; block < 2; ++block) {
            const uint32_t from = ring + stage * Cfg::stage_b;
            get_value_scales(from);
            softmax(pos0 + warp * 32 + block * 16, masked);
            // the values, and the scores of the next 16 keys if they are of the same rows
            const int next = stage + 1 == S ? 0 : stage + 1;
            if (__builtin_expect(block == 0 || (kt + 1 < nkt && it + 1 < count), 1)) {
                landed(next, (none >> 2) & 3);
                const uint32_t ahead = ring + next * Cfg::stage_b;
                clear_scores();
                for_each<(KS > VS ? KS : VS)>([&](auto x) {
                    constexpr int i = decltype(x)::value;
                    if constexpr (i < KS) add_scores(ahead, x);
                    if constexpr (i < VS) add_values(from, x);
                });
            } else {
                for_each<VS>([&](auto x) { add_values(from, x); });
            }
            __syncwarp();
            none >>= 2;
            stage = next;
            send();   // into the stage that has been read
        }
        if (__builtin_expect(++kt < nkt && it < count - 1, 1)) continue;

        // ---- end of the segment, or of this CTA's run: warps 2 and 3 join 0 and 1, then 1 joins 0, which puts the rows out ----
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], d);
                if (g == 0) s_ml[warp][i * 8 + 2 * t + j] = make_float2(m[i][j], l[i][j]);
            }
        __syncthreads();
        const Cursor c = s_seg;
        const int rows = min(RT, c.r.n * p.group - c.rt * RT);
        const bool whole = kt_first == 0 && kt == nkt;
        float sum[NT][2];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float keep[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < Cfg::warps; ++w) top = fmaxf(top, s_ml[w][i * 8 + 2 * t + j].x);
                const float base = top == -INFINITY ? 0.0f : top;
                sum[i][j] = 0.0f;
#pragma unroll
                for (int w = 0; w < Cfg::warps; ++w) sum[i][j] += s_ml[w][i * 8 + 2 * t + j].y * exp2_fast(s_ml[w][i * 8 + 2 * t + j].x - base);
                keep[j] = exp2_fast(m[i][j] - base) * (!whole ? 1.0f : sum[i][j] == 0.0f ? 0.0f : 1.0f / sum[i][j]);
                m[i][j] = top;
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
        float* mine = so + (warp & 1) * kO * 32 + lane;
        if (warp >= 2) {
#pragma unroll
            for (int i = 0; i < kO; ++i) mine[i * 32] = (&o[0][0][0][0][0])[i];
        }
        __syncthreads();
        if (warp < 2) {
#pragma unroll
            for (int i = 0; i < kO; ++i) (&o[0][0][0][0][0])[i] += mine[i * 32];
            if (warp == 1) {
#pragma unroll
                for (int i = 0; i < kO; ++i) mine[i * 32] = (&o[0][0][0][0][0])[i];
            }
        }
        __syncthreads();
        const int slot = 2 * blockIdx.x + (kt_first > 0 ? 0 : 1);   // a part: its segment began in an earlier run, or not
        if (warp == 0) {
            float4* part = reinterpret_cast<float4*>(p.part_o + (int64_t)slot * RT * DIM);   // [column / 4][row]
#pragma unroll
            for (int i = 0; i < kO; ++i) (&o[0][0][0][0][0])[i] += mine[kO * 32 + i * 32];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = i * 8 + 2 * t + j;
                    if (row >= rows) continue;
                    const uint32_t nan = s_nan[0][row] | s_nan[1][row] | s_nan[2][row] | s_nan[3][row];
                    const int at = c.rt * RT + row, n = p.group_div.div(at), hq = c.h * p.group + at - n * p.group;
                    T* out = static_cast<T*>(p.out) + (int64_t)(c.r.q0 + n) * p.out_stride_token + (int64_t)hq * p.out_stride_head;
#pragma unroll
                    for (int a = 0; a < VS; ++a)
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            const int col = a * Cfg::vcols + g * 8 * VW + w * 8;
                            if (col >= DIM) continue;
                            float v[8];
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                v[2 * b] = o[a][w][b][i][j], v[2 * b + 1] = o[a][w][b][i][2 + j];
                                if ((nan >> (col / kKv4Chunk)) & 1) v[2 * b] = v[2 * b + 1] = NAN;
                            }
                            if (whole) {
                                *reinterpret_cast<uint4*>(out + col) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
                            } else {
                                part[col / 4 * RT + row] = make_float4(v[0], v[1], v[2], v[3]);
                                part[(col / 4 + 1) * RT + row] = make_float4(v[4], v[5], v[6], v[7]);
                            }
                        }
                    if (g > 0) continue;
                    if (!whole) p.part_ml[(int64_t)slot * RT + row] = make_float2(m[i][j], sum[i][j]);
                    else if (p.lse)
                        p.lse[(int64_t)(c.r.q0 + n) * p.q_heads + hq] = sum[i][j] == 0.0f ? -INFINITY : (m[i][j] + log2f(sum[i][j])) * 0.6931471805599453f;
                }
        }
        if (!whole) {
            const int64_t v_seg = s_place;
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
                join_rows<T, NC, NT>(p, c, rows, fc, lc, so);
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
            s_place += nkt + Cfg::extra;
        }
        if (tid < Cfg::warps * RT) s_nan[tid / RT][tid % RT] = 0;
        __syncthreads();
        enter();
        load_rows();
        clear();
        cp_async_wait<0>();
        __syncthreads();
        landed(stage, none & 3);
        scores(stage);
    }
    cp_async_wait<0>();
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
