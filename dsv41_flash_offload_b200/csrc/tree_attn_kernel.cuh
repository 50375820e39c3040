// Attention of drafted tokens over a paged cache on the fifth-generation tensor cores (tree_attn.cu has the
// mathematics, the rows and the cut of the work into runs).
//
// One CTA per SM walks its run of (request, KV head, row tile, key tile) units:
//   producers            (over a cache in 4 bits: four or eight warps that decode codes into the same tiles)
//                        key and value tiles (128 keys; 64 for head sizes over 128) into a ring of units, in the
//                        128-byte swizzle the tensor cores read. Whole pages go by tensor copies (one or two warps, a lane
//                        per page and 64 columns); page sizes that do not make up a tile are gathered key by key by four
//                        warps of cp.async, whose issue rate then bounds a call (16 tokens x 8 rows over 4 x 64-128k keys:
//                        332 us for 270)
//   Q loaders            the rows of the segment
//   two issuers (1 thread each)  S = Q K^T (A and B from shared memory) and O += P V (A from tensor memory, V read
//                        as it lies, N-major), fp32 accumulators in tensor memory. One thread for both left the tensor
//                        pipe idle between its waits and commits (2900 cycles of issuing per tile)
//   softmax (4 or 8 warps per 128 rows; one or two threads per row, who share its keys)  S out of tensor memory,
//                        running maximum and sum, P back into tensor memory as 16-bit pairs; at the end of a segment
//                        O out. A single warp per sub-partition spends most of its time on latencies: with 4 warps a
//                        tile of 128 rows took 4700 cycles for 128 exponentials a thread
// The product of tile i + 1 runs while tile i is in the softmax (two S and P buffers for up to 128 rows; two row
// tiles take turns for up to 256).
//
// Few rows (REP 4 or 2): the tensor cores compute 128 rows whatever they hold, so 32 (64) rows are repeated 4
// (2) times and each repeat takes a quarter (half) of a tile's keys: its P is zero elsewhere, so the four warps
// share the exponentials of the few rows, and the repeats are joined like any split over keys.
//
// The accumulator is rescaled only when a row's maximum grows by more than 2^8: P stays below 2^8, its rounding
// is relative, and the sums are fp32, so the deferral costs no accuracy; a rescale has to wait for the product
// in flight, the deferral makes that rare. P is rounded to the cache's type (the second product's operand), which is
// half a unit of each weight, as much as the output's own rounding; the sum of weights is of the unrounded ones. Exponentials
// are the hardware's ex2 (2^-22 relative, results under 2^-126 are 0): far below P's rounding.
//
// Measured, 4 requests of 32-64k keys, 8 KV heads of 128, bf16, pages of 64 (floor 120 us of HBM): 32 rows 145 us,
// 5.4 TB/s; 128 rows 156 us, 5.0 TB/s, 643 TFLOP/s; 256 rows 251 us, 802 TFLOP/s. The first two are bound by the key
// stream and, at the ends of a run, by latency; the last waits: no pipe is full (a third of the issue slots, exponentials
// at 36% of theirs, tensor pipe 35%), its softmax warps stand at loads from tensor memory, where S is read twice, and at one
// another. Over a cache in 4 bits, same lengths: 24 or 32 rows 145 us, 64 rows 160 us, 128 rows 182 us, 256 rows 264 us; heads of 256 384,
// 401, 473 and 897 us (codes of one unit at a time); 32 x 64 tokens of 4 rows over 1-8k keys 240 us (16 bits: 223). Through a window of
// 2048: prompt chunks of 6000 and 8192 tokens, 32/8 heads of 128, 856 us, 520 TFLOP/s of the pairs that are seen (3 of the 19 tiles
// that a row tile walks are masked).
// Heads of 256 (floor 240 us): 266 us, 5.9 TB/s; 288 us; 523 us (two tiles of
// 128 rows, a second trip of the keys), 769 TFLOP/s; 192: 245 us, 4.8 TB/s (a quarter of the ring idle). Warp-level
// matrix instructions took 780 us for the first of 256 and reached 120 TFLOP/s in the last. A call of one tile takes
// 14 us, most of it latencies one after the other: lengths, page numbers, keys, two products, the row out.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "internal.h"
#include "kv4.cuh"
#include "tree_attn.cuh"

namespace dsv41 {

// where keys and values come from
enum Source { kGather, kPages, kPacked };

template <int DT, int MT, int REP, int SRC>
struct TcCfg {
    static constexpr bool TMA = SRC == kPages;
    static_assert(MT == 1 || REP == 1, "repeats are for a single tile of 128 rows");
    static_assert(MT == 1 || DT <= 128, "tensor memory holds one row tile of 256 columns");
    static constexpr int kt = DT == 256 ? 64 : 128;          // keys per tile (256 columns of O leave room for two S of 64)
    static constexpr int rt = MT * 128 / REP;                // rows per tile
    static constexpr int split = REP == 4 ? 1 : 2;           // softmax threads that share a row's keys
    static constexpr int kw = kt / REP / split;              // keys of a tile per softmax thread
    static constexpr int hold = MT == 2 ? 32 : kw;           // scores a thread holds at a time (registers)
    static constexpr int group = 128 * split;                // softmax threads per 128 rows
    static constexpr int soft_warps = 4 * split * MT;
    // one warp's tensor copies of 16-token pages (16 a unit) take 1200 cycles to issue; two share them where there is room
    static constexpr int prod_warps = TMA ? (MT == 2 ? 1 : 2) : SRC == kPacked && REP > 1 ? 8 : 4, q_warps = TMA && MT == 2 ? 1 : 2;
    static constexpr int w_prod = soft_warps, w_q = w_prod + prod_warps, w_s = w_q + q_warps, w_o = w_s + 1;
    static constexpr int threads = (w_o + 1) * 32;
    static constexpr int blocks = DT / 64;                   // blocks of 64 columns (128 bytes), swizzled
    static constexpr int block_b = kt * 128;
    static constexpr int unit_b = blocks * block_b;          // a key or value tile
    static constexpr int q_block_b = 128 * 128, q_tile_b = blocks * q_block_b;
    static constexpr int q_b = MT * q_tile_b;
    static constexpr int own = 32 / REP;                     // of 32 columns of O, those a repeat's warps put out
    static constexpr int stage_b = soft_warps * (32 - own) * 32 * 4;   // the others', on their way to their repeat
    // what a segment costs beside its tiles (rows' loads, its end), in tiles. 2, 3, 5: 32 x 64 tokens of 4 rows over
    // 1-8k keys 237, 228, 224 us (before the join's last step); 16 x 5-13 tokens over 0.1-4k keys 50, 50, 54 us; long lengths within 1%
    static constexpr int extra = 3;
    static constexpr int off_b = SRC == kPacked ? 0 : 4 * kt * 8;   // byte offsets of the keys of four tiles
    static constexpr int raw_unit_b = kt * DT / kKv4Chunk * 20, raw_units = DT == 256 ? 1 : 2,
                         raw_b = SRC == kPacked ? raw_units * raw_unit_b : 0;   // codes and scales of a tile's keys, values (of either: 256 columns)
    static constexpr int ml_b = MT * 2 * 128 * 8;
    static constexpr int mx_b = MT * 4 * 128 * 4;            // tile maxima of the threads that share a row
    static constexpr int bars_b = 1024;
    static constexpr int fixed_b = 1024 + q_b + stage_b + off_b + raw_b + ml_b + mx_b + bars_b;
    static constexpr int units_fit = (232448 - fixed_b) / unit_b;
    static constexpr int units = units_fit < 10 ? units_fit : 10;
    static constexpr int lag = units - 2;                    // cp.async: units in flight when the next is issued
    static constexpr int smem = fixed_b + units * unit_b;
    static_assert(units >= 4 && lag <= 8, "ring length");
    // tensor memory columns
    __host__ __device__ static constexpr int s_col(int b) { return b * kt; }
    // P of key x of buffer b (two keys a column). Two row tiles leave no room of its own: P then lies over S, each
    // softmax thread's over its own keys', which it alone reads.
    __host__ __device__ static constexpr int p_col(int b, int x)
    {
        return MT == 1 ? 2 * kt + b * (kt / 2) + x / 2 : b * kt + (x / kw) * kw + (x % kw) / 2;
    }
    __host__ __device__ static constexpr int o_col(int t) { return DT == 256 ? 256 : MT == 1 ? 384 : 256 + t * 128; }
};

__device__ __forceinline__ void st_shared16(uint32_t at, const uint4& v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_shared4(uint32_t at)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live)
{
    const int n = live ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// whether a phase is complete, without waiting for it
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}

// ---- tcgen05 ----------------------------------------------------------------------------------
__device__ __forceinline__ void tcf_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcf_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Operand descriptors: swizzled-128B, rows of 128 bytes, 8-row atoms of 1024 bytes. The low word holds the address
// and, for N-major operands, the distance of the 64-column blocks (K-major: unused); both in units of 16 bytes.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc_desc_low(uint32_t saddr, uint32_t block) { return ((saddr & 0x3FFFFu) >> 4) | ((block >> 4) << 16); }
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, float* v)
{
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        " tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// N (16, or a multiple of 32) columns of this thread's lane: all loads, one wait. The empty statements after the wait tie
// the registers to it, so no use of them is scheduled before.
template <int N>
__device__ __forceinline__ void tc_ld(uint32_t taddr, float* v)
{
    if constexpr (N == 16) {
        tc_ld16(taddr, v);
        return;
    } else {
    uint32_t r[N];
#pragma unroll
    for (int c = 0; c < N; c += 32)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
            "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]), "=r"(r[c + 6]),
              "=r"(r[c + 7]), "=r"(r[c + 8]), "=r"(r[c + 9]), "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]), "=r"(r[c + 13]),
              "=r"(r[c + 14]), "=r"(r[c + 15]), "=r"(r[c + 16]), "=r"(r[c + 17]), "=r"(r[c + 18]), "=r"(r[c + 19]),
              "=r"(r[c + 20]), "=r"(r[c + 21]), "=r"(r[c + 22]), "=r"(r[c + 23]), "=r"(r[c + 24]), "=r"(r[c + 25]),
              "=r"(r[c + 26]), "=r"(r[c + 27]), "=r"(r[c + 28]), "=r"(r[c + 29]), "=r"(r[c + 30]), "=r"(r[c + 31])
            : "r"(taddr + c)
            : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < N; c += 8)
        asm volatile("" : "+r"(r[c]), "+r"(r[c + 1]), "+r"(r[c + 2]), "+r"(r[c + 3]), "+r"(r[c + 4]), "+r"(r[c + 5]),
                          "+r"(r[c + 6]), "+r"(r[c + 7]));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
    }
}
// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// The paths that few tiles take are functions of their own: inlined, they crowd the common path out of the
// instruction cache.

// Infinities and NaN among new tokens' values would reach rows that do not see them (0 * NaN): zero those of this
// thread's pieces of a tile and say whether there were any; the softmax warps give them to the rows that do see them at
// the end of the segment (see_nonfinite). A first look only: a half-word's exponent bits, turned, are zero in a value that is not finite, and the minimum over
// all words finds one.
template <typename T, int ROWS>
__device__ __noinline__ bool clear_nonfinite(unsigned char* base, int row0, int step, int chunk)
{
    constexpr uint32_t kExp = exp_bits<T>() * 0x10001u;
    auto piece = [&](int i) {
        const int row = row0 + i * step;
        return reinterpret_cast<uint4*>(base + row * 128 + ((chunk ^ (row & 7)) << 4));
    };
    uint32_t least = 0xffffffffu;
#pragma unroll 8
    for (int i = 0; i < ROWS; ++i) {
        const uint4 v = *piece(i);
        least = __vminu2(least, __vminu2(__vminu2((v.x & kExp) ^ kExp, (v.y & kExp) ^ kExp), __vminu2((v.z & kExp) ^ kExp, (v.w & kExp) ^ kExp)));
    }
    if ((least & 0xffffu) != 0 && (least >> 16) != 0) return false;
#pragma unroll 1
    for (int i = 0; i < ROWS; ++i) {
        uint4 v = *piece(i);
        v.x = finite2<T>(v.x), v.y = finite2<T>(v.y), v.z = finite2<T>(v.z), v.w = finite2<T>(v.w);
        *piece(i) = v;
    }
    return true;
}

// The same for a tile of whole pages, by `threads` threads together, before its product: values past the last key
// (rows from `rows` on, which may hold anything) are cleared too; `mark` is for keys that rows can see, `touched` for all.
// Both are set before a value is cleared: who finds it cleared (another group of threads looks at the same tile)
// finds them set.
template <typename T, int KT, int N>
__device__ __noinline__ void clear_tile(unsigned char* unit, int thread, int threads, int rows, volatile int* mark, volatile int* touched, int value)
{
    constexpr uint32_t kExp = exp_bits<T>() * 0x10001u;
    uint32_t least = 0xffffffffu;
    uint4* at = reinterpret_cast<uint4*>(unit) + thread;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint4 v = at[i * threads];
        least = __vminu2(least, __vminu2(__vminu2((v.x & kExp) ^ kExp, (v.y & kExp) ^ kExp), __vminu2((v.z & kExp) ^ kExp, (v.w & kExp) ^ kExp)));
    }
    if ((least & 0xffffu) == 0 || (least >> 16) == 0) {
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            uint4 v = at[i * threads];
            if (!any_nonfinite<T>(v)) continue;
            *touched = value;
            if (((thread + i * threads) >> 3) % KT < rows) *mark = value;   // 128-byte rows, KT of them a block
            __threadfence_block();
            v.x = finite2<T>(v.x), v.y = finite2<T>(v.y), v.z = finite2<T>(v.z), v.w = finite2<T>(v.w);
            at[i * threads] = v;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Infinities and NaN of a row's sums, from the cache itself. In the products 0 * inf is NaN where the definition has no
// such term: a repeat's P is zero outside its share of a tile's keys, a weight or a rescale may be zero in 16 or 32 bits only.
// And values that not all rows see entered them as zeros. Here a weight counts as more than zero unless its score is -inf, and
// then 0 * inf is NaN (products of finite numbers are taken as finite). By a whole warp, a row a lane (where `live`): columns that hold
// an infinity or NaN are put out anew, to the output or (not null) to the part at `part`. Keys x0 .. x1 - 1 of the list of tiles, 32 at a
// time, a lane each, then those with such values in turn, for all rows. The warp's own columns are OWN of each 32 from col0 to
// end; `bad` has a bit for each 32 in which they are not finite. The others can hold only what new tokens' tiles were cleared
// of. Only segments that have either come here: 160 requests of 60000 keys, one infinity in one of them, take 2.1 ms for 0.8 (64
// rows: 3.4); 4 tokens over 20000 keys that are full of them 0.6 ms. 16 columns at a time and nothing read back: what
// registers this function takes, the caller spills (32 columns at a time: 32 x 64 tokens over 1-8k keys 1% slower).
template <typename T, int RT, int KT, int OWN, bool WIN>
__device__ __noinline__ void settle_nonfinite(const TreeAttnParams& p, const UnitCursor<RT, KT, WIN>* cursor, int row, bool live, uint32_t bad, bool cleared,
                                              int x0, int x1, int col0, int end, float4* part)
{
    const UnitCursor<RT, KT, WIN> c = *cursor;
    const int lane = threadIdx.x & 31, ctx = c.r.seq - c.r.n;
    const int at = c.rt * RT + row, i = p.group_div.div(at), g = at - i * p.group;
    const T* q = static_cast<const T*>(p.q) + (int64_t)(c.r.q0 + i) * p.q_stride_token + (int64_t)(c.h * p.group + g) * p.q_stride_head;
    const T* k_head = static_cast<const T*>(p.k_cache) + c.h * p.stride_head;
    auto nonfinite = [](const T* from, int count) {
        bool bad = false;
        for (int d = 0; d < count; d += 8) bad |= any_nonfinite<T>(*reinterpret_cast<const uint4*>(from + d));
        return bad;
    };
    const bool q_bad = live && nonfinite(q, p.head_dim);
#pragma unroll 1
    for (int col = col0; col < min(end, p.head_dim); col += OWN < 32 ? 32 : 16) {
        const bool sums = __any_sync(0xffffffffu, live && (bad >> (col >> 5)) & 1);
        if (!sums && !cleared) continue;
        const int cols = min(p.head_dim - col, OWN < 16 ? OWN : 16), from = sums || WIN ? x0 : max(x0, ctx / KT * KT);
        const T* v_head = static_cast<const T*>(p.v_cache) + c.h * p.stride_head + col;
        const uint32_t all = (1u << cols) - 1;
        uint32_t plus = 0, minus = 0;   // bit j: column col + j holds +inf, -inf; both: NaN
#pragma unroll 1
        for (int x = from; x < x1; x += 32) {
            if (!__any_sync(0xffffffffu, live && (plus & minus) != all)) break;
            const int base = c.keys.tile(x / KT) * KT + x % KT, pos = base + lane;
            int64_t off = 0;
            bool hit = false, k_bad = false;
            if (pos < c.r.seq) {
                const int pg = p.page_div.div(pos), id = p.block_table[(int64_t)c.b * p.table_stride + pg];
                if ((unsigned)id < (unsigned)p.num_pages) {
                    off = id * p.stride_page + (pos - pg * p.page_size) * p.stride_slot;
                    hit = nonfinite(v_head + off, cols);
                    if (hit) k_bad = nonfinite(k_head + off, p.head_dim);
                }
            }
            uint32_t hits = __ballot_sync(0xffffffffu, hit);
            const uint32_t bad_keys = __ballot_sync(0xffffffffu, k_bad);
            while (hits) {
                const int l = __ffs(hits) - 1;
                hits &= hits - 1;
                const int64_t key = __shfl_sync(0xffffffffu, off, l);
                if (!live || !(seen_keys<WIN>(p, c.r, i, base + l) & 1)) continue;
                bool zero = false;
                if (q_bad || ((bad_keys >> l) & 1)) {
                    float score = 0.0f;
#pragma unroll 1
                    for (int d = 0; d < p.head_dim; d += 2) {
                        const float2 u = unpack2<T>(*reinterpret_cast<const uint32_t*>(q + d)),
                                     w = unpack2<T>(*reinterpret_cast<const uint32_t*>(k_head + key + d));
                        score = fmaf(u.x, w.x, fmaf(u.y, w.y, score));
                    }
                    zero = (p.flip ? -score : score) == -INFINITY;
                }
#pragma unroll 1
                for (int j = 0; j < cols; j += 2) {
                    const uint32_t raw = *reinterpret_cast<const uint32_t*>(v_head + key + j);
                    if (raw == finite2<T>(raw)) continue;
                    const float2 w = unpack2<T>(raw);
                    if (!(fabsf(w.x) < INFINITY)) plus |= w.x < 0 && !zero ? 0u : 1u << j, minus |= w.x > 0 && !zero ? 0u : 1u << j;
                    if (!(fabsf(w.y) < INFINITY)) plus |= w.y < 0 && !zero ? 0u : 2u << j, minus |= w.y > 0 && !zero ? 0u : 2u << j;
                }
            }
            __syncwarp();
        }
        __syncwarp();
        T* out = static_cast<T*>(p.out) + (int64_t)(c.r.q0 + i) * p.out_stride_token + (int64_t)(c.h * p.group + g) * p.out_stride_head + col;
        for (uint32_t odd = plus | minus; odd; odd &= odd - 1) {
            const int j = __ffs(odd) - 1;
            const float v = (plus & minus) >> j & 1 ? NAN : plus >> j & 1 ? INFINITY : -INFINITY;
            if (part) reinterpret_cast<float*>(part + (col + j) / 4 * RT + row)[(col + j) & 3] = v;
            else reinterpret_cast<uint16_t*>(out)[j] = (uint16_t)pack2<T>(v, v);
        }
    }
    __syncwarp();
}

// The same for a cache in 4 bits, whose chunks stand for NaN in all columns or in none: in tiles that all rows see such a chunk reaches
// them by itself, what was cleared of the others (tiles kt0 .. kt1 of the list) makes the chunk's columns NaN in the rows that see it.
template <typename T, int RT, int KT, int OWN, bool WIN>
__device__ __noinline__ void settle_packed(const TreeAttnParams& p, const UnitCursor<RT, KT, WIN>* cursor, int row, bool live, int kt0, int kt1, int col0,
                                           int end, float4* part)
{
    const UnitCursor<RT, KT, WIN> c = *cursor;
    const int lane = threadIdx.x & 31, nc = p.head_dim / kKv4Chunk;
    const int at = c.rt * RT + row, i = p.group_div.div(at), g = at - i * p.group;
    const MaskedKeys<WIN> mask = masked_keys<RT, WIN>(p, c);
    uint32_t chunks = 0;
#pragma unroll 1
    for (int x = kt0; x <= kt1; ++x) {
        const int pos0 = c.keys.tile(x) * KT;
        if (!mask.template tile<KT>(p, pos0)) continue;
#pragma unroll 1
        for (int base = pos0; base < pos0 + KT; base += 32) {
            const int pos = base + lane;
            uint32_t nan = 0;
            if (pos < c.r.seq) {
                const int pg = p.page_div.div(pos), id = p.block_table[(int64_t)c.b * p.table_stride + pg], in_page = pos - pg * p.page_size;
                if ((unsigned)id < (unsigned)p.num_pages) {
                    const unsigned char* rec = p.packed + (((int64_t)id * p.kv_heads + c.h) * 2 + 1) * kv4_block(p.page_size, nc) +
                                               (in_page / kKv4Tokens) * kv4_record(nc) + nc * kKv4Codes + (in_page % kKv4Tokens) * 4;
                    for (int j = 0; j < nc; ++j) nan |= (uint32_t)kv4_nan<T>(*reinterpret_cast<const uint32_t*>(rec + j * kKv4Scales)) << j;
                }
            }
            uint32_t hits = __ballot_sync(0xffffffffu, nan != 0);
            while (hits) {
                const int l = __ffs(hits) - 1;
                hits &= hits - 1;
                const uint32_t of = __shfl_sync(0xffffffffu, nan, l);
                if (live && (seen_keys<WIN>(p, c.r, i, base + l) & 1)) chunks |= of;
            }
            __syncwarp();
        }
    }
    T* out = static_cast<T*>(p.out) + (int64_t)(c.r.q0 + i) * p.out_stride_token + (int64_t)(c.h * p.group + g) * p.out_stride_head;
#pragma unroll 1
    for (int col = col0; live && col < min(end, p.head_dim); col += OWN < 32 ? 32 : 16) {
        if (!((chunks >> (col / kKv4Chunk)) & 1)) continue;
        for (int j = col; j < col + (OWN < 16 ? OWN : 16); ++j) {
            if (part) reinterpret_cast<float*>(part + j / 4 * RT + row)[j & 3] = NAN;
            else reinterpret_cast<uint16_t*>(out)[j] = (uint16_t)pack2<T>(NAN, NAN);
        }
    }
    __syncwarp();
}

template <typename T, int DT, int MT, int REP, int SRC, bool WIN>
__global__ void __launch_bounds__(TcCfg<DT, MT, REP, SRC>::threads, 1) tree_attn_tc_kernel(const __grid_constant__ TreeAttnParams p, const __grid_constant__ CUtensorMap tm_k,
                                                                                      const __grid_constant__ CUtensorMap tm_v)
{
    using Cfg = TcCfg<DT, MT, REP, SRC>;
    constexpr bool TMA = Cfg::TMA;
    // without a tree mask, tiles of new tokens before all of the row tile's are ordinary ones (plain calls over a 16-bit cache
    // mask every tile with new tokens)
    constexpr bool kRowMasks = WIN || SRC == kPacked;
    constexpr int KT = Cfg::kt, RT = Cfg::rt, KW = Cfg::kw, NU = Cfg::units, LAG = Cfg::lag, CPR = DT / 8;
    using Cursor = UnitCursor<RT, KT, WIN>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sq = smem;
    unsigned char* su = sq + Cfg::q_b;
    float* stage = reinterpret_cast<float*>(su + NU * Cfg::unit_b);
    int64_t* key_off = reinterpret_cast<int64_t*>(reinterpret_cast<unsigned char*>(stage) + Cfg::stage_b);
    unsigned char* raw = reinterpret_cast<unsigned char*>(stage) + Cfg::stage_b + Cfg::off_b;
    float2* ml = reinterpret_cast<float2*>(raw + Cfg::raw_b);
    float* mx = reinterpret_cast<float*>(ml + MT * 2 * 128);
    uint64_t* bars = reinterpret_cast<uint64_t*>(mx + MT * 4 * 128);
    uint64_t* full = bars;                 // [NU] a unit's copies have landed (4 producer warps)
    uint64_t* empty = full + NU;           // [NU] its products are done (keys: told by a softmax thread, values: by the S issuer)
    uint64_t* q_full = empty + NU;         // the segment's rows have landed
    uint64_t* q_free = q_full + 1;         // its last S product is done
    uint64_t* s_full = q_free + 1;         // [2] S buffer computed
    uint64_t* p_full = s_full + 2;         // [2] P buffer written (every softmax warp of the row tile)
    uint64_t* pv_done = p_full + 2;        // [2] the product of a P buffer is done
    uint64_t* all_done = pv_done + 2;      // [2] per issuer
    int* dirty = reinterpret_cast<int*>(all_done + 2);   // [NU] 1 + ring position of a unit that held infinities or NaN
    int* touched = dirty + NU;             // [NU] the same, of one in which any were cleared
    int* s_last = touched + NU;            // [2]
    volatile int* abort_flag = s_last + 2;
    uint32_t* tmem_slot = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(abort_flag)) + 1;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < NU; ++i) {
            mbar_init(&full[i], Cfg::prod_warps);
            mbar_init(&empty[i], 1);
            dirty[i] = touched[i] = 0;
        }
        mbar_init(q_full, Cfg::q_warps);
        mbar_init(q_free, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4 * Cfg::split);
            mbar_init(&pv_done[i], 1);
            mbar_init(&all_done[i], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == Cfg::w_s) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- this CTA's run ----
    // Parts of 4 (8) tiles: joining parts costs about 5 us, a tile of a CTA alone 1: 3 requests of 50 rows over 13 tiles, 2 KV
    // heads, took 43 us in parts of one tile and take 22 us, over 2 tiles 22 and 16 us; 8 segments of 16 tiles and 4 rows
    // 20.5 both ways.
    constexpr int kSmall = 4;
    __shared__ CutShared<Cfg::threads / 32> cut;
    struct SegState {
        Cursor c;
        int64_t v_seg;   // place on the line where the segment begins
        int cleared;     // its tiles held infinities or NaN that not all rows see
        MaskedKeys<WIN> mask;
    };
    __shared__ SegState s_seg[Cfg::soft_warps];
    int64_t run, v0;
    int part_tiles;   // R (0: runs of the line)
    cut_runs<RT, KT, WIN, Cfg::extra, kSmall>(p, cut, run, v0, part_tiles);
    if (p.head_dim % 16) {   // the last 16-column step of Q K^T reads past the head size: zeros there
        uint4* z = reinterpret_cast<uint4*>(sq);
        for (int i = tid; i < (Cfg::q_b + NU * Cfg::unit_b) / 16; i += Cfg::threads) z[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_smem();
    }
    tcf_before();
    __syncthreads();
    tcf_after();
    const uint32_t tmem = *tmem_slot;
    const int count = (int)(cut.end - cut.tiles0);   // tiles of the run
    if (count <= 0) {
        if (warp == Cfg::w_s) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        return;
    }
    Cursor cur;
    cur.b = (int)cut.first[0];
    cur.enter(p);
    cur.h = (int)cut.first[1] / cur.nrt;
    cur.rt = (int)cut.first[1] - cur.h * cur.nrt;
    cur.kt = part_tiles ? (int)cut.tiles0 : max((int)cut.first[2] - Cfg::extra, 0);
    cur.place(p);
    const int ksteps = (p.head_dim + 15) / 16;
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t kIdesc = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(128 >> 4) << 24);   // fp32 sums, M = 128
    auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, abort_flag, p.status); };
    // whether rows differ in what they see of the cursor's tile (new tokens, a window's edge)
    auto masked = [&](const Cursor& c) {
        if constexpr (kRowMasks) return masked_keys<RT, WIN>(p, c).template tile<KT>(p, c.tile() * KT);
        else return c.kt * KT + KT > c.r.seq - c.r.n;
    };
    // by a whole warp, which goes on converged (the tensor memory instructions need that)
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        wait(bar, parity);
        __syncwarp();
    };
    // ring position of tile i's keys and values: K0 K1 V0 K2 V1 ... (the order in which they are needed)
    auto k_pos = [&](int i) { return i == 0 ? 0 : 2 * i - 1; };
    auto v_pos = [&](int i) { return i == count - 1 ? 2 * i + 1 : 2 * i + 2; };

    if (TMA && warp >= Cfg::w_prod && warp < Cfg::w_q) {
        // ---------------------------------- producer, whole pages ----------------------------------
        // A tile is boxes of `box` tokens (a page, or a tile's tokens of a larger one) and 64 columns; lane: one of them.
        // Boxes past the last key are left out: their keys are masked, their values are cleared by the softmax warps.
        const int per = KT / p.box, mine = lane * Cfg::prod_warps + warp - Cfg::w_prod, in_tile = mine % per, block = mine / per;
        const uint32_t dst0 = smem_addr(su) + block * Cfg::block_b + in_tile * p.box * 128;
        struct Box {
            int page, slot, head, live;
        };
        auto look_up = [&](const Cursor& c) {
            Box b;
            const int pos = c.tile() * KT + in_tile * p.box, pg = p.page_div.div(pos);
            b.live = block * 64 < p.head_dim && pos < c.r.seq;
            b.page = b.live ? __ldg(p.block_table + (int64_t)c.b * p.table_stride + pg) : 0;
            b.slot = pos - pg * p.page_size;
            b.head = c.h;
            return b;
        };
        auto issue = [&](int n, const CUtensorMap* map, const Box& b) {
            const int slot = n % NU;
            wait_warp(&empty[slot], ((n / NU) & 1) ^ 1);
            const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, b.live));
            if (lane == 0) mbar_arrive_expect_tx(&full[slot], boxes * p.box * 128);
            __syncwarp();
            if (b.live && !*abort_flag) {
                // (a page that is not the cache's lies outside the map: zeros)
                asm volatile(
                    "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                        dst0 + slot * Cfg::unit_b),
                    "l"(reinterpret_cast<uint64_t>(map)), "r"(block * 64), "r"(p.slot_first ? b.slot : b.head), "r"(p.slot_first ? b.head : b.slot), "r"(b.page), "r"(smem_addr(&full[slot]))
                    : "memory");
            }
            __syncwarp();
        };
        // pages are looked up two tiles ahead (a length, then a table entry: two trips to L2 where a request begins)
        Box box[3] = {look_up(cur), Box{}, Box{}};   // this tile, the next, the one before
        auto look_ahead = [&](int tile) {
            if (tile >= count) return;
            cur.next(p);
            box[1] = look_up(cur);
        };
        look_ahead(1);
        int n = 0;
        for (int step = 0; step <= count; ++step) {
            if (step < count) issue(n++, &tm_k, box[0]);
            if (step > 0) issue(n++, &tm_v, box[2]);
            box[2] = box[0];
            box[0] = box[1];
            look_ahead(step + 2);
        }
        // on an abort, let the copies already issued land before the CTA exits
        for (int u = max(n - NU, 0); u < n && *abort_flag; ++u) {
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait(&full[u % NU], (u / NU) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {}
        }
        __syncwarp();
    } else if (SRC == kPacked && warp >= Cfg::w_prod && warp < Cfg::w_q) {
        if constexpr (SRC == kPacked) {
        // ---------------------------------- producers, codes ----------------------------------
        // A thread decodes the chunks of one key that are its group's. Their codes and scales go to places of its own in shared memory
        // (cp.async) a tile ahead, keys and values in turn. (In registers they were read as early, but two tiles' pieces left
        // too few of them where 256 rows share a CTA, and decoding them had to be written out for every chunk, twice: code
        // that the instruction cache did not hold: 32 x 64 tokens of 4 rows over 1-8k keys 328 us for 242, 16 small trees over
        // 0.1-16k keys 137 us for 127.)
        // Eight neighbouring keys' 16-byte pieces fall into different banks by the swizzle.
        constexpr int PT = Cfg::prod_warps * 32, G = PT / KT, C = DT / kKv4Chunk / G;   // groups of threads; chunks of each
        static_assert(G >= 1 && C >= 1 && G * C * kKv4Chunk == DT, "chunks are dealt out evenly");
        const int pt = tid - Cfg::w_prod * 32, key = pt % KT, c0 = pt / KT * C;
        const int nc = p.head_dim / kKv4Chunk, ps8 = p.page_size / kKv4Tokens, record_b = kv4_record(nc);
        const int chunks = min(C, nc - c0);   // of this thread (none: past the head size)
        const uint32_t raw_codes = smem_addr(raw) + pt * 16, raw_scales = smem_addr(raw) + PT * C * 16 + pt * 4;   // [chunk][thread]
        const uint32_t row = smem_addr(su) + (c0 >> 1) * Cfg::block_b + key * 128 + ((((c0 & 1) * 4) ^ (key & 7)) << 4);
        // this thread's key of the cursor's tile: a page number that is on its way, and which record of the page
        const int* pages = p.block_table + (int64_t)cur.b * p.table_stride;
        int id = -1, in_page = 0, head = 0;
        MaskedKeys<WIN> masks = masked_keys<RT, WIN>(p, cur);
        bool mask = false;
        auto look_up = [&]() {
            const int pos0 = cur.tile() * KT, pos = pos0 + key, pg = p.page_div.div(pos);
            id = pos < cur.r.seq ? __ldg(pages + pg) : -1;
            in_page = (pos - pg * p.page_size) / kKv4Tokens;
            head = cur.h;
            mask = masks.template tile<KT>(p, pos0);
        };
        auto look_ahead = [&](int tile) {
            if (tile >= count) return;
            if (__builtin_expect(cur.kt + 1 < cur.nkt, 1)) {
                ++cur.kt;
            } else {
                cur.next(p);
                masks = masked_keys<RT, WIN>(p, cur);
                pages = p.block_table + (int64_t)cur.b * p.table_stride;
            }
            look_up();
        };
        // its keys' record by number; -1: past the end, or not a page of this cache (zeros)
        auto record = [&]() { return (unsigned)id < (unsigned)p.num_pages ? (id * p.kv_heads + head) * 2 * ps8 + in_page : -1; };
        auto send = [&](int unit, int rec) {   // unit: 0 keys, 1 values
            const unsigned char* at = p.packed + (int64_t)max(rec, 0) * record_b;
            const int token = key % kKv4Tokens;
#pragma unroll 1
            for (int i = 0; i < chunks; ++i) {
                const int c = c0 + i;
                cp_async16(raw_codes + unit * Cfg::raw_unit_b + i * PT * 16, at + c * kKv4Codes + kv4_place(c, token) * 16, rec >= 0);
                cp_async4(raw_scales + unit * Cfg::raw_unit_b + i * PT * 4, at + nc * kKv4Codes + c * kKv4Scales + token * 4, rec >= 0);
            }
            cp_async_commit();
        };
        auto put = [&](int n, int unit, bool check) {
            const int slot = n % NU;
            cp_async_wait<Cfg::raw_units - 1>();   // (the last sent for may still be on their way)
            wait_warp(&empty[slot], ((n / NU) & 1) ^ 1);
            const uint32_t to = row + slot * Cfg::unit_b, codes = raw_codes + unit * Cfg::raw_unit_b, scales = raw_scales + unit * Cfg::raw_unit_b;
#pragma unroll 1
            for (int i = 0; i < chunks; ++i) {
                uint32_t sv = ld_shared4(scales + i * PT * 4);
                const uint4 u = ld_shared16(codes + i * PT * 16);
                if (__builtin_expect(check && kv4_nan<T>(sv), 0)) {   // not all rows see it: zeros (settle_packed)
                    *reinterpret_cast<volatile int*>(dirty + slot) = n + 1;
                    sv = 0;
                }
                const Scale2<T> sc(sv);
                // (an even number of chunks a thread begins at an even one)
                const uint32_t at = (to ^ ((i & 1) << 6)) + (i >> 1) * Cfg::block_b;
                st_shared16(at, kv4_word<T>(u.x, sc));
                st_shared16(at ^ 16, kv4_word<T>(u.y, sc));
                st_shared16(at ^ 32, kv4_word<T>(u.z, sc));
                st_shared16(at ^ 48, kv4_word<T>(u.w, sc));
            }
            fence_proxy_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            __syncwarp();
        };
        // a tile's pages are looked up a tile ahead of sending for it, which is a tile (one place for both: half a tile) ahead of
        // its decoding
        constexpr bool kBoth = Cfg::raw_units == 2;
        constexpr int kValues = kBoth ? 1 : 0;
        auto values = [&](int rec) { send(kValues, rec < 0 ? -1 : rec + ps8); };
        look_up();
        int rec = record(), rec_v = -1;   // of tile `step`, and the one before
        bool mask_k = mask, mask_v = false;
        send(0, rec);
        if (kBoth) cp_async_commit();     // (no values yet)
        look_ahead(1);
        int n = 0;
        for (int step = 0; step <= count; ++step) {
            const bool more = step + 1 < count;
            const int next = more ? record() : -1;
            if (step < count) {
                put(n++, 0, false);
                if (kBoth || (step == 0 && more)) send(0, next);
                else values(step > 0 ? rec_v : rec);
            } else if (kBoth) {
                cp_async_commit();        // (no keys after the last values)
            }
            if (step > 0) {
                put(n++, kValues, mask_v);
                if (!kBoth && more) send(0, next);
                else if (!kBoth && step < count) values(rec);
            }
            if (kBoth && step < count) values(rec);
            rec_v = rec;
            mask_v = mask_k;
            rec = next;
            mask_k = mask;
            look_ahead(step + 2);
        }
        }
    } else if (SRC == kGather && warp >= Cfg::w_prod && warp < Cfg::w_q) {
        // ---------------------------------- producers ----------------------------------
        const int pt = tid - Cfg::w_prod * 32, chunk = pt % CPR, row0 = pt / CPR;
        constexpr int kRowStep = 128 / CPR;
        const bool col_live = chunk * 8 < p.head_dim;
        const uint32_t col_at = (chunk >> 3) * Cfg::block_b;
        const uint32_t ring = smem_addr(su);
        int arrived = 0;     // units handed over
        uint32_t hist = 0;   // bit k: the unit issued k units ago holds values that not all rows see
        auto arrive = [&](int n, bool check) {   // this thread's copies of unit n have landed
            const int slot = n % NU;
            if (__builtin_expect(check && col_live, 0)) {
                if (clear_nonfinite<T, KT / kRowStep>(su + slot * Cfg::unit_b + col_at, row0, kRowStep, chunk & 7))
                    *reinterpret_cast<volatile int*>(dirty + slot) = n + 1;
            }
            fence_proxy_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            __syncwarp();
        };
        // hand over the units in flight before unit n, each as soon as it has landed, until stop()
        auto flush = [&](int n, auto stop) {
            bool stopped = false;
            auto one = [&](auto left) {
                constexpr int k = decltype(left)::value;   // units that may still be in flight
                if (stopped || arrived > n - 1 - k) return;
                cp_async_wait<k>();
                arrive(arrived++, (hist >> k) & 1);
                stopped = stop();
            };
            if (LAG > 7) one(std::integral_constant<int, 7>());
            if (LAG > 6) one(std::integral_constant<int, 6>());
            if (LAG > 5) one(std::integral_constant<int, 5>());
            if (LAG > 4) one(std::integral_constant<int, 4>());
            if (LAG > 3) one(std::integral_constant<int, 3>());
            if (LAG > 2) one(std::integral_constant<int, 2>());
            one(std::integral_constant<int, 1>());
            one(std::integral_constant<int, 0>());
            return stopped;
        };
        auto issue = [&](int n, const void* cache, const int64_t* offs, bool check) {
            const int slot = n % NU;
            const uint32_t par = ((n / NU) & 1) ^ 1;
            // A full ring: hand over what is on its way while waiting, the consumers may need it to go on.
            auto vacant = [&]() { return __all_sync(0xffffffffu, mbar_test(&empty[slot], par)); };
            if (!vacant() && !flush(n, vacant)) wait_warp(&empty[slot], par);
            if (col_live) {
                const uint32_t dst = ring + slot * Cfg::unit_b + col_at;
                constexpr int kBatch = 8;   // offsets of a batch of rows first: a copy is a barrier to the compiler's loads
#pragma unroll
                for (int r = 0; r < KT / kRowStep; r += kBatch) {
                    int64_t off[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) off[i] = offs[row0 + (r + i) * kRowStep];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const int row = row0 + (r + i) * kRowStep;
                        cp_async16(dst + row * 128 + (((chunk & 7) ^ (row & 7)) << 4),
                                   static_cast<const T*>(cache) + (off[i] < 0 ? 0 : off[i] + chunk * 8), off[i] >= 0);
                    }
                }
            }
            cp_async_commit();
            hist = (hist << 1) | (check ? 1u : 0u);
            cp_async_wait<LAG>();
            if (arrived <= n - LAG) arrive(arrived++, (hist >> LAG) & 1);
        };
        // element offset of key `pt` of the cursor's tile (-1: past the end, or not a page of this cache)
        auto offset_of = [&](const Cursor& c) -> int64_t {
            const int pos = c.tile() * KT + pt;
            if (pt >= KT || pos >= c.r.seq) return -1;
            const int pg = p.page_div.div(pos);
            const int id = __ldg(p.block_table + (int64_t)c.b * p.table_stride + pg);
            if ((unsigned)id >= (unsigned)p.num_pages) return -1;
            return id * p.stride_page + (pos - pg * p.page_size) * p.stride_slot + c.h * p.stride_head;
        };
        // offsets are looked up two tiles ahead (a length, then a table entry: two trips to L2 where a request begins)
        int64_t off[2] = {offset_of(cur), -1};
        bool tail[2] = {masked(cur), false}, tail_before = false;
        auto look_ahead = [&](int tile) {
            if (tile >= count) return;
            cur.next(p);
            off[1] = offset_of(cur);
            tail[1] = masked(cur);
        };
        look_ahead(1);
        int n = 0;
        for (int step = 0; step <= count; ++step) {
            if (step < count) {
                if (pt < KT) key_off[(step & 3) * KT + pt] = off[0];
                named_bar_sync(3, 128);
                issue(n++, p.k_cache, key_off + (step & 3) * KT, false);
            }
            if (step > 0) issue(n++, p.v_cache, key_off + ((step - 1) & 3) * KT, tail_before);
            tail_before = tail[0];
            off[0] = off[1];
            tail[0] = tail[1];
            look_ahead(step + 2);
        }
        flush(n, [] { return false; });
    } else if (warp < Cfg::w_s && warp >= Cfg::w_q) {
        // ---------------------------------- Q loaders ----------------------------------
        const int ql = tid - Cfg::w_q * 32, chunk = ql % CPR;
        constexpr int kRowStep = 32 * Cfg::q_warps / CPR;
        const uint32_t dst = smem_addr(sq) + (chunk >> 3) * Cfg::q_block_b;
        int seg = 0;
        for (int it = 0; it < count; ++it) {
            if (it == 0 || cur.kt == 0) {
                wait_warp(q_free, (seg & 1) ^ 1);
                // rows of no token stay what they are: nothing of them is read
                const int rows = min(RT, cur.r.n * p.group - cur.rt * RT);
                if (chunk * 8 < p.head_dim) {
                    const T* base = static_cast<const T*>(p.q) + (int64_t)cur.r.q0 * p.q_stride_token +
                                    (int64_t)(cur.h * p.group) * p.q_stride_head + chunk * 8;
#pragma unroll 4
                    for (int row = ql / CPR; row < rows; row += kRowStep) {
                        const int at = cur.rt * RT + row, i = p.group_div.div(at), g = at - i * p.group;
                        const T* src = base + i * p.q_stride_token + g * p.q_stride_head;
#pragma unroll
                        for (int r = row; r < MT * 128; r += RT)
                            cp_async16(dst + (r >> 7) * Cfg::q_tile_b + (r & 127) * 128 + (((chunk & 7) ^ (r & 7)) << 4), src, true);
                    }
                }
                cp_async_commit();
                cp_async_wait<0>();
                fence_proxy_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
                ++seg;
            }
            cur.next(p);
        }
    } else if (warp == Cfg::w_s) {
        // ---------------------------------- S issuer ----------------------------------
        // Buffers: two per row tile for up to 128 rows (tile i uses buffer i % 2), one each for two row tiles. A buffer's
        // S, then P, are free once its product is done.
        if (lane == 0) {
            const uint32_t idesc = kIdesc | ((uint32_t)(KT >> 3) << 17);
            const uint32_t q_at = smem_addr(sq), ring = smem_addr(su);
            bool ok = true;
            int seg = 0, used[2] = {0, 0};   // segments so far; S products per buffer
            int freed = 0;                   // tiles whose values' slot has been handed back
            for (int i = 0; i < count && ok; ++i, cur.next(p)) {
                const int rows = min(RT, cur.r.n * p.group - cur.rt * RT), tiles = MT == 2 && rows > 128 ? 2 : 1;
                const bool fresh = i == 0 || cur.kt == 0;
                const int n = k_pos(i);
                for (int t = 0; t < tiles && ok; ++t) {
                    const int buf = MT == 1 ? i & 1 : t;
                    if (used[buf] > 0) ok = wait(&pv_done[buf], (used[buf] - 1) & 1);
                    if (t == tiles - 1 && ok) {
                        if (MT == 2 && tiles == 1 && used[1] > 0) ok = wait(&pv_done[1], (used[1] - 1) & 1);
                        // products of tiles before i (two row tiles) or i - 1 have ended: their values' slots are free
                        for (; freed < (MT == 1 ? i - 1 : i); ++freed) mbar_arrive(&empty[v_pos(freed) % NU]);
                    }
                    if (t == 0 && fresh) ok = ok && wait(q_full, seg++ & 1);
                    if (t == 0) ok = ok && wait(&full[n % NU], (n / NU) & 1);
                    if (!ok) break;
                    tcf_after();
                    const uint32_t kd = tc_desc_low(ring + (n % NU) * Cfg::unit_b, 16), qd = tc_desc_low(q_at + t * Cfg::q_tile_b, 16);
                    const uint32_t dst = tmem + Cfg::s_col(buf);
#pragma unroll
                    for (int kk = 0; kk < DT / 16; ++kk) {
                        const int block = kk >> 2, step = (kk & 3) * (32 >> 4);
                        if (kk < ksteps)
                            tc_mma_ss(dst, qd + block * (Cfg::q_block_b >> 4) + step, kd + block * (Cfg::block_b >> 4) + step, idesc, kk > 0);
                    }
                    tc_commit(&s_full[buf]);
                    ++used[buf];
                }
            }
            tc_commit(&all_done[0]);
        }
        __syncwarp();
    } else if (warp == Cfg::w_o) {
        // ---------------------------------- O issuer ----------------------------------
        if (lane == 0) {
            const uint32_t idesc = kIdesc | (1u << 16) | ((uint32_t)(ksteps * 16 >> 3) << 17);   // V is N-major
            const uint32_t ring = smem_addr(su);
            bool ok = true;
            int used[2] = {0, 0};
            for (int i = 0; i < count && ok; ++i, cur.next(p)) {
                const int rows = min(RT, cur.r.n * p.group - cur.rt * RT), tiles = MT == 2 && rows > 128 ? 2 : 1;
                const bool first = i == 0 || cur.kt == 0;
                const int n = v_pos(i);
                ok = wait(&full[n % NU], (n / NU) & 1);
                for (int t = 0; t < tiles && ok; ++t) {
                    const int buf = MT == 1 ? i & 1 : t;
                    ok = wait(&p_full[buf], used[buf] & 1);
                    if (!ok) break;
                    tcf_after();
                    const uint32_t vd = tc_desc_low(ring + (n % NU) * Cfg::unit_b, Cfg::block_b);
                    const uint32_t dst = tmem + Cfg::o_col(t);
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        tc_mma_ts(dst, tmem + Cfg::p_col(buf, kk * 16), vd + kk * (2048 >> 4), idesc, !(first && kk == 0));
                    tc_commit(&pv_done[buf]);
                    ++used[buf];
                }
            }
            tc_commit(&all_done[1]);
        }
        __syncwarp();
    } else {
        // ---------------------------------- softmax ----------------------------------
        constexpr int SPLIT = Cfg::split, HB = Cfg::hold, GT = Cfg::group;
        const int t = warp / (4 * SPLIT), half = (warp >> 2) % SPLIT, wq = warp & 3;   // row tile, share, lane quarter
        const int rep = wq / (4 / REP), tw = wq % (4 / REP);          // repeat, 32-row group
        const int kq = rep * (KT / REP) + half * KW;                  // first key of this thread's share of a tile
        const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16);
        const int row = t * 128 + tw * 32 + lane;                     // row within the row tile
        const int gtid = tid - t * GT;                                // thread within the row tile's group
        const int bar_group = 1 + t, bar_pair = 4 + t * 4 + wq, bar_half = 12 + half;   // 3: the producers, 14: both row tiles
        if (REP > 1 && half == 0) {   // P is zero outside the repeat's keys, for good
            uint32_t z[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) {   // a quarter of a tile's keys in a buffer
                if ((c & 3) / (4 / REP) == rep) continue;
                if constexpr (KT == 128) tc_st16(lanes + Cfg::p_col(c >> 2, (c & 3) * (KT / 4)), z);
                else tc_st8(lanes + Cfg::p_col(c >> 2, (c & 3) * (KT / 4)), z);
            }
            tc_wait_st();
        }
        float m = -INFINITY, l = 0.0f;
        // What changes only with the segment lies in shared memory, one copy per warp: registers are short here, and
        // spilled ones cost a trip to L2 each (the ring leaves no L1).
        SegState* const seg = s_seg + warp;
        seg->c = cur;
        seg->v_seg = v0 - cut.first[2];
        seg->cleared = 0;
        if (kRowMasks) seg->mask = masked_keys<RT, WIN>(p, cur);
        __syncwarp();
        int kt = cur.kt, nkt = cur.nkt, kt_first = kt;
        int rows = min(RT, cur.r.n * p.group - cur.rt * RT);
        int ctx = cur.r.seq - cur.r.n;   // negative for a refused request (no keys)
        int done = 0;                    // tiles of this row tile
        for (int it = 0; it < count; ++it) {
            if (__builtin_expect(it > 0 && ++kt == nkt, 0)) {
                __syncwarp();
                Cursor c = seg->c;
                c.kt = nkt - 1;
                c.next(p);
                seg->c = c;
                seg->v_seg += nkt + Cfg::extra;
                seg->cleared = 0;
                if (kRowMasks) seg->mask = masked_keys<RT, WIN>(p, c);
                __syncwarp();
                kt = kt_first = 0;
                nkt = c.nkt;
                rows = min(RT, c.r.n * p.group - c.rt * RT);
                ctx = c.r.seq - c.r.n;
            }
            if (MT == 2 && t == 1 && rows <= 128) continue;
            const int buf = MT == 1 ? it & 1 : t;
            const uint32_t par = (MT == 1 ? it >> 1 : done) & 1;   // of every barrier of this buffer
            const bool last = kt == nkt - 1 || it == count - 1;
            const bool live = t * 128 + tw * 32 < rows;
            const bool first = kt == kt_first;
            if (first) m = -INFINITY, l = 0.0f;
            const int pos0 = WIN ? seg->c.keys.tile(kt) * KT : kt * KT;
            // rows differ in what they see of the tile (new tokens, a window's edge)
            const bool tail = kRowMasks ? seg->mask.template tile<KT>(p, pos0) : pos0 + KT > ctx;
            static_assert(KW <= 64, "one mask window per thread");
            uint64_t win = 0;
            // this row's new token
            auto token = [&]() { return p.group_div.div(min(seg->c.rt * RT + row, seg->c.r.n * p.group - 1)); };
            if (tail && seg->c.r.seq > 0) win = seen_keys<WIN>(p, seg->c.r, token(), pos0 + kq);
            wait_warp(&s_full[buf], par);
            tcf_after();
            if (wq == 0 && half == 0 && lane == 0 && (MT == 1 || t == 1 || rows <= 128)) {   // the tile's S products have all ended
                mbar_arrive(&empty[k_pos(it) % NU]);
                if (last) mbar_arrive(q_free);
            }
            __syncwarp();
            if (live) {
                const uint32_t s_at = lanes + Cfg::s_col(buf) + kq, p_at = lanes + Cfg::p_col(buf, kq);
                // Tiles that reach the new tokens or a window's edge: keys that the row does not see become -inf in place, before the common
                // path below (a negative scale is turned around there too, so that a maximum stays a maximum).
                if (__builtin_expect(tail || p.flip, 0)) {
#pragma unroll 1
                    for (int c = 0; c < KW; c += 16) {
                        float w[16];
                        uint32_t u[16];
                        tc_ld16(s_at + c, w);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const bool see = !tail || ((win >> (c + j)) & 1);
                            u[j] = __float_as_uint(see ? (p.flip ? -w[j] : w[j]) : -INFINITY);
                        }
                        tc_st16(s_at + c, u);
                    }
                    tc_wait_st();
                }
                const float f = p.scale_log2;
                float v[HB];
                float mt = -INFINITY;
#pragma unroll
                for (int c = 0; c < KW; c += HB) {
                    tc_ld<HB>(s_at + c, v);
                    float a[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = v[j];
#pragma unroll
                    for (int j = 4; j + 8 <= HB; j += 8)
#pragma unroll
                        for (int q = 0; q < 4; ++q) a[q] = max3(a[q], v[j + 2 * q], v[j + 2 * q + 1]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) a[q] = fmaxf(a[q], v[HB - 4 + q]);
                    mt = fmaxf(mt, fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
                }
                mt *= f;
                if (SPLIT == 2) {   // the row's other thread
                    float* at = mx + ((t * 2 + (done & 1)) * 2 + half) * 128 + wq * 32 + lane;
                    *at = mt;
                    named_bar_sync(bar_pair, 64);
                    mt = fmaxf(mt, mx[((t * 2 + (done & 1)) * 2 + (half ^ 1)) * 128 + wq * 32 + lane]);
                }
                if (first) {
                    m = mt;
                } else {
                    const bool grow = mt > m + 8.0f || (m == -INFINITY && mt > m);
                    if (__builtin_expect(__any_sync(0xffffffffu, grow), 0)) {
                        const float alpha = grow ? exp2_fast(m - mt) : 1.0f;
                        if (grow) m = mt;
                        l *= alpha;
                        // the previous tile's product: the other buffer's, or this one's last
                        if (MT == 1) wait_warp(&pv_done[buf ^ 1], ((it - 1) >> 1) & 1);
                        tcf_after();
#pragma unroll 1
                        for (int c = half; c < ksteps; c += SPLIT) {
                            float o[16];
                            tc_ld16(lanes + Cfg::o_col(t) + c * 16, o);
                            uint32_t u[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(o[j] * alpha);
                            tc_st16(lanes + Cfg::o_col(t) + c * 16, u);
                        }
                        tc_wait_st();
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m;
                const uint64_t f2 = pair(f, f), base2 = pair(-base, -base);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < KW; c += HB) {
                    if (HB < KW) tc_ld<HB>(s_at + c, v);
#pragma unroll
                    for (int x0 = 0; x0 < HB; x0 += 16) {
                        uint32_t u[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int x = x0 + 2 * j;
                            float a, b;
                            unpair(fma_pair(pair(v[x], v[x + 1]), f2, base2), a, b);
                            a = exp2_fast(a), b = exp2_fast(b);
                            sum[j & 1] = add_pair(sum[j & 1], pair(a, b));
                            u[j] = pack2<T>(a, b);
                        }
                        tc_st8(p_at + (c + x0) / 2, u);
                    }
                }
                float s0, s1, s2, s3;
                unpair(sum[0], s0, s1);
                unpair(sum[1], s2, s3);
                l += (s0 + s1) + (s2 + s3);
                tc_wait_st();
            }
            if (__builtin_expect(tail, 0)) {
                const int n = v_pos(it);
                wait_warp(&full[n % NU], (n / NU) & 1);
                if (TMA) {
                    clear_tile<T, KT, Cfg::unit_b / 16 / GT>(su + (n % NU) * Cfg::unit_b, gtid, GT, ctx + seg->c.r.n - pos0, dirty + n % NU,
                                                             touched + n % NU, n + 1);
                    named_bar_sync(bar_group, GT);
                    // Where two groups look at the same tile, what one cleared the other finds cleared, but only the one that did
                    // has ordered it before the tensor cores' reads: neither goes on before both have. (In every tile
                    // with new tokens, cleared or not, that wait cost 222 -> 231 us on 32 x 64 tokens over 1-8k keys.)
                    if (MT == 2 && rows > 128 && *reinterpret_cast<volatile int*>(touched + n % NU) == n + 1) named_bar_sync(14, 2 * GT);
                    __syncwarp();
                }
                if (*reinterpret_cast<volatile int*>(dirty + n % NU) == n + 1) seg->cleared = 1;
            }
            tcf_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[buf]);
            __syncwarp();
            ++done;
            if (__builtin_expect(!last, 1)) continue;

            // ---- end of the segment, or of this CTA's run ----
            wait_warp(&pv_done[buf], par);
            tcf_after();
            float mm = m, ll = l, scale_o = 1.0f;   // of the row; scale_o: of this thread's O row
            if (REP > 1 || SPLIT == 2) {
                float2* mine = ml + t * 256;        // [share][repeat and row]
                mine[half * 128 + wq * 32 + lane] = make_float2(m, l);
                named_bar_sync(bar_group, GT);
                mm = -INFINITY, ll = 0.0f;
                const int r0 = REP == 1 ? wq * 32 + lane : tw * 32 + lane;
#pragma unroll
                for (int r = 0; r < REP; ++r) mm = fmaxf(mm, mine[r * RT * (REP > 1) + r0].x);
                const float safe = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
                for (int r = 0; r < REP; ++r) {
                    float2 v = mine[r * RT * (REP > 1) + r0];
                    if (SPLIT == 2) v.y += mine[128 + r * RT * (REP > 1) + r0].y;
                    ll += v.y * exp2_fast(v.x - safe);
                }
                scale_o = exp2_fast(m - safe);
            }
            const Cursor c = seg->c;
            const bool whole = kt_first == 0 && kt == nkt - 1;
            if (whole) scale_o = ll == 0.0f ? 0.0f : scale_o / ll;
            const int slot = 2 * blockIdx.x + (kt_first > 0 ? 0 : 1);   // a part: its segment began in an earlier run, or not
            float4* part = reinterpret_cast<float4*>(p.part_o + (int64_t)slot * RT * DT);   // [column / 4][row]
            auto out_ptr = [&](int r, int d) {
                const int at = c.rt * RT + r, i = p.group_div.div(at), g = at - i * p.group;
                return static_cast<T*>(p.out) + (int64_t)(c.r.q0 + i) * p.out_stride_token +
                       (int64_t)(c.h * p.group + g) * p.out_stride_head + d;
            };
            auto put_lse = [&](int r, float top, float sum) {
                const int at = c.rt * RT + r, i = p.group_div.div(at), g = at - i * p.group;
                p.lse[(int64_t)(c.r.q0 + i) * p.q_heads + c.h * p.group + g] =
                    sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
            };
            constexpr int kCols = DT / SPLIT;   // of this thread
            // 32 columns at a time, the row's two threads half the columns each. A thread's columns of a row are whole
            // 16-byte pieces, so they go out from its registers.
            T* out_row = row < rows ? out_ptr(row, 0) : nullptr;
            float test;          // NaN if one of 32 columns is not finite
            uint32_t bad = 0;    // a bit for each 32 columns of which one is not
            auto put8 = [&](int d, const float* v) {
                if (row >= rows || d >= p.head_dim) return;
#pragma unroll
                for (int j = 0; j < 8; ++j) test = fmaf(v[j], 0.0f, test);
                if (whole) {
                    *reinterpret_cast<uint4*>(out_row + d) =
                        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
                } else {
                    part[d / 4 * RT + row] = make_float4(v[0], v[1], v[2], v[3]);
                    part[(d / 4 + 1) * RT + row] = make_float4(v[4], v[5], v[6], v[7]);
                }
            };
#pragma unroll 1
            for (int col = half * kCols; col < half * kCols + kCols; col += 32) {
                float o[32];
                test = 0.0f;
                __syncwarp();
                tc_ld<32>(lanes + Cfg::o_col(t) + col, o);   // columns past the head size hold anything: not put out
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] *= scale_o;
                if (REP == 1) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) put8(col + j, o + j);
                } else {
                    // each repeat sums and puts out its own `own` of the 32 columns: [warp][other repeat][column][lane]
                    constexpr int OWN = Cfg::own, NX = REP - 1;
                    float sum[OWN];
#pragma unroll
                    for (int q = 0; q < REP; ++q) {
                        if (q == rep) {
#pragma unroll
                            for (int j = 0; j < OWN; ++j) sum[j] = o[q * OWN + j];
                        } else {
                            float* to = stage + ((warp * NX + (q - rep - 1 + REP) % REP) * OWN) * 32 + lane;
#pragma unroll
                            for (int j = 0; j < OWN; ++j) to[j * 32] = o[q * OWN + j];
                        }
                    }
                    named_bar_sync(bar_half, 128);
#pragma unroll
                    for (int q = 0; q < REP; ++q) {
                        if (q == rep) continue;
                        const int from = half * 4 + q * (4 / REP) + tw;
                        const float* src = stage + ((from * NX + (rep - q - 1 + REP) % REP) * OWN) * 32 + lane;
#pragma unroll
                        for (int j = 0; j < OWN; ++j) sum[j] += src[j * 32];
                    }
#pragma unroll
                    for (int j = 0; j < OWN; j += 8) put8(col + rep * OWN + j, sum + j);
                    named_bar_sync(bar_half, 128);
                }
                if (test != 0.0f) bad |= 1u << (col >> 5);
            }
            // (a sum of weights that is NaN makes the row NaN by itself)
            const bool cleared = seg->cleared, odd = ((SRC != kPacked && bad != 0) || (cleared && row < rows)) && ll == ll;
            if (SRC == kPacked && __builtin_expect(cleared, 0))
                settle_packed<T, RT, KT, Cfg::own, WIN>(p, &seg->c, min(row, rows - 1), odd, kt_first, kt, half * kCols + rep * Cfg::own,
                                                        half * kCols + kCols, whole ? nullptr : part);
            else if (SRC != kPacked && __builtin_expect(__any_sync(0xffffffffu, odd), 0))
                settle_nonfinite<T, RT, KT, Cfg::own, WIN>(p, &seg->c, min(row, rows - 1), odd, bad, cleared, kt_first * KT, (kt + 1) * KT,
                                                      half * kCols + rep * Cfg::own, half * kCols + kCols, whole ? nullptr : part);
            const bool owner = half == 0 && rep == 0 && row < rows;   // one thread per row
            if (whole) {
                if (owner && p.lse) put_lse(row, mm, ll);
                __syncwarp();
                tcf_before();
                continue;
            }
            if (owner) p.part_ml[(int64_t)slot * RT + row] = make_float2(mm, ll);
            const int64_t v_seg = seg->v_seg;
            const int fc = part_tiles ? (int)v_seg : (int)((v_seg + Cfg::extra) / run);   // runs with tiles of it
            const int lc = part_tiles ? fc + cut_parts(nkt, part_tiles) - 1 : (int)((v_seg + nkt + Cfg::extra - 1) / run);
            int* counter = p.counters + 2 * fc + t;
            named_bar_sync(bar_group, GT);
            if (gtid == 0) {
                __threadfence();   // the group's stores, ordered before this thread by the barrier
                const bool all_in = atomicAdd(counter, 1) == lc - fc;
                if (all_in) __threadfence();
                s_last[t] = all_in;
            }
            named_bar_sync(bar_group, GT);
            if (*reinterpret_cast<volatile int*>(s_last + t)) {
                JoinArgs a;
                a.ml = p.part_ml;
                a.o = reinterpret_cast<const float4*>(p.part_o);
                a.out = static_cast<T*>(p.out) + c.r.q0 * p.out_stride_token + (int64_t)c.h * p.group * p.out_stride_head;
                a.lse = p.lse ? p.lse + (int64_t)c.r.q0 * p.q_heads + c.h * p.group : nullptr;
                a.stride_token = p.out_stride_token, a.stride_head = p.out_stride_head;
                a.group_div = p.group_div;
                a.group = p.group, a.q_heads = p.q_heads, a.head_dim = p.head_dim, a.row0 = c.rt * RT;
                join_parts<T, DT, RT>(a, fc, lc, t * 128, min(rows - t * 128, 128), gtid, GT);
                if (gtid == 0) *counter = 0;   // ready for the next call
            }
            named_bar_sync(bar_group, GT);
            __syncwarp();
            tcf_before();
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    if (warp == Cfg::w_s) {
        // every product has ended before the tensor memory goes back (also after a wait that ran out)
        const uint64_t t0 = globaltimer_ns();
        for (int i = 0; i < 2; ++i)
            while (!mbar_try_wait(&all_done[i], 0) && globaltimer_ns() - t0 < kWaitLimitNs) {}
        tcf_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_fn()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void* f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// a cache as [page][slot][head][column] (or heads outside the slots, by their strides: each stride of a map is to be a
// multiple of the one before), boxes of 64 columns, one head, `box` slots; zeros outside
static bool cache_map(CUtensorMap* m, const void* base, const TreeAttnParams& p, bool bf16)
{
    auto fn = tensor_map_fn();
    if (!fn) return false;
    auto bytes = [](int64_t s) { return (cuuint64_t)(s > 8 ? s : 8) * 2; };   // (0 is left to dimensions of one, whose stride counts for nothing)
    const int h = p.slot_first ? 2 : 1, t = 3 - h;   // dimension of heads, of slots
    cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, 0, 0, (cuuint64_t)p.num_pages}, strides[3] = {0, 0, bytes(p.stride_page)};
    cuuint32_t box[4] = {64, 1, 1, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    dims[h] = (cuuint64_t)p.kv_heads, dims[t] = (cuuint64_t)p.page_size;
    strides[h - 1] = bytes(p.stride_head), strides[t - 1] = bytes(p.stride_slot);
    box[t] = (cuuint32_t)p.box;
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides,
              box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DT, int MT, int REP, int SRC, bool WIN>
static cudaError_t launch_tc(const TreeAttnParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st)
{
    using Cfg = TcCfg<DT, MT, REP, SRC>;
    auto kernel = tree_attn_tc_kernel<T, DT, MT, REP, SRC, WIN>;
    static bool ready[64] = {};   // the attribute is per device and kernel, and stays
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !ready[dev]) {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    kernel<<<num_sms(), Cfg::threads, Cfg::smem, st>>>(p, tm_k, tm_v);
    return cudaGetLastError();
}

template <typename T, int DT, int SRC, bool WIN>
static cudaError_t launch_tc_rows(const TreeAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int rows, cudaStream_t st)
{
    if (rows <= 32) return launch_tc<T, DT, 1, 4, SRC, WIN>(p, k, v, st);
    if (rows <= 64) return launch_tc<T, DT, 1, 2, SRC, WIN>(p, k, v, st);
    if constexpr (DT <= 128) {
        if (rows > 128) return launch_tc<T, DT, 2, 1, SRC, WIN>(p, k, v, st);
    }
    return launch_tc<T, DT, 1, 1, SRC, WIN>(p, k, v, st);
}

template <typename T, int DT, bool WIN>
static cudaError_t launch_tc_dim(TreeAttnParams p, int max_rows, cudaStream_t st)
{
    // Whole pages go by tensor copies where a tile is whole pages (or a page whole tiles) of at least a swizzle atom's
    // 8 rows; other page sizes are gathered key by key, and so are caches that repeat in memory (a view whose heads, slots
    // or pages are one: a map has no stride of 0).
    constexpr int kt = TcCfg<DT, 1, 1, kPages>::kt;
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    CUtensorMap k{}, v{};
    p.box = p.page_size < kt ? p.page_size : kt;
    p.slot_first = p.stride_slot < p.stride_head;
    const bool repeats = (p.stride_head == 0 && p.kv_heads > 1) || (p.stride_slot == 0 && p.page_size > 1) ||
                         (p.stride_page == 0 && p.num_pages > 1);
    const bool pages = p.num_pages > 0 && !repeats && p.box >= 8 && kt % p.box == 0 && p.page_size % p.box == 0 &&
                       cache_map(&k, p.k_cache, p, bf16) && cache_map(&v, p.v_cache, p, bf16);
    return pages ? launch_tc_rows<T, DT, kPages, WIN>(p, k, v, max_rows, st) : launch_tc_rows<T, DT, kGather, WIN>(p, k, v, max_rows, st);
}

template <typename T, bool WIN>
static cudaError_t launch_tree_attn_typed(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    if (p.head_dim <= 64) return launch_tc_dim<T, 64, WIN>(p, max_rows, st);
    if (p.head_dim <= 128) return launch_tc_dim<T, 128, WIN>(p, max_rows, st);
    return launch_tc_dim<T, 256, WIN>(p, max_rows, st);
}

// over a cache in 4 bits
template <typename T, bool WIN>
static cudaError_t launch_tree_attn4_typed(const TreeAttnParams& p, int max_rows, cudaStream_t st)
{
    const CUtensorMap none{};
    if (p.head_dim <= 64) return launch_tc_rows<T, 64, kPacked, WIN>(p, none, none, max_rows, st);
    if (p.head_dim <= 128) return launch_tc_rows<T, 128, kPacked, WIN>(p, none, none, max_rows, st);
    return launch_tc_rows<T, 256, kPacked, WIN>(p, none, none, max_rows, st);
}

}  // namespace dsv41
