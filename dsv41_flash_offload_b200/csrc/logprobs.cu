// Scores of rows of logits (dsv41_token_logprobs): log probabilities of given tokens, entropy, and the `top` likeliest tokens.
//
// For a row x of V logits, with m its maximum:
//     L = sum_v e^(x_v - m),  lse = m + log L,  logprob(t) = (x_t - m) - log L,
//     entropy = log L - (1 / L) sum_v e^(x_v - m) (x_v - m)
// in one pass: running maximum, sum and weighted sum in fp32 per thread. Differences to the maximum are formed before they are
// scaled, so rows of the type's lowest value are ordinary rows. Terms that vanish in 32 bits (logits of -inf among them)
// add nothing to either sum. A NaN or +inf makes the sums NaN by itself.
//
// Alternatives. A key of 64 bits orders tokens by logit, ties by the lowest index. Every thread knows the largest key of its own
// elements; the k-th largest of these is no larger than the k-th largest key of all, and only the k threads at or above it
// can hold the k largest. Their elements (k / threads of the row) are read once more, from L2, and those at or above that key are the candidates:
// hardly more than k of them where logits lie in no special order, and never more than the list has room for (it is cut down
// to its k largest when it runs full). The candidates' order in the list does not change what comes out.
//
// Bound: reading the logits once (16-bit ones nearly as much by instructions: five an element, and its exponential). 2048 rows of 100001
// fp32 logits 158 us, 5.2 TB/s; 2048 of 128000 bf16 119 us, 4.4 TB/s, with 32 alternatives 182 us; 512 of them 45 and 61 us (1.7 CTAs for
// each place: half of the SMs idle at the end); one row of 100001 10 us, with 5 alternatives 16 us. Alternatives cost a CTA 6 to 8 us,
// sorts and three trips to L2 one after the other, half hidden behind the SM's other CTA. One CTA a row where there are many rows; where there are few, a row's CTAs are a cluster
// and the first joins the others' sums and keys through distributed shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "logprobs.h"

namespace cg = cooperative_groups;

namespace dsv41 {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kPlainCtas = 3;    // CTAs on an SM where no alternatives are asked for
constexpr int kLpRoom = 6144;    // keys of the list of candidates
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLpNone = -140.0f;   // e^-140 is 0 in fp32 (results under 2^-126 are)

__device__ __forceinline__ float lp_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lp_exp(float x) { return lp_exp2(x * kLog2e); }
// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t pair2(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)   // NaN if one is
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
struct LpVec {
    static constexpr int n = 16 / sizeof(T);
    static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;   // -inf
    float v[n];
    // the largest element (NaN counts for nothing)
    __device__ __forceinline__ static float largest(const uint4& u)
    {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2* h = reinterpret_cast<const __half2*>(&u);
            const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
            return fmaxf(f.x, f.y);
        } else {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
            const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
            return fmaxf(f.x, f.y);
        }
    }
    __device__ __forceinline__ static uint4 none() { return make_uint4(kNone, kNone, kNone, kNone); }
    __device__ __forceinline__ void unpack(const uint4& u)
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};

// A row as aligned 16-byte vectors: element e lies at place e + head. The vectors at its ends may be partial: those are read
// element by element, what lies outside the row counts as -inf.
template <typename T>
struct LpRow {
    static constexpr int n = LpVec<T>::n;
    const T* x;        // element 0
    int head, vocab, vectors, whole0, whole1;   // (vectors whole0 .. whole1 - 1 are)
    __device__ __forceinline__ LpRow(const void* logits, int64_t at, int vocab_) : x(static_cast<const T*>(logits) + at), vocab(vocab_)
    {
        head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        vectors = (int)(((int64_t)vocab + head + n - 1) / n);
        whole0 = head > 0, whole1 = (int)(((int64_t)vocab + head) / n);
    }
    __device__ __forceinline__ const uint4* at(int i) const { return reinterpret_cast<const uint4*>(x - head + (int64_t)i * n); }
    __device__ __forceinline__ int first(int i) const { return i * n - head; }   // element of the vector's first place (may be outside)
    __device__ __noinline__ uint4 partial(int i) const
    {
        uint32_t w[4] = {LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone, LpVec<T>::kNone};
        for (int j = 0; j < n; ++j) {
            const int64_t e = (int64_t)i * n - head + j;
            if (e < 0 || e >= vocab) continue;
            if constexpr (sizeof(T) == 4) {
                w[j] = __float_as_uint(x[e]);
            } else {
                const uint32_t h = reinterpret_cast<const uint16_t*>(x)[e];
                w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | h << 16 : (w[j / 2] & 0xffff0000u) | h;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ uint4 load(int i) const { return __builtin_expect(i >= whole0 && i < whole1, 1) ? __ldg(at(i)) : partial(i); }
};

// orders tokens by logit, then by the lowest index; 0: none (a logit of -inf)
__device__ __forceinline__ uint64_t lp_key(float v, int e)
{
    const uint32_t b = __float_as_uint(v + 0.0f);   // (-0 and 0 tie)
    const uint32_t o = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
    return v > -INFINITY ? (uint64_t)o << 32 | (0xffffffffu - (uint32_t)e) : 0ull;
}
__device__ __forceinline__ float lp_key_value(uint64_t k)
{
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ uint64_t lp_swap(uint64_t k, int lane, int d, bool larger_low)
{
    const uint64_t o = __shfl_xor_sync(0xffffffffu, k, d);
    return (((lane & d) == 0) == larger_low) == (k > o) ? k : o;   // (keys of 0 alone are equal)
}
// a warp's keys, the largest in lane 0
__device__ __forceinline__ uint64_t lp_sort(uint64_t k, int lane)
{
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size / 2; d > 0; d >>= 1) k = lp_swap(k, lane, d, (lane & size) == 0);
    return k;
}
// the 32 largest of two sorted sets of 32
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b_reversed, int lane)
{
    uint64_t k = a > b_reversed ? a : b_reversed;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) k = lp_swap(k, lane, d, true);
    return k;
}

struct LpShared {
    float m[kLpWarps], l[kLpWarps], e[kLpWarps];
    uint64_t best[kLpWarps][32];   // [0]: the CTA's (or the row's) largest keys, in order
    int hot[kMaxTop], hots, count;
    float sum_m, sum_l, sum_e;     // of the CTA
};

// best[0] = the 32 largest of keys[0 .. count), in order; by the whole CTA
__device__ __noinline__ void lp_select(LpShared& s, const uint64_t* keys, int count)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t mine = 0;
    for (int i = warp * 32; i < count; i += kLpThreads) {
        const uint64_t k = lp_sort(i + lane < count ? keys[i + lane] : 0ull, lane);
        mine = i == warp * 32 ? k : lp_merge(mine, __shfl_sync(0xffffffffu, k, 31 - lane), lane);
    }
    s.best[warp][lane] = mine;
    __syncthreads();
#pragma unroll 1
    for (int half = kLpWarps / 2; half > 0; half >>= 1) {
        if (warp < half) {
            mine = lp_merge(mine, s.best[warp + half][31 - lane], lane);
            s.best[warp][lane] = mine;
        }
        __syncthreads();
    }
}

// joins (m, l, e) of another share of the row
__device__ __forceinline__ void lp_join(float& m, float& l, float& e, float m2, float l2, float e2)
{
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
    const float d1 = max_nan(m - base, kLpNone), d2 = max_nan(m2 - base, kLpNone), w1 = lp_exp(d1), w2 = lp_exp(d2);
    e = fmaf(l, d1, e) * w1 + fmaf(l2, d2, e2) * w2;
    l = l * w1 + l2 * w2;
    m = top;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, TOP ? 2 : kPlainCtas) logprobs_kernel(const LogprobParams p)
{
    using Row = LpRow<T>;
    constexpr int n = Row::n, kBatch = 4;
    extern __shared__ uint64_t keys[];   // [kLpRoom] (TOP)
    __shared__ LpShared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), r = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Row row(p.logits, r * p.row_stride, p.vocab);
    const int step = kLpThreads * ranks, i0 = rank * kLpThreads + tid;   // this thread's vectors: i0, i0 + step, ...

    // ---- sums ----
    float m = -INFINITY;                       // the largest logit so far
    uint64_t l2 = 0, e2 = 0;                   // sums, as pairs
    int at = -1;                               // first vector of the batch that it came with
    for (int i = i0; i < row.vectors; i += kBatch * step) {   // (a row has less than 2^30 vectors, kBatch * step is 2^14 at most)
        uint4 u[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int v = i + b * step;
            u[b] = v < row.vectors ? row.load(v) : LpVec<T>::none();
        }
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) top = fmaxf(top, LpVec<T>::largest(u[b]));
        if (top > m) at = i;
        const float now = fmaxf(m, top), base = now == -INFINITY ? 0.0f : now;
        const float d = max_nan(m - base, kLpNone), keep = lp_exp(d);
        e2 = mul2(fma2(l2, pair2(d, d), e2), pair2(keep, keep));
        l2 = mul2(l2, pair2(keep, keep));
        m = now;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            LpVec<T> x;
            x.unpack(u[b]);
#pragma unroll
            for (int j = 0; j < n; j += 2) {
                float z0, z1;
                split2(add2(pair2(x.v[j], x.v[j + 1]), pair2(-base, -base)), z0, z1);
                const uint64_t z = pair2(max_nan(z0, kLpNone), max_nan(z1, kLpNone));
                split2(mul2(z, pair2(kLog2e, kLog2e)), z0, z1);
                const uint64_t w = pair2(lp_exp2(z0), lp_exp2(z1));
                l2 = add2(l2, w);
                e2 = fma2(w, z, e2);
            }
        }
    }
    float l, e, other;
    split2(l2, l, other);
    l += other;
    split2(e2, e, other);
    e += other;
    float jm = m, jl = l, je = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        lp_join(jm, jl, je, __shfl_xor_sync(0xffffffffu, jm, o), __shfl_xor_sync(0xffffffffu, jl, o), __shfl_xor_sync(0xffffffffu, je, o));
    if (lane == 0) s.m[warp] = jm, s.l[warp] = jl, s.e[warp] = je;
    if (tid == 0) s.hots = s.count = 0;

    // ---- alternatives ----
    if (TOP) {
        uint64_t mine = 0;   // the largest key of this thread's elements
        if (at >= 0) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = at + b * step;
                u[b] = i < row.vectors ? row.load(i) : LpVec<T>::none();
            }
#pragma unroll
            for (int b = kBatch - 1; b >= 0; --b) {   // (the first one that has it is the last to be set)
                LpVec<T> x;
                x.unpack(u[b]);
#pragma unroll
                for (int j = n - 1; j >= 0; --j)
                    if (x.v[j] == m) mine = lp_key(m, row.first(at + b * step) + j);
            }
        }
        keys[tid] = mine;
        __syncthreads();
        lp_select(s, keys, kLpThreads);
        const uint64_t least = s.best[0][p.top - 1];   // 0: fewer threads than that hold any
        if (mine >= least && mine > 0) s.hot[atomicAdd(&s.hots, 1)] = tid;
        __syncthreads();
        const int per = (row.vectors + step - 1) / step, work = s.hots * per;
        auto vector_of = [&](int w) { return w < work ? rank * kLpThreads + s.hot[w / per] + w % per * step : row.vectors; };
        constexpr int kRounds = 4;   // whose vectors are read together
        for (int w0 = 0; w0 < work; w0 += kRounds * kLpThreads) {
            uint4 u[kRounds];
            int first[kRounds];
#pragma unroll
            for (int q = 0; q < kRounds; ++q) {
                const int i = vector_of(w0 + q * kLpThreads + tid);
                u[q] = i < row.vectors ? row.load(i) : LpVec<T>::none();
                first[q] = row.first(i);
            }
#pragma unroll
            for (int q = 0; q < kRounds; ++q) {
                if (w0 + q * kLpThreads >= work) break;
                const int have = s.count;
                __syncthreads();   // (all have read it before any adds to it)
                if (have > kLpRoom - kLpThreads * n - 32) {   // no room for what these vectors may hold
                    lp_select(s, keys, have);
                    if (warp == 0) keys[lane] = s.best[0][lane];
                    if (tid == 0) s.count = 32;
                    __syncthreads();
                }
                LpVec<T> x;
                x.unpack(u[q]);
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const uint64_t k = lp_key(x.v[j], first[q] + j);
                    if (k >= least && k > 0) keys[atomicAdd(&s.count, 1)] = k;
                }
                __syncthreads();
            }
        }
        lp_select(s, keys, s.count);
    }
    __syncthreads();
    if (tid == 0) {
        float a = s.m[0], b = s.l[0], c = s.e[0];
        for (int w = 1; w < kLpWarps; ++w) lp_join(a, b, c, s.m[w], s.l[w], s.e[w]);
        s.sum_m = a, s.sum_l = b, s.sum_e = c;
    }
    cluster.sync();

    // ---- the row, by its first CTA ----
    if (rank == 0) {
        if (TOP && ranks > 1) {
            for (int i = tid; i < ranks * 32; i += kLpThreads) keys[i] = cluster.map_shared_rank(&s, i / 32)->best[0][i & 31];
            __syncthreads();
            lp_select(s, keys, ranks * 32);
        }
        float a = s.sum_m, b = s.sum_l, c = s.sum_e;
        for (int i = 1; i < ranks; ++i) {
            const LpShared* o = cluster.map_shared_rank(&s, i);
            lp_join(a, b, c, o->sum_m, o->sum_l, o->sum_e);
        }
        const bool none = b == 0.0f;   // no token has a weight
        const float log_l = none ? 0.0f : logf(b);
        auto score = [&](float x) { return (x - a) - log_l; };
        if (tid == 0) {
            p.lse[r] = b == b ? a + log_l : NAN;
            p.entropy[r] = none ? 0.0f : log_l - c / b;
        }
        for (int i = tid; i < p.given; i += kLpThreads) {
            const int64_t t = p.tokens[(int64_t)r * p.given + i];
            float v = b == b ? -INFINITY : NAN;
            if (b > 0.0f && t >= 0 && t < p.vocab) {
                float x;
                if constexpr (sizeof(T) == 4) x = row.x[t];
                else if constexpr (std::is_same<T, __half>::value) x = __half2float(row.x[t]);
                else x = __bfloat162float(row.x[t]);
                v = score(x);
            }
            p.logprobs[(int64_t)r * p.given + i] = v;
        }
        if (TOP && tid < p.top) {
            const uint64_t k = b == b ? s.best[0][tid] : 0ull;
            p.top_ids[(int64_t)r * p.top + tid] = k ? (int64_t)(0xffffffffu - (uint32_t)k) : -1;
            p.top_logprobs[(int64_t)r * p.top + tid] = k ? score(lp_key_value(k)) : b == b ? -INFINITY : NAN;
        }
    }
    cluster.sync();   // the first CTA has read the others' shared memory
}

template <typename T, bool TOP>
static cudaError_t launch_lp(const LogprobParams& p, cudaStream_t st)
{
    auto kernel = logprobs_kernel<T, TOP>;
    const int smem = TOP ? kLpRoom * 8 : 0;
    static bool ready[64] = {};   // the attribute is per device and kernel, and stays
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (TOP && (dev >= 64 || !ready[dev])) {
        if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return err;
        if (dev < 64) ready[dev] = true;
    }
    // Few rows are shared by up to 8 CTAs each, of at least 4096 logits. With alternatives as long as every CTA has an SM of its own, for
    // what a CTA does beside its sums does not shrink with its share: with 5 alternatives, 37 rows of 128000 bf16 logits take 23 us in
    // four CTAs each and 31 in eight, 74 rows 23 in two and 33 in four, 100 rows of 32768 17 in one and 21 in two (75 rows of
    // 128000 fp32 logits lose: 30 for 28). Without alternatives up to two CTAs on an SM: 100 rows of 128000 fp32 logits take 21 us in
    // two each, 27 in one.
    const int64_t places = (TOP ? 1 : 2) * (int64_t)num_sms();
    int ranks = 1;
    while (ranks < 8 && (int64_t)p.rows * ranks * 2 <= places && p.vocab / (2 * ranks) >= 4096) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows * ranks));
    cfg.blockDim = dim3(kLpThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

cudaError_t launch_logprobs(const LogprobParams& p, int dtype, cudaStream_t st)
{
    if (dtype == 0) return p.top ? launch_lp<__half, true>(p, st) : launch_lp<__half, false>(p, st);
    if (dtype == 1) return p.top ? launch_lp<__nv_bfloat16, true>(p, st) : launch_lp<__nv_bfloat16, false>(p, st);
    return p.top ? launch_lp<float, true>(p, st) : launch_lp<float, false>(p, st);
}

}  // namespace dsv41
