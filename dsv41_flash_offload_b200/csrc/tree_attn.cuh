// Device helpers of the attention kernel: 16-bit pairs, asynchronous
// copies, the kernel's view of a request, positions in the list of units, and the mask windows.
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

// Position in the list of units: request, KV head, row tile, key tile.
template <int RT, int KT>
struct UnitCursor {
    int b, h, rt, kt, nrt, nkt;
    AttnReq r;
    __device__ __forceinline__ void enter(const TreeAttnParams& p)
    {
        r = attn_req(p, b);
        nrt = (r.n * p.group + RT - 1) / RT;
        nkt = max((r.seq + KT - 1) / KT, 1);
    }
    __device__ __forceinline__ void next(const TreeAttnParams& p)
    {
        if (++kt < nkt) return;
        kt = 0;
        if (++rt < nrt) return;
        rt = 0;
        if (++h < p.kv_heads) return;
        h = 0;
        while (++b < p.batch) {
            enter(p);
            if (r.n > 0) return;
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

}  // namespace dsv41
