// Store of keys and values into a cache in 4 bits, reading back, and moving (dsv41_kv4_store, dsv41_kv4_load, dsv41_kv4_move).
//
// Store. For 32 columns x of a token's head, lo and hi their smallest and largest:
//     s = T((hi - lo) / 15),   code = round((x - lo) / s) in 0..15 (halves to even; s = 0: 0),   x stands for T(lo + s code)
// lo is one of the values and exact. Where the 15th code would round past T's largest number s is the next smaller one. A
// chunk whose values or whose s are not finite stands for NaN throughout: it has no codes that say which of its columns are not.
// x - lo is formed in fp32 with its rounding error, the quotient from a reciprocal; where that comes near a half, the remainder of the
// half decides, so every code is the exact quotient's.
//
// Four threads share a chunk, 8 columns (16 bytes) each: loads are whole, and a chunk's codes leave as 16 contiguous bytes. Bound by
// HBM: 64 bytes in and 20 out a chunk.
//
// Load is the reverse, and move copies codes and scales as they are (a drafted path that is accepted keeps its bits): all
// are read before any is written, so slots may be both source and destination of one call.
#include "internal.h"
#include "kv4.cuh"
#include "tree_attn.cuh"

namespace dsv41 {

constexpr int kKv4Threads = 256;

// where chunk c of token slot lies: codes, and scales
struct Kv4At {
    unsigned char *codes, *scales;
};
__device__ __forceinline__ Kv4At kv4_at(const Kv4Params& p, int64_t slot, int head, int which, int c)
{
    const int64_t page = slot / p.page_size;
    const int in_page = (int)(slot - page * p.page_size), t = in_page % kKv4Tokens;
    unsigned char* rec = p.data + ((page * p.kv_heads + head) * 2 + which) * kv4_block(p.page_size, p.chunks) +
                         (int64_t)(in_page / kKv4Tokens) * kv4_record(p.chunks);
    return {rec + c * kKv4Codes + kv4_place(c, t) * 16, rec + p.chunks * kKv4Codes + c * kKv4Scales + t * 4};
}

template <typename T>
__device__ __forceinline__ uint32_t bits16(float v)
{
    return pack2<T>(v, 0.0f) & 0xffffu;
}
template <typename T>
__device__ __forceinline__ float of_bits16(uint32_t v)
{
    return unpack2<T>(v).x;
}

// code of x in a chunk from lo with steps of s (not 0), inv about 1 / s
__device__ __forceinline__ uint32_t kv4_code(float x, float lo, float s, float inv)
{
    const float d = x - lo, r = d * inv;
    float n = rintf(r);
    if (__builtin_expect(fabsf(r - n) > 0.4999f, 0)) {   // near a half (r is off by a few units of 2^-23): which side is the exact one on?
        const float h = floorf(r) + 0.5f, low = d + lo, err = (x - low) + ((low - d) - lo);   // x - lo is d + err exactly
        const float rest = fmaf(-h, s, d) + err;
        n = rest > 0.0f ? h + 0.5f : rest < 0.0f ? h - 0.5f : rintf(h);
    }
    return (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f);
}

template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_store_kernel(const Kv4Params p)
{
    const int64_t per_token = (int64_t)p.kv_heads * 2 * p.chunks * 4, units = per_token * p.num_tokens, slots = (int64_t)p.num_pages * p.page_size;
    const int64_t stride = (int64_t)gridDim.x * kKv4Threads;
    // whole warps go round together: the four threads of a chunk exchange their extremes
    for (int64_t u0 = (int64_t)blockIdx.x * kKv4Threads + (threadIdx.x & ~31); u0 < units; u0 += stride) {
        const int64_t u = u0 + (threadIdx.x & 31);
        const int part = (int)(u & 3);
        const int64_t t = u / per_token;
        const int rest = (int)(u - t * per_token) >> 2, c = rest % p.chunks, wh = rest / p.chunks, which = wh / p.kv_heads, head = wh - which * p.kv_heads;
        const int64_t slot = u < units ? p.slots[t] : -1;
        const bool live = slot >= 0 && slot < slots;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (live)
            raw = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(which ? p.v : p.k) + t * (which ? p.v_stride_token : p.k_stride_token) +
                                                        head * (which ? p.v_stride_head : p.k_stride_head) + c * kKv4Chunk + part * 8));
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
        float lo = x[0], hi = x[0], test = 0.0f;   // test: NaN if one is not finite
#pragma unroll
        for (int i = 0; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]), test = fmaf(x[i], 0.0f, test);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            test += __shfl_xor_sync(0xffffffffu, test, o);
        }
        uint32_t sb = bits16<T>(__fdiv_rn(hi - lo, 15.0f));
        float s = of_bits16<T>(sb);
        const bool fine = test == 0.0f && fabsf(s) < INFINITY;
        if (fine && (bits16<T>(fmaf(15.0f, s, lo)) & exp_bits<T>()) == exp_bits<T>()) s = of_bits16<T>(--sb);
        uint32_t code = 0;
        if (fine && s > 0.0f) {
            const float up = s < 1e-30f ? 0x1p64f : 1.0f, inv = 1.0f / (s * up);   // (1 / s would pass fp32)
#pragma unroll
            for (int i = 0; i < 8; ++i) code |= kv4_code(x[i] * up, lo * up, s * up, inv) << (4 * (i >> 1) + 16 * (i & 1));
        }
        if (!live) continue;
        const Kv4At at = kv4_at(p, slot, head, which, c);
        reinterpret_cast<uint32_t*>(at.codes)[part] = code;
        if (part == 0) *reinterpret_cast<uint32_t*>(at.scales) = fine ? sb | bits16<T>(lo) << 16 : 0x7fff0000u;   // (0x7fff: NaN in both types)
    }
}

template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_load_kernel(const Kv4Params p)
{
    const int64_t per_token = (int64_t)p.kv_heads * 2 * p.chunks * 4, units = per_token * p.num_tokens, slots = (int64_t)p.num_pages * p.page_size;
    for (int64_t u = (int64_t)blockIdx.x * kKv4Threads + threadIdx.x; u < units; u += (int64_t)gridDim.x * kKv4Threads) {
        const int part = (int)(u & 3);
        const int64_t t = u / per_token;
        const int rest = (int)(u - t * per_token) >> 2, c = rest % p.chunks, wh = rest / p.chunks, which = wh / p.kv_heads, head = wh - which * p.kv_heads;
        const int64_t slot = p.slots[t];
        uint4 v = make_uint4(0, 0, 0, 0);
        if (slot >= 0 && slot < slots) {
            const Kv4At at = kv4_at(p, slot, head, which, c);
            const uint32_t w = reinterpret_cast<const uint32_t*>(at.codes)[part], sc = *reinterpret_cast<const uint32_t*>(at.scales);
            v = kv4_word<T>(w, Scale2<T>(sc));
        }
        T* dst = static_cast<T*>(const_cast<void*>(which ? p.v : p.k)) + t * (which ? p.v_stride_token : p.k_stride_token) +
                 head * (which ? p.v_stride_head : p.k_stride_head) + c * kKv4Chunk + part * 8;
        *reinterpret_cast<uint4*>(dst) = v;
    }
}

// out: from the cache to `moved` ([token][head, keys or values][chunk] codes, then scales), or back
template <bool OUT>
__global__ void __launch_bounds__(kKv4Threads) kv4_move_kernel(const Kv4Params p, const int64_t* other)
{
    const int per_token = p.kv_heads * 2 * p.chunks;
    const int64_t units = (int64_t)per_token * p.num_tokens, slots = (int64_t)p.num_pages * p.page_size;
    uint4* codes = reinterpret_cast<uint4*>(p.moved);
    uint32_t* scales = reinterpret_cast<uint32_t*>(codes + units);
    for (int64_t u = (int64_t)blockIdx.x * kKv4Threads + threadIdx.x; u < units; u += (int64_t)gridDim.x * kKv4Threads) {
        const int64_t t = u / per_token, slot = p.slots[t], far = other[t];
        if (slot < 0 || slot >= slots || far < 0 || far >= slots) continue;   // both or neither
        const int rest = (int)(u - t * per_token), c = rest % p.chunks, wh = rest / p.chunks, which = wh / p.kv_heads, head = wh - which * p.kv_heads;
        const Kv4At at = kv4_at(p, slot, head, which, c);
        if (OUT) {
            codes[u] = *reinterpret_cast<const uint4*>(at.codes);
            scales[u] = *reinterpret_cast<const uint32_t*>(at.scales);
        } else {
            *reinterpret_cast<uint4*>(at.codes) = codes[u];
            *reinterpret_cast<uint32_t*>(at.scales) = scales[u];
        }
    }
}

static int kv4_grid(int64_t units)
{
    const int64_t ctas = (units + kKv4Threads - 1) / kKv4Threads, cap = 16 * (int64_t)num_sms();
    return (int)(ctas > cap ? cap : ctas);
}

cudaError_t launch_kv4_store(const Kv4Params& p, int dtype, cudaStream_t st)
{
    const int grid = kv4_grid((int64_t)p.num_tokens * p.kv_heads * 2 * p.chunks * 4);
    if (dtype == 0) kv4_store_kernel<__half><<<grid, kKv4Threads, 0, st>>>(p);
    else kv4_store_kernel<__nv_bfloat16><<<grid, kKv4Threads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_kv4_load(const Kv4Params& p, int dtype, cudaStream_t st)
{
    const int grid = kv4_grid((int64_t)p.num_tokens * p.kv_heads * 2 * p.chunks * 4);
    if (dtype == 0) kv4_load_kernel<__half><<<grid, kKv4Threads, 0, st>>>(p);
    else kv4_load_kernel<__nv_bfloat16><<<grid, kKv4Threads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_kv4_move(const Kv4Params& p, const int64_t* to, cudaStream_t st)
{
    const int grid = kv4_grid((int64_t)p.num_tokens * p.kv_heads * 2 * p.chunks);
    kv4_move_kernel<true><<<grid, kKv4Threads, 0, st>>>(p, to);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    Kv4Params back = p;
    back.slots = to;
    kv4_move_kernel<false><<<grid, kKv4Threads, 0, st>>>(back, p.slots);
    return cudaGetLastError();
}

}  // namespace dsv41
