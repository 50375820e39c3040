// Store of keys and values into a cache in 4 bits, reading back, and moving (dsv41_kv4_store, dsv41_kv4_load, dsv41_kv4_move).
//
// Store. For 32 columns x of a token's head, lo and hi their smallest and largest:
//     s = T((hi - lo) / 15),   code = round((x - lo) / s) in 0..15 (halves to even; s = 0: 0),   x stands for T(lo + s code)
// lo is one of the values and exact. Where the 15th code would round past T's largest number s is the next smaller one. A
// chunk with a value that is not finite stands for NaN throughout: it has no codes that say which of its columns are not. So does
// one whose hi - lo passes fp32, where s is formed: bf16 chunks of 3.4e38 and more from end to end.
// x - lo is formed in fp32 with its rounding error, the quotient from a reciprocal; where that comes near a half, the remainder of the
// half decides, so every code is the exact quotient's.
//
// Four threads share a chunk, 8 columns (16 bytes) of keys and of values each: loads are whole, and a chunk's codes leave as 16 contiguous
// bytes. 64 bytes in and 20 out a chunk: 16384 tokens of 8 heads of 128 in 43 us (floor 13 us), bound by instructions (73% of the issue
// slots, 16 a value); reading back 27 us, moving 33 us; 100 tokens 8, 6 and 10 us.
//
// Load is the reverse, and move copies codes and scales as they are (a drafted path that is accepted keeps its bits): all
// are read before any is written, so slots may be both source and destination of one call.
#include "internal.h"
#include "kv4.cuh"
#include "tree_attn.cuh"

namespace dsv41 {

constexpr int kKv4Threads = 256;

// where chunk c of a slot's key lies: codes, and scales (the value's: `values` bytes further)
struct Kv4At {
    unsigned char *codes, *scales;
    int64_t values;
};
__device__ __forceinline__ Kv4At kv4_at(const Kv4Params& p, int64_t slot, int head, int c)
{
    const int page = p.few_slots ? p.page_div.div((int)slot) : (int)(slot / p.page_size);
    const int in_page = (int)(slot - (int64_t)page * p.page_size), t = in_page % kKv4Tokens, ps8 = p.page_size / kKv4Tokens;
    const int record = (page * p.kv_heads + head) * 2 * ps8 + in_page / kKv4Tokens, bytes = kv4_record(p.chunks);   // (records are below 2^31)
    unsigned char* at = p.data + (int64_t)record * bytes;
    return {at + c * kKv4Codes + kv4_place(c, t) * 16, at + p.chunks * kKv4Codes + c * kKv4Scales + t * 4, (int64_t)ps8 * bytes};
}

// f(token, head, chunk, quarter of the chunk, in a token) for every quarter (8 columns) of the call's chunks. A CTA takes as many tokens
// at a time as it has threads for; all its threads go round together, those without a token or a quarter with a token of -1.
template <typename F>
__device__ __forceinline__ void each_quarter(const Kv4Params& p, F f)
{
    const int per_token = p.kv_heads * p.chunks * 4, many = max(kKv4Threads / per_token, 1);
    const int mine = per_token < kKv4Threads ? threadIdx.x / per_token : 0, first = threadIdx.x - mine * per_token;
    for (int64_t t0 = (int64_t)blockIdx.x * many; t0 < p.num_tokens; t0 += (int64_t)gridDim.x * many) {
        const int64_t t = mine < many && t0 + mine < p.num_tokens ? t0 + mine : -1;
        for (int u0 = 0; u0 < per_token; u0 += kKv4Threads) {
            const int u = u0 + first, hc = u >> 2, head = hc / p.chunks;
            f(u < per_token ? t : -1, head, hc - head * p.chunks, u & 3);
        }
    }
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

// The word of 8 codes of x in a chunk from lo with steps of s (not 0). A quotient from the reciprocal is off by a few units of 2^-23:
// where one comes near a half, all 8 are decided exactly.
__device__ __noinline__ uint32_t kv4_word_exact(float4 a, float4 b, float lo, float s)
{
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const float up = s < 1e-30f ? 0x1p64f : 1.0f;   // (1 / s would pass fp32)
    lo *= up, s *= up;
    const float inv = 1.0f / s;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = x[i] * up, d = v - lo, r = d * inv;
        float n = rintf(r);
        if (fabsf(r - n) > 0.4999f) {   // which side of the half is the exact quotient on?
            const float h = floorf(r) + 0.5f, low = d + lo, err = (v - low) + ((low - d) - lo);   // v - lo is d + err exactly
            const float rest = fmaf(-h, s, d) + err;
            n = rest > 0.0f ? h + 0.5f : rest < 0.0f ? h - 0.5f : rintf(h);
        }
        word |= (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f) << (4 * (i >> 1) + 16 * (i & 1));
    }
    return word;
}
__device__ __forceinline__ uint32_t kv4_word_of(const float* x, float lo, float s)
{
    constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: a sum's low bits are the rounded number
    const float inv = 1.0f / s;
    float worst = s < 1e-30f ? 1.0f : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = fminf((x[i] - lo) * inv, 15.0f), t = r + kRound;
        worst = fmaxf(worst, fabsf(r - (t - kRound)));
        word |= (__float_as_uint(t) & 15u) << (4 * (i >> 1) + 16 * (i & 1));
    }
    return __builtin_expect(worst > 0.4999f, 0) ? kv4_word_exact(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), lo, s) : word;
}

template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_store_kernel(const Kv4Params p)
{
    const int64_t slots = (int64_t)p.num_pages * p.page_size;
    each_quarter(p, [&](int64_t t, int head, int c, int part) {
        const int64_t slot = t >= 0 ? p.slots[t] : -1;
        const bool live = slot >= 0 && slot < slots;
        uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};   // of keys, values
        if (live) {
            raw[0] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + t * p.k_stride_token + head * p.k_stride_head + c * kKv4Chunk + part * 8));
            raw[1] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + t * p.v_stride_token + head * p.v_stride_head + c * kKv4Chunk + part * 8));
        }
        const Kv4At at = kv4_at(p, live ? slot : 0, head, c);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint32_t w[4] = {raw[which].x, raw[which].y, raw[which].z, raw[which].w};
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
            if (fine && s > 0.0f) code = kv4_word_of(x, lo, s);
            if (!live) continue;
            reinterpret_cast<uint32_t*>(at.codes + which * at.values)[part] = code;
            if (part == 0) *reinterpret_cast<uint32_t*>(at.scales + which * at.values) = fine ? sb | bits16<T>(lo) << 16 : 0x7fff0000u;   // (0x7fff: NaN in both types)
        }
    });
}

template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_load_kernel(const Kv4Params p)
{
    const int64_t slots = (int64_t)p.num_pages * p.page_size;
    each_quarter(p, [&](int64_t t, int head, int c, int part) {
        if (t < 0) return;
        const int64_t slot = p.slots[t];
        uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (slot >= 0 && slot < slots) {
            const Kv4At at = kv4_at(p, slot, head, c);
            uint32_t w[2], sc[2];
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                w[which] = reinterpret_cast<const uint32_t*>(at.codes + which * at.values)[part];
                sc[which] = *reinterpret_cast<const uint32_t*>(at.scales + which * at.values);
            }
#pragma unroll
            for (int which = 0; which < 2; ++which) v[which] = kv4_word<T>(w[which], Scale2<T>(sc[which]));
        }
        T *k = static_cast<T*>(const_cast<void*>(p.k)), *val = static_cast<T*>(const_cast<void*>(p.v));
        *reinterpret_cast<uint4*>(k + t * p.k_stride_token + head * p.k_stride_head + c * kKv4Chunk + part * 8) = v[0];
        *reinterpret_cast<uint4*>(val + t * p.v_stride_token + head * p.v_stride_head + c * kKv4Chunk + part * 8) = v[1];
    });
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
        Kv4At at = kv4_at(p, slot, head, c);
        at.codes += which * at.values, at.scales += which * at.values;
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
static int quarters_grid(const Kv4Params& p)
{
    const int per_token = p.kv_heads * p.chunks * 4, many = per_token < kKv4Threads ? kKv4Threads / per_token : 1;
    const int64_t ctas = ((int64_t)p.num_tokens + many - 1) / many, cap = 16 * (int64_t)num_sms();
    return (int)(ctas > cap ? cap : ctas);
}

cudaError_t launch_kv4_store(const Kv4Params& p, int dtype, cudaStream_t st)
{
    if (dtype == 0) kv4_store_kernel<__half><<<quarters_grid(p), kKv4Threads, 0, st>>>(p);
    else kv4_store_kernel<__nv_bfloat16><<<quarters_grid(p), kKv4Threads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_kv4_load(const Kv4Params& p, int dtype, cudaStream_t st)
{
    if (dtype == 0) kv4_load_kernel<__half><<<quarters_grid(p), kKv4Threads, 0, st>>>(p);
    else kv4_load_kernel<__nv_bfloat16><<<quarters_grid(p), kKv4Threads, 0, st>>>(p);
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
