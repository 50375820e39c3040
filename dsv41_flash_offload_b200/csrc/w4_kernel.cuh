// The product kernel of the 4-bit weights (see w4.cu), instantiated per input type in w4_f16.cu and w4_bf16.cu.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "../../include/dsv41_b200.h"
#include "common.cuh"
#include "internal.h"
#include "w4.h"

namespace dsv41 {

// ---------------------------------------------------------------------------------------------
// codes of one word -> the A fragment {row r: k 0,1 | row r + 8: k 0,1 | row r: k 2,3 | row r + 8: k 2,3} of
// q - z. za, zb: the rows' zero points in the form that the type's decode subtracts (w4_zero).
// ---------------------------------------------------------------------------------------------
template <typename T>
struct W4Dec;
// (w & mask) | magic in one instruction (two from the plain expression, and the ALU pipe bounds the decode)
__device__ __forceinline__ uint32_t w4_place(uint32_t w, uint32_t mask, uint32_t magic)
{
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(magic));
    return v;
}
template <>
struct W4Dec<__half> {
    // 0x6400 | q is 1024 + q; with the code four bits up, 1024 + 16 q, which one fused multiply-add brings
    // to q - z (all steps exact)
    uint32_t za, zb;   // -(1024 + z), -(64 + z) twice
    __device__ __forceinline__ void zero(int z0, int z1)
    {
        za = half2_as_u32(__float2half2_rn(-1024.0f - z0));
        zb = half2_as_u32(__float2half2_rn(-64.0f - z1));
    }
    __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&a)[4]) const
    {
        const __half2 sixteenth = __float2half2_rn(0.0625f);
        const uint32_t v = w >> 8;
        a[0] = half2_as_u32(__hadd2(u32_as_half2(w4_place(w, 0x000f000fu, 0x64006400u)), u32_as_half2(za)));
        a[1] = half2_as_u32(__hfma2(u32_as_half2(w4_place(w, 0x00f000f0u, 0x64006400u)), sixteenth, u32_as_half2(zb)));
        a[2] = half2_as_u32(__hadd2(u32_as_half2(w4_place(v, 0x000f000fu, 0x64006400u)), u32_as_half2(za)));
        a[3] = half2_as_u32(__hfma2(u32_as_half2(w4_place(v, 0x00f000f0u, 0x64006400u)), sixteenth, u32_as_half2(zb)));
    }
};
template <>
struct W4Dec<__nv_bfloat16> {
    // 0x4300 | q is 128 + q (7 mantissa bits hold it exactly), and 128 + z <= 143 is exact too
    uint32_t za, zb;   // -(128 + z) twice, per row
    __device__ __forceinline__ static uint32_t dup(float f)
    {
        const __nv_bfloat162 h = __float2bfloat162_rn(f);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ __forceinline__ void zero(int z0, int z1)
    {
        za = dup(-128.0f - z0);
        zb = dup(-128.0f - z1);
    }
    __device__ __forceinline__ static uint32_t sub(uint32_t q, uint32_t z)
    {
        const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&q), *reinterpret_cast<const __nv_bfloat162*>(&z));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&a)[4]) const
    {
        a[0] = sub(w4_place(w, 0x000f000fu, 0x43004300u), za);
        a[1] = sub(w4_place(w >> 4, 0x000f000fu, 0x43004300u), zb);
        a[2] = sub(w4_place(w >> 8, 0x000f000fu, 0x43004300u), za);
        a[3] = sub(w4_place(w >> 12, 0x000f000fu, 0x43004300u), zb);
    }
};

// d = a b + c; c = 0 where `fresh`
template <typename T>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool fresh)
{
    const float c0 = fresh ? 0.0f : d[0], c1 = fresh ? 0.0f : d[1], c2 = fresh ? 0.0f : d[2], c3 = fresh ? 0.0f : d[3];
    if constexpr (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ float w4_scale(uint32_t bits16, int bf16)
{
    return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}

// the weight stream passes L1 by: it keeps the inputs and the scales
__device__ __forceinline__ uint4 w4_stream(const uint4* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// N words in one load
template <int N>
__device__ __forceinline__ void w4_words(const uint32_t* p, uint32_t (&v)[N])
{
    if constexpr (N == 1) {
        v[0] = __ldg(p);
    } else if constexpr (N == 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        v[0] = u.x, v[1] = u.y;
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    }
}

// min(silu(g), L) * clamp(u, -L, L), L = 0: no clamps. Clamps by comparison: minimum and maximum would turn a NaN product
// into a limit. The fast exp and division are off by 2^-17 at gates of -60: nothing to a 16-bit output (half a unit is 2^-12 or
// 2^-9), too much for a fp32 one, which takes the full ones.
static __device__ __noinline__ float w4_silu_full(float g) { return g / (1.0f + expf(-g)); }
template <bool FULL>
__device__ __forceinline__ float w4_swiglu(float g, float u, float limit)
{
    float s = FULL ? w4_silu_full(g) : __fdividef(g, 1.0f + __expf(-g));
    if (limit != 0.0f) {
        s = s > limit ? limit : s;
        u = u > limit ? limit : u < -limit ? -limit : u;
    }
    return s * u;
}

// Work: one CTA per SM takes a run of whole row tiles, its warps equal runs of that run's steps (of 128 inputs), so
// the warps of a small matrix share one tile's inputs and those of a large one take tiles of their own, by the same
// rule. Codes, scales and zero points of a CTA's steps are contiguous; a warp keeps D steps on their way in
// registers, across the ends of tiles. A tile that one warp holds whole goes out from its registers; the parts of a
// shared one lie in shared memory and its first warp adds them in order once all have ended.
// TB: token blocks of 8 per CTA (blockIdx.y: further ones). GATED: a step is one of gate and one of up.
// Measured: 100001 x 4096, groups of 128, 4 tokens: 49 us, 4.3 TB/s of codes and scales (floor 32 us). No pipe is full (ALU 62%,
// issue slots 61%, tensor pipe 26%), and 8, 16, 20 and 24 warps and 2 to 6 steps in flight are within 5%: a warp's loads and its
// decoding wait on one another. CTAs of 8 warps x 4 row tiles without a stream took 86 us. Small ones (4096 x 2048,
// 1 token, 10 us) are a launch and one trip of the codes. From 17 tokens on a fragment of weights feeds four products of 8 tokens
// and a group's scales as many additions: 32 tokens of 2 x 2048 x 4096 12 us, 22 tokens of 2 x 5970 x 8864 in groups of 32 51 us,
// 91 TFLOP/s. Every further 32 tokens read and unpack the weights again: 144 tokens of 2 x 2048 x 4096 53 us, 512 139 us.
// Whole row tiles to a CTA leave SMs idle where the tiles are not a multiple of their number (2560 outputs: 160 tiles, 12 CTAs with two).
template <int TB, bool GATED>
struct W4Cfg {
    static constexpr int nt = GATED ? 2 : 1;
    static constexpr int warps = GATED && TB == 4 ? 8 : 16;
    static constexpr int depth = GATED || TB == 4 ? 2 : 4;
    static constexpr int part = nt * TB * 4 * 32;            // values of a part
    static constexpr int smem = warps * 2 * part * 4;        // a warp's first and last part
};

template <typename T, int GS, int TB, bool GATED, bool ZEROS>
__global__ void __launch_bounds__(W4Cfg<TB, GATED>::warps * 32, 1) w4_kernel(const W4Params p)
{
    using Cfg = W4Cfg<TB, GATED>;
    constexpr int NT = Cfg::nt, D = Cfg::depth, W = Cfg::warps, G = 128 / GS, kPer = GS / 32;
    extern __shared__ float parts[];   // [warp][first, last][tile][block][4][lane]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    const int tile0 = (int)((int64_t)p.n16 * blockIdx.x / gridDim.x), tile1 = (int)((int64_t)p.n16 * (blockIdx.x + 1) / gridDim.x);
    const int K = p.k128, S = (tile1 - tile0) * K;   // steps of the CTA (bounded: checked on the host)
    const int s0 = (int)((int64_t)S * warp / W), s1 = (int)((int64_t)S * (warp + 1) / W);
    const int t0 = blockIdx.y * 8 * TB;

    // this lane's token of each block; lanes past the last token repeat it (their sums are not put out)
    const T* xr[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b)
        xr[b] = static_cast<const T*>(p.x) + (int64_t)min(t0 + b * 8 + r, p.tokens - 1) * p.x_stride + c * 8;
    struct Step {
        uint4 w[NT][2];
        uint32_t sc[NT][G];
        uint16_t z[NT][ZEROS ? G : 1];
    } st[D];
    const int64_t base = (int64_t)tile0 * K;
    auto fetch = [&](int s, Step& d) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const W4Mat& m = GATED && t ? p.b : p.a;
            const uint4* src = m.codes + base * 64 + lane + s * 64;
            d.w[t][0] = w4_stream(src);
            d.w[t][1] = w4_stream(src + 32);
            w4_words<G>(m.scales + (base * 8 + r) * G + s * (8 * G), d.sc[t]);
            if (ZEROS) {
#pragma unroll
                for (int g = 0; g < G; ++g) d.z[t][g] = __ldg(m.zeros + (base * 8 + r) * G + s * (8 * G) + g);
            }
        }
    };
    float tot[NT][TB][4];
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int b = 0; b < TB; ++b) tot[t][b][0] = tot[t][b][1] = tot[t][b][2] = tot[t][b][3] = 0.0f;
    };
    auto multiply = [&](int j, const Step& d) {
        float acc[NT][TB][4];
        // inputs left in the row: fewer than 128 in the last step of a row that ends inside it (groups of 32 and 64).
        // The inputs past its end are read from before it, and their groups are not added.
        const int left = GS == 128 ? 128 : p.k - j * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {   // 32 inputs
            const int g = q / kPer;
            uint4 xv[TB];
#pragma unroll
            for (int b = 0; b < TB; ++b)
                xv[b] = __ldg(reinterpret_cast<const uint4*>(xr[b] + j * 128 + (GS == 128 ? q * 32 : min(q * 32, left - 32))));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                W4Dec<T> dec;
                if (ZEROS) dec.zero(d.z[t][g] & 255, d.z[t][g] >> 8);
                else dec.zero(8, 8);
                const uint4 v = d.w[t][q >> 1];
                uint32_t a[4];
                dec(q & 1 ? v.z : v.x, a);
#pragma unroll
                for (int b = 0; b < TB; ++b) w4_mma<T>(acc[t][b], a, xv[b].x, xv[b].y, q % kPer == 0);
                dec(q & 1 ? v.w : v.y, a);
#pragma unroll
                for (int b = 0; b < TB; ++b) w4_mma<T>(acc[t][b], a, xv[b].z, xv[b].w, false);
                if (q % kPer == kPer - 1 && g * GS < left) {
                    const float f0 = w4_scale(d.sc[t][g] & 0xffffu, p.scale_bf16), f1 = w4_scale(d.sc[t][g] >> 16, p.scale_bf16);
#pragma unroll
                    for (int b = 0; b < TB; ++b) {
                        tot[t][b][0] = fmaf(f0, acc[t][b][0], tot[t][b][0]);
                        tot[t][b][1] = fmaf(f0, acc[t][b][1], tot[t][b][1]);
                        tot[t][b][2] = fmaf(f1, acc[t][b][2], tot[t][b][2]);
                        tot[t][b][3] = fmaf(f1, acc[t][b][3], tot[t][b][3]);
                    }
                }
            }
        }
    };
    // the sums of a whole tile to the output: a lane has rows r, r + 8 and tokens 2c, 2c + 1 of each block
    // (SwiGLU before the stores, in loops of its own: within them it cost 32 tokens of 2 x 2048 x 4096 11.5 us for 10.6)
    auto put = [&](int tile) {
        auto gate = [&](auto full) {
#pragma unroll
            for (int b = 0; b < TB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) tot[0][b][e] = w4_swiglu<decltype(full)::value>(tot[0][b][e], tot[NT - 1][b][e], p.limit);
        };
        if (GATED && p.out_dtype == DSV41_DTYPE_F32) gate(std::true_type());
        else if (GATED) gate(std::false_type());
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = t0 + b * 8 + 2 * c + (e & 1), n = tile * 16 + r + 8 * (e >> 1);
                if (t >= p.tokens || n >= p.n) continue;
                const float y = tot[0][b][e];
                const int64_t at = (int64_t)t * p.out_stride + n;
                if (p.out_dtype == DSV41_DTYPE_F32) {
                    float* o = static_cast<float*>(p.out) + at;
                    *o = p.accumulate ? *o + y : y;
                } else if (p.out_dtype == DSV41_DTYPE_BF16) {
                    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
                } else {
                    static_cast<__half*>(p.out)[at] = __float2half_rn(y);
                }
            }
    };
    auto part_of = [&](int w, int which) { return parts + (w * 2 + which) * Cfg::part + lane; };

    clear();
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (s0 + d < s1) fetch(s0 + d, st[d]);
    int tile = s0 / K, j = s0 - tile * K, j_first = j;
    for (int s = s0; s < s1; s += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (s + d >= s1) break;
            multiply(j, st[d]);
            if (s + d + D < s1) fetch(s + d + D, st[d]);
            if (++j == K || s + d + 1 == s1) {   // the end of the tile, or of the warp's run
                if (j_first == 0 && j == K) {
                    put(tile0 + tile);
                } else {   // a part: of a tile that began in an earlier warp, or that goes on in the next
                    float* to = part_of(warp, j_first > 0 ? 0 : 1);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int b = 0; b < TB; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) to[((t * TB + b) * 4 + e) * 32] = tot[t][b][e];
                }
                clear();
                ++tile;
                j = j_first = 0;
            }
        }
    }
    __syncthreads();
    // a tile that begins in this warp's run and goes on past it
    if (s0 < s1 && s1 % K != 0 && (s1 / K) * K >= s0) {
        const int own = s1 / K, end = (own + 1) * K;
        for (int w = warp; w < W; ++w) {
            const int a = (int)((int64_t)S * w / W), b1 = (int)((int64_t)S * (w + 1) / W);
            if (a >= end) break;
            if (a == b1) continue;
            const float* from = part_of(w, w == warp ? 1 : 0);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) tot[t][b][e] += from[((t * TB + b) * 4 + e) * 32];
        }
        put(tile0 + own);
    }
}

template <typename T, int GS, int TB, bool GATED, bool ZEROS>
static cudaError_t launch_w4_shape(const W4Params& p, cudaStream_t st)
{
    using Cfg = W4Cfg<TB, GATED>;
    auto kernel = w4_kernel<T, GS, TB, GATED, ZEROS>;
    if (Cfg::smem > 48 * 1024) {
        static bool ready[64] = {};   // the attribute is per device and kernel, and stays
        int dev = 0;
        cudaError_t err = cudaGetDevice(&dev);
        if (err != cudaSuccess) return err;
        if (dev >= 64 || !ready[dev]) {
            if ((err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem)) != cudaSuccess) return err;
            if (dev < 64) ready[dev] = true;
        }
    }
    const int sms = num_sms(), gy = (p.tokens + 8 * TB - 1) / (8 * TB);
    kernel<<<dim3(p.n16 < sms ? p.n16 : sms, gy), Cfg::warps * 32, Cfg::smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int GS, bool GATED, bool ZEROS>
static cudaError_t launch_w4_tb(const W4Params& p, cudaStream_t st)
{
    if (p.tokens <= 8) return launch_w4_shape<T, GS, 1, GATED, ZEROS>(p, st);
    if (p.tokens <= 16) return launch_w4_shape<T, GS, 2, GATED, ZEROS>(p, st);
    return launch_w4_shape<T, GS, 4, GATED, ZEROS>(p, st);
}

template <typename T, bool GATED, bool ZEROS>
static cudaError_t launch_w4_group(const W4Params& p, int group, cudaStream_t st)
{
    if (group == 32) return launch_w4_tb<T, 32, GATED, ZEROS>(p, st);
    if (group == 64) return launch_w4_tb<T, 64, GATED, ZEROS>(p, st);
    return launch_w4_tb<T, 128, GATED, ZEROS>(p, st);
}

template <typename T>
cudaError_t launch_w4_typed(const W4Params& p, int group, bool gated, cudaStream_t st)
{
    if (p.a.zeros) return gated ? launch_w4_group<T, true, true>(p, group, st) : launch_w4_group<T, false, true>(p, group, st);
    return gated ? launch_w4_group<T, true, false>(p, group, st) : launch_w4_group<T, false, false>(p, group, st);
}

}  // namespace dsv41
