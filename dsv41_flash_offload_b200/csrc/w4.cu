// Products of a few tokens with 4-bit weights and group scales (dsv41_w4_linear, dsv41_w4_gated).
//
//     y[t, n] = sum_g s[n, g] * sum_{k in group g} (q[n, k] - z[n, g]) * x[t, k]
// gated: y = min(silu(gate), limit) * clamp(up, -limit, limit) of two such products.
//
// Arithmetic: q - z is a whole number of -15..15, exact in fp16 and bf16, so the tensor
// cores multiply the codes themselves with the unrounded inputs and accumulate in fp32; each group's sum is
// scaled in fp32. Nothing is rounded to 16 bits before the output.
//
// Bound: HBM, half a byte per weight (plus scales). One warp streams whole 512-byte chunks (16 features x 64
// inputs, one 16-byte load per lane) that were laid out once so that a lane's word holds exactly its mma
// fragment: the weights are the A operand (16 features x 16 inputs), the tokens the B operand (8 tokens).
// The inputs of a chunk are assigned to fragment positions such that a lane's B registers are 16 contiguous
// bytes of a token's row: x needs no shared memory and no shuffle.
#include <cuda_bf16.h>

#include "../../include/dsv41_b200.h"
#include "common.cuh"
#include "internal.h"
#include "w4.h"

namespace dsv41 {

constexpr int kW4Warps = 8;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4Unroll = 4;   // chunks of each of the two row tiles in flight per warp

// chunk position of (mma w, lane column c, i of 0..3): the four k of a lane's fragment in mma w
__host__ __device__ constexpr int w4_k_of(int w, int c, int i) { return (w >> 1) * 32 + c * 8 + (w & 1) * 4 + i; }

__global__ void w4_pack_kernel(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group,
                               W4Layout l, unsigned char* dst)
{
    const int64_t words = (int64_t)l.n16 * l.k64 * 128, pairs = (int64_t)l.n16 * l.groups * 8;
    const int g_in = k / group;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words + pairs;
         i += (int64_t)gridDim.x * blockDim.x) {
        if (i < words) {
            const int w = (int)(i & 3), lane = (int)(i >> 2) & 31, r = lane >> 2, c = lane & 3;
            const int64_t chunk = i >> 7;
            const int tile = (int)(chunk / l.k64), j = (int)(chunk - (int64_t)tile * l.k64);
            uint32_t v = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {   // e: k pair element (e & 1), register a0..a3 (e >> 1)
                const int reg = e >> 1, row = tile * 16 + r + (reg & 1) * 8;
                const int kk = j * 64 + w4_k_of(w, c, (reg >> 1) * 2 + (e & 1));
                uint32_t code = 0;
                if (row < n && kk < k) code = (q[(int64_t)row * (k / 2) + kk / 2] >> (4 * (kk & 1))) & 15u;
                v |= code << (4 * reg + 16 * (e & 1));
            }
            reinterpret_cast<uint32_t*>(dst)[i] = v;
        } else {
            const int64_t s = i - words;
            const int r = (int)(s & 7);
            const int64_t tg = s >> 3;
            const int tile = (int)(tg / l.groups), g = (int)(tg - (int64_t)tile * l.groups);
            uint32_t sv = 0;
            uint16_t zv = 0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = tile * 16 + r + 8 * half;
                if (row >= n || g >= g_in) continue;
                sv |= (uint32_t)scales[(int64_t)row * g_in + g] << (16 * half);
                if (zeros) zv |= (uint16_t)(zeros[(int64_t)row * g_in + g] << (8 * half));
            }
            reinterpret_cast<uint32_t*>(dst + l.scales_off)[s] = sv;
            if (zeros) reinterpret_cast<uint16_t*>(dst + l.zeros_off)[s] = zv;
        }
    }
}

cudaError_t launch_w4_pack(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group,
                           void* dst, cudaStream_t st)
{
    const W4Layout l = W4Layout::make(n, k, group, zeros != nullptr);
    const int64_t items = (int64_t)l.n16 * l.k64 * 128 + (int64_t)l.n16 * l.groups * 8;
    const int64_t ctas = (items + 255) / 256, cap = 32 * num_sms();
    w4_pack_kernel<<<(int)(ctas > cap ? cap : ctas), 256, 0, st>>>(q, scales, zeros, n, k, group, l,
                                                                   static_cast<unsigned char*>(dst));
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------
// codes of one word -> the A fragment {row r: k 0,1 | row r + 8: k 0,1 | row r: k 2,3 | row r + 8: k 2,3} of
// q - z. za, zb: the rows' zero points in the form that the type's decode subtracts (w4_zero).
// ---------------------------------------------------------------------------------------------
template <typename T>
struct W4Dec;
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
        a[0] = half2_as_u32(__hadd2(u32_as_half2((w & 0x000f000fu) | 0x64006400u), u32_as_half2(za)));
        a[1] = half2_as_u32(__hfma2(u32_as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, u32_as_half2(zb)));
        a[2] = half2_as_u32(__hadd2(u32_as_half2((v & 0x000f000fu) | 0x64006400u), u32_as_half2(za)));
        a[3] = half2_as_u32(__hfma2(u32_as_half2((v & 0x00f000f0u) | 0x64006400u), sixteenth, u32_as_half2(zb)));
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
        a[0] = sub((w & 0x000f000fu) | 0x43004300u, za);
        a[1] = sub(((w >> 4) & 0x000f000fu) | 0x43004300u, zb);
        a[2] = sub(((w >> 8) & 0x000f000fu) | 0x43004300u, za);
        a[3] = sub(((w >> 12) & 0x000f000fu) | 0x43004300u, zb);
    }
};

template <typename T>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value) {
        mma_16816(d, a, b0, b1);
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ float w4_scale(uint32_t bits16, int bf16)
{
    return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}

// One CTA: two row tiles (gated: the same tile of gate and up), the 8 warps split the inputs and add their
// sums in shared memory in warp order. TB: token blocks of 8 per CTA (blockIdx.y: further ones).
template <typename T, int GS, int TB, bool GATED>
__global__ void __launch_bounds__(kW4Threads) w4_kernel(const W4Params p)
{
    constexpr int kCols = 8 * TB;
    __shared__ float red[kW4Warps][2][16][kCols + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    const int t0 = blockIdx.y * kCols;
    int tile[2];
    tile[0] = GATED ? blockIdx.x : 2 * blockIdx.x;
    tile[1] = GATED ? blockIdx.x : min(2 * (int)blockIdx.x + 1, p.n16 - 1);
    const int j0 = (int)((int64_t)p.k64 * warp / kW4Warps), j1 = (int)((int64_t)p.k64 * (warp + 1) / kW4Warps);

    float tot[2][TB][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int b = 0; b < TB; ++b) tot[t][b][0] = tot[t][b][1] = tot[t][b][2] = tot[t][b][3] = 0.0f;

    const T* xr[TB];
    bool live[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
        const int t = t0 + b * 8 + r;
        live[b] = t < p.tokens;
        xr[b] = static_cast<const T*>(p.x) + (live[b] ? (int64_t)t * p.x_stride : 0) + c * 8;
    }
    for (int j = j0; j < j1; j += kW4Unroll) {
        uint4 w[2][kW4Unroll];
#pragma unroll
        for (int u = 0; u < kW4Unroll; ++u) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const W4Mat& m = GATED && t ? p.b : p.a;
                if (j + u < j1) w[t][u] = __ldcs(m.codes + ((int64_t)tile[t] * p.k64 + j + u) * 32 + lane);
            }
        }
#pragma unroll
        for (int u = 0; u < kW4Unroll; ++u) {
            if (j + u >= j1) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 xv[TB];
                const int k = (j + u) * 64 + h * 32;
#pragma unroll
                for (int b = 0; b < TB; ++b)
                    xv[b] = (live[b] && k < p.k) ? __ldg(reinterpret_cast<const uint4*>(xr[b] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const W4Mat& m = GATED && t ? p.b : p.a;
                    const int g = GS == 32 ? (j + u) * 2 + h : GS == 64 ? j + u : (j + u) >> 1;
                    const int64_t gi = ((int64_t)tile[t] * p.groups + g) * 8 + r;
                    const uint32_t sc = __ldg(m.scales + gi);
                    const float s0 = w4_scale(sc & 0xffffu, p.scale_bf16), s1 = w4_scale(sc >> 16, p.scale_bf16);
                    W4Dec<T> dec;
                    if (m.zeros) {
                        const uint32_t z = __ldg(m.zeros + gi);
                        dec.zero(z & 255, z >> 8);
                    } else {
                        dec.zero(8, 8);
                    }
                    float acc[TB][4];
#pragma unroll
                    for (int b = 0; b < TB; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.0f;
                    uint32_t a[4];
                    dec(h ? w[t][u].z : w[t][u].x, a);
#pragma unroll
                    for (int b = 0; b < TB; ++b) w4_mma<T>(acc[b], a, xv[b].x, xv[b].y);
                    dec(h ? w[t][u].w : w[t][u].y, a);
#pragma unroll
                    for (int b = 0; b < TB; ++b) w4_mma<T>(acc[b], a, xv[b].z, xv[b].w);
#pragma unroll
                    for (int b = 0; b < TB; ++b) {
                        tot[t][b][0] = fmaf(s0, acc[b][0], tot[t][b][0]);
                        tot[t][b][1] = fmaf(s0, acc[b][1], tot[t][b][1]);
                        tot[t][b][2] = fmaf(s1, acc[b][2], tot[t][b][2]);
                        tot[t][b][3] = fmaf(s1, acc[b][3], tot[t][b][3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            red[warp][t][r][b * 8 + 2 * c] = tot[t][b][0];
            red[warp][t][r][b * 8 + 2 * c + 1] = tot[t][b][1];
            red[warp][t][r + 8][b * 8 + 2 * c] = tot[t][b][2];
            red[warp][t][r + 8][b * 8 + 2 * c + 1] = tot[t][b][3];
        }
    __syncthreads();
    constexpr int kOuts = (GATED ? 16 : 32) * kCols;
    for (int e = threadIdx.x; e < kOuts; e += kW4Threads) {
        const int row = e & 15, tt = GATED ? 0 : (e >> 4) & 1, col = GATED ? e >> 4 : e >> 5;
        const int t = t0 + col, n = tile[tt] * 16 + row;
        if (t >= p.tokens || n >= p.n || (!GATED && tt && 2 * (int)blockIdx.x + 1 >= p.n16)) continue;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w) y += red[w][tt][row][col];
        if (GATED) {
            float up = 0.0f;
#pragma unroll
            for (int w = 0; w < kW4Warps; ++w) up += red[w][1][row][col];
            y = act_gu(y, up, p.limit);
        }
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
}

template <typename T, int GS, bool GATED>
static cudaError_t launch_w4_tb(const W4Params& p, cudaStream_t st)
{
    const int gx = GATED ? p.n16 : (p.n16 + 1) / 2;
    if (p.tokens <= 8) w4_kernel<T, GS, 1, GATED><<<dim3(gx, 1), kW4Threads, 0, st>>>(p);
    else if (p.tokens <= 16) w4_kernel<T, GS, 2, GATED><<<dim3(gx, 1), kW4Threads, 0, st>>>(p);
    else w4_kernel<T, GS, 4, GATED><<<dim3(gx, (p.tokens + 31) / 32), kW4Threads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, bool GATED>
static cudaError_t launch_w4_group(const W4Params& p, int group, cudaStream_t st)
{
    if (group == 32) return launch_w4_tb<T, 32, GATED>(p, st);
    if (group == 64) return launch_w4_tb<T, 64, GATED>(p, st);
    return launch_w4_tb<T, 128, GATED>(p, st);
}

cudaError_t launch_w4(const W4Params& p, int x_dtype, int group, bool gated, cudaStream_t st)
{
    if (x_dtype == DSV41_DTYPE_F16)
        return gated ? launch_w4_group<__half, true>(p, group, st) : launch_w4_group<__half, false>(p, group, st);
    return gated ? launch_w4_group<__nv_bfloat16, true>(p, group, st) : launch_w4_group<__nv_bfloat16, false>(p, group, st);
}

}  // namespace dsv41
