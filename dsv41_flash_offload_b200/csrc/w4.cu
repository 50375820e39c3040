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
#include "../../include/dsv41_b200.h"
#include "common.cuh"
#include "internal.h"
#include "w4.h"

namespace dsv41 {

// chunk position of (mma w, lane column c, i of 0..3): the four k of a lane's fragment in mma w
__host__ __device__ constexpr int w4_k_of(int w, int c, int i) { return (w >> 1) * 32 + c * 8 + (w & 1) * 4 + i; }

__global__ void w4_pack_kernel(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group,
                               W4Layout l, unsigned char* dst)
{
    const int64_t steps = (int64_t)l.n16 * l.k128, words = steps * 256, pairs = steps * 8 * l.groups;
    const int g_in = k / group;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words + pairs;
         i += (int64_t)gridDim.x * blockDim.x) {
        if (i < words) {
            const int w = (int)(i & 3), lane = (int)(i >> 2) & 31, chunk = (int)(i >> 7) & 1, r = lane >> 2, c = lane & 3;
            const int64_t step = i >> 8;
            const int tile = (int)(step / l.k128), j = (int)(step - (int64_t)tile * l.k128);
            uint32_t v = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {   // e: k pair element (e & 1), register a0..a3 (e >> 1)
                const int reg = e >> 1, row = tile * 16 + r + (reg & 1) * 8;
                const int kk = j * 128 + chunk * 64 + w4_k_of(w, c, (reg >> 1) * 2 + (e & 1));
                uint32_t code = 0;
                if (row < n && kk < k) code = (q[(int64_t)row * (k / 2) + kk / 2] >> (4 * (kk & 1))) & 15u;
                v |= code << (4 * reg + 16 * (e & 1));
            }
            reinterpret_cast<uint32_t*>(dst)[i] = v;
        } else {
            const int64_t s = i - words;
            const int in_step = (int)(s % l.groups), r = (int)(s / l.groups) & 7;
            const int64_t step = s / (8 * l.groups);
            const int tile = (int)(step / l.k128), g = (int)(step - (int64_t)tile * l.k128) * l.groups + in_step;
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
    const int64_t items = (int64_t)l.n16 * l.k128 * (256 + 8 * l.groups);
    const int64_t ctas = (items + 255) / 256, cap = 32 * num_sms();
    w4_pack_kernel<<<(int)(ctas > cap ? cap : ctas), 256, 0, st>>>(q, scales, zeros, n, k, group, l,
                                                                   static_cast<unsigned char*>(dst));
    return cudaGetLastError();
}

cudaError_t launch_w4(const W4Params& p, int x_dtype, int group, bool gated, cudaStream_t st)
{
    return x_dtype == DSV41_DTYPE_F16 ? launch_w4_f16(p, group, gated, st) : launch_w4_bf16(p, group, gated, st);
}

}  // namespace dsv41
