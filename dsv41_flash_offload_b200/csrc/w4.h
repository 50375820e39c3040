// Launch interface of the 4-bit weight products (w4.cu) for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dsv41 {

// Laid-out matrix (one device buffer): row tiles of 16 output features, k steps of 128 inputs (two chunks of 64).
//   codes  [n16][k128][2][32 lanes] x 16 bytes                       a lane's 32 codes of a chunk
//   scales [n16][k128][8][groups of a step] x {row r, row r + 8} 16-bit
//   zeros  [n16][k128][8][groups of a step] x {row r, row r + 8} 8-bit (only with zero points)
// so that each of them is one load per lane and step. Rows past n and inputs past k have scale 0.
struct W4Layout {
    int n16, k128, groups;   // groups: per step
    size_t scales_off, zeros_off, total;
    static W4Layout make(int n, int k, int group, bool zeros)
    {
        W4Layout l;
        l.n16 = (n + 15) / 16;
        l.k128 = (k + 127) / 128;
        l.groups = 128 / group;
        auto up = [](size_t v) { return (v + 255) / 256 * 256; };
        const size_t steps = (size_t)l.n16 * l.k128;
        l.scales_off = steps * 1024;
        l.zeros_off = l.scales_off + up(steps * l.groups * 32);
        l.total = l.zeros_off + (zeros ? up(steps * l.groups * 16) : 0);
        return l;
    }
};

struct W4Mat {
    const uint4* codes;
    const uint32_t* scales;
    const uint16_t* zeros;   // NULL: every zero point is 8
};

struct W4Params {
    W4Mat a, b;              // b: the up matrix of the gated form
    const void* x;           // [tokens][x_stride]
    void* out;               // [tokens][out_stride]
    int64_t x_stride, out_stride;
    int tokens, n, k, n16, k128;
    int scale_bf16;          // scales are bf16 (else fp16)
    int out_dtype;           // DSV41_DTYPE_*
    int accumulate;          // out += (fp32 outputs)
    float limit;             // gated: clamp of SwiGLU, 0 = none
};

cudaError_t launch_w4(const W4Params& p, int x_dtype, int group, bool gated, cudaStream_t st);
cudaError_t launch_w4_f16(const W4Params& p, int group, bool gated, cudaStream_t st);
cudaError_t launch_w4_bf16(const W4Params& p, int group, bool gated, cudaStream_t st);
cudaError_t launch_w4_pack(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group,
                           void* dst, cudaStream_t st);

}  // namespace dsv41
