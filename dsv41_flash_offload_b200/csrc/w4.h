// Launch interface of the 4-bit weight products (w4.cu) for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dsv41 {

// Laid-out matrix (one device buffer): row tiles of 16 output features, k chunks of 64 inputs.
//   codes  [n16][k64][32 lanes] x 16 bytes     a lane's 32 codes of a chunk
//   scales [n16][groups][8] x {row r, row r + 8} 16-bit
//   zeros  [n16][groups][8] x {row r, row r + 8} 8-bit (only with zero points)
// Rows past n and inputs past k have scale 0.
struct W4Layout {
    int n16, k64, groups;
    size_t scales_off, zeros_off, total;
    static W4Layout make(int n, int k, int group, bool zeros)
    {
        W4Layout l;
        l.n16 = (n + 15) / 16;
        l.k64 = (k + 63) / 64;
        l.groups = group == 128 ? (l.k64 + 1) / 2 : l.k64 * (64 / group);
        auto up = [](size_t v) { return (v + 255) / 256 * 256; };
        l.scales_off = (size_t)l.n16 * l.k64 * 512;
        l.zeros_off = l.scales_off + up((size_t)l.n16 * l.groups * 32);
        l.total = l.zeros_off + (zeros ? up((size_t)l.n16 * l.groups * 16) : 0);
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
    int tokens, n, k, n16, k64, groups;
    int scale_bf16;          // scales are bf16 (else fp16)
    int out_dtype;           // DSV41_DTYPE_*
    int accumulate;          // out += (fp32 outputs)
    float limit;             // gated: clamp of SwiGLU, 0 = none
};

cudaError_t launch_w4(const W4Params& p, int x_dtype, int group, bool gated, cudaStream_t st);
cudaError_t launch_w4_pack(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group,
                           void* dst, cudaStream_t st);

}  // namespace dsv41
