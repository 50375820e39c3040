// A cache in 4 bits: its layout, and how codes become 16-bit values.
//
// A token's head is cut into groups ("chunks") of 32 columns. A chunk stands for T(lo + s * code) in the cache's type T, codes
// 0..15, lo and s of type T. One (page, KV head) holds its keys, then its values: records of 8 tokens, so that a warp that wants
// 8 tokens finds each chunk's codes in 128 contiguous bytes at a constant offset:
//     [chunk][token][16 bytes of codes], then [chunk][token][s, lo]          160 bytes a chunk
// A word of 8 codes: columns 0 2 4 6 in its low half-word from the low bits on, 1 3 5 7 in the high one. Masked to 4 bits per half-word
// it is a pair of neighbouring columns.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.h"

namespace dsv41 {

constexpr int kKv4Tokens = 8;          // of a record
constexpr int kKv4Chunk = 32;          // columns
constexpr int kKv4Codes = 128, kKv4Scales = 32;   // bytes of a chunk's codes and scales in a record

__host__ __device__ constexpr int kv4_record(int chunks) { return chunks * (kKv4Codes + kKv4Scales); }
// bytes of the keys (or values) of one page and head
__host__ __device__ inline int64_t kv4_block(int page_size, int chunks) { return (int64_t)page_size / kKv4Tokens * kv4_record(chunks); }

template <typename T>
struct Pair16;
template <>
struct Pair16<__half> {
    using type = __half2;
    static constexpr uint32_t magic = 0x64006400u;   // 1024: the codes lie in the low bits of its significand
};
template <>
struct Pair16<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static constexpr uint32_t magic = 0x43004300u;   // 128
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// (w & mask) | magic in one instruction
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask, uint32_t magic)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
    return r;
}

// The pair whose codes are in bits 4 i .. 4 i + 3 of w's half-words, as lo + s * code, rounded once: the code is exact in T (an
// integer over 1024 or 128 less that number), the product and the sum are one fused operation.
template <typename T, int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, uint32_t s2, uint32_t lo2)
{
    using P = typename Pair16<T>::type;
    const uint32_t m = Pair16<T>::magic, c = mask_or(w >> (4 * I), 0x000f000fu, m);
    const P code = __hsub2(*reinterpret_cast<const P*>(&c), *reinterpret_cast<const P*>(&m));
    const P v = __hfma2(code, *reinterpret_cast<const P*>(&s2), *reinterpret_cast<const P*>(&lo2));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Loads that stay where they are written, ahead of the work that hides their latency (a plain one may be moved to its first use).
__device__ __forceinline__ uint4 load_early16(const void* from)
{
    uint4 v;
    asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from));
    return v;
}
__device__ __forceinline__ uint2 load_early8(const void* from)
{
    uint2 v;
    asm volatile("ld.global.nc.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(from));
    return v;
}
__device__ __forceinline__ uint32_t load_early4(const void* from)
{
    uint32_t v;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(from));
    return v;
}

// whether a chunk stands for NaN (lo is)
template <typename T>
__device__ __forceinline__ bool kv4_nan(uint32_t scales)
{
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c000000u : 0x7f800000u;
    return (scales & e) == e;
}

}  // namespace dsv41
