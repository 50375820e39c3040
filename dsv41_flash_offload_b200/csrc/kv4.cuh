// A cache in 4 bits: its layout, and how codes become 16-bit values.
//
// A token's head is cut into groups ("chunks") of 32 columns. A chunk stands for T(lo + s * code) in the cache's type T, codes
// 0..15, lo and s of type T. One (page, KV head) holds its keys, then its values: records of 8 tokens, which go to shared memory
// whole and are read there as they lie:
//     [chunk][place][16 bytes of codes], then [chunk][token][s, lo]          160 bytes a chunk
// Token t of chunk c has its codes at place t ^ (0, 5, 2, 7)[c % 4], so that the lanes of a warp, which read one token in several chunks
// and several tokens in one, find them in different banks.
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

__host__ __device__ constexpr int kv4_place(int chunk, int token) { return token ^ ((chunk & 3) | (chunk & 1) << 2); }
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

// Scales of a chunk, or of two keys' chunks, as pairs.
template <typename T>
struct Scale2 {
    using P = typename Pair16<T>::type;
    P s, s4, lo;   // s4: 4 s (bf16: it is finite where the range of the chunk is)
    __device__ __forceinline__ Scale2(uint32_t a, uint32_t b, uint32_t s_sel, uint32_t lo_sel)
    {
        const uint32_t sv = prmt(a, b, s_sel), lv = prmt(a, b, lo_sel), four = 0x40804080u;
        s = *reinterpret_cast<const P*>(&sv), lo = *reinterpret_cast<const P*>(&lv);
        if constexpr (!std::is_same<T, __half>::value) s4 = __hmul2(s, *reinterpret_cast<const P*>(&four));
    }
    __device__ __forceinline__ explicit Scale2(uint32_t one) : Scale2(one, one, 0x1010, 0x3232) {}          // of one chunk, twice
    __device__ __forceinline__ Scale2(uint32_t a, uint32_t b) : Scale2(a, b, 0x5410, 0x7632) {}             // of a, b
};

// The pair whose codes are in bits 4 I .. 4 I + 3 of w's half-words, as lo + s * code, rounded once: the code is exact in T and
// the product and the sum are one fused operation. Even places: the code as the low bits of 1024 or 128, less that number. Odd ones without a
// shift of their own: fp16 has room for bits 4 to 7 of its significand as well (16 times the code, scaled back with the
// subtraction); in bf16 a half-word of 0 .. 255 is the number 2^-133 times that, across the end of the subnormals, and times
// 2^127 a quarter of the code.
template <typename T, int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, const Scale2<T>& sc)
{
    using P = typename Pair16<T>::type;
    constexpr uint32_t m = Pair16<T>::magic;
    auto pair = [](uint32_t v) { return *reinterpret_cast<const P*>(&v); };
    const uint32_t at = w >> (8 * (I / 2));
    P v;
    if constexpr (I % 2 == 0) v = __hfma2(__hsub2(pair(mask_or(at, 0x000f000fu, m)), pair(m)), sc.s, sc.lo);
    else if constexpr (std::is_same<T, __half>::value)
        v = __hfma2(__hfma2(pair(mask_or(at, 0x00f000f0u, m)), pair(0x2c002c00u), pair(0xd400d400u)), sc.s, sc.lo);   // / 16 - 64
    else v = __hfma2(__hmul2(pair(at & 0x00f000f0u), pair(0x7f007f00u)), sc.s4, sc.lo);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ uint4 kv4_word(uint32_t w, const Scale2<T>& sc)   // its 8 columns
{
    return make_uint4(kv4_pair<T, 0>(w, sc), kv4_pair<T, 1>(w, sc), kv4_pair<T, 2>(w, sc), kv4_pair<T, 3>(w, sc));
}

// whether a chunk stands for NaN (lo is)
template <typename T>
__device__ __forceinline__ bool kv4_nan(uint32_t scales)
{
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c000000u : 0x7f800000u;
    return (scales & e) == e;
}

}  // namespace dsv41
