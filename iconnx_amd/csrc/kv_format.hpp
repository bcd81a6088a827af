// The quantized key / value cache in memory.
//
// A block of 32 consecutive values of one head of one token has a power-of-two scale 2^e, held as
// the byte e + 127 (255: the block held an infinity or a NaN, and reads back as NaN), and a code of
// 4 bits (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) or 8 bits (4 of exponent, 3 of mantissa, up to 448)
// for each value.  The CU converts both to bfloat16 pairs, scale included, in one instruction
// (v_cvt_scalef32_pk_bf16_fp4 / _fp8), and the result is exact: a code has at most 4 significant
// bits, and e stays where neither end of the range leaves bfloat16's normal numbers, so the matrix
// cores multiply what the cache holds.  The instruction reads the exponent bits of its f32 scale
// operand and nothing else, so a byte of four is put in place by one shift.
//
// Memory is laid out for the attention kernels' matrix instructions.  A page holds page_size tokens
// of every head; each head's part is cut into chunks of 16 tokens, and a chunk of G = D / 32 blocks
// a token is
//   keys' codes    lane (token t, quarter j) of an operand reads the D / 4 codes of its quarter of the
//                  head, G * bits bytes at (4 t + j) * G * bits: token by token, as written
//   values' codes  lane (d = 0..15, quad j) reads the codes of tokens 4 j .. 4 j + 3 and of the values
//                  32 g + d and 32 g + 16 + d of every block g: bits bytes for each (j, d, g), the two
//                  values of a token side by side (low and high nibble, or two bytes)
//   keys' scales   byte t * G + g
//   values' scales byte (j * G + g) * 4 + (t & 3), j = t / 4
// so that an operand of either product is one wide load a lane, keys without a transpose in the
// way and values already transposed.
#pragma once

#include "elem.hpp"

namespace icx {

struct KvLayout {
    int64_t page_bytes;
    int head_bytes, chunk_bytes;
    int chunks;  // of 16 tokens, a page
    int heads, G, bits;
};

inline KvLayout kv_layout(const icx_kv_cache& c) {
    KvLayout l;
    l.G = c.head_size / 32;
    l.bits = c.bits;
    l.heads = c.kv_heads;
    l.chunks = c.page_size / 16;
    l.chunk_bytes = 2 * (64 * l.G * c.bits + 16 * l.G);
    l.head_bytes = l.chunks * l.chunk_bytes;
    l.page_bytes = (int64_t)l.heads * l.head_bytes;
    return l;
}

// Whether the descriptor is one that the kernels take (a message in icx_last_error if not).
int check_kv_cache(const icx_kv_cache* c, const char* who);

// Byte offsets inside a chunk.
__host__ __device__ __forceinline__ int kv_codes(int G, int bits) { return 64 * G * bits; }
__host__ __device__ __forceinline__ int kv_key_scales(int G, int bits) { return 2 * kv_codes(G, bits); }
__host__ __device__ __forceinline__ int kv_value_scales(int G, int bits) { return 2 * kv_codes(G, bits) + 16 * G; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// The f32 whose exponent bits are byte `b` (0..3) of w; its other bits are whatever w holds there.
__device__ __forceinline__ float scale_of(uint32_t w, int b) {
    return __uint_as_float(b == 3 ? w >> 1 : w << (23 - 8 * b));
}

// Two values as packed bfloat16: 4 bits, byte `sel` of w; 8 bits, half `sel` of w.
template <int BITS, int SEL>
__device__ __forceinline__ uint32_t decode2(uint32_t w, float scale) {
    if constexpr (BITS == 4)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, SEL != 0));
}

// The biased exponent of a block's scale from the bits of its largest magnitude: the least one for
// which that magnitude does not round past the largest code.  In 4 bits the line is at 7, half way
// from 6 to the 8 that the next code would be (a tie goes to the even code, that one); in 8 bits at
// 464, half way from 448 to 480 (the tie goes to 448).  Below 2^-126 the exponent field is 0 and
// the least scale is taken anyway.
template <int BITS>
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
    const int e = (int)(top >> 23);
    const uint32_t m = top & 0x7fffffu;
    if (e == 255) return 255u;
    const int r = BITS == 4 ? e - 2 + (m >= 0x600000u) : e - 8 + (m > 0x680000u);
    return (uint32_t)(BITS == 4 ? min(max(r, 2), 252) : min(max(r, 10), 246));
}

}  // namespace icx
