// kv4.hpp -- the 4-bit cache's layout (include/trhip.h): pieces of sixteen places, 9 * dim bytes of codes and scales each.
//
// The codes lie as the attention's matrix operands want them (attn4.hip): lane r + 16 q of a wave takes its dim / 8 bytes of a piece of
// keys (place r, elements 32 b + 8 q ... of every block b) and of a piece of values (elements 32 b + 2 r and 2 r + 1, places 4 q ...
// 4 q + 3) as they stand, 64 lanes one run of memory.
#pragma once

#include "trhip_internal.hpp"

namespace trhip {

// Where a place of a page lies, and where its scale of block b is in its piece.
struct Kv4Place {
    int64_t piece;  // the piece's byte offset in its plane
    int r;          // the place in it
};
__device__ __forceinline__ Kv4Place kv4_place(int64_t slot, int page_log2, int heads, int head, int dim) {
    const int64_t pg = slot >> page_log2, in = slot & ((1 << page_log2) - 1);
    return {((((pg * heads + head) << page_log2) + (in & ~15)) >> 4) * (9 * dim), (int)(in & 15)};
}
__device__ __forceinline__ int kv4_scale_at(int r, int b, int dim) { return 8 * dim + 2 * ((((r >> 2) * (dim >> 5)) + b) * 4 + (r & 3)); }

// The scale of a block whose element of largest magnitude is m: m / -8 rounded to five significant bits, then to f16, at most 7936;
// NaN where m is not finite.
__device__ __forceinline__ uint32_t kv4_scale(float m) {
    const uint32_t b = __float_as_uint(m) & 0x7FFFFFFFu;
    if (b >= 0x7F800000u) return 0x7E00u;
    const uint32_t a = __float_as_uint(__uint_as_float(b) * 0.125f);  // exact, or too small for f16
    const float r = fminf(__uint_as_float((a + 0x3FFFFu + ((a >> 19) & 1u)) & 0xFFF80000u), 7936.0f);
    return __builtin_bit_cast(uint16_t, (_Float16)r) | (m > 0.0f ? 0x8000u : 0u);
}
// clamp(rint(x / d), -8, 7) + 8, plus kCode (a float's bits: the sum with 1.5 * 2^23 + 8 rounds, to even at a half, and its last bits are
// the code). inv is 1 / d rounded, d has five significant bits. What is rounded, q, is x / d but for 2^-46 of it, rounded once: the
// remainder x - q0 d has few bits and is exact. Where x / d is half a whole number, q is it. Where it is not, q is not either: x is a
// neighbour of the half's x or farther, that is 2^-24 (1 + 2^-9) of it at least (such an x has nine bits), and q's rounding is 2^-24 of it
// at most (less below a power of two, where x's neighbours are as near).
constexpr uint32_t kCode = 0x4B400000u;
__device__ __forceinline__ uint32_t kv4_code(float x, float d, float inv) {
    const float q0 = x * inv, q = fmaf(fmaf(-q0, d, x), inv, q0);
    return __float_as_uint(__builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 12582920.0f);
}

}  // namespace trhip
