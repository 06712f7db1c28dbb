// kv4.hpp -- the 4-bit cache's layout (include/trhip.h): pieces of sixteen places, 9 * dim bytes of codes and scales each.
//
// The codes lie as the attention's matrix operands want them (attn4.hip): lane r + 16 q of a wave takes its dim / 8 bytes of a piece of
// keys (place r, elements 32 b + 8 q ... of every block b) and of a piece of values (elements 32 b + 2 r and 2 r + 1, places 4 q ...
// 4 q + 3) as they stand, 64 lanes one run of memory.
#pragma once

#include "trhip_internal.hpp"

namespace trhip {

// Where the codes and scales of one place of a page start in its piece, and where an element's nibble lies.
struct Kv4Place {
    int64_t piece;  // the piece's byte offset in its plane
    int r;          // the place in it
};
__device__ __forceinline__ Kv4Place kv4_place(int64_t slot, int page_log2, int heads, int head, int dim) {
    const int64_t pg = slot >> page_log2, in = slot & ((1 << page_log2) - 1);
    return {((((pg * heads + head) << page_log2) + (in & ~15)) >> 4) * (9 * dim), (int)(in & 15)};
}
__device__ __forceinline__ int kv4_scale_at(int r, int b, int dim) { return 8 * dim + 2 * ((((r >> 2) * (dim >> 5)) + b) * 4 + (r & 3)); }
// Byte (from the piece's start) of element e of a value at place r; its nibble is e % 2.
__device__ __forceinline__ int kv4_value_at(int r, int e, int dim) {
    return 4 * (((r >> 2) * 16 + ((e & 31) >> 1)) * (dim >> 5) + (e >> 5)) + (((r & 1) << 1) | ((r >> 1) & 1));
}
// Byte of dword that holds elements e ... e + 7 of a key at place r (e a multiple of 8).
__device__ __forceinline__ int kv4_key_at(int r, int e, int dim) { return 4 * ((((e & 31) >> 3) * 16 + r) * (dim >> 5) + (e >> 5)); }

// The scale of a block whose element of largest magnitude is m: m / -8 rounded to five significant bits, then to f16, at most 7936;
// NaN where m is not finite.
__device__ __forceinline__ uint32_t kv4_scale(float m) {
    const uint32_t b = __float_as_uint(m) & 0x7FFFFFFFu;
    if (b >= 0x7F800000u) return 0x7E00u;
    const uint32_t a = __float_as_uint(__uint_as_float(b) * 0.125f);  // exact, or too small for f16
    const float r = fminf(__uint_as_float((a + 0x3FFFFu + ((a >> 19) & 1u)) & 0xFFF80000u), 7936.0f);
    return __builtin_bit_cast(uint16_t, (_Float16)r) | (m > 0.0f ? 0x8000u : 0u);
}
// clamp(rint(x / d), -8, 7) + 8 without any error before the rounding: r = rint(x * (1 / d)) is one off at most, and x - r d is exact
// (fused, and x and r d are within a factor of two of each other or r is 0), so comparing it with d / 2 corrects r.
__device__ __forceinline__ int kv4_code(float x, float d, float inv) {
    float r = rintf(x * inv);
    r = fminf(fmaxf(r, -9.0f), 9.0f);
    const float a = fabsf(d), e = fmaf(-r, d, x), s = d < 0.0f ? -1.0f : 1.0f, over = 2.0f * e * s;  // in units of |d|, twice what is left
    const bool odd = ((int)r & 1) != 0;
    if (over > a || (over == a && odd)) r += 1.0f;
    else if (over < -a || (over == -a && odd)) r -= 1.0f;
    r = fminf(fmaxf(r, -8.0f), 7.0f);
    return d == 0.0f || a != a ? 8 : (int)r + 8;
}
__device__ __forceinline__ float kv4_value(int code, uint32_t d) { return (float)(code - 8) * f16_to_f32((uint16_t)d); }

}  // namespace trhip
