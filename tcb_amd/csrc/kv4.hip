// kv4.hip -- the 4-bit cache: rows in, quantized, and out again.
//
// A workgroup takes a token, or the four tokens of four places in a row (a quarter of a piece), whose value codes share dwords: written
// together they are dwords, by themselves bytes. A lane has eight elements of each token's row, four lanes a block. Every element moves
// once, so bytes bound it; of few tokens it is a launch. 8192 tokens of 8 heads of 128, bf16, what is read in the last cache: in 15.3 us (2.8 TB/s; 18
// vector instructions an element took 23), out 12.2 (3.5 TB/s); from memory 16.0 and 15.6, in fp32 23 (3.3 TB/s) and 27. Tokens one by one, whose
// value codes are written as bytes: in and out 140 us against 29.
#include "attn_common.hpp"
#include "kv4.hpp"
#include "kv4_runs.hpp"

namespace trhip {
namespace {

struct Kv4Args {
    uint8_t *kc, *vc;
    int page_log2, heads, dim;
    int64_t places, stride;
    uint32_t tokens, run;  // run: tokens of a workgroup
    int wide;              // rows are aligned to 16 bytes
    const int *slots;
};

template <int CTRL> __device__ __forceinline__ uint32_t quad(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}

template <int IO> __device__ __forceinline__ void get8(const void *src, int64_t at, bool wide, float (&f)[8]) {
    if constexpr (IO == TRHIP_F32) {
        const float *s = static_cast<const float *>(src) + at;
        if (wide) {
            *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(s);
            *reinterpret_cast<float4 *>(f + 4) = *reinterpret_cast<const float4 *>(s + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = s[i];
        }
    } else {
        const uint16_t *s = static_cast<const uint16_t *>(src) + at;
        if (wide) {
            const uint4 y = *reinterpret_cast<const uint4 *>(s);
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 4; j++) f[2 * j] = wide_lo<IO == TRHIP_BF16>(w[j]), f[2 * j + 1] = wide_hi<IO == TRHIP_BF16>(w[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = wide_lo<IO == TRHIP_BF16>(s[i]);
        }
    }
}
template <int IO> __device__ __forceinline__ void put8(void *dst, int64_t at, bool wide, const float (&f)[8]) {
    if constexpr (IO == TRHIP_F32) {
        float *d = static_cast<float *>(dst) + at;
        if (wide) {  // four lanes' 128 bytes in two runs of 64: first the first two lanes' eights
            const int lane = threadIdx.x & 3;
            d -= 8 * lane;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t lo = i == 0 ? quad<0x50>(__float_as_uint(f[j])) : quad<0xFA>(__float_as_uint(f[j]));  // lanes 0 0 1 1, 2 2 3 3
                    const uint32_t hi = i == 0 ? quad<0x50>(__float_as_uint(f[4 + j])) : quad<0xFA>(__float_as_uint(f[4 + j]));
                    y[j] = __uint_as_float(lane & 1 ? hi : lo);
                }
                *reinterpret_cast<float4 *>(d + 16 * i + 4 * lane) = make_float4(y[0], y[1], y[2], y[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) d[i] = f[i];
        }
    } else {
        uint16_t *d = static_cast<uint16_t *>(dst) + at;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = pack2<IO == TRHIP_BF16>(f[2 * j], f[2 * j + 1]);
        if (wide) {
            *reinterpret_cast<uint4 *>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) d[2 * j] = (uint16_t)w[j], d[2 * j + 1] = (uint16_t)(w[j] >> 16);
        }
    }
}

// The block's element of largest magnitude, the first of equal ones, from each of its four lanes' eight. As whole numbers the positive
// ones are in order, and without a sign the negative ones; infinities and NaN are above all others. Only where the largest of both
// signs are the same size (in a block of 32 normally distributed bf16 numbers one time in sixty) the elements are looked through.
__device__ __forceinline__ float largest(const float (&f)[8]) {
    int p = (int)__float_as_uint(f[0]);
    uint32_t n = __float_as_uint(f[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) {
        const uint32_t b = __float_as_uint(f[i]);
        p = p > (int)b ? p : (int)b, n = n > b ? n : b;
    }
    int a = (int)quad<0xB1>((uint32_t)p);  // lanes 1, 0, 3, 2
    uint32_t c = quad<0xB1>(n);
    p = p > a ? p : a, n = n > c ? n : c;
    a = (int)quad<0x4E>((uint32_t)p), c = quad<0x4E>(n);  // lanes 2, 3, 0, 1
    p = p > a ? p : a, n = n > c ? n : c;
    const uint32_t size = n & 0x7FFFFFFFu;  // of the most negative where there is one
    bool neg = (int)n < 0 && (p < 0 || size > (uint32_t)p);
    if (__any((int)n < 0 && size == (uint32_t)p)) {
        uint32_t sign = 2;  // of this lane's first of that size
#pragma unroll
        for (int i = 7; i >= 0; i--) {
            const uint32_t b = __float_as_uint(f[i]);
            sign = (b & 0x7FFFFFFFu) == size ? b >> 31 : sign;
        }
        const uint32_t s0 = quad<0x00>(sign), s1 = quad<0x55>(sign), s2 = quad<0xAA>(sign), s3 = quad<0xFF>(sign);
        const uint32_t first = s0 != 2 ? s0 : s1 != 2 ? s1 : s2 != 2 ? s2 : s3;
        if ((int)n < 0 && size == (uint32_t)p) neg = first == 1;
    }
    return __uint_as_float(neg ? n : (uint32_t)p);
}

constexpr int kKeyNibble[8] = {0, 4, 1, 5, 2, 6, 3, 7};

// T tokens from token t, whose places start at r of a piece; this lane's eights of their rows.
template <int IO, int T>
__device__ __forceinline__ void append_rows(const Kv4Args &p, const void *src, uint8_t *piece, bool value, int64_t from, int r, int b, int q) {
    const int blocks = p.dim >> 5;
    float f[T][8];
#pragma unroll
    for (int i = 0; i < T; i++) get8<IO>(src, from + i * p.stride, p.wide, f[i]);
    uint32_t h[T], code[T][8];
#pragma unroll
    for (int i = 0; i < T; i++) {
        h[i] = kv4_scale(largest(f[i]));
        const float d = f16_to_f32((uint16_t)h[i]);
        const bool none = !(fabsf(d) > 0.0f);  // a scale of 0, or a block that is not finite: code 8 throughout
        const float inv = none ? 0.0f : 1.0f / d;
        if (__any(h[i] == 0x7E00u)) {
#pragma unroll
            for (int j = 0; j < 8; j++) f[i][j] = none ? 0.0f : f[i][j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) code[i][j] = kv4_code(f[i][j], none ? 0.0f : d, inv);
    }
    uint16_t *scale = reinterpret_cast<uint16_t *>(piece + kv4_scale_at(r, b, p.dim));
    if (q == 0) {
        if constexpr (T == 4) *reinterpret_cast<uint2 *>(scale) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        else *scale = (uint16_t)h[0];
    }
    if (!value) {
#pragma unroll
        for (int i = 0; i < T; i++) {
            constexpr int element[8] = {0, 2, 4, 6, 1, 3, 5, 7};  // of each nibble
            uint32_t w = code[i][element[7]];
#pragma unroll
            for (int j = 6; j >= 0; j--) w = (w << 4) + code[i][element[j]];
            w -= kCode * 0x11111111u;
            reinterpret_cast<uint32_t *>(piece)[(q * 16 + r + i) * blocks + b] = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {  // elements 8 q + 2 j and the next
            uint32_t *dst = reinterpret_cast<uint32_t *>(piece) + ((r >> 2) * 16 + 4 * q + j) * blocks + b;
            if constexpr (T == 4) {
                constexpr int token[4] = {0, 2, 1, 3};  // of each byte
                uint32_t w = 0;
#pragma unroll
                for (int i = 3; i >= 0; i--) w = (((w << 4) + code[token[i]][2 * j + 1]) << 4) + code[token[i]][2 * j];
                *dst = w - kCode * 0x11111111u;
            } else {
                reinterpret_cast<uint8_t *>(dst)[((r & 1) << 1) | ((r >> 1) & 1)] = (uint8_t)((code[0][2 * j] & 15) | (code[0][2 * j + 1] << 4));
            }
        }
    }
}

__device__ __forceinline__ float byte_of(uint32_t w, int i) { return (float)((w >> (8 * i)) & 0xFFu); }

template <int IO, int T>
__device__ __forceinline__ void read_rows(const Kv4Args &p, void *dst, const uint8_t *piece, bool value, int64_t to, int r, int b, int q) {
    const int blocks = p.dim >> 5;
    const uint16_t *scale = reinterpret_cast<const uint16_t *>(piece + kv4_scale_at(r, b, p.dim));
    float f[T][8], d[T];
#pragma unroll
    for (int i = 0; i < T; i++) {
        const uint32_t h = scale[i];
        d[i] = ((h >> 10) & 31) == 31 ? __builtin_nanf("") : f16_to_f32((uint16_t)h);
    }
#pragma unroll
    for (int i = 0; i < (value ? 4 : T); i++) {
        // (the even nibbles and the odd ones, a byte each)
        if (!value) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(piece)[(q * 16 + r + i) * blocks + b], lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
#pragma unroll
            for (int j = 0; j < 8; j++) f[i < T ? i : 0][j] = byte_of((kKeyNibble[j] & 1) ? hi : lo, kKeyNibble[j] >> 1);
        } else {
            const uint32_t w = reinterpret_cast<const uint32_t *>(piece)[((r >> 2) * 16 + 4 * q + i) * blocks + b], lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
#pragma unroll
            for (int t = 0; t < T; t++) {
                const int at = T == 4 ? t : r & 3, byte = ((at & 1) << 1) | (at >> 1);
                f[t][2 * i] = byte_of(lo, byte), f[t][2 * i + 1] = byte_of(hi, byte);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < T; i++) {
        const float off = -8.0f * d[i];  // c d - 8 d is (c - 8) d: the scale has 11 bits, the code 4
#pragma unroll
        for (int j = 0; j < 8; j++) f[i][j] = fmaf(f[i][j], d[i], off);
        put8<IO>(dst, to + i * p.stride, p.wide, f[i]);
    }
}

// APPEND: rows k, v into the cache; else out of it.
// (Registers for eight waves a SIMD hold 8192 tokens at once, in 15.3 us against 15.8 with seven waves, in and out by other inputs each time 27.5 against
// 29.2; rows out to fp32 would spill more than that gives, 26.7 us against 18.8, both with the codes in the last cache.)
template <int IO, bool APPEND> __global__ __launch_bounds__(256, APPEND || IO != TRHIP_F32 ? 8 : 5) void kv4_rows_kernel(const Kv4Args p, void *k, void *v) {
    const int blocks = p.dim >> 5, row = 4 * p.heads * blocks;  // eights of a row
    const int x = blockIdx.x * blockDim.x + threadIdx.x;
    const bool value = x >= row;
    const int y = value ? x - row : x, head = y / (4 * blocks), e = y - head * (4 * blocks), b = e >> 2, q = e & 3;
    // (a workgroup a token would leave all work to every fourth, and workgroups are dealt to the XCDs in turn: two of eight would do it)
    for (uint32_t t0 = blockIdx.y * p.run; t0 < p.tokens; t0 = kv4_next(t0, gridDim.y, p.run))
    for (uint32_t t = t0; t < t0 + p.run && t < p.tokens; t++) {
        int64_t slot;
        const int n = kv4_together(p.slots, p.tokens, p.places, t, slot);
        if (n == 0 || x >= 2 * row) continue;
        const Kv4Place at = kv4_place(slot, p.page_log2, p.heads, head, p.dim);
        uint8_t *piece = (value ? p.vc : p.kc) + at.piece;
        const int64_t from = (int64_t)t * p.stride + head * p.dim + 32 * b + 8 * q;
        void *rows = value ? v : k;
        if constexpr (APPEND) {
            if (n == 4) append_rows<IO, 4>(p, rows, piece, value, from, at.r, b, q);
            else append_rows<IO, 1>(p, rows, piece, value, from, at.r, b, q);
        } else {
            if (n == 4) read_rows<IO, 4>(p, rows, piece, value, from, at.r, b, q);
            else read_rows<IO, 1>(p, rows, piece, value, from, at.r, b, q);
        }
    }
}

template <bool APPEND>
int launch(trhip_ctx *ctx, const trhip_kv4 *kv, int64_t tokens, void *k, void *v, int io, int64_t stride, const int *slots) {
    const int64_t size = io == TRHIP_F32 ? 4 : 2;
    const bool wide = reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && stride * size % 16 == 0;
    // (8192 tokens: in 15.8 us, with one token a workgroup 34; few tokens go faster on a workgroup each, 6.0 us against 6.2)
    const uint32_t run = tokens >= 256 ? 4 : 1;
    const Kv4Args p = {static_cast<uint8_t *>(kv->k), static_cast<uint8_t *>(kv->v), __builtin_ctz((unsigned)kv->page), kv->heads, kv->dim,
                       kv->pages * kv->page, stride, (uint32_t)tokens, run, wide, slots};
    const int eights = kv->heads * kv->dim / 4, threads = eights >= 256 ? 256 : (eights + 63) / 64 * 64;
    const int64_t y = (tokens + run - 1) / run;
    const dim3 grid((unsigned)((eights + threads - 1) / threads), (unsigned)(y < kKv4Groups ? y : kKv4Groups));
    if (io == TRHIP_F32) hipLaunchKernelGGL((kv4_rows_kernel<TRHIP_F32, APPEND>), grid, dim3(threads), 0, ctx->stream, p, k, v);
    else if (io == TRHIP_F16) hipLaunchKernelGGL((kv4_rows_kernel<TRHIP_F16, APPEND>), grid, dim3(threads), 0, ctx->stream, p, k, v);
    else hipLaunchKernelGGL((kv4_rows_kernel<TRHIP_BF16, APPEND>), grid, dim3(threads), 0, ctx->stream, p, k, v);
    return launch_check(ctx, APPEND ? "kv4_append" : "kv4_read");
}

}  // namespace

int launch_kv4_append(trhip_ctx *ctx, const trhip_kv4 *kv, int64_t tokens, const void *k, const void *v, int io, int64_t stride,
                      const int *slots) {
    return launch<true>(ctx, kv, tokens, const_cast<void *>(k), const_cast<void *>(v), io, stride, slots);
}
int launch_kv4_read(trhip_ctx *ctx, const trhip_kv4 *kv, int64_t tokens, void *k, void *v, int io, int64_t stride, const int *slots) {
    return launch<false>(ctx, kv, tokens, k, v, io, stride, slots);
}

}  // namespace trhip
