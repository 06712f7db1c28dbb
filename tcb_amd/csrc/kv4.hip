// kv4.hip -- the 4-bit cache: rows in, quantized, and out again.
//
// A workgroup takes a token, or the four tokens of four places in a row (a quarter of a piece), whose value codes share dwords: written
// together they are dwords, by themselves bytes. A lane has eight elements of each token's row, four lanes a block. Every element moves
// once, so bytes bound it; of few tokens it is a launch.
#include "kv4.hpp"

namespace trhip {
namespace {

struct Kv4Args {
    uint8_t *kc, *vc;
    int page_log2, heads, dim;
    int64_t places, stride;
    int tokens, wide, run;  // wide: rows are aligned to 16 bytes; run: tokens of a workgroup
    const int *slots;
};

// The token's slot and how many tokens the workgroup of token t takes: 4 where t is the first of four in a row from a multiple of four,
// 0 where an earlier workgroup takes it.
__device__ __forceinline__ int together(const Kv4Args &p, int t, int64_t &slot) {
    slot = p.slots[t];
    if ((uint64_t)slot >= (uint64_t)p.places) return 0;
    const int at = (int)(slot & 3), first = t - at;
    if (first < 0 || first + 3 >= p.tokens) return 1;
    bool row = true;
#pragma unroll
    for (int i = 0; i < 4; i++) row = row && (int64_t)p.slots[first + i] == slot - at + i;
    return !row ? 1 : at == 0 ? 4 : 0;
}

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
            for (int j = 0; j < 4; j++) f[2 * j] = h16_to_f32(w[j] & 0xFFFFu, IO), f[2 * j + 1] = h16_to_f32(w[j] >> 16, IO);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = h16_to_f32(s[i], IO);
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
        for (int j = 0; j < 4; j++) w[j] = f32_to_h16(f[2 * j], IO) | (f32_to_h16(f[2 * j + 1], IO) << 16);
        if (wide) {
            *reinterpret_cast<uint4 *>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) d[2 * j] = (uint16_t)w[j], d[2 * j + 1] = (uint16_t)(w[j] >> 16);
        }
    }
}

// The block's element of largest magnitude, the first of equal ones, from each of its four lanes' eight. (As whole numbers magnitudes
// are in the same order, infinities and NaN above all others.)
__device__ __forceinline__ float largest(const float (&f)[8]) {
    uint32_t m = __float_as_uint(f[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) {
        const uint32_t b = __float_as_uint(f[i]);
        m = (b & 0x7FFFFFFFu) > (m & 0x7FFFFFFFu) ? b : m;
    }
    const int lane = threadIdx.x & 3;
    const uint32_t a = quad<0xB1>(m);  // lanes 1, 0, 3, 2
    m = (a & 0x7FFFFFFFu) > (m & 0x7FFFFFFFu) || ((a & 0x7FFFFFFFu) == (m & 0x7FFFFFFFu) && (lane & 1)) ? a : m;
    const uint32_t b = quad<0x4E>(m);  // lanes 2, 3, 0, 1
    m = (b & 0x7FFFFFFFu) > (m & 0x7FFFFFFFu) || ((b & 0x7FFFFFFFu) == (m & 0x7FFFFFFFu) && (lane & 2)) ? b : m;
    return __uint_as_float(m);
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
        const float d = f16_to_f32((uint16_t)h[i]), inv = 1.0f / d;
#pragma unroll
        for (int j = 0; j < 8; j++) code[i][j] = (uint32_t)kv4_code(f[i][j], d, inv);
    }
    uint16_t *scale = reinterpret_cast<uint16_t *>(piece + kv4_scale_at(r, b, p.dim));
    if (q == 0) {
        if constexpr (T == 4) *reinterpret_cast<uint2 *>(scale) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        else *scale = (uint16_t)h[0];
    }
    if (!value) {
#pragma unroll
        for (int i = 0; i < T; i++) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) w |= code[i][j] << (4 * kKeyNibble[j]);
            reinterpret_cast<uint32_t *>(piece)[(q * 16 + r + i) * blocks + b] = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {  // elements 8 q + 2 j and the next
            uint32_t *dst = reinterpret_cast<uint32_t *>(piece) + ((r >> 2) * 16 + 4 * q + j) * blocks + b;
            if constexpr (T == 4) {
                constexpr int byte[4] = {0, 2, 1, 3};
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) w |= (code[i][2 * j] | (code[i][2 * j + 1] << 4)) << (8 * byte[i]);
                *dst = w;
            } else {
                reinterpret_cast<uint8_t *>(dst)[((r & 1) << 1) | ((r >> 1) & 1)] = (uint8_t)(code[0][2 * j] | (code[0][2 * j + 1] << 4));
            }
        }
    }
}

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
        if (!value) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(piece)[(q * 16 + r + i) * blocks + b];
#pragma unroll
            for (int j = 0; j < 8; j++) f[i < T ? i : 0][j] = (float)((int)((w >> (4 * kKeyNibble[j])) & 15) - 8);
        } else {
            const uint32_t w = reinterpret_cast<const uint32_t *>(piece)[((r >> 2) * 16 + 4 * q + i) * blocks + b];
#pragma unroll
            for (int t = 0; t < T; t++) {
                const int at = T == 4 ? t : r & 3, sh = 8 * (((at & 1) << 1) | (at >> 1));
                f[t][2 * i] = (float)((int)((w >> sh) & 15) - 8);
                f[t][2 * i + 1] = (float)((int)((w >> (sh + 4)) & 15) - 8);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < T; i++) {
#pragma unroll
        for (int j = 0; j < 8; j++) f[i][j] *= d[i];
        put8<IO>(dst, to + i * p.stride, p.wide, f[i]);
    }
}

// APPEND: rows k, v into the cache; else out of it.
template <int IO, bool APPEND> __global__ __launch_bounds__(256) void kv4_rows_kernel(const Kv4Args p, void *k, void *v) {
    const int blocks = p.dim >> 5, row = 4 * p.heads * blocks;  // eights of a row
    const int x = blockIdx.x * blockDim.x + threadIdx.x;
    const bool value = x >= row;
    const int y = value ? x - row : x, head = y / (4 * blocks), e = y - head * (4 * blocks), b = e >> 2, q = e & 3;
    // (a workgroup a token would leave all work to every fourth, and workgroups are dealt to the XCDs in turn: two of eight would do it)
    for (int t0 = blockIdx.y * p.run; t0 < p.tokens; t0 += gridDim.y * p.run)
    for (int t = t0; t < t0 + p.run && t < p.tokens; t++) {
        int64_t slot;
        const int n = together(p, t, slot);
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
    const int run = tokens >= 256 ? 4 : 1;
    const Kv4Args p = {static_cast<uint8_t *>(kv->k), static_cast<uint8_t *>(kv->v), __builtin_ctz((unsigned)kv->page), kv->heads, kv->dim,
                       kv->pages * kv->page, stride, (int)tokens, wide, run, slots};
    const int eights = kv->heads * kv->dim / 4, threads = eights >= 256 ? 256 : (eights + 63) / 64 * 64;
    const int64_t y = (tokens + run - 1) / run;
    const dim3 grid((unsigned)((eights + threads - 1) / threads), (unsigned)(y < 65535 ? y : 65535));
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
