// kv4.hip -- the 4-bit cache: rows in, quantized, and out again.
#include "kv4.hpp"

namespace trhip {
namespace {

struct Kv4Args {
    uint8_t *kc, *vc;
    int page_log2, heads, dim, io;
    int64_t places, tokens, stride;
    const int *slots;
};

__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4Args p, const void *k, const void *v) {
    const int blocks = p.dim / 32, per = 2 * p.heads * blocks;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < p.tokens * per; at += (int64_t)gridDim.x * 256) {
        const int64_t t = at / per, slot = p.slots[t];
        if ((uint64_t)slot >= (uint64_t)p.places) continue;
        const int x = (int)(at - t * per), value = x >= p.heads * blocks, y = value ? x - p.heads * blocks : x, head = y / blocks, b = y - head * blocks;
        const void *src = value ? v : k;
        float f[32], m = 0.0f;
        bool odd = false;
        for (int i = 0; i < 32; i++) {
            const int64_t e = t * p.stride + head * p.dim + 32 * b + i;
            f[i] = p.io == TRHIP_F32 ? static_cast<const float *>(src)[e] : h16_to_f32(static_cast<const uint16_t *>(src)[e], p.io);
            if (fabsf(f[i]) > fabsf(m)) m = f[i];
            odd = odd || !(fabsf(f[i]) < __builtin_inff());
        }
        if (odd) m = __builtin_nanf("");
        const uint32_t h = kv4_scale(m);
        const float d = f16_to_f32((uint16_t)h), inv = 1.0f / d;
        const Kv4Place at0 = kv4_place(slot, p.page_log2, p.heads, head, p.dim);
        uint8_t *piece = (value ? p.vc : p.kc) + at0.piece;
        *reinterpret_cast<uint16_t *>(piece + kv4_scale_at(at0.r, b, p.dim)) = (uint16_t)h;
        if (value) {
            for (int i = 0; i < 32; i += 2)
                piece[kv4_value_at(at0.r, 32 * b + i, p.dim)] = (uint8_t)(kv4_code(f[i], d, inv) | (kv4_code(f[i + 1], d, inv) << 4));
        } else {
            constexpr int nib[8] = {0, 4, 1, 5, 2, 6, 3, 7};
            for (int q = 0; q < 4; q++) {
                uint32_t w = 0;
                for (int i = 0; i < 8; i++) w |= (uint32_t)kv4_code(f[8 * q + i], d, inv) << (4 * nib[i]);
                *reinterpret_cast<uint32_t *>(piece + kv4_key_at(at0.r, 32 * b + 8 * q, p.dim)) = w;
            }
        }
    }
}

__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4Args p, void *k, void *v) {
    const int row = p.heads * p.dim, per = 2 * row;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < p.tokens * per; at += (int64_t)gridDim.x * 256) {
        const int64_t t = at / per, slot = p.slots[t];
        if ((uint64_t)slot >= (uint64_t)p.places) continue;
        const int x = (int)(at - t * per), value = x >= row, y = value ? x - row : x, head = y / p.dim, e = y - head * p.dim;
        const Kv4Place at0 = kv4_place(slot, p.page_log2, p.heads, head, p.dim);
        const uint8_t *piece = (value ? p.vc : p.kc) + at0.piece;
        const uint32_t h = *reinterpret_cast<const uint16_t *>(piece + kv4_scale_at(at0.r, e / 32, p.dim));
        int code;
        if (value) {
            code = (piece[kv4_value_at(at0.r, e, p.dim)] >> (4 * (e & 1))) & 15;
        } else {
            constexpr int nib[8] = {0, 4, 1, 5, 2, 6, 3, 7};
            code = (*reinterpret_cast<const uint32_t *>(piece + kv4_key_at(at0.r, e & ~7, p.dim)) >> (4 * nib[e & 7])) & 15;
        }
        const float f = ((h >> 10) & 31) == 31 ? __builtin_nanf("") : kv4_value(code, h);
        const int64_t to = t * p.stride + y;
        void *dst = value ? v : k;
        if (p.io == TRHIP_F32) static_cast<float *>(dst)[to] = f;
        else static_cast<uint16_t *>(dst)[to] = (uint16_t)f32_to_h16(f, p.io);
    }
}

Kv4Args args(const trhip_kv4 *kv, int64_t tokens, int io, int64_t stride, const int *slots) {
    return {static_cast<uint8_t *>(kv->k), static_cast<uint8_t *>(kv->v), __builtin_ctz((unsigned)kv->page), kv->heads, kv->dim, io,
            kv->pages * kv->page, tokens, stride, slots};
}
unsigned grid(int64_t threads) {
    const int64_t n = (threads + 255) / 256;
    return (unsigned)(n < 65536 ? n : 65536);
}

}  // namespace

int launch_kv4_append(trhip_ctx *ctx, const trhip_kv4 *kv, int64_t tokens, const void *k, const void *v, int io, int64_t stride,
                      const int *slots) {
    hipLaunchKernelGGL(kv4_append_kernel, dim3(grid(tokens * kv->heads * kv->dim / 16)), dim3(256), 0, ctx->stream,
                       args(kv, tokens, io, stride, slots), k, v);
    return launch_check(ctx, "kv4_append");
}
int launch_kv4_read(trhip_ctx *ctx, const trhip_kv4 *kv, int64_t tokens, void *k, void *v, int io, int64_t stride, const int *slots) {
    hipLaunchKernelGGL(kv4_read_kernel, dim3(grid(tokens * kv->heads * kv->dim * 2)), dim3(256), 0, ctx->stream,
                       args(kv, tokens, io, stride, slots), k, v);
    return launch_check(ctx, "kv4_read");
}

}  // namespace trhip
