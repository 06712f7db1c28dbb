// rope.hip -- rotary positions with up to four axes: pair i of a head's elements is turned by pos[axis(i)][t] * frequency(i).
#include "trhip_internal.hpp"

#include <cmath>

namespace trhip {
namespace {

constexpr int kMostPairs = 256;

// Per pair: the axis, and the turns (of 2 pi) a position of 1 makes.
struct RopePairs {
    double turns[kMostPairs];
    uint8_t axis[kMostPairs];
};

struct RopeArgs {
    const void *x;
    void *out;
    int64_t x_stride, out_stride, tokens, pos_stride;
    int heads, dim, pairs, io, neighbours;
    const int *pos;
    const float *factors;
};

__device__ __forceinline__ float load_io(const void *p, int64_t i, int io) {
    if (io == TRHIP_F32) return static_cast<const float *>(p)[i];
    return h16_to_f32(static_cast<const uint16_t *>(p)[i], io);
}
__device__ __forceinline__ void store_io(void *p, int64_t i, int io, float v) {
    if (io == TRHIP_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)f32_to_h16(v, io);
}

// Sine and cosine of `turns` whole turns. The turns are reduced to a quarter in 64 bits, the rest y (|y| <= 1/8 turn) goes through the
// Taylor series of x = 2 pi y, |x| <= pi / 4: what they leave out is below 2^-28, so fp32's own roundings are what is off.
__device__ __forceinline__ float2 cos_sin(double turns) {
    const double q = 4.0 * (turns - rint(turns)), k = rint(q);
    const float x = (float)(q - k) * 1.57079632679f, z = x * x;
    const float s = fmaf(z * x, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f), x);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.48015873e-5f, -1.38888889e-3f), 4.16666667e-2f), -0.5f), 1.0f);
    const int n = (int)k & 3;
    const float a = n & 1 ? s : c, b = n & 1 ? c : s;
    return make_float2(n == 1 || n == 2 ? -a : a, n >= 2 ? -b : b);
}

__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs p, const RopePairs by) {
    const int rest = p.dim - 2 * p.pairs, per = p.pairs + rest;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < p.tokens * per; at += (int64_t)gridDim.x * 256) {
        const int64_t t = at / per;
        const int i = (int)(at - t * per);
        if (i >= p.pairs) {
            for (int h = 0; h < p.heads; h++) {
                const int64_t e = (int64_t)h * p.dim + p.pairs + i;
                if (p.io == TRHIP_F32) static_cast<uint32_t *>(p.out)[t * p.out_stride + e] = static_cast<const uint32_t *>(p.x)[t * p.x_stride + e];
                else static_cast<uint16_t *>(p.out)[t * p.out_stride + e] = static_cast<const uint16_t *>(p.x)[t * p.x_stride + e];
            }
            continue;
        }
        double turns = (double)p.pos[by.axis[i] * p.pos_stride + t] * by.turns[i];
        if (p.factors) turns *= (double)p.factors[i];
        const float2 w = cos_sin(turns);
        const int a = p.neighbours ? 2 * i : i, b = p.neighbours ? 2 * i + 1 : i + p.pairs;
        for (int h = 0; h < p.heads; h++) {
            const int64_t e = (int64_t)h * p.dim;
            const float x = load_io(p.x, t * p.x_stride + e + a, p.io), y = load_io(p.x, t * p.x_stride + e + b, p.io);
            store_io(p.out, t * p.out_stride + e + a, p.io, fmaf(x, w.x, -(y * w.y)));
            store_io(p.out, t * p.out_stride + e + b, p.io, fmaf(x, w.y, y * w.x));
        }
    }
}

}  // namespace

int launch_rope(trhip_ctx *ctx, const trhip_rope_spec &spec, const void *x, int64_t x_stride, void *out, int64_t out_stride, int io,
                int64_t tokens, int heads, int dim, const int *pos, int64_t pos_stride) {
    RopePairs by = {};
    int left[4], total = 0;
    for (int a = 0; a < spec.axes; a++) total += left[a] = spec.pairs[a];
    for (int i = 0, a = 0; i < total; i++) {
        while (left[a] == 0) a = a + 1 == spec.axes ? 0 : a + 1;
        const double s = spec.flags & TRHIP_ROPE_LADDERS ? (double)(spec.pairs[a] - left[a]) / spec.pairs[a] : (double)i / total;
        by.axis[i] = (uint8_t)a;
        by.turns[i] = std::pow(spec.base, -s) * 0.15915494309189533577;
        left[a]--;
        if (spec.flags & TRHIP_ROPE_DEALT) a = a + 1 == spec.axes ? 0 : a + 1;
    }
    const RopeArgs p = {x, out, x_stride, out_stride, tokens, pos_stride, heads, dim, total, io, spec.flags & TRHIP_ROPE_NEIGHBOURS, pos, spec.factors};
    int64_t blocks = (tokens * (dim - total) + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    hipLaunchKernelGGL(rope_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, p, by);
    return launch_check(ctx, "rope");
}

}  // namespace trhip
