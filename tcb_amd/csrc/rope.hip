// rope.hip -- rotary positions with up to four axes: pair i of a head's elements is turned by pos[axis(i)][t] * frequency(i).
//
// A workgroup takes one or four tokens and some of their heads: first the sines and cosines of the tokens' pairs, once for all heads, into
// LDS, then the heads, 16 bytes a load. Every element moves once in and once out, which is what bounds it: 8192 tokens of 40 heads of 128 in bf16
// take 35 us from memory (4.8 TB/s; three axes and factors 38), in place 36.5, in fp32 63 (5.3 TB/s); 16 tokens 4.8, a launch. (Angles by every head
// anew, 64-bit arithmetic each: 72 us.)
#include "rope.hpp"
#include "trhip_internal.hpp"

#include <cmath>

namespace trhip {
namespace {

constexpr int kMostPairs = 256, kThreads = kRopeThreads;

struct RopeArgs {
    const void *x;
    void *out;
    int64_t x_stride, out_stride, pos_stride;
    int tokens, heads, dim, pairs, each;  // each: heads of a workgroup
    int axes, n[4];                       // pairs of each axis
    int dealt, ladders, neighbours, copy; // copy: out is not x, what is not turned has to be copied
    double log_hi, log_lo;                // log2 of the base, in two parts
    const int *pos;
    const float *factors;
};

// Sine and cosine of `turns` whole turns. The turns are reduced to a quarter in 64 bits, the rest y (|y| <= 1/8 turn) goes through the
// series of x = 2 pi y, |x| <= pi / 4: what they leave out is below 2^-29, so fp32's own roundings are what is off.
__device__ __forceinline__ float2 cos_sin(double turns) {
    const double q = 4.0 * (turns - rint(turns)), k = rint(q);
    const float x = (float)(q - k) * 1.57079632679f, z = x * x;
    const float s = rope_sin(x, z), c = rope_cos(z);
    const int n = (int)k & 3;
    const float a = n & 1 ? s : c, b = n & 1 ? c : s;
    return make_float2(n == 1 || n == 2 ? -a : a, n >= 2 ? -b : b);
}

// The axis of pair i and its place among the axis's pairs.
__device__ __forceinline__ int2 axis_of(const RopeArgs &p, int i) {
    if (!p.dealt) {
        int a = 0;
        while (a < p.axes - 1 && i >= p.n[a]) i -= p.n[a], a++;
        return make_int2(a, i);
    }
    int done = 0;  // rounds so far: in each, one pair to every axis that has more
    for (;;) {
        int m = 0, least = 0x7FFFFFFF;
        for (int a = 0; a < p.axes; a++)
            if (p.n[a] > done) m++, least = p.n[a] < least ? p.n[a] : least;
        if (i < m * (least - done)) {
            int want = i % m;
            for (int a = 0; a < p.axes; a++)
                if (p.n[a] > done && want-- == 0) return make_int2(a, done + i / m);
        }
        i -= m * (least - done);
        done = least;
    }
}

// Turns that a position of 1 makes of pair i: base^-s / 2 pi, s the pair's place over the number of pairs. s and the logarithm are taken in
// two parts each, or the exponent's rounding would be that many times as much of far angles.
__device__ __forceinline__ double turns_of(const RopeArgs &p, int i, int2 at) {
    const double a = p.ladders ? at.y : i, b = p.ladders ? p.n[at.x] : p.pairs;
    const double s = a / b, s_lo = fma(-s, b, a) / b, e = s * p.log_hi;
    const double rest = fma(s, p.log_hi, -e) + fma(s, p.log_lo, s_lo * p.log_hi);
    const double f = exp2(-e) * 0.15915494309189533577;
    return fma(f, -0.69314718055994530942 * rest, f) * (p.factors ? (double)p.factors[i] : 1.0);
}

template <int IO> struct Elem {
    static constexpr int SIZE = IO == TRHIP_F32 ? 4 : 2;
};
// N elements (16 bytes, or one)
template <int IO, int N> __device__ __forceinline__ void get(const void *p, int64_t i, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = IO == TRHIP_F32 ? static_cast<const float *>(p)[i] : h16_to_f32(static_cast<const uint16_t *>(p)[i], IO);
    } else if constexpr (IO == TRHIP_F32) {
        *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    } else {
        const uint4 y = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; j++) f[2 * j] = h16_to_f32(w[j] & 0xFFFFu, IO), f[2 * j + 1] = h16_to_f32(w[j] >> 16, IO);
    }
}
template <int IO, int N> __device__ __forceinline__ void put(void *p, int64_t i, const float (&f)[N]) {
    if constexpr (N == 1) {
        if (IO == TRHIP_F32) static_cast<float *>(p)[i] = f[0];
        else static_cast<uint16_t *>(p)[i] = (uint16_t)f32_to_h16(f[0], IO);
    } else if constexpr (IO == TRHIP_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = f32_to_h16(f[2 * j], IO) | (f32_to_h16(f[2 * j + 1], IO) << 16);
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int IO, bool WIDE, int TOKENS> __global__ __launch_bounds__(kThreads) void rope_kernel(const RopeArgs p) {
    constexpr int N = WIDE ? 16 / Elem<IO>::SIZE : 1;  // pairs, or copied elements, of an item
    __shared__ float2 s_turn[TOKENS][kMostPairs];
    const int tid = threadIdx.x, t0 = blockIdx.x * TOKENS, h0 = blockIdx.y * p.each;
    const int tokens = p.tokens - t0 < TOKENS ? p.tokens - t0 : TOKENS, heads = p.heads - h0 < p.each ? p.heads - h0 : p.each;
    for (int i = tid; i < p.pairs; i += kThreads) {
        const int2 at = axis_of(p, i);
        const double f = turns_of(p, i, at);
#pragma unroll
        for (int t = 0; t < TOKENS; t++)
            if (t < tokens) s_turn[t][i] = cos_sin((double)p.pos[at.x * p.pos_stride + t0 + t] * f);
    }
    __syncthreads();
    const int turn = p.pairs / N, rest = p.copy ? (p.dim - 2 * p.pairs) / N : 0, per = turn + rest;
#pragma unroll 2
    for (int i = tid; i < tokens * heads * per; i += kThreads) {
        const int row = i / per, c = i - row * per, t = row / heads, h = h0 + row - t * heads;
        const int64_t from = (int64_t)(t0 + t) * p.x_stride + (int64_t)h * p.dim, to = (int64_t)(t0 + t) * p.out_stride + (int64_t)h * p.dim;
        if (c >= turn) {
            const int e = 2 * p.pairs + (c - turn) * N;
            if constexpr (WIDE) {
                *reinterpret_cast<uint4 *>(static_cast<char *>(p.out) + (to + e) * Elem<IO>::SIZE) =
                    *reinterpret_cast<const uint4 *>(static_cast<const char *>(p.x) + (from + e) * Elem<IO>::SIZE);
            } else if constexpr (IO == TRHIP_F32) {
                static_cast<uint32_t *>(p.out)[to + e] = static_cast<const uint32_t *>(p.x)[from + e];
            } else {
                static_cast<uint16_t *>(p.out)[to + e] = static_cast<const uint16_t *>(p.x)[from + e];
            }
            continue;
        }
        const int i0 = c * N, ea = p.neighbours ? 2 * i0 : i0, eb = p.neighbours ? 2 * i0 + N : i0 + p.pairs;
        float a[N], b[N], u[N], v[N];
        get<IO, N>(p.x, from + ea, a);
        get<IO, N>(p.x, from + eb, b);
        if (p.neighbours && N > 1) {  // pairs lie side by side: the first half of them in a, the second in b
#pragma unroll
            for (int j = 0; j < N / 2; j++) {
                const float2 w = s_turn[t][i0 + j], z = s_turn[t][i0 + N / 2 + j];
                u[2 * j] = fmaf(a[2 * j], w.x, -(a[2 * j + 1] * w.y));
                u[2 * j + 1] = fmaf(a[2 * j], w.y, a[2 * j + 1] * w.x);
                v[2 * j] = fmaf(b[2 * j], z.x, -(b[2 * j + 1] * z.y));
                v[2 * j + 1] = fmaf(b[2 * j], z.y, b[2 * j + 1] * z.x);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float2 w = s_turn[t][i0 + j];
                u[j] = fmaf(a[j], w.x, -(b[j] * w.y));
                v[j] = fmaf(a[j], w.y, b[j] * w.x);
            }
        }
        put<IO, N>(p.out, to + ea, u);
        put<IO, N>(p.out, to + eb, v);
    }
}

template <int IO, bool WIDE> void launch(trhip_ctx *ctx, const RopeArgs &p, bool four, unsigned groups, unsigned splits) {
    if (four) hipLaunchKernelGGL((rope_kernel<IO, WIDE, 4>), dim3(groups, splits), dim3(kThreads), 0, ctx->stream, p);
    else hipLaunchKernelGGL((rope_kernel<IO, WIDE, 1>), dim3(groups, splits), dim3(kThreads), 0, ctx->stream, p);
}

}  // namespace

int launch_rope(trhip_ctx *ctx, const trhip_rope_spec &spec, const void *x, int64_t x_stride, void *out, int64_t out_stride, int io,
                int64_t tokens, int heads, int dim, const int *pos, int64_t pos_stride) {
    RopeArgs p = {};
    p.x = x, p.out = out, p.x_stride = x_stride, p.out_stride = out_stride, p.pos_stride = pos_stride;
    p.heads = heads, p.dim = dim, p.axes = spec.axes;
    for (int a = 0; a < spec.axes; a++) p.pairs += p.n[a] = spec.pairs[a];
    p.dealt = spec.flags & TRHIP_ROPE_DEALT, p.ladders = spec.flags & TRHIP_ROPE_LADDERS, p.neighbours = spec.flags & TRHIP_ROPE_NEIGHBOURS;
    p.copy = x != out;
    const long double log = std::log2((long double)spec.base);
    p.log_hi = (double)log;
    p.log_lo = (double)(log - (long double)p.log_hi);
    p.pos = pos, p.factors = spec.factors;
    const int size = io == TRHIP_F32 ? 4 : 2, n = 16 / size;
    const auto whole = [&](int64_t bytes) { return bytes % 16 == 0; };
    const bool wide = whole(reinterpret_cast<uintptr_t>(x)) && whole(reinterpret_cast<uintptr_t>(out)) && (tokens == 1 || (whole(x_stride * size) && whole(out_stride * size))) &&
                      whole((int64_t)dim * size) && whole((int64_t)p.pairs * size);
    // Four tokens a workgroup where there are many whose items do not fill one (8192 tokens of 10 heads of 128, the same rows each time, which
    // the last cache holds: 10.5 us against 14.5 with one; of 40 heads, which do, 29.1 against 27.7); of few tokens the heads are dealt out, an
    // item a thread (a token of 128 heads, fp32: 4.4 against 5.0).
    const int64_t cus = ctx->sm_count > 0 ? ctx->sm_count : 256;
    const int per = wide ? p.pairs / n + (p.copy ? (dim - 2 * p.pairs) / n : 0) : p.pairs + (p.copy ? dim - 2 * p.pairs : 0);
    const bool four = tokens >= 16 * cus && heads * per <= kThreads;
    int64_t splits = 1;
    if (tokens < 4 * cus) {
        const int64_t items = ((int64_t)heads * per + kThreads - 1) / kThreads, room = (4 * cus + tokens - 1) / tokens;
        splits = items < room ? items : room;
        splits = splits > heads ? heads : splits;
    }
    p.each = (int)((heads + splits - 1) / splits);
    const unsigned s = (unsigned)((heads + p.each - 1) / p.each);
    for (int64_t t = 0; t < tokens; t += kRopeTokens) {
        const RopeLaunch l = rope_launch(tokens - t, four ? 4 : 1);
        p.tokens = l.tokens;
        if (io == TRHIP_F32) wide ? launch<TRHIP_F32, true>(ctx, p, four, l.groups, s) : launch<TRHIP_F32, false>(ctx, p, four, l.groups, s);
        else if (io == TRHIP_F16) wide ? launch<TRHIP_F16, true>(ctx, p, four, l.groups, s) : launch<TRHIP_F16, false>(ctx, p, four, l.groups, s);
        else wide ? launch<TRHIP_BF16, true>(ctx, p, four, l.groups, s) : launch<TRHIP_BF16, false>(ctx, p, four, l.groups, s);
        const int st = launch_check(ctx, "rope");
        if (st != TRHIP_OK) return st;
        p.x = static_cast<const char *>(p.x) + kRopeTokens * x_stride * size;
        p.out = static_cast<char *>(p.out) + kRopeTokens * out_stride * size;
        p.pos += kRopeTokens;
    }
    return TRHIP_OK;
}

}  // namespace trhip
