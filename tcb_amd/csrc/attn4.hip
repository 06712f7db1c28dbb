// attn4.hip -- attention over the 4-bit paged cache.
#include "attn_common.hpp"
#include "kv4.hpp"

namespace trhip {
namespace {

struct Attn4Args {
    const uint16_t *q;
    uint16_t *out;
    const uint8_t *k, *v;
    int64_t q_stride, out_stride, max_pages, pages;
    const int *q_start, *kv_len, *table;
    int tokens, nreq, heads, kv_heads, dim, page_log2, window, sinks, io;
    float scale;
};

__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// One wave a token and head, a key at a time, up to four elements a lane.
__global__ __launch_bounds__(64) void attn4_simple(const Attn4Args p) {
    const int t = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, kvh = head / (p.heads / p.kv_heads);
    int req = -1, start = 0, end = 0;
    for (int i = 0; i < p.nreq; i++) {
        int a = p.q_start[i], b = p.q_start[i + 1];
        a = a < 0 ? 0 : a > p.tokens ? p.tokens : a;
        b = b < a ? a : b > p.tokens ? p.tokens : b;
        if (t >= a && t < b) req = i, start = a, end = b;
    }
    if (req < 0) return;
    const int64_t cap = p.max_pages << p.page_log2;
    int kv = p.kv_len[req];
    kv = kv < 0 ? 0 : (int64_t)kv > cap ? (int)cap : kv;
    const int pos = kv - (end - start) + (t - start);
    constexpr int nib[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    float q[4] = {}, o[4] = {}, m = -__builtin_inff(), l = 0.0f;
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < p.dim) q[u] = h16_to_f32(p.q[(int64_t)t * p.q_stride + head * p.dim + lane + 64 * u], p.io);
    for (int j = 0; j <= pos; j++) {
        if (p.window > 0 && j <= pos - p.window && j >= p.sinks) {
            j = pos - p.window;
            continue;
        }
        const int page = p.table[(int64_t)req * p.max_pages + (j >> p.page_log2)];
        float s = 0.0f, v[4] = {};
        if ((uint32_t)page < (uint32_t)p.pages) {
            const Kv4Place at = kv4_place(((int64_t)page << p.page_log2) + (j & ((1 << p.page_log2) - 1)), p.page_log2, p.kv_heads, kvh, p.dim);
            for (int u = 0; u < 4; u++) {
                const int e = lane + 64 * u;
                if (e >= p.dim) continue;
                const uint32_t kd = *reinterpret_cast<const uint16_t *>(p.k + at.piece + kv4_scale_at(at.r, e / 32, p.dim));
                const uint32_t vd = *reinterpret_cast<const uint16_t *>(p.v + at.piece + kv4_scale_at(at.r, e / 32, p.dim));
                const int kc = *reinterpret_cast<const uint32_t *>(p.k + at.piece + kv4_key_at(at.r, e & ~7, p.dim)) >> (4 * nib[e & 7]) & 15;
                const int vc = p.v[at.piece + kv4_value_at(at.r, e, p.dim)] >> (4 * (e & 1)) & 15;
                const float nan = __builtin_nanf("");
                s = fmaf(q[u], (kd >> 10 & 31) == 31 ? nan : kv4_value(kc, kd), s);
                v[u] = (vd >> 10 & 31) == 31 ? nan : kv4_value(vc, vd);
            }
        }
        s = wave_sum(s) * p.scale;
        const float n = fmaxf(m, s), a = m == n ? 1.0f : __builtin_amdgcn_exp2f((m - n) * 1.44269504f), e = __builtin_amdgcn_exp2f((s - n) * 1.44269504f);
        m = n;
        l = l * a + e;
        for (int u = 0; u < 4; u++) o[u] = o[u] * a + e * v[u];
    }
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < p.dim)
            p.out[(int64_t)t * p.out_stride + head * p.dim + lane + 64 * u] = (uint16_t)f32_to_h16(pos >= 0 ? o[u] / l : 0.0f, p.io);
}

}  // namespace

int launch_kv4_attn(trhip_ctx *ctx, const trhip_kv4 *kv, const AttnCall &c, int io) {
    const Attn4Args p = {static_cast<const uint16_t *>(c.q), static_cast<uint16_t *>(c.out), static_cast<const uint8_t *>(kv->k),
                         static_cast<const uint8_t *>(kv->v), c.q_stride, c.out_stride, c.max_pages, kv->pages, c.q_start, c.kv_len, c.table,
                         (int)c.tokens, (int)c.nreq, c.heads, kv->heads, kv->dim, __builtin_ctz((unsigned)kv->page), (int)c.window, (int)c.sinks, io, c.scale};
    hipLaunchKernelGGL(attn4_simple, dim3((unsigned)c.tokens, (unsigned)c.heads), dim3(64), 0, ctx->stream, p);
    return launch_check(ctx, "kv4_attn");
}

}  // namespace trhip
