// attn4_image.hip -- the 4-bit cache's keys of long requests, opened once into the workspace in 16 bits, for the kernel of many rows.
//
// A long prompt reads every key of its request once for each 128 of its rows, and its time is that of the products; opening the codes
// anew each time would take as long. Every value that an append wrote is exact in f16 and bf16, so the products see what the cache
// stands for. It moves 4.6 times the codes' bytes (4.5 bits an element in, 16 out), 8192 keys of 8 heads of 128 in 12 us; loading a piece's
// blocks one after the other took 17.
#include "attn4_image.hpp"
#include "attn_common.hpp"
#include "kv4.hpp"

namespace trhip {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Workgroup (x, head, rank): pieces x, x + gridDim.x, ... of the keys of the rank-th long request, a wave a piece.
template <int NG, bool BF> __global__ __launch_bounds__(256) void attn4_image(const Image4 p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), head = blockIdx.y, rank = blockIdx.z;
    // the request
    int req = -1, nq = 0, kv = 0;
    const int64_t cap = p.max_pages << p.page_log2;
    for (int base = 0, seen = 0; base < p.nreq; base += 64) {
        const int i = base + lane;
        int a = 0, b = 0, n = 0;
        if (i < p.nreq) {
            a = p.q_start[i], b = p.q_start[i + 1], n = p.kv_len[i];
            a = a < 0 ? 0 : a > p.tokens ? p.tokens : a;
            b = b < a ? a : b > p.tokens ? p.tokens : b;
            n = n < 0 ? 0 : (int64_t)n > cap ? (int)cap : n;
        }
        const bool is = (b - a) * p.group > p.row_lo;
        const uint64_t m = __ballot(is);
        const int before = seen + __popcll(m & (((uint64_t)1 << lane) - 1));
        const uint64_t hit = __ballot(is && before == rank);
        seen += __popcll(m);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            req = base + src;
            nq = __builtin_amdgcn_readlane(b - a, src);
            kv = __builtin_amdgcn_readlane(n, src);
            break;
        }
    }
    if (req < 0) return;
    const int *table = p.table + (int64_t)req * p.max_pages;
    int *out_table = p.out_table + (int64_t)req * p.max_pages;
    constexpr int DIM = 32 * NG;
    const int r = lane & 15, q = lane >> 4, pieces = (int)(((int64_t)kv + 15) >> 4), per = 1 << (p.page_log2 - 4);
    const int first = kv - nq, low = p.window > 0 && first >= p.window ? first - p.window + 1 : 0;  // the first key of the first token's window
    const float nan = __builtin_nanf("");
    for (int at = blockIdx.x * 4 + w; at < pieces; at += gridDim.x * 4) {
        const int key = 16 * at, j = key >> p.page_log2;
        const int page_first = j << p.page_log2, page_end = page_first + (1 << p.page_log2);
        const bool page_seen = page_end > low || page_first < p.sinks;  // (entries of pages that no token sees are not read)
        if (!page_seen) continue;
        const int page = __builtin_amdgcn_readfirstlane(table[j]);
        const bool there = (uint32_t)page < (uint32_t)p.pages;
        const int64_t to = (int64_t)rank * p.max_pages + j;
        if (head == 0 && lane == 0 && (at & (per - 1)) == 0) out_table[j] = there ? (int)to : -1;
        if (!there || (key + 16 <= low && key >= p.sinks)) continue;
        const int64_t piece = (((int64_t)page * p.heads + head) * per + (at & (per - 1))) * (9 * DIM);
        const int64_t dst = (((to * p.heads + head) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) * DIM;
        // (all of a piece's loads are in flight together)
        uint32_t codes[2][NG], at_key[NG];
        u32x2 at_value[NG];
#pragma unroll
        for (int b = 0; b < NG; b++) {
            codes[0][b] = reinterpret_cast<const uint32_t *>(p.k + piece)[lane * NG + b];
            codes[1][b] = reinterpret_cast<const uint32_t *>(p.v + piece)[lane * NG + b];
            at_key[b] = reinterpret_cast<const uint16_t *>(p.k + piece + 8 * DIM)[((r >> 2) * NG + b) * 4 + (r & 3)];
            at_value[b] = reinterpret_cast<const u32x2 *>(p.v + piece + 8 * DIM)[q * NG + b];
        }
        auto scale = [&](uint32_t h) { return ((h >> 10) & 31) == 31 ? nan : f16_to_f32((uint16_t)h); };
        auto code = [](uint32_t x, int n) { return (float)((int)((x >> (4 * n)) & 15) - 8); };
#pragma unroll
        for (int b = 0; b < NG; b++) {
            const float d = scale(at_key[b]);
            u32x4 y;
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = pack2<BF>(code(codes[0][b], i) * d, code(codes[0][b], i + 4) * d);  // nibbles 0 4, 1 5, 2 6, 3 7
            *reinterpret_cast<u32x4 *>(p.out_k + dst + r * DIM + 32 * b + 8 * q) = y;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            constexpr int nib[4] = {0, 4, 2, 6};
#pragma unroll
            for (int b = 0; b < NG; b++) {
                const float d = scale((at_value[b][i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
                *reinterpret_cast<uint32_t *>(p.out_v + dst + (4 * q + i) * DIM + 32 * b + 2 * r) =
                    pack2<BF>(code(codes[1][b], nib[i]) * d, code(codes[1][b], nib[i] + 1) * d);
            }
        }
    }
}

}  // namespace

int launch_attn4_image(trhip_ctx *ctx, const Image4 &p, int most) {
    const int64_t pieces = (p.max_pages << p.page_log2) >> 4, cus = ctx->sm_count > 0 ? ctx->sm_count : 256;
    int64_t x = (pieces + 3) / 4, each = 8 * cus / ((int64_t)p.heads * most) + 1;
    if (x > each) x = each;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)x, (unsigned)p.heads, (unsigned)most), dim3(256), 0, ctx->stream, p); };
    switch (p.dim / 32) {
    case 1: go(p.bf ? attn4_image<1, true> : attn4_image<1, false>); break;
    case 2: go(p.bf ? attn4_image<2, true> : attn4_image<2, false>); break;
    case 3: go(p.bf ? attn4_image<3, true> : attn4_image<3, false>); break;
    case 4: go(p.bf ? attn4_image<4, true> : attn4_image<4, false>); break;
    case 5: go(p.bf ? attn4_image<5, true> : attn4_image<5, false>); break;
    case 6: go(p.bf ? attn4_image<6, true> : attn4_image<6, false>); break;
    case 7: go(p.bf ? attn4_image<7, true> : attn4_image<7, false>); break;
    default: go(p.bf ? attn4_image<8, true> : attn4_image<8, false>);
    }
    return launch_check(ctx, "kv4_attn");
}

}  // namespace trhip
