// attn4_image.hip -- the 4-bit cache's keys of long requests, opened once into the workspace in 16 bits, for the kernel of many rows.
//
// A long prompt reads every key of its request once for each 128 of its rows, and its time is that of the products; opening the codes
// anew each time would take as long. Every value is exact in f16 and bf16, so what the products see is what the cache stands for.
// It moves 2.56 times the codes' bytes (4.5 bits an element in, 16 out).
#include "kv4.hpp"
#include "attn4_image.hpp"

namespace trhip {
namespace {

typedef uint32_t u32x4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack16(float a, float b, bool bf) {
    if (bf) return (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xFFFF0000u);  // exact: no bits below
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2){(_Float16)a, (_Float16)b});
}

// Workgroup (x, head, rank): pieces x, x + gridDim.x, ... of the keys of the rank-th long request, a wave a piece, plane after plane.
__global__ __launch_bounds__(256) void attn4_image(const Image4 p) {
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
    const int blocks = p.dim >> 5, r = lane & 15, q = lane >> 4, pieces = (int)(((int64_t)kv + 15) >> 4), per = 1 << (p.page_log2 - 4);
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
        const int64_t piece = (((int64_t)page * p.heads + head) * per + (at & (per - 1))) * (9 * p.dim);
        uint16_t *dst = nullptr;
        for (int plane = 0; plane < 2; plane++) {
            const uint8_t *src = (plane ? p.v : p.k) + piece;
            const uint32_t *codes = reinterpret_cast<const uint32_t *>(src) + lane * blocks;
            const uint16_t *scales = reinterpret_cast<const uint16_t *>(src + 8 * p.dim);
            dst = (plane ? p.out_v : p.out_k) + (((to * p.heads + head) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) * p.dim;
            auto scale = [&](int row, int b) {
                const uint32_t h = scales[((row >> 2) * blocks + b) * 4 + (row & 3)];
                return ((h >> 10) & 31) == 31 ? nan : f16_to_f32((uint16_t)h);
            };
            for (int b = 0; b < blocks; b++) {
                const uint32_t x = codes[b];
                auto code = [&](int n) { return (float)((int)((x >> (4 * n)) & 15) - 8); };
                if (plane == 0) {
                    const float d = scale(r, b);
                    u32x4i y;
                    for (int i = 0; i < 4; i++) y[i] = pack16(code(i) * d, code(i + 4) * d, p.bf);  // nibbles 0 4, 1 5, 2 6, 3 7
                    *reinterpret_cast<u32x4i *>(dst + r * p.dim + 32 * b + 8 * q) = y;
                } else {
                    constexpr int nib[4] = {0, 4, 2, 6};
                    for (int i = 0; i < 4; i++) {
                        const float d = scale(4 * q + i, b);
                        *reinterpret_cast<uint32_t *>(dst + (4 * q + i) * p.dim + 32 * b + 2 * r) = pack16(code(nib[i]) * d, code(nib[i] + 1) * d, p.bf);
                    }
                }
            }
        }
    }
}

}  // namespace

int launch_attn4_image(trhip_ctx *ctx, const Image4 &p, int most) {
    const int64_t pieces = (p.max_pages << p.page_log2) >> 4, cus = ctx->sm_count > 0 ? ctx->sm_count : 256;
    int64_t x = (pieces + 3) / 4, each = 8 * cus / ((int64_t)p.heads * most) + 1;
    if (x > each) x = each;
    hipLaunchKernelGGL(attn4_image, dim3((unsigned)x, (unsigned)p.heads, (unsigned)most), dim3(256), 0, ctx->stream, p);
    return launch_check(ctx, "kv4_attn");
}

}  // namespace trhip
