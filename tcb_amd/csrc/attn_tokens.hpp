// attn_tokens.hpp -- attention over a paged cache for few rows: a workgroup takes a tile of up to 32 rows (the heads of a few
// tokens of one request, attn_common.hpp) and a piece of its keys. Its four waves hold all rows each and take every fourth
// block of 32 keys, which they copy into LDS rings of their own (no barrier until the end), then join their references and
// sums. A token step reads every key and value once, so what bounds it is the cache's bytes: 64 requests of up to 8192 keys
// (1.08 GB) take 203 us, 5.3 TB/s, one request of 131071 (537 MB) 104 us. The pieces' length deals the keys over
// all CUs, and two workgroups a CU keep copies in flight while the other starts or ends (128 requests of up to 1000 keys: 62
// us, 80 with one of twice the ring). Below some hundred keys a CU what counts is the chain of instructions: lengths, item, page,
// copy 3 us, 1.3 us for each of a wave's blocks, joining 1 us (one request of 300 keys: 9 us in the kernel). The weights
// are multiplied in two 16-bit terms, as near as fp32 ones: the matrix units have time. Pieces of one tile go to the
// workspace, and the workgroup that finishes last joins them (behind a shared prefix, a launch of its own).
#pragma once

#include "attn_common.hpp"

namespace trhip {
namespace {

constexpr int kTokRows = 32, kTokBlock = 32, kTokWaves = 4, kTokLeast = 8, kTokOver = 6;

template <int DP> struct TokLds {
    static constexpr int SLOT = 32 * DP * 2;  // 32 keys or values
    static constexpr int SLOTS = 2;  // a block's keys and its values; each is filled anew as soon as it has been read
    static constexpr int OSTRIDE = DP + 4;  // floats between rows of a wave's results
    static constexpr int RING = SLOT * SLOTS, OUT = 32 * OSTRIDE * 4;
    static constexpr int WAVE = RING > OUT ? RING : OUT;
    static constexpr int BYTES = kTokWaves * (WAVE + 32 * 8) + 16;
};

// PREFIX: rows are all tokens' and keys the shared prefix's; results go to prefix_part.
template <int DP, bool BF, bool PREFIX> __device__ __forceinline__ void tokens_of(const AttnArgs &p, int wg, int grid) {
    using L = TokLds<DP>;
    extern __shared__ __attribute__((aligned(1024))) uint4 smem[];  // nothing else is shared: the rows' swizzle needs them aligned
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
    Item it;
    const int *table;
    int keys;
    if (PREFIX) {
        const int x = p.by_heads(wg);
        it.head = wg - x * p.kv_heads;
        it.tile = x / p.prefix_splits;
        it.split = x - it.tile * p.prefix_splits;
        it.nsplit = p.prefix_splits;
        it.q0 = 0;
        it.nq = p.tokens;
        it.kv = it.slot = it.counter = 0;
        table = p.prefix_table;
        keys = p.prefix_len;
    } else {
        const bool some = find_item<kTokRows, kTokBlock, kTokLeast, kTokOver>(p, wg, grid, it);
        leave_count(p, it, wg);
        if (!some) return;
        table = p.table + (int64_t)it.req * p.max_pages;
        keys = it.kv;
    }
    const int r0 = it.tile * kTokRows, left = it.nq * p.group - r0, n = left < kTokRows ? left : kTokRows;
    Rows rw;
    if (PREFIX) rw = {keys - 1, 0, keys - 1, keys - 1, 0, 0, 0};
    else rw = rows_of(p, r0, n, it.nq, keys);
    const Span sp = span_of<kTokBlock>(rw.hi_max, rw.lo_min, rw.sinks);
    const int nb = sp.count(), piece = it.nsplit == 1 ? nb : (nb + it.nsplit - 1) / it.nsplit;
    const int b0 = it.split * piece, b1 = b0 + piece < nb ? b0 + piece : nb;
    // some rows see keys that others do not, or keys that none sees are copied with those before or behind them
    const bool mixed = rw.hi_min != rw.hi_max || rw.lo_min != rw.lo_max || rw.lo_min > rw.sinks;

    const uint32_t ring = lds_addr(smem) + w * L::WAVE;
    Lanes16<DP> lanes;
    lanes.init(p.dim);
    uint4 q[DP / 16];
    load_q<DP>(p, q, it.q0, r0, n, it.head);

    auto key_of = [&](int b) { return 32 * sp.block(b); };
    // Block b's two pages, fetched a step before they are used, and its pieces; past the last block nothing but zeros.
    auto pages_of = [&](int b) {
        const int t = b < b1 ? key_of(b) : 0, hi = b < b1 ? rw.hi_max : -1;
        return make_int2(page16(p, table, t, hi), page16(p, table, t + 16, hi));
    };
    auto pieces = [&](int b, int2 pages, Piece16 (&s)[2]) {
        const int t = b < b1 ? key_of(b) : 0, hi = b < b1 ? rw.hi_max : -1;
        s[0] = piece16(p, pages.x, it.head, t, hi, rw.lo_min, rw.sinks);
        s[1] = piece16(p, pages.y, it.head, t + 16, hi, rw.lo_min, rw.sinks);
    };
    auto copy_k = [&](const Piece16 (&s)[2], int slot) {
#pragma unroll
        for (int i = 0; i < 2; i++) lanes.copy(s[i].k, ring + slot * L::SLOT + i * (L::SLOT / 2));
    };
    auto copy_v = [&](const Piece16 (&s)[2], int slot) {
#pragma unroll
        for (int i = 0; i < 2; i++) lanes.copy(s[i].v, ring + slot * L::SLOT + i * (L::SLOT / 2));
    };
    constexpr int D = L::SLOTS / 2, AHEAD = (L::SLOTS - 1) * (DP / 16);
    Piece16 s[2];
    int2 pages[D + 1];
#pragma unroll
    for (int i = 0; i <= D; i++) pages[i] = pages_of(b0 + w + i * kTokWaves);
#pragma unroll
    for (int i = 0; i < D; i++) {
        pieces(b0 + w + i * kTokWaves, pages[i], s);
        copy_k(s, 2 * i);
        copy_v(s, 2 * i + 1);
    }
    int2 pg = pages[D];
    Acc<DP> A;
    A.init();
    int slot = 0;
    for (int b = b0 + w; b < b1; b += kTokWaves) {
        const int t = key_of(b);
        pieces(b + D * kTokWaves, pg, s);
        pg = pages_of(b + (D + 1) * kTokWaves);
        wait_vmcnt(AHEAD);
        a16f x = scores<DP, BF>(ring + slot * L::SLOT, q);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
        copy_k(s, slot);
        const bool all = all_see(rw, t, 32);
        if (!all) mask(x, rw, t);
        softmax_step<DP, BF>(A, x, p.scale);
        wait_vmcnt(AHEAD);
        const uint32_t v = ring + (slot + 1) * L::SLOT;
        if (!all && mixed && odd_values<DP, BF>(v)) values_one_by_one<DP, BF>(A.o, x, v, rw.hi, rw.lo, rw.sinks, t);
        else values<DP, BF, true, true>(A.o, x, v);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        copy_v(s, slot + 1);
        slot = slot + 2 == L::SLOTS ? 0 : slot + 2;
    }
    wait_vmcnt(0);
    // the four waves' results, through LDS
    const float l = half_sum(A.l);
    float *mine = reinterpret_cast<float *>(reinterpret_cast<char *>(smem) + w * L::WAVE);
    float2 *ml = reinterpret_cast<float2 *>(reinterpret_cast<char *>(smem) + kTokWaves * L::WAVE);
    const int r = lane & 31, h = lane >> 5;
    if (r < n) {
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<float4 *>(mine + r * L::OSTRIDE + 32 * d + 8 * g + 4 * h) =
                    make_float4(A.o[d][4 * g], A.o[d][4 * g + 1], A.o[d][4 * g + 2], A.o[d][4 * g + 3]);
        if (h == 0) ml[w * 32 + r] = make_float2(A.m, l);
    }
    __syncthreads();
    const bool direct = !PREFIX && it.nsplit == 1 && p.prefix_splits == 0;
    for (int idx = tid; idx < n * (DP / 4); idx += 64 * kTokWaves) {
        const int r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4, row = r0 + r, t = p.by_group(row);
        if (d >= p.dim) continue;
        Join j;
        j.init();
#pragma unroll
        for (int u = 0; u < kTokWaves; u++) {
            const float4 o = *reinterpret_cast<const float4 *>(reinterpret_cast<const char *>(smem) + u * L::WAVE +
                                                              (r * L::OSTRIDE + d) * 4);
            j.add(ml[u * 32 + r].x, ml[u * 32 + r].y, o.x, o.y, o.z, o.w);
        }
        if (direct) {
            put4<BF>(p, it.q0, row, it.head, d, j.o, j.l, keys - it.nq + t >= 0);
        } else if (PREFIX) {
            float *dst = p.prefix_part + ((int64_t)it.split * p.tokens * p.heads + (int64_t)t * p.heads + it.head * p.group +
                                          (row - t * p.group)) * (DP + 2);
            *reinterpret_cast<float2 *>(dst + d) = make_float2(j.o[0], j.o[1]);
            *reinterpret_cast<float2 *>(dst + d + 2) = make_float2(j.o[2], j.o[3]);
            if (d == 0) *reinterpret_cast<float2 *>(dst + DP) = make_float2(j.m, j.l);
        } else {
            float *dst = p.part + ((int64_t)it.slot * kTokRows + r) * (DP + 2);
            agent_store(dst + d, j.o[0], j.o[1]);
            agent_store(dst + d + 2, j.o[2], j.o[3]);
            if (d == 0) agent_store(dst + DP, j.m, j.l);
        }
    }
    if (direct || PREFIX) return;
    if (p.parts) {
        leave_place(p, it, r0, n);
        return;
    }
    if (last_piece(p, it, reinterpret_cast<int *>(ml + kTokWaves * 32)))
        join_tile<DP, kTokRows, BF, kTokWaves>(p, it, r0, n, reinterpret_cast<float *>(smem), kTokWaves * L::WAVE);
}

}  // namespace
}  // namespace trhip
