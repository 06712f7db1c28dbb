// attn_rows.hpp -- the kernel of attention over a paged cache for many rows: prompts, and a shared prefix under a batch's tokens.
//
// A workgroup takes a tile of 128 rows, 32 a wave (attn_common.hpp), and goes through its keys in blocks of 64 that its waves
// copy into LDS together. What bounds it are the matrix instructions, the softmax's instructions beside them and the
// power that both draw: a causal prompt of 8192 tokens, 32 heads of 128, takes 502 to 543 us (it differs by the card), 1.0 to 1.1 PFLOP/s,
// at a clock of 1.67 GHz (2.4 without load), where a large library product reaches 1.63 PFLOP/s. Blocks are taken in a skewed loop: step j
// multiplies K of block j + 1 and V of block j - 1 while it takes the exponentials of block j, three independent pieces of work
// in one run of instructions, and two waves share a SIMD. Masks only touch the scores there. Every instruction in it
// counts: choosing each copied row by the mask took 32 of 165 vector instructions and 3.5% of the time. Rows that see few
// keys, and what is left of an odd number of blocks, go through a plain step in a loop of its own: as a branch of the skewed one
// it made the compiler copy O^T between registers at every join, a third of the instructions (616 us, 597 without).
//
// The softmax's reference (what is subtracted from a row's scores) is a whole power of two, raised only when a block's
// maximum exceeds it by more than 2^8: then the sums, O^T and the pending weights are multiplied by a power of two, exactly (f16
// weights below its normal numbers lose bits). The weights stay below 2^9 in bf16 and 2^16 in f16, where they stand 2^7 higher: below 2^-14 f16
// loses bits, below 2^-25 everything, so a weight is held to 2^-11 of itself or 2^-31 of the row's largest. The row's sum is
// taken of the weights in fp32; for the product with V the skewed loop rounds them to 16 bits, to nearest, so that many
// keys' roundings average out. Rows that see fewer than kFewKeys keys go through the plain step, which multiplies a second
// term of each weight (what the rounding dropped): as near as with weights in fp32, for half again as many products (the
// whole prompt would take 798 us so, 596 in plain steps of one term, 521 in the skewed loop of the same run).
#pragma once

#include "attn_common.hpp"

namespace trhip {
namespace {

constexpr int kFewKeys = 256;

template <int V> struct Const {
    static constexpr int value = V;
};

template <int DP> struct RowsShape {
    static constexpr int WAVES = 4, BK = 64, NT = BK / 32;
    // Heads of over 128: their accumulators leave no registers for a second block's scores and weights, so a plain step, one
    // workgroup a CU, operands eight products ahead (prompt of 4096, 16 heads of 256: 250 us).
    static constexpr bool SKEW = DP != 256;
    static constexpr int PER_CU = DP == 256 ? 1 : 2;  // workgroups a CU: by registers, for heads of 256 by LDS as well (128 KB)
    static constexpr int THREADS = 64 * WAVES, TR = 32 * WAVES;
    static constexpr int TILE = BK * DP * 2;       // bytes of a block's keys or values
    static constexpr int PI = DP / 32;             // copies a wave makes of a block: a sixteen-row piece
    static constexpr int BYTES = 4 * TILE + 16;  // two blocks of each are in LDS
};

// PREFIX: rows are all tokens' and keys the shared prefix's; results go to prefix_part.
template <int DP, bool BF, bool PREFIX> __device__ __forceinline__ void rows_of_tile(const AttnArgs &p, int wg, int grid) {
    using L = RowsShape<DP>;
    constexpr int BK = L::BK, NT = L::NT;
    extern __shared__ __attribute__((aligned(1024))) uint4 smem[];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), h = lane >> 5;
    Item it;
    const int *table;
    int keys;
    if (PREFIX) {
        const int x = p.by_heads(wg);
        it.head = wg - x * p.kv_heads;
        it.tile = x / p.prefix_splits;
        it.split = x - it.tile * p.prefix_splits;
        it.nsplit = p.prefix_splits;
        it.q0 = it.kv = it.slot = it.counter = 0;
        it.nq = p.tokens;
        table = p.prefix_table;
        keys = p.prefix_len;
    } else {
        const bool some = find_item<L::TR, BK, kRowsLeast, kRowsOver>(p, wg, grid, it);
        leave_count(p, it, wg);
        if (!some) return;
        table = p.table + (int64_t)it.req * p.max_pages;
        keys = it.kv;
    }
    const int r0 = it.tile * L::TR, left = it.nq * p.group - r0, n = left < L::TR ? left : L::TR;
    // the tile's masks, then this wave's rows'
    Rows all, rw;
    const int wr = w * 32, wn = n - wr < 0 ? 0 : n - wr < 32 ? n - wr : 32;  // this wave's first row in the tile, its rows
    if (PREFIX) {
        all = rw = {keys - 1, 0, keys - 1, keys - 1, 0, 0, 0};
    } else {
        all = rows_of(p, r0, n, it.nq, keys);
        rw = wn > 0 ? rows_of(p, r0 + wr, wn, it.nq, keys) : rows_of(p, r0 + n - 1, 1, it.nq, keys);
    }
    const bool mixed = all.hi_min != all.hi_max || all.lo_min != all.lo_max;
    const Span sp = span_of<BK>(all.hi_max, all.lo_min, all.sinks);
    const int total = sp.count(), piece = it.nsplit == 1 ? total : (total + it.nsplit - 1) / it.nsplit;
    const int b0 = it.split * piece, left_b = total - b0, nb = left_b < 0 ? 0 : left_b < piece ? left_b : piece;

    const uint32_t ring = lds_addr(smem);
    Lanes16<DP> share;
    share.init(p.dim);
    const int prow = 16 * w;  // its piece's first row in a block

    uint4 q[DP / 16];
    load_q<DP>(p, q, it.q0, wn > 0 ? r0 + wr : r0, wn, it.head);
    auto key_of = [&](int j) { return BK * sp.block(b0 + j); };
    // Block j's piece of this wave; past the last block: zeros. The page's number is fetched a step before it is used.
    auto page_of = [&](int j) { return j < nb ? page16(p, table, key_of(j) + prow, all.hi_max) : 0; };
    auto piece_of = [&](int j, int page) {
        return piece16(p, page, it.head, (j < nb ? key_of(j) : 0) + prow, j < nb ? all.hi_max : -1, all.lo_min, all.sinks);
    };
    // block j's places: keys at k_at, values at v_at
    auto k_at = [&](int j) { return ring + (j & 1) * L::TILE; };
    auto v_at = [&](int j) { return ring + (2 + (j & 1)) * L::TILE; };
    const uint32_t mine = w * (32 * DP);
    auto copy_k = [&](const Piece16 &c, int j) { share.copy(c.k, k_at(j) + mine); };
    auto copy_v = [&](const Piece16 &c, int j) { share.copy(c.v, v_at(j) + mine); };

    a16f o[DP / 32], s[NT];
    uint32_t pk[NT][8];  // weights of the block before, two a register, in the order of its score registers
    float ms = -__builtin_inff(), mf = ms, l = 0.0f, top;  // reference (log2 units), the score it came from, the sum, the block's maximum
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 8; i++) pk[t][i] = 0;
    // lane parts of the operands' addresses
    const int kr = lane & 31, vi = lane & 15, vr = 4 * h + (vi >> 2), vc = 2 * ((lane >> 4) & 1) + ((vi >> 1) & 1);
    const uint32_t ka = kr * (2 * DP) + ((h ^ swz<DP>(kr)) << 4), va = vr * (2 * DP) + ((vc ^ swz<DP>(vr)) << 4) + 8 * (vi & 1);
    constexpr int NK = DP / 16, NV = DP / 16;

    auto maximum = [&](const a16f (&x)[NT]) {
        float m = x[0][0];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) m = fmaxf(m, x[t][i]);
        return m;
    };
    auto k_frag = [&](uint32_t at, int i) { return lds16(ring + (ka ^ ((i / NT) << 5)) + (at + (i % NT) * 64 * DP)); };  // the NT sums in turn
    auto v_frag = [&](uint32_t at, int i) {
        const int d = i % (DP / 32), c = i / (DP / 32);  // dimensions 32 d ..., keys 16 c ...
        const uint2 x = lds_tr(ring + (va ^ (d << 6)) + (at + c * 32 * DP)), y = lds_tr(ring + (va ^ (d << 6) ^ 32) + (at + c * 32 * DP + 16 * DP));
        return (u32x4){x.x, x.y, y.x, y.y};
    };
    auto p_frag = [&](const uint32_t (&x)[NT][8], int i) {
        const int c = i / (DP / 32), t = c / 2, e = 4 * (c & 1);
        return make_uint4(x[t][e], x[t][e + 1], x[t][e + 2], x[t][e + 3]);
    };
    // The reference: raised to a block's maximum where that exceeds it by more than 2^8. neg: minus the reference, for the
    // exponentials' fused step; 0 where scores are too large for that (far) and are made relative first. Far scores can lie more
    // than 2^8 apart and next to each other, so their difference is looked at, not a sum that rounds to the next one.
    float neg = 0.0f;
    bool far = false;
    auto exceeds = [&] { return (top - mf) * p.scale > 8.0f; };
    auto raise = [&](uint32_t (&pk)[NT][8], bool weights) {
        const float y = top * p.scale;
        const bool up = exceeds(), to_far = fabsf(y) > kFar;
        const float r = to_far ? y : ceilf(y) - kLift<BF>;
        const float a = up ? exp2_hw(far && to_far ? (mf - top) * p.scale : ms - r) : 1.0f;  // from -Inf: 0
        ms = up ? r : ms;
        mf = up ? top : mf;
        l *= a;
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= a;
        if (weights) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 8; i++) pk[t][i] = pack2<BF>(wide_lo<BF>(pk[t][i]) * a, wide_hi<BF>(pk[t][i]) * a);
        }
        far = up ? to_far : far;
        neg = far || ms == -__builtin_inff() ? 0.0f : -ms;
    };
    auto relative = [&](a16f (&x)[NT]) {
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[t][i] -= far ? mf : 0.0f;
        }
    };

    {
        const Piece16 c = piece_of(0, page_of(0));
        copy_k(c, 0);
        copy_v(c, 0);
    }

    // Whether a key that some rows see and others do not, or one that none sees in a piece of sixteen that some see, has a value
    // that is not finite (0 times it would reach all rows): its tile goes through plain steps, which look out for that. Those
    // keys are the ones behind the first token's last and before the last token's window, one for each token of the
    // tile, and up to fifteen before the window and behind the first tokens.
    bool odd = false;
    const bool gap = all.lo_min > all.sinks;
    if (!PREFIX && (mixed || gap)) {
        constexpr uint32_t E = BF ? 0x7F807F80u : 0x7C007C00u, U = BF ? 0x00800080u : 0x04000400u;
        const int l0 = gap ? (all.lo_min & ~15) < all.sinks ? all.sinks : all.lo_min & ~15 : all.lo_min;
        const uint32_t e0 = ((uint32_t)all.sinks + 15) & ~15u;
        const int e1 = e0 < (uint32_t)l0 ? (int)e0 : l0;
        const int chunks = p.dim / 8, n0 = all.hi_max - all.hi_min, n1 = all.lo_max - l0, n2 = gap ? e1 - all.sinks : 0;
        uint32_t any = 0;
        for (int i = tid; i < (n0 + n1 + n2) * chunks; i += L::THREADS) {
            const int k = i / chunks, c = i - k * chunks, t = k < n0 ? all.hi_min + 1 + k : k < n0 + n1 ? l0 + (k - n0) : all.sinks + (k - n0 - n1);
            if (t < 0) continue;
            const int page = table[t >> p.page_log2];
            if ((uint32_t)page >= (uint32_t)p.npages) continue;
            const uint4 x = *reinterpret_cast<const uint4 *>(p.v + (int64_t)page * p.page_bytes + (int64_t)it.head * p.head_bytes +
                                                             (int64_t)((t & ((1 << p.page_log2) - 1)) * p.dim * 2 + c * 16));
            any |= ((x.x & E) + U) | ((x.y & E) + U) | ((x.z & E) + U) | ((x.w & E) + U);
        }
        int *flag = reinterpret_cast<int *>(smem) + 4 * L::TILE / 4;
        if (tid == 0) *flag = 0;
        lds_barrier();
        if (any & 0x80008000u) *flag = 1;
        lds_barrier();
        odd = *flag != 0;
    }
    // Blocks go through the skewed loop in pairs (an odd one last through a plain step), except where rows see few keys and in a
    // short request (one that a wrong hint of the sizes brought here), whose weights have two terms in attn_tokens too.
    const bool few = all.hi_min + 1 < kFewKeys || (p.window > 0 && p.window < kFewKeys) || (!PREFIX && it.nq * p.group <= kTokMost);
    const int pairs = !L::SKEW || few || odd ? 0 : nb & ~1;
    auto qk = [&](a16f (&x)[NT], int place) {
        if constexpr (L::SKEW) {
#pragma unroll
            for (int i = 0; i < NT * NK; i++) x[i % NT] = mma<BF>(k_frag(place * L::TILE, i), q[i / NT], i < NT ? a16f{} : x[i % NT]);
        } else {  // alone on its SIMD: operands eight ahead
            u32x4 f[NT * NK];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = k_frag(place * L::TILE, i);
#pragma unroll
            for (int i = 0; i < NT * NK; i++) {
                __builtin_amdgcn_sched_barrier(0);
                if (i + 8 < NT * NK) f[i + 8] = k_frag(place * L::TILE, i + 8);
                x[i % NT] = mma<BF>(f[i], q[i / NT], i < NT ? a16f{} : x[i % NT]);
            }
        }
    };
    auto plain = [&](int j) {
        const int page = page_of(j + 1);
        wait_vmcnt(0);
        lds_barrier();  // block j is there, and block j - 1 has been read
        {
            const Piece16 c = piece_of(j + 1, page);
            copy_k(c, j + 1);
            copy_v(c, j + 1);
        }
        qk(s, j & 1);
        const uint32_t vat = v_at(j);
        const int t0 = key_of(j);
        const bool see = all_see(rw, t0, BK);
        if (!see) {
#pragma unroll
            for (int t = 0; t < NT; t++) mask(s[t], rw, t0 + 32 * t);
        }
        top = half_max(maximum(s));
        if (__any(exceeds())) raise(pk, false);
        relative(s);
        bool odd_here = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[t][i] = exp2_hw(fmaf(s[t][i], p.scale, neg));
                l += s[t][i];
            }
            if (!see && odd) odd_here = odd_here || odd_values<DP, BF>(vat + t * 64 * DP);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (odd_here) values_one_by_one<DP, BF>(o, s[t], vat + t * 64 * DP, rw.hi, rw.lo, rw.sinks, t0 + 32 * t);
            else if (few || (!L::SKEW && !see)) values<DP, BF, true, false>(o, s[t], vat + t * 64 * DP);
            else values<DP, BF, false, false>(o, s[t], vat + t * 64 * DP);
        }
    };
    int j = 0;
    if constexpr (L::SKEW)
    if (pairs > 0) {
        Piece16 c0 = piece_of(j, page_of(j)), c1 = piece_of(j + 1, page_of(j + 1));
        int page2 = page_of(j + 2);
        wait_vmcnt(0);
        lds_barrier();
        // no weights are pending: zeros in the place of block j - 1's values
        for (int i = tid; i < L::TILE / 16; i += L::THREADS) smem[3 * L::TILE / 16 + i] = make_uint4(0, 0, 0, 0);
        copy_k(c1, 1);
        qk(s, 0);
        top = half_max(maximum(s));
        bool higher = exceeds();
        a16f s1[NT];
        uint32_t p1[NT][8];
        // Step j, P = j % 2: scores x, weights y of block j - 1; leaves the next scores in xn, this block's weights in yn.
        auto step = [&](auto P, a16f (&x)[NT], a16f (&xn)[NT], uint32_t (&y)[NT][8], uint32_t (&yn)[NT][8]) {
            constexpr int here = decltype(P)::value, there = 1 - here;
            const int page3 = page_of(j + 3);
            wait_vmcnt(0);
            lds_barrier();  // keys of block j + 1 and values of j - 1 are there; keys of j and values of j - 2 have been read
            const int t0 = key_of(j);
            if (!all_see(rw, t0, BK)) {
#pragma unroll
                for (int t = 0; t < NT; t++) mask(x[t], rw, t0 + 32 * t);
                top = half_max(maximum(x));
                higher = exceeds();
            }
            if (__any(higher)) raise(y, true);
            relative(x);
            // three independent runs, dealt over one another: products with K, exponentials, products with V; between
            // them the copies of keys j + 2 and values j, and behind the first the next scores' maximum
            const Piece16 c2 = piece_of(j + 2, page2);
            float sum = 0.0f, best = 0.0f;
            constexpr int M = NT * (NK + NV), NW = 8 * NT, AHEAD = 3;  // products, pairs of weights, operands read ahead
            u32x4 f[AHEAD + 1];
            auto frag = [&](int i) { return i < NT * NK ? k_frag(there * L::TILE, i) : v_frag((2 + there) * L::TILE, i - NT * NK); };
#pragma unroll
            for (int i = 0; i < AHEAD; i++) f[i] = frag(i);
#pragma unroll
            for (int i = 0; i < M; i++) {
                __builtin_amdgcn_sched_barrier(0);  // in this order: the compiler would read operands late and add up last
                if (i + AHEAD < M) f[(i + AHEAD) % (AHEAD + 1)] = frag(i + AHEAD);
                const u32x4 a = f[i % (AHEAD + 1)];
                if (i < NT * NK) xn[i % NT] = mma<BF>(a, q[i / NT], i < NT ? a16f{} : xn[i % NT]);
                else o[(i - NT * NK) % (DP / 32)] = mma<BF>(a, p_frag(y, i - NT * NK), o[(i - NT * NK) % (DP / 32)]);
                if (i % 2 == 0 && i / 2 < L::PI) share.copy_one(c2.k, ring + here * L::TILE + mine, i / 2);
                if (i % 2 == 0 && i / 2 >= L::PI && i / 2 < 2 * L::PI) share.copy_one(c0.v, ring + (2 + here) * L::TILE + mine, i / 2 - L::PI);
#pragma unroll
                for (int e = i * NW / M; e < (i + 1) * NW / M; e++) {
                    const int t = e >> 3, k = e & 7;
                    const float u = exp2_hw(fmaf(x[t][2 * k], p.scale, neg)), v = exp2_hw(fmaf(x[t][2 * k + 1], p.scale, neg));
                    yn[t][k] = opaque(pack2<BF>(u, v));  // (made here: the compiler would move it to the next step, where it is used)
                    sum += u;
                    sum += v;
                    asm("" : "+v"(sum));  // (likewise)
                }
                const int m0 = NT * NK + 2, m1 = M - 2;  // maxima of pairs [from, to)
                if (i >= m0 && i < m1) {
#pragma unroll
                    for (int e = (i - m0) * 8 * NT / (m1 - m0); e < (i - m0 + 1) * 8 * NT / (m1 - m0); e++) {
                        const float u = xn[e / 8][2 * (e % 8)], v = xn[e / 8][2 * (e % 8) + 1];
                        best = e == 0 ? fmaxf(u, v) : fmaxf(fmaxf(best, u), v);
                    }
                }
                if (i == M - 2) {
                    top = half_max(best);
                    higher = exceeds();
                }
            }
            l += sum;
            c0 = c1, c1 = c2, page2 = page3;
            j++;
        };
        while (j < pairs) {
            step(Const<0>{}, s, s1, pk, p1);
            step(Const<1>{}, s1, s, p1, pk);
        }
        wait_vmcnt(0);
        lds_barrier();
        copy_v(c0, 0);
#pragma unroll
        for (int i = 0; i < NT * NV; i++) o[i % (DP / 32)] = mma<BF>(v_frag(3 * L::TILE, i), p_frag(pk, i), o[i % (DP / 32)]);
    }
    for (; j < nb; j++) plain(j);
    wait_vmcnt(0);

    const bool direct = !PREFIX && it.nsplit == 1 && p.prefix_splits == 0;
    const float sum = half_sum(l);
    if ((lane & 31) < wn) {
        const int r = wr + (lane & 31), row = r0 + r, t = p.by_group(row);
        float *part = PREFIX ? p.prefix_part + ((int64_t)it.split * p.tokens * p.heads + (int64_t)t * p.heads + it.head * p.group +
                                                (row - t * p.group)) * (DP + 2)
                             : p.part + ((int64_t)it.slot * L::TR + r) * (DP + 2);
        const bool sees = keys - it.nq + t >= 0;
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int at = 32 * d + 8 * g + 4 * h;
                const float y[4] = {o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                if (direct) {
                    put4<BF>(p, it.q0, row, it.head, at, y, sum, sees);
                } else {
                    *reinterpret_cast<float2 *>(part + at) = make_float2(y[0], y[1]);
                    *reinterpret_cast<float2 *>(part + at + 2) = make_float2(y[2], y[3]);
                }
            }
        if (!direct && h == 0) *reinterpret_cast<float2 *>(part + DP) = make_float2(ms, sum);
    }
    if (!direct && !PREFIX) leave_place(p, it, r0, n);
}

template <int DP, bool BF, bool PREFIX>
__global__ __launch_bounds__(RowsShape<DP>::THREADS, RowsShape<DP>::PER_CU) void attn_rows(const AttnArgs p) {
    rows_of_tile<DP, BF, PREFIX>(p, blockIdx.x, gridDim.x);
}

template <int DP, bool BF, bool PREFIX> int launch_rows(trhip_ctx *ctx, const AttnArgs &p, int64_t grid) {
    const void *fn = reinterpret_cast<const void *>(attn_rows<DP, BF, PREFIX>);
    const int st = allow_dyn_lds(ctx, fn, RowsShape<DP>::BYTES, "attention");
    if (st != TRHIP_OK) return st;
    hipLaunchKernelGGL((attn_rows<DP, BF, PREFIX>), dim3((unsigned)grid), dim3(RowsShape<DP>::THREADS), RowsShape<DP>::BYTES, ctx->stream, p);
    return launch_check(ctx, "attention");
}

}  // namespace
}  // namespace trhip
