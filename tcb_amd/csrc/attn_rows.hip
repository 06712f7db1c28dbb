// attn_rows.hip -- attention over a paged cache for many rows: prompts, and a shared prefix under a batch's tokens.
//
// A workgroup takes a tile of 32 rows a wave (attn_common.hpp) and goes through its keys in blocks of BK that its waves copy
// into LDS together. What bounds it are the matrix instructions and, nearly as much, the softmax's instructions, which
// have to run under them. Blocks that every row sees whole are taken in a skewed loop: step j multiplies K of block j + 1 and V of
// block j - 1 while it takes the exponentials of block j, three independent pieces of work in one run of instructions, and two
// waves share a SIMD. Blocks with a mask go through a plain step. The two are loops of their own: with masks as branches of one loop the
// compiler copied O^T between registers at every join, a third of the loop's instructions.
//
// The softmax's reference (what is subtracted from a row's scores) is a whole power of two, raised only when a block's
// maximum exceeds it by more than 2^8: then the sums, O^T and the pending weights are multiplied by a power of two, exactly.
// The weights stay below 2^9, inside f16 and bf16, and lose no precision to a reference that is a little low. In the skewed
// loop they are rounded to 16 bits for the product with V, and the row's sum is taken of the rounded ones, so that many keys'
// rounding averages out. The plain step, which all blocks of rows that see fewer than kFewKeys keys take, multiplies a second
// term of each weight (what the rounding dropped): as near as with weights in fp32.
#include "attn_common.hpp"

namespace trhip {
namespace {

constexpr int kFewKeys = 128;

template <int DP> struct RowsShape {
    static constexpr int WAVES = DP == 256 ? 4 : 8, BK = DP == 256 ? 32 : 64, NT = BK / 32;  // two waves a SIMD where the registers allow
    static constexpr int THREADS = 64 * WAVES, TR = 32 * WAVES;
    static constexpr int TILE = BK * DP * 2;       // bytes of a block's keys or values
    static constexpr int SLOTS = 3;                // blocks of each in LDS
    static constexpr int PI = DP / 64;             // copies a wave makes of a block: eight rows
    static constexpr int ZERO = 2 * SLOTS * TILE;  // a block of zeros behind the rings
    static constexpr int BYTES = ZERO + TILE + 16;
};

// A wave's share of a block: eight rows of a sixteen-row piece, from row `r0` of it.
template <int DP> struct Share {
    static constexpr int N = DP / 64, CH = DP / 8, RPI = 64 / CH;
    uint32_t voff[N];
    int row;
    __device__ __forceinline__ void init(int dim, int r0) {
        const int lane = threadIdx.x & 63;
        row = r0 + lane / CH;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = row + i * RPI, c = (lane % CH) ^ swz<DP>(r);
            voff[i] = 8 * c < dim ? (uint32_t)(r * dim * 2 + c * 16) : 0x80000000u;
        }
    }
    __device__ __forceinline__ void copy(dma_rsrc d, uint32_t dst, int ha, int hb) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t o = voff[i];
            if (hb > ha) o = (uint32_t)(row + i * RPI - ha) < (uint32_t)(hb - ha) ? 0x80000000u : o;
            dma16(d, dst + i * 1024, o, 0);
        }
    }
};

template <int DP, bool BF, bool PREFIX>
__global__ __launch_bounds__(RowsShape<DP>::THREADS, RowsShape<DP>::WAVES / 4) void attn_rows(const AttnArgs p) {
    using L = RowsShape<DP>;
    constexpr int BK = L::BK, NT = L::NT;
    extern __shared__ __attribute__((aligned(1024))) uint4 smem[];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), h = lane >> 5;
    Item it;
    const int *table;
    int keys;
    if (PREFIX) {
        const int x = blockIdx.x / p.kv_heads;
        it.head = blockIdx.x - x * p.kv_heads;
        it.tile = x / p.prefix_splits;
        it.split = x - it.tile * p.prefix_splits;
        it.nsplit = p.prefix_splits;
        it.q0 = it.kv = it.slot = it.counter = 0;
        it.nq = p.tokens;
        table = p.prefix_table;
        keys = p.prefix_len;
    } else {
        if (!find_item<L::TR, BK, 4, kRowsOver>(p, blockIdx.x, it)) return;
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
    const int total = sp.count(), piece = (total + it.nsplit - 1) / it.nsplit;
    const int b0 = it.split * piece, left_b = total - b0, nb = left_b < 0 ? 0 : left_b < piece ? left_b : piece;

    const uint32_t ring = lds_addr(smem);
    Share<DP> share;
    share.init(p.dim, 8 * (w & 1));
    const int prow = 16 * (w >> 1);  // its piece's first row in a block
    for (int i = tid; i < L::TILE / 16; i += L::THREADS) smem[L::ZERO / 16 + i] = make_uint4(0, 0, 0, 0);

    uint4 q[DP / 16];
    load_q<DP>(p, q, it.q0, wn > 0 ? r0 + wr : r0, wn, it.head);
    auto key_of = [&](int j) { return BK * sp.block(b0 + j); };
    auto piece_of = [&](int j) {  // past the last block: zeros
        return piece16(p, table, it.head, (j < nb ? key_of(j) : 0) + prow, j < nb ? all.hi_max : -1, all.lo_min, all.sinks);
    };
    const uint32_t dst = ring + w * (16 * DP);
    auto copy_k = [&](const Piece16 &s, int slot) { share.copy(s.k, dst + slot * L::TILE, s.ha, s.hb); };
    auto copy_v = [&](const Piece16 &s, int slot) { share.copy(s.v, dst + (L::SLOTS + slot) * L::TILE, s.ha, s.hb); };

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
    auto k_frag = [&](uint32_t base, int i) { return lds16(base + (ka ^ ((i % NK) << 5)) + (i / NK) * 64 * DP); };
    auto v_frag = [&](uint32_t base, int i) {
        const int d = i % (DP / 32), c = i / (DP / 32);  // dimensions 32 d ..., keys 16 c ...
        const uint2 x = lds_tr(base + (va ^ (d << 6)) + c * 32 * DP), y = lds_tr(base + (va ^ (d << 6) ^ 16) + c * 32 * DP + 16 * DP);
        return make_uint4(x.x, x.y, y.x, y.y);
    };
    auto p_frag = [&](const uint32_t (&x)[NT][8], int i) {
        const int c = i / (DP / 32), t = c / 2, e = 4 * (c & 1);
        return make_uint4(x[t][e], x[t][e + 1], x[t][e + 2], x[t][e + 3]);
    };
    // Raises the reference to a block's maxima where they exceed it by more than 2^8; returns minus the reference for the
    // exponentials' fused step (0 where scores x were too large for it and have been made relative here).
    auto refer = [&](a16f (&x)[NT], bool weights) -> float {
        top = half_max(top);
        if (__any(top * p.scale > ms + 8.0f)) {
            const float y = top * p.scale, r = fabsf(y) > 1048576.0f ? y : ceilf(y);
            const bool up = r > ms + 8.0f;
            const float a = up ? exp2_hw(ms - r) : 1.0f;  // from -Inf: 0
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
        }
        const float neg = ms == -__builtin_inff() ? 0.0f : -ms;
        const bool far = fabsf(neg) > 1048576.0f;
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[t][i] -= far ? mf : 0.0f;
        }
        return far ? 0.0f : neg;
    };

    // Blocks [f0, f1) are seen whole by every row of the tile.
    const int at0 = sp.ns - sp.w0 - b0;
    int f0 = at0 + (all.lo_max + BK - 1) / BK, f1 = at0 + (all.hi_min + 1) / BK;
    f0 = f0 < 0 ? 0 : f0;
    f1 = f1 > nb ? nb : f1;
    if (f1 < f0 + 2 || all.hi_min + 1 < kFewKeys || (p.window > 0 && p.window < kFewKeys)) f0 = f1 = nb;

    // Copies run ahead of step j by K of block j + 3 and V of block j + 1.
    Piece16 c1 = piece_of(1), c2 = piece_of(2);
    {
        const Piece16 c0 = piece_of(0);
        copy_k(c0, 0);
        copy_k(c1, 1);
        copy_k(c2, 2);
        copy_v(c0, 0);
    }
    int k0 = 0;  // ring place of block j, keys and values
    auto next = [&](int k) { return k + 1 == L::SLOTS ? 0 : k + 1; };
    auto ahead = [&](int j) {
        const Piece16 c3 = piece_of(j + 3);
        copy_v(c1, next(k0));
        copy_k(c3, k0);
        c1 = c2, c2 = c3;
    };
    auto plain = [&](int j) {
        wait_vmcnt(0);
        lds_barrier();
        const uint32_t kat = ring + k0 * L::TILE, vat = ring + (L::SLOTS + k0) * L::TILE;
#pragma unroll
        for (int i = 0; i < NT * NK; i++) s[i / NK] = mma<BF>(k_frag(kat, i), q[i % NK], i % NK == 0 ? a16f{} : s[i / NK]);
        lds_barrier();  // the keys have been read
        ahead(j);
        const int t0 = key_of(j);
        const bool see = all_see(rw, t0, BK);
        if (!see) {
#pragma unroll
            for (int t = 0; t < NT; t++) mask(s[t], rw, t0 + 32 * t);
        }
        top = maximum(s);
        const float neg = refer(s, false);
        bool odd = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[t][i] = exp2_hw(fmaf(s[t][i], p.scale, neg));
                l += s[t][i];
            }
            if (!see && mixed) odd = odd || odd_values<DP, BF>(vat + t * 64 * DP);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (odd) values_one_by_one<DP, BF>(o, s[t], vat + t * 64 * DP, rw.hi, rw.lo, rw.sinks, t0 + 32 * t);
            else values<DP, BF, true>(o, s[t], vat + t * 64 * DP);
        }
        k0 = next(k0);
    };
    int j = 0;
    for (; j < f0; j++) plain(j);
    if (j < f1) {
        wait_vmcnt(2 * L::PI);
        lds_barrier();
        {
            const uint32_t kat = ring + k0 * L::TILE;
#pragma unroll
            for (int i = 0; i < NT * NK; i++) s[i / NK] = mma<BF>(k_frag(kat, i), q[i % NK], i % NK == 0 ? a16f{} : s[i / NK]);
        }
        top = maximum(s);
        uint32_t vat = ring + L::ZERO;  // V of block j - 1
        for (; j < f1; j++) {
            wait_vmcnt(2 * L::PI);
            lds_barrier();  // keys of block j + 1 and values of j - 1 are there, and what the next copies replace has been read
            ahead(j);
            const uint32_t kat = ring + next(k0) * L::TILE;
            const float neg = refer(s, true);
            // three independent runs, dealt over one another: products with K, exponentials, products with V
            a16f sn[NT];
            uint32_t pn[NT][8];
            float sum = 0.0f;
            constexpr int M = NT * (NK + NV), NW = 8 * NT, AHEAD = 3;  // products, pairs of weights, operands read ahead
            uint4 f[AHEAD + 1];
            auto frag = [&](int i) { return i < NT * NK ? k_frag(kat, i) : v_frag(vat, i - NT * NK); };
#pragma unroll
            for (int i = 0; i < AHEAD; i++) f[i] = frag(i);
#pragma unroll
            for (int i = 0; i < M; i++) {
                if (i + AHEAD < M) f[(i + AHEAD) % (AHEAD + 1)] = frag(i + AHEAD);
                const uint4 a = f[i % (AHEAD + 1)];
                if (i < NT * NK) sn[i / NK] = mma<BF>(a, q[i % NK], i % NK == 0 ? a16f{} : sn[i / NK]);
                else o[(i - NT * NK) % (DP / 32)] = mma<BF>(a, p_frag(pk, i - NT * NK), o[(i - NT * NK) % (DP / 32)]);
#pragma unroll
                for (int e = i * NW / M; e < (i + 1) * NW / M; e++) {
                    const int t = e >> 3, k = e & 7;
                    pn[t][k] = pack2<BF>(exp2_hw(fmaf(s[t][2 * k], p.scale, neg)), exp2_hw(fmaf(s[t][2 * k + 1], p.scale, neg)));
                    sum = add2<BF>(pn[t][k], sum);  // of the rounded weights
                }
            }
            l += sum;
            top = maximum(sn);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                s[t] = sn[t];
#pragma unroll
                for (int i = 0; i < 8; i++) pk[t][i] = pn[t][i];
            }
            vat = ring + (L::SLOTS + k0) * L::TILE;
            k0 = next(k0);
        }
        wait_vmcnt(0);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NT * NV; i++) o[i % (DP / 32)] = mma<BF>(v_frag(vat, i), p_frag(pk, i), o[i % (DP / 32)]);
    }
    for (; j < nb; j++) plain(j);
    wait_vmcnt(0);

    const bool direct = !PREFIX && it.nsplit == 1 && p.prefix_splits == 0;
    const float sum = half_sum(l);
    if ((lane & 31) < wn) {
        const int r = wr + (lane & 31), row = r0 + r, t = row / p.group;
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
                } else if (PREFIX) {
                    *reinterpret_cast<float2 *>(part + at) = make_float2(y[0], y[1]);
                    *reinterpret_cast<float2 *>(part + at + 2) = make_float2(y[2], y[3]);
                } else {
                    agent_store(part + at, y[0], y[1]);
                    agent_store(part + at + 2, y[2], y[3]);
                }
            }
        if (!direct && h == 0) {
            if (PREFIX) *reinterpret_cast<float2 *>(part + DP) = make_float2(ms, sum);
            else agent_store(part + DP, ms, sum);
        }
    }
    if (direct || PREFIX) return;
    if (last_piece(p, it, reinterpret_cast<int *>(smem) + (L::BYTES - 16) / 4)) join_tile<DP, L::TR, BF>(p, it, r0, n, L::THREADS);
}

template <int DP, bool BF, bool PREFIX> int launch_rows(trhip_ctx *ctx, const AttnArgs &p, int64_t grid) {
    const void *fn = reinterpret_cast<const void *>(attn_rows<DP, BF, PREFIX>);
    const int st = allow_dyn_lds(ctx, fn, RowsShape<DP>::BYTES, "attention");
    if (st != TRHIP_OK) return st;
    hipLaunchKernelGGL((attn_rows<DP, BF, PREFIX>), dim3((unsigned)grid), dim3(RowsShape<DP>::THREADS), RowsShape<DP>::BYTES, ctx->stream, p);
    return launch_check(ctx, "attention");
}

}  // namespace

int attn_rows_tile(int dp) { return dp == 256 ? RowsShape<256>::TR : RowsShape<128>::TR; }
int attn_rows_block(int dp) { return dp == 256 ? RowsShape<256>::BK : RowsShape<128>::BK; }

template <bool PREFIX> static int by_type(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, int64_t grid) {
    if (dp == 64) return bf ? launch_rows<64, true, PREFIX>(ctx, p, grid) : launch_rows<64, false, PREFIX>(ctx, p, grid);
    if (dp == 128) return bf ? launch_rows<128, true, PREFIX>(ctx, p, grid) : launch_rows<128, false, PREFIX>(ctx, p, grid);
    return bf ? launch_rows<256, true, PREFIX>(ctx, p, grid) : launch_rows<256, false, PREFIX>(ctx, p, grid);
}
int launch_attn_rows(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, bool prefix, int64_t grid) {
    return prefix ? by_type<true>(ctx, p, dp, bf, grid) : by_type<false>(ctx, p, dp, bf, grid);
}

}  // namespace trhip
