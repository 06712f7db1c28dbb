// attn.hip -- attention over a paged key/value cache for rows of new tokens: causal, optionally with a sliding window and
// first tokens that stay visible; and behind a prefix that all requests share.
//
//   out[t, head] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  j over the keys the token sees
//
// attn_tokens: a workgroup takes a tile of up to 32 rows (the heads of a few tokens of one request, attn_common.hpp) and
// a piece of its keys. Its four waves hold all rows each and take every fourth block of 32 keys, which they copy into
// LDS rings of their own (no barrier until the end), then join their running maxima and sums. A token step reads every
// key and value once, so what bounds it is the cache's bytes; the piece's length deals them over all CUs. Pieces of one
// tile go to the workspace, and the workgroup that finishes last joins them.
#include "attn_common.hpp"

namespace trhip {
namespace {

constexpr int kTokRows = 32, kTokBlock = 32, kTokWaves = 4;

template <int DP> struct TokLds {
    static constexpr int SLOT = 32 * DP * 2;  // 32 keys or values
    static constexpr int SLOTS = DP == 64 ? 8 : DP == 128 ? 4 : 2;
    static constexpr int OSTRIDE = DP + 4;  // floats between rows of a wave's results
    static constexpr int RING = SLOT * SLOTS, OUT = 32 * OSTRIDE * 4;
    static constexpr int WAVE = RING > OUT ? RING : OUT;
    static constexpr int BYTES = kTokWaves * (WAVE + 32 * 8) + 16;
};

// Joins nsplit pieces of a row (agent-coherent loads: other workgroups of this launch wrote them) and the prefix's (an earlier launch).
template <int DP, int TR, bool BF>
__device__ __forceinline__ void join_tile(const AttnArgs &p, const Item &it, int r0, int n, int threads) {
    constexpr int ST = DP + 2;
    for (int idx = threadIdx.x; idx < n * (DP / 4); idx += threads) {
        const int r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4, row = r0 + r, t = row / p.group;
        if (d >= p.dim) continue;
        Join j;
        j.init(p.scale);
        const float *src = p.part + ((int64_t)it.first * TR + r) * ST;
        const int64_t step = (int64_t)p.kv_heads * TR * ST;
        for (int s0 = 0; s0 < it.nsplit; s0 += 4) {
            float2 a[4], b[4], ml[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float *x = src + (s0 + u < it.nsplit ? s0 + u : s0) * step;
                a[u] = agent_load(x + d);
                b[u] = agent_load(x + d + 2);
                ml[u] = agent_load(x + DP);
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (s0 + u < it.nsplit) j.add(ml[u].x, ml[u].y, a[u].x, a[u].y, b[u].x, b[u].y);
        }
        const float *pre = p.prefix_part + ((int64_t)(it.q0 + t) * p.heads + it.head * p.group + (row - t * p.group)) * ST;
        for (int s = 0; s < p.prefix_splits; s++) {
            const float *x = pre + (int64_t)s * p.tokens * p.heads * ST;
            const float2 a = *reinterpret_cast<const float2 *>(x + d), b = *reinterpret_cast<const float2 *>(x + d + 2);
            const float2 ml = *reinterpret_cast<const float2 *>(x + DP);
            j.add(ml.x, ml.y, a.x, a.y, b.x, b.y);
        }
        put4<BF>(p, it.q0, row, it.head, d, j.o, j.l, p.prefix_splits > 0 || it.kv - it.nq + t >= 0);
    }
}

// Partial results are written: whether this workgroup is the last of its tile's pieces.
__device__ __forceinline__ bool last_piece(const AttnArgs &p, const Item &it, int *flag) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this thread's stores have completed
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (it.nsplit == 1) return true;
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(&p.arrivals[it.first], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                          (uint32_t)(it.nsplit - 1);
        if (last) __hip_atomic_store(&p.arrivals[it.first], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    return *flag != 0;
}

// PREFIX: rows are all tokens' and keys the shared prefix's; results go to prefix_part.
template <int DP, bool BF, bool PREFIX> __global__ __launch_bounds__(64 * kTokWaves) void attn_tokens(const AttnArgs p) {
    using L = TokLds<DP>;
    extern __shared__ __attribute__((aligned(1024))) uint4 smem[];  // nothing else is shared: the rows' swizzle needs them aligned
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), wg = blockIdx.x;
    Item it;
    const int *table;
    int keys;
    if (PREFIX) {
        const int x = wg / p.kv_heads;
        it.head = wg - x * p.kv_heads;
        it.tile = x / p.prefix_splits;
        it.split = x - it.tile * p.prefix_splits;
        it.nsplit = p.prefix_splits;
        it.q0 = 0;
        it.nq = p.tokens;
        it.kv = it.first = 0;
        table = p.prefix_table;
        keys = p.prefix_len;
    } else {
        if (!find_item<kTokRows, kTokBlock, kTokWaves>(p, wg, it)) return;
        table = p.table + (int64_t)it.req * p.max_pages;
        keys = it.kv;
    }
    const int r0 = it.tile * kTokRows, left = it.nq * p.group - r0, n = left < kTokRows ? left : kTokRows;
    Rows rw;
    if (PREFIX) rw = {keys - 1, 0, keys - 1, keys - 1, 0, 0, 0};
    else rw = rows_of(p, r0, n, it.nq, keys);
    const Span sp = span_of<kTokBlock>(rw.hi_max, rw.lo_min, rw.sinks);
    const int nb = sp.count(), piece = (nb + it.nsplit - 1) / it.nsplit;
    const int b0 = it.split * piece, b1 = b0 + piece < nb ? b0 + piece : nb;
    const bool mixed = rw.hi_min != rw.hi_max || rw.lo_min != rw.lo_max;  // some rows see keys that others do not

    const uint32_t ring = lds_addr(smem) + w * L::WAVE;
    Lanes16<DP> lanes;
    lanes.init(p.dim);
    uint4 q[DP / 16];
    load_q<DP>(p, q, it.q0, r0, n, it.head);

    auto key_of = [&](int b) { return 32 * sp.block(b); };
    auto pieces = [&](int b, Piece16 (&s)[2]) {  // past the last block: nothing but zeros
        const int t = b < b1 ? key_of(b) : 0, hi = b < b1 ? rw.hi_max : -1;
#pragma unroll
        for (int i = 0; i < 2; i++) s[i] = piece16(p, table, it.head, t + 16 * i, hi, rw.lo_min, rw.sinks);
    };
    auto copy_k = [&](const Piece16 (&s)[2], int slot) {
#pragma unroll
        for (int i = 0; i < 2; i++) lanes.copy(s[i].k, ring + slot * L::SLOT + i * (L::SLOT / 2), s[i].ha, s[i].hb);
    };
    auto copy_v = [&](const Piece16 (&s)[2], int slot) {
#pragma unroll
        for (int i = 0; i < 2; i++) lanes.copy(s[i].v, ring + slot * L::SLOT + i * (L::SLOT / 2), s[i].ha, s[i].hb);
    };
    constexpr int D = L::SLOTS / 2, AHEAD = (L::SLOTS - 1) * (DP / 16);
    Piece16 s[2];
#pragma unroll
    for (int i = 0; i < D; i++) {
        pieces(b0 + w + i * kTokWaves, s);
        copy_k(s, 2 * i);
        copy_v(s, 2 * i + 1);
    }
    Acc<DP> A;
    A.init();
    int slot = 0;
    for (int b = b0 + w; b < b1; b += kTokWaves) {
        const int t = key_of(b);
        pieces(b + D * kTokWaves, s);
        wait_vmcnt(AHEAD);
        a16f x[1];
        x[0] = scores<DP, BF>(ring + slot * L::SLOT, q);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
        copy_k(s, slot);
        const bool all = all_see(rw, t, 32);
        if (!all) mask(x[0], rw, t);
        softmax_step<DP, 1>(A, x, p.scale);
        wait_vmcnt(AHEAD);
        const uint32_t v = ring + (slot + 1) * L::SLOT;
        if (!all && mixed && odd_values<DP, BF>(v)) values_one_by_one<DP, BF>(A.o, x[0], v, rw.hi, rw.lo, rw.sinks, t);
        else values<DP, BF, true>(A.o, x[0], v);
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
        const int r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4, row = r0 + r, t = row / p.group;
        if (d >= p.dim) continue;
        Join j;
        j.init(p.scale);
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
            float *dst = p.part + ((int64_t)wg * kTokRows + r) * (DP + 2);
            agent_store(dst + d, j.o[0], j.o[1]);
            agent_store(dst + d + 2, j.o[2], j.o[3]);
            if (d == 0) agent_store(dst + DP, j.m, j.l);
        }
    }
    if (direct || PREFIX) return;
    if (last_piece(p, it, reinterpret_cast<int *>(ml + kTokWaves * 32))) join_tile<DP, kTokRows, BF>(p, it, r0, n, 64 * kTokWaves);
}

template <int DP, bool BF, bool PREFIX> int launch_tokens(trhip_ctx *ctx, const AttnArgs &p, int64_t grid) {
    const void *fn = reinterpret_cast<const void *>(attn_tokens<DP, BF, PREFIX>);
    const int st = allow_dyn_lds(ctx, fn, TokLds<DP>::BYTES, "attention");
    if (st != TRHIP_OK) return st;
    hipLaunchKernelGGL((attn_tokens<DP, BF, PREFIX>), dim3((unsigned)grid), dim3(64 * kTokWaves), TokLds<DP>::BYTES,
                       ctx->stream, p);
    return launch_check(ctx, "attention");
}

template <bool PREFIX> int launch_tokens(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, int64_t grid) {
    if (dp == 64) return bf ? launch_tokens<64, true, PREFIX>(ctx, p, grid) : launch_tokens<64, false, PREFIX>(ctx, p, grid);
    if (dp == 128) return bf ? launch_tokens<128, true, PREFIX>(ctx, p, grid) : launch_tokens<128, false, PREFIX>(ctx, p, grid);
    return bf ? launch_tokens<256, true, PREFIX>(ctx, p, grid) : launch_tokens<256, false, PREFIX>(ctx, p, grid);
}

}  // namespace

int launch_attn(trhip_ctx *ctx, const trhip_kv *kv, const AttnCall &c) {
    const int dp = kv->dim <= 64 ? 64 : kv->dim <= 128 ? 128 : 256;
    const bool bf = kv->dtype == TRHIP_BF16;
    AttnArgs p = {};
    p.q = static_cast<const uint16_t *>(c.q);
    p.out = static_cast<uint16_t *>(c.out);
    p.q_stride = c.q_stride;
    p.out_stride = c.out_stride;
    p.k = static_cast<const uint8_t *>(kv->k);
    p.v = static_cast<const uint8_t *>(kv->v);
    p.head_bytes = kv->page * kv->dim * 2;
    p.page_bytes = (int64_t)p.head_bytes * kv->heads;
    p.npages = kv->pages;
    p.page_log2 = __builtin_ctz((unsigned)kv->page);
    p.table = c.table;
    p.max_pages = c.max_pages;
    p.q_start = c.q_start;
    p.kv_len = c.kv_len;
    p.prefix_table = c.prefix_table;
    p.prefix_len = (int)c.prefix_len;
    p.nreq = (int)c.nreq;
    p.tokens = (int)c.tokens;
    p.heads = c.heads;
    p.kv_heads = kv->heads;
    p.group = c.heads / kv->heads;
    p.dim = kv->dim;
    p.window = (int)c.window;
    p.sinks = (int)c.sinks;
    p.scale = c.scale * 1.44269504088896341f;
    p.q_aligned = (reinterpret_cast<uintptr_t>(c.q) % 16 == 0) && c.q_stride % 8 == 0;
    p.out_aligned = (reinterpret_cast<uintptr_t>(c.out) % 8 == 0) && c.out_stride % 4 == 0;
    p.target = 2 * (ctx->sm_count > 0 ? ctx->sm_count : 256);
    p.row_lo = 0;
    p.row_hi = 0x7FFFFFFF;
    p.arrivals = ctx->arrivals;
    // workgroups: every tile of rows once, and as many again as pieces may be cut (find_item)
    const int64_t rows = c.tokens * p.group, tiles = rows / kTokRows + c.nreq;
    int64_t grid = tiles * p.kv_heads;
    p.split_ok = grid + p.target + p.kv_heads <= trhip_ctx::kArrivalSlots;
    if (p.split_ok) grid += p.target + p.kv_heads;
    if (grid >= ((int64_t)1 << 31)) return fail(ctx, TRHIP_ERR_INVALID, "attention: too many rows");
    const int64_t ptiles = (rows + kTokRows - 1) / kTokRows;
    if (p.prefix_len > 0) {
        const int64_t nb = (p.prefix_len + kTokBlock - 1) / kTokBlock, items = ptiles * p.kv_heads;
        int64_t s = (p.target + items - 1) / items;
        if (s > (nb + kTokWaves - 1) / kTokWaves) s = (nb + kTokWaves - 1) / kTokWaves;
        const int64_t piece = (nb + s - 1) / s;
        p.prefix_splits = (int)((nb + piece - 1) / piece);
    }
    const bool parts = p.split_ok || p.prefix_splits > 0;
    const int64_t part = parts ? grid * kTokRows * (dp + 2) : 0;
    const int64_t pre = (int64_t)p.prefix_splits * c.tokens * c.heads * (dp + 2);
    if (part + pre > 0) {
        int st = TRHIP_OK;
        p.part = static_cast<float *>(workspace(ctx, (size_t)(part + pre) * sizeof(float), &st));
        if (!p.part) return st;
        p.prefix_part = p.part + part;
    }
    if (p.prefix_len > 0) {
        const int st = launch_tokens<true>(ctx, p, dp, bf, ptiles * p.prefix_splits * p.kv_heads);
        if (st != TRHIP_OK) return st;
    }
    return launch_tokens<false>(ctx, p, dp, bf, grid);
}

}  // namespace trhip
