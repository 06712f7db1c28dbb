// attn.hip -- attention over a paged key/value cache for rows of new tokens: causal, optionally with a sliding window and
// first tokens that stay visible; and behind a prefix that all requests share.
//
//   out[t, head] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  j over the keys the token sees
//
// Here: the kernel of few rows (attn_tokens.hpp), the joining launch, and the call's plan. Many rows: attn_rows.hpp. Both in one
// launch, for batches that have both and for a shared prefix beside its requests' own keys: attn_two.hip.
#include "attn_tokens.hpp"

namespace trhip {
namespace {

template <int DP, bool BF, bool PREFIX> __global__ __launch_bounds__(64 * kTokWaves) void attn_tokens(const AttnArgs p) {
    tokens_of<DP, BF, PREFIX>(p, blockIdx.x, gridDim.x);
}

// Joins the pieces of a tile's rows, and the shared prefix's: a workgroup for `each` rows of a place (workgroups of places that
// hold no tile's first piece end at once). All it does is read the pieces, eight in flight a thread.
template <int DP, bool BF> __global__ __launch_bounds__(256) void attn_join(const AttnArgs p, int tr, int each) {
    constexpr int ST = DP + 2, AT = 8;
    if ((int)blockIdx.x >= p.parts[0]) return;
    const Place t = reinterpret_cast<const Place *>(p.parts + 8)[blockIdx.x];
    const int g = each * blockIdx.y, rows = t.n - g < each ? t.n - g : each;
    if (t.pieces == 0 || rows <= 0) return;
    const int64_t step = (int64_t)p.kv_heads * tr * ST, pstep = (int64_t)p.tokens * p.heads * ST;
    for (int idx = threadIdx.x; idx < rows * (DP / 4); idx += 256) {
        const int r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4, row = t.r0 + g + r, tok = p.by_group(row);
        if (d >= p.dim) continue;
        const float *x = p.part + ((int64_t)blockIdx.x * tr + g + r) * ST;
        const float *pre = p.prefix_part + ((int64_t)(t.q0 + tok) * p.heads + t.head * p.group + (row - tok * p.group)) * ST;
        Join j;
        j.init();
        const int all = t.pieces + p.prefix_splits;
        for (int s0 = 0; s0 < all; s0 += AT) {
            float2 a[AT], b[AT], ml[AT];
#pragma unroll
            for (int u = 0; u < AT; u++) {
                const int s = s0 + u < all ? s0 + u : s0;
                const float *y = s < t.pieces ? x + s * step : pre + (s - t.pieces) * pstep;
                a[u] = *reinterpret_cast<const float2 *>(y + d);
                b[u] = *reinterpret_cast<const float2 *>(y + d + 2);
                ml[u] = *reinterpret_cast<const float2 *>(y + DP);
            }
#pragma unroll
            for (int u = 0; u < AT; u++)
                if (s0 + u < all) j.add(ml[u].x, ml[u].y, a[u].x, a[u].y, b[u].x, b[u].y);
        }
        put4<BF>(p, t.q0, row, t.head, d, j.o, j.l, p.prefix_splits > 0 || t.kv - t.nq + tok >= 0);
    }
}

template <int DP, bool BF> int launch_join(trhip_ctx *ctx, const AttnArgs &p, int tr, int each) {
    hipLaunchKernelGGL((attn_join<DP, BF>), dim3((unsigned)p.part_slots, (unsigned)(tr / each)), dim3(256), 0, ctx->stream, p, tr, each);
    return launch_check(ctx, "attention");
}
// Sixteen rows a workgroup, four where that would leave CUs without one (a chunk of 64 tokens over 16000 keys: 57.0 us, 48.2 with
// four; a prompt of 512: 22.5, 25.0, for its idle workgroups).
int launch_join(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, int tr, int64_t tiles, int cus) {
    const int each = tiles * (tr / 16) < cus ? 4 : 16;
    if (dp == 64) return bf ? launch_join<64, true>(ctx, p, tr, each) : launch_join<64, false>(ctx, p, tr, each);
    if (dp == 128) return bf ? launch_join<128, true>(ctx, p, tr, each) : launch_join<128, false>(ctx, p, tr, each);
    return bf ? launch_join<256, true>(ctx, p, tr, each) : launch_join<256, false>(ctx, p, tr, each);
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

constexpr int kAnyRows = 0x7FFFFFFF;

// Tiles of a batch of these sizes, at most.
int64_t tiles_of(const AttnArgs &p, const AttnCall &c, int tile_rows) {
    int64_t tiles = c.tokens * p.group / tile_rows + c.nreq;
    if (p.row_hi != kAnyRows) {
        const int64_t few = (p.row_hi + tile_rows - 1) / tile_rows * c.nreq;
        tiles = tiles < few ? tiles : few;
    }
    return tiles * p.kv_heads;
}

// The launch's workgroups: as many items as a batch of these sizes can have (find_item), whatever its lengths are. The rounds
// that pieces may take go by the tiles there will be: a tile a request beside longer ones.
int64_t plan_items(AttnArgs &p, const AttnCall &c, int tile_rows, int block, int least) {
    const int64_t tiles = tiles_of(p, c, tile_rows), one = c.nreq * p.kv_heads, usual = p.row_hi != kAnyRows && one < tiles ? one : tiles;
    const int64_t blocks = ((c.max_pages << p.page_log2) + block - 1) / block, most = tiles * ((blocks + least - 1) / least + 1);
    const int64_t k = (2 * usual + p.target - 1) / p.target;
    p.rounds = (int)(k < kMostRounds ? k : kMostRounds);
    p.part_slots = p.rounds * p.target;
    int64_t items = p.part_slots < most ? p.part_slots : most;
    if (tiles > items) items = tiles;
    if (c.prefix_len > 0) p.part_slots = (int)items;
    return items;
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
    p.by_group.of(p.group);
    p.by_heads.of(p.kv_heads);
    p.out_aligned = (reinterpret_cast<uintptr_t>(c.out) % 8 == 0) && c.out_stride % 4 == 0;
    p.arrivals = ctx->arrivals;
    const int cus = ctx->sm_count > 0 ? ctx->sm_count : 256;
    const int64_t rows = c.tokens * p.group;
    // Requests of up to kTokMost rows go to attn_tokens, longer ones to attn_rows, which multiplies 128 rows whatever there are:
    // 64 requests of up to 12 tokens over 2000 keys, 4 heads a kv head, took 72.6 us there, 63.9 here; of up to 24 tokens (96 rows)
    // 79.6 and 80.4. Which there are is known only from the hint, so both are launched unless it (or the sizes) rules one
    // out. Each takes the requests of its own length, or all of them when it is alone.
    const int64_t most_new = c.max_new < c.tokens ? c.max_new : c.tokens;
    const bool tokens_alone = most_new * p.group <= kTokMost, rows_alone = !tokens_alone && c.tokens == c.nreq * most_new;
    AttnArgs pt = p, pr = p;
    pt.target = cus * (dp <= 128 ? 2 : 1);
    pt.row_lo = 0;
    pt.row_hi = tokens_alone ? kAnyRows : kTokMost;
    pr.target = cus * attn_rows_per_cu(dp);
    pr.row_lo = rows_alone ? 0 : kTokMost;
    pr.row_hi = kAnyRows;
    const int tr = attn_rows_tile(), br = attn_rows_block();
    const bool prefix = c.prefix_len > 0;
    // Pieces of long tiles are joined by a launch of their own (a workgroup that joined a tile of 128 rows alone would take
    // longer than the pieces); there are none where the tiles fill the device by themselves. A token's few rows are joined
    // by the last workgroup of their tile, in the same launch, except behind a prefix.
    const int64_t tiles_r = tiles_of(pr, c, tr);
    const bool cut = !tokens_alone && (prefix || tiles_r < pr.target);
    const int64_t grid_t = plan_items(pt, c, kTokRows, kTokBlock, kTokLeast), grid_r = cut ? plan_items(pr, c, tr, br, kRowsLeast) : tiles_r;
    if (grid_t >= ((int64_t)1 << 31) || grid_r >= ((int64_t)1 << 31)) return fail(ctx, TRHIP_ERR_INVALID, "attention: too many rows");
    const int64_t part_t = rows_alone ? 0 : (int64_t)pt.part_slots * kTokRows, part_r = tokens_alone ? 0 : (int64_t)pr.part_slots * tr;
    const int64_t part = (part_t + part_r) * (dp + 2);
    const int64_t places = 8 + 8 * (int64_t)(pt.part_slots > pr.part_slots ? pt.part_slots : pr.part_slots);
    // the prefix: all tokens' rows are one tall product, its keys cut to fill the device
    // (24 tokens of 4 heads behind 20000 keys: 40.8 us as rows, 35.5). Rows of short requests get weights of one term there; with two, 192 x 2
    // tokens behind 30001 keys would take 330 us, not 246, and 32 behind 4096 23.7, not 21.9.
    const bool tall = rows > kTokMost;
    const int ptr = tall ? tr : kTokRows, pbk = tall ? br : kTokBlock;
    const int64_t ptiles = (rows + ptr - 1) / ptr;
    int splits = 0;
    if (prefix) {
        const int64_t nb = (c.prefix_len + pbk - 1) / pbk, items = ptiles * p.kv_heads;
        const int64_t piece = piece_blocks((float)items * (float)nb, (int)items, (int)nb, tall ? pr.target : pt.target, kMostRounds, tall ? kRowsLeast : kTokLeast, tall ? kRowsOver : kTokOver);
        splits = piece >= nb ? 1 : (int)((nb + piece - 1) / piece);
    }
    int st = TRHIP_OK;
    float *ws = static_cast<float *>(workspace(ctx, (size_t)(places + part + (int64_t)splits * c.tokens * c.heads * (dp + 2)) * sizeof(float), &st));
    if (!ws) return st;
    for (AttnArgs *a : {&pt, &pr}) {
        a->part = ws + places + (a == &pr ? part_t * (dp + 2) : 0);
        a->prefix_part = ws + places + part;
        a->prefix_splits = splits;
    }
    const int64_t grid_p = prefix ? ptiles * splits * p.kv_heads : 0;
    if (grid_p + grid_t + grid_r >= ((int64_t)1 << 30)) return fail(ctx, TRHIP_ERR_INVALID, "attention: too many rows");
    pt.parts = prefix ? reinterpret_cast<int *>(ws) : nullptr;
    pr.parts = cut ? reinterpret_cast<int *>(ws) : nullptr;
    // Two kinds of work in one launch: the one waits for memory while the other multiplies. Prompts and tokens take turns in
    // runs of a workgroup a CU, a prefix goes first (its pieces are the long ones), and so do prompts of three times as many tiles
    // as there are tokens', which then fill the prompts' last round (8 prompts of up to 901 with a window of 1024 beside 32
    // tokens: 129 us in turns, 119; 16 prompts of up to 500 beside 16 tokens 120, 113; 2 of up to 4000 beside 32 tokens with up
    // to 6000 keys 387, 397; but 4 of up to 2000 beside 128 tokens with up to 8000 keys, twice as many tiles, 647, 716).
    const bool two = dp <= 128 && (prefix ? !rows_alone : !tokens_alone && !rows_alone);
    bool rows_left = !tokens_alone, tokens_left = !rows_alone;
    if (two && prefix) {
        st = launch_attn_two(ctx, tall ? pr : pt, (int)grid_p, tall ? TwoKind::PrefixRows : TwoKind::PrefixTokens, pt, (int)grid_t, dp, bf, (int)grid_p);
        if (st == TRHIP_OK) st = launch_join(ctx, pt, dp, bf, kTokRows, tiles_of(pt, c, kTokRows), cus);
        tokens_left = false;
    } else if (two) {
        const bool rows_first = c.tokens * p.group / tr >= 3 * c.nreq;
        st = launch_attn_two(ctx, pr, (int)grid_r, TwoKind::Rows, pt, (int)grid_t, dp, bf, rows_first ? (int)grid_r : cus);
        if (st == TRHIP_OK && cut) st = launch_join(ctx, pr, dp, bf, tr, tiles_r, cus);
        return st;
    } else if (prefix) {
        st = tall ? launch_attn_rows(ctx, pr, dp, bf, true, grid_p) : launch_tokens<true>(ctx, pt, dp, bf, grid_p);
    }
    if (st != TRHIP_OK) return st;
    if (tokens_left) {
        st = launch_tokens<false>(ctx, pt, dp, bf, grid_t);
        if (st == TRHIP_OK && prefix) st = launch_join(ctx, pt, dp, bf, kTokRows, tiles_of(pt, c, kTokRows), cus);
        if (st != TRHIP_OK) return st;
    }
    if (rows_left) {
        st = launch_attn_rows(ctx, pr, dp, bf, false, grid_r);
        if (st == TRHIP_OK && cut) st = launch_join(ctx, pr, dp, bf, tr, tiles_r, cus);
    }
    return st;
}

}  // namespace trhip
