// attn_two.hip -- two kinds of attention work in one launch, two workgroups a CU: few rows, which wait for the cache's bytes,
// beside many rows (a batch of prompts and tokens) or a shared prefix under its requests' own keys. One after the other, each
// leaves half the device idle (32 tokens behind 4096 shared keys: 32 us in two launches, 24 in this when it came in). The kinds take turns in
// runs of `turn` workgroups, so that with as many as there are CUs each CU starts with one of either.
#include "attn_rows.hpp"
#include "attn_tokens.hpp"

namespace trhip {
namespace {

static_assert(RowsShape<128>::THREADS == 64 * kTokWaves && RowsShape<64>::PER_CU == 2 && RowsShape<128>::PER_CU == 2, "one launch shape");

template <int DP, bool BF, TwoKind KIND>
__global__ __launch_bounds__(64 * kTokWaves, 2) void attn_two(const AttnArgs a, int na, const AttnArgs b, int nb, int turn) {
    const int runs = (na + turn - 1) / turn, other = (nb + turn - 1) / turn, both = runs < other ? runs : other;  // runs of either
    const int run = blockIdx.x / turn, in = blockIdx.x - run * turn;
    const bool first = run < 2 * both ? run % 2 == 0 : runs > other;
    const int at = (run < 2 * both ? run / 2 : run - both) * turn + in;
    if (first) {
        if (at >= na) return;
        if constexpr (KIND == TwoKind::PrefixTokens) tokens_of<DP, BF, true>(a, at, na);
        else rows_of_tile<DP, BF, KIND == TwoKind::PrefixRows>(a, at, na);
    } else {
        if (at >= nb) return;
        tokens_of<DP, BF, false>(b, at, nb);
    }
}

template <int DP, bool BF, TwoKind KIND>
int launch(trhip_ctx *ctx, const AttnArgs &a, int na, const AttnArgs &b, int nb, int turn) {
    constexpr int BYTES = TokLds<DP>::BYTES > RowsShape<DP>::BYTES ? TokLds<DP>::BYTES : RowsShape<DP>::BYTES;
    const int st = allow_dyn_lds(ctx, reinterpret_cast<const void *>(attn_two<DP, BF, KIND>), BYTES, "attention");
    if (st != TRHIP_OK) return st;
    const int runs = (na + turn - 1) / turn + (nb + turn - 1) / turn;
    hipLaunchKernelGGL((attn_two<DP, BF, KIND>), dim3((unsigned)(runs * turn)), dim3(64 * kTokWaves), BYTES, ctx->stream, a, na, b, nb, turn);
    return launch_check(ctx, "attention");
}
template <int DP, bool BF>
int by_kind(trhip_ctx *ctx, const AttnArgs &a, int na, TwoKind kind, const AttnArgs &b, int nb, int turn) {
    if (kind == TwoKind::Rows) return launch<DP, BF, TwoKind::Rows>(ctx, a, na, b, nb, turn);
    if (kind == TwoKind::PrefixRows) return launch<DP, BF, TwoKind::PrefixRows>(ctx, a, na, b, nb, turn);
    return launch<DP, BF, TwoKind::PrefixTokens>(ctx, a, na, b, nb, turn);
}

}  // namespace

int launch_attn_two(trhip_ctx *ctx, const AttnArgs &a, int na, TwoKind kind, const AttnArgs &b, int nb, int dp, bool bf, int turn) {
    if (dp == 64) return bf ? by_kind<64, true>(ctx, a, na, kind, b, nb, turn) : by_kind<64, false>(ctx, a, na, kind, b, nb, turn);
    return bf ? by_kind<128, true>(ctx, a, na, kind, b, nb, turn) : by_kind<128, false>(ctx, a, na, kind, b, nb, turn);
}

}  // namespace trhip
