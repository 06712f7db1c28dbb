// attn_rows.hip -- attention over a paged cache for many rows: the launch, and the kernel for heads of up to 128 elements.
#include "attn_rows.hpp"

namespace trhip {

int attn_rows_per_cu(int dp) { return dp == 256 ? RowsShape<256>::PER_CU : RowsShape<128>::PER_CU; }
int attn_rows_tile() { return RowsShape<128>::TR; }
int attn_rows_block() { return RowsShape<128>::BK; }

template <bool PREFIX> static int by_type(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, int64_t grid) {
    if (dp == 64) return bf ? launch_rows<64, true, PREFIX>(ctx, p, grid) : launch_rows<64, false, PREFIX>(ctx, p, grid);
    return bf ? launch_rows<128, true, PREFIX>(ctx, p, grid) : launch_rows<128, false, PREFIX>(ctx, p, grid);
}
int launch_attn_rows(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, bool prefix, int64_t grid) {
    if (dp == 256) return launch_attn_rows256(ctx, p, bf, prefix, grid);
    return prefix ? by_type<true>(ctx, p, dp, bf, grid) : by_type<false>(ctx, p, dp, bf, grid);
}

}  // namespace trhip
