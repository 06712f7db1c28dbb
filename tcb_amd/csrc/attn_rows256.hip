// attn_rows256.hip -- the kernel of attention for many rows for heads of 136 to 256 elements, in a file of its own: it is compiled
// with matrix accumulators in architectural registers (build.py), which the narrower ones do by themselves.
#include "attn_rows.hpp"

namespace trhip {

int launch_attn_rows256(trhip_ctx *ctx, const AttnArgs &p, bool bf, bool prefix, int64_t grid) {
    if (prefix) return bf ? launch_rows<256, true, true>(ctx, p, grid) : launch_rows<256, false, true>(ctx, p, grid);
    return bf ? launch_rows<256, true, false>(ctx, p, grid) : launch_rows<256, false, false>(ctx, p, grid);
}

}  // namespace trhip
