// attn4_image.hpp -- long requests' keys of a 4-bit cache in 16 bits (attn4_image.hip).
#pragma once

#include "trhip_internal.hpp"

namespace trhip {

struct Image4 {
    const uint8_t *k, *v;
    uint16_t *out_k, *out_v;  // planes [long request][max_pages][head][page][dim], as a 16-bit cache's
    int *out_table;           // [request][max_pages]: page numbers in them
    const int *q_start, *kv_len, *table;
    int64_t max_pages, pages;
    int nreq, tokens, group, heads, dim, page_log2, row_lo, window, sinks;
    bool bf;
};
// Opens the keys that the first `most` requests of more than row_lo rows see.
int launch_attn4_image(trhip_ctx *ctx, const Image4 &p, int most);

}  // namespace trhip
