// attn_plan.hpp -- how many workgroups a launch of attention work items needs (attn.hip, attn4.hip).
#pragma once

#include "attn_common.hpp"

namespace trhip {
namespace {

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
}  // namespace trhip
