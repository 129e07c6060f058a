// The paged key/value cache: its layout, and the workspace of the attention over it, shared by the kernels
// (kernels_paged.hip), their contract and the C ABI.
#pragma once

#include <cstddef>
#include <cstdint>

namespace lrm {
namespace paged {

// A page holds `page` positions (a power of two, 16 to 256) of every KV head. The key cache is [pages][kv_heads][page]
// [head_dim] and the value cache [pages][kv_heads][page / 8][head_dim][8]: position p of a page at (p / 8) 8 head_dim +
// dim 8 + p % 8 of its head's part. The values' product reads 8 positions of one dim per lane, so with 8 positions
// innermost every such read is 16 bytes, 16 lanes read 256 contiguous ones, and the layout is the same for every page size.

// No page, no slot.
constexpr uint32_t kNone = 0xFFFFFFFFu;

// Requests of one dispatch: every workgroup scans their lengths in LDS.
constexpr uint32_t kMaxRequests = 4096;

inline bool page_ok(uint32_t page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }

// attention_paged shares its work out in units, a block of keys of one item (query columns of one request on one KV head).
// Either every item has workgroups of its own, or workgroup w of G takes the units [w units / G, (w + 1) units / G) of all
// items in order (for tiles weighted, kTileStart); both follow the lengths on the device. An item of several workgroups is joined from partials in the
// workspace, two slots per workgroup: 2 w for the part of an item that w finds begun (or the part of its own), 2 w + 1 for
// the part of the one that it begins and does not end. Before them stand kGroups words, in which the items count their parts
// in where the last one to arrive joins them (word w for the one that w begins; zero between launches), and for the tiles what
// a join in a launch of its own has to know, eight words per workgroup.
constexpr uint32_t kGroups = 512;  // the most workgroups that share out the work
// Items of few columns (a request's rows x the heads of a group up to 16): two workgroups per CU, units of 128 keys.
constexpr uint32_t kRowsGroups = 512, kRowsKeys = 128, kRowsCols = 16;
// Items of many columns: tiles of 32 columns per wave, units of 64 keys, 2048 waves in all (times of calls back to back): workgroups of eight, one per CU, or of
// four, two per CU, so that one's start, end and barriers run beside the other's products, and a single token among the
// chunks holds half as much. Four for heads of 64 (40 mixed requests 31.6 us against 37.8, 3621 rows on 2581 positions 78.5 and
// 80.8), and for heads of 128, whose blocks then have a place less in LDS, where most requests bring few rows (29 requests
// with 3 chunks 24.6 us against 31.9, 48 of up to 8 rows 56.7 and 67.0, 16 21-row ones 31.0 and 31.5; but a prompt of 2048 31.7
// and 29.9, 4096 rows on 28,672 positions 1009 and 954, and with fewer requests 14 of up to 30 rows 16.5 and 13.6). A row's heads
// of a group have to fit a tile.
constexpr uint32_t kTileKeys = 64, kMaxTileCols = 256;
constexpr uint32_t tile_waves(uint64_t requests, uint64_t tokens, uint64_t head_dim, uint64_t group) {
    return group <= 128 && (head_dim == 64 || (requests >= 16 && tokens <= 64 * requests)) ? 4 : 8;
}
// The tiles' split items are joined by their last workgroup where the table holds no more than this many positions, so that
// parts are few, and by a second launch over all CUs otherwise (64-row prompts 5.5 us and 7.7, 41 rows among 24 requests of up
// to 655 positions 15.3 and 17.1, a prompt of 2263 28.3 and 27.8; but 13 rows on 3576 positions 23.8 and 16.8, 24 on 11,275 74 and
// 26: the last one reads the parts alone, 1.5 us each).
constexpr uint32_t kJoinHere = 2048;
constexpr uint32_t tile_cols(uint32_t waves) { return 32 * waves; }
constexpr uint32_t tile_groups(uint32_t waves) { return 2048 / waves; }
// What the start of a tile weighs in even shares of the units, in units: its queries, its first blocks and the end of the tile
// before it (6 against 0: 30 prompts of 300 to 1500 rows 245 us against 257, one of 4096 89 against 93).
constexpr uint32_t kTileStart = 6;
constexpr uint32_t tile_slots(uint32_t waves) { return kGroups + 8 * tile_groups(waves); }  // the word of the first slot
// a slot: per column its maximum, its sum and its products
constexpr uint64_t slot_words(uint64_t cols, uint64_t head_dim) { return cols * (2 + head_dim); }

// u32 words of attention_paged's workspace. The lengths of a launch come from the device, so any launch of a batch may
// split between all its workgroups, however many requests it has: 68 MB for heads of 128 and 34 for heads of 64; one whose
// requests could not together have more than 16 columns on a KV head never takes the tiles, 8.5 and 4.3 MB.
inline uint64_t workspace_words(uint64_t requests, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads,
                                uint64_t head_dim) {
    (void)requests;
    const uint64_t rows = kGroups + 2 * kRowsGroups * slot_words(kRowsCols, head_dim);
    uint64_t tiles = 0;
    for (uint32_t waves : {4u, 8u}) {  // (which of them a dispatch of fewer requests or tokens takes is its own)
        const uint64_t n = tile_slots(waves) + 2 * tile_groups(waves) * slot_words(tile_cols(waves), head_dim);
        tiles = n > tiles ? n : tiles;
    }
    return kv_heads && tokens * (q_heads / kv_heads) <= kRowsCols ? rows : (tiles > rows ? tiles : rows);
}

}  // namespace paged
}  // namespace lrm
