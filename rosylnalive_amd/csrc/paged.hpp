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
constexpr int kVTile = 8;

// No page, no slot.
constexpr uint32_t kNone = 0xFFFFFFFFu;

// Requests of one dispatch: every workgroup scans their lengths in LDS.
constexpr uint32_t kMaxRequests = 4096;

inline bool page_ok(uint32_t page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }

// attention_paged shares its work out in units of kUnitKeys keys of one item (a request's rows on one KV head): workgroup w of
// G = min(kGroups, units) takes the units [w units / G, (w + 1) units / G) of all items in order, whatever the lengths are.
// An item that ends in another workgroup than it began in is joined from partials in the workspace: words 0 .. items - 1
// count an item's partials in (zero between launches), then two slots per workgroup hold them: slot 2 w the part of the item
// that w finds begun, slot 2 w + 1 the part of the item that w begins and does not end.
constexpr uint32_t kGroups = 512;
constexpr uint32_t kUnitKeys = 128;
constexpr uint32_t kCols = 16;  // query columns (rows of a request x heads of a group) of an item
constexpr uint64_t slot_words(uint64_t head_dim) { return 2 * kCols + kCols * head_dim; }  // maxima, sums, products

// u32 words of attention_paged's workspace.
inline uint64_t workspace_words(uint64_t requests, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads,
                                uint64_t head_dim) {
    (void)tokens, (void)q_heads;
    const uint64_t counters = (requests * kv_heads + 63) / 64 * 64;
    return counters + 2 * kGroups * slot_words(head_dim);
}

}  // namespace paged
}  // namespace lrm
