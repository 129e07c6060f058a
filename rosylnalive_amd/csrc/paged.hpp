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

// u32 words of attention_paged's workspace.
inline uint64_t workspace_words(uint64_t requests, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads,
                                uint64_t head_dim) {
    (void)requests, (void)tokens, (void)q_heads, (void)kv_heads, (void)head_dim;
    return 64;
}

}  // namespace paged
}  // namespace lrm
