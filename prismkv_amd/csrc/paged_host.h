// Host checks of the paged cache's C entries, alike in all of them.
#pragma once

#include "paged.h"
#include "prismkv_hip.h"

namespace prismkv {
namespace {

inline PageDiv page_div(int page_size) {
  int log = 0;
  while ((1ll << log) < page_size) ++log;
  const int shift = 31 + log;
  return PageDiv{(unsigned)(((1ull << shift) + page_size - 1) / page_size), shift};
}

// Bytes of an element of the rows that go in and out; of the pages (bytes of codes in
// 4 bits); elements of a page's row.
inline int element_bytes(int dtype) { return (dtype & 15) == kFp32 ? 4 : 2; }
inline int page_element_bytes(int dtype) { return dtype >= kFour ? 1 : element_bytes(dtype); }
inline int page_row(const prismkv_paged_cache& c) { return c.dtype >= kFour ? c.head_dim / 2 : c.head_dim; }

// The second cache's lengths, tokens seen, scores and positions are all the first's or
// lie apart from all of them: a launch reads the first's while it writes the second's.
inline bool results_fit(const prismkv_paged_cache& c, const prismkv_paged_cache& to) {
  if (to.lengths == c.lengths && to.seen == c.seen && to.scores == c.scores && to.positions == c.positions) return true;
  const uint64_t few = 4ull * c.sequences, many = few * c.kv_heads * c.page_size * c.max_pages;
  const uint64_t from[4] = {c.lengths, c.seen, c.scores, c.positions}, into[4] = {to.lengths, to.seen, to.scores, to.positions};
  const uint64_t size[4] = {few, few, many, many};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (from[i] && into[j] && from[i] < into[j] + size[j] && into[j] < from[i] + size[i]) return false;
  return true;
}

// The cache and where its results go, checked alike by every entry point: rows,
// heads and pages lie at 16-byte multiples, and a page's last row within 2^32
// 16-byte units.  0, or the code to return.
inline int check_cache(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, bool scored) {
  if (!cache || !into) return kBadSize;
  const prismkv_paged_cache& c = *cache;
  const prismkv_paged_cache& to = *into;
  const bool four = c.dtype == (kFour | kBf16) || c.dtype == (kFour | kFp16);
  if (!four && (c.dtype < kBf16 || c.dtype > kFp32)) return kBadMode;
  if (c.sequences < 1 || c.sequences > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.page_size < 1 ||
      c.max_pages < 1 || c.pages < 1 || c.pages > INT32_MAX)
    return kBadSize;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  if (slots > (1 << 30) || slots * c.sequences > INT32_MAX) return kBadSize;
  const int64_t es = page_element_bytes(c.dtype), limit = 1ll << 36;  // bytes
  if (c.page_stride < 0 || c.head_stride < 0 || c.slot_stride < page_row(c)) return kBadSize;
  if (c.page_stride > limit || c.head_stride > limit || c.slot_stride > limit) return kBadSize;
  if ((c.page_stride * es | c.head_stride * es | c.slot_stride * es) & 15) return kBadSize;
  if (c.page_stride * es > limit / c.pages || c.slot_stride * es > limit / c.page_size) return kBadSize;
  if ((c.pages - 1) * c.page_stride * es + (c.page_size - 1) * c.slot_stride * es >= limit) return kBadSize;
  if (to.k != c.k || to.v != c.v || to.table != c.table || to.pages != c.pages || to.page_stride != c.page_stride ||
      to.head_stride != c.head_stride || to.slot_stride != c.slot_stride || to.sequences != c.sequences ||
      to.kv_heads != c.kv_heads || to.head_dim != c.head_dim || to.page_size != c.page_size ||
      to.max_pages != c.max_pages || to.dtype != c.dtype)
    return kBadSize;
  if (!c.k || !c.v || !c.table || !c.lengths || !to.lengths || !c.err) return kBadSize;
  if ((c.k | c.v) & 15 || c.err & 7 ||
      (c.table | c.lengths | c.seen | c.scores | c.positions | to.lengths | to.seen | to.scores | to.positions) & 3)
    return kBadSize;
  if (four) {  // the scales: a row's D / 32 bytes are read together
    const int64_t row = c.head_dim / 32;
    if (!c.k_scales || !c.v_scales || (c.k_scales | c.v_scales) % row) return kBadSize;
    if (to.k_scales != c.k_scales || to.v_scales != c.v_scales || to.scale_page_stride != c.scale_page_stride ||
        to.scale_head_stride != c.scale_head_stride || to.scale_slot_stride != c.scale_slot_stride)
      return kBadSize;
    if (c.scale_page_stride < 0 || c.scale_head_stride < 0 || c.scale_slot_stride < row) return kBadSize;
    const int64_t most = 1ll << 33;  // (a row's place is counted in 32 bits)
    if (c.scale_page_stride > most / c.pages || c.scale_head_stride > most || c.scale_slot_stride > most / c.page_size ||
        (c.pages - 1) * c.scale_page_stride + (c.page_size - 1) * c.scale_slot_stride >= most)
      return kBadSize;
    if ((c.scale_page_stride | c.scale_head_stride | c.scale_slot_stride) % row) return kBadSize;
  }
  const bool some = c.seen || c.scores || c.positions || to.seen || to.scores || to.positions;
  const bool all = c.seen && c.scores && c.positions && to.seen && to.scores && to.positions;
  return some != all || (scored && !all) || !results_fit(c, to) ? kBadSize : 0;
}

}  // namespace
}  // namespace prismkv
