// How the work of a prompt is cut into items, by the device from the lengths, and how
// many there can be, by the host from the sizes: plain C++, so that the two can be held
// against each other without a device.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIP__
#define PRISMKV_BOTH __host__ __device__ __forceinline__
#else
#define PRISMKV_BOTH inline
#endif

namespace prismkv {
namespace {

constexpr int kTileRows = 128;  // rows of the queries' matrix, of one KV head
// Keys and values that are staged at a time, by the bytes of a row in LDS.
constexpr int tile_tokens(int row_bytes) { return row_bytes > 256 ? 32 : 64; }

// The work of all tiles is cut so that no item is more than 1 / 2^kItemsLog of it, but
// no item is less than kLeastTiles tiles of keys.  Twice as many items are slower (2048
// rows of 8 x 4 heads 92 us against 60, 48 rows over 65000 slots 116 against 94).  A sequence
// is cut only where that saves its longest tile more tiles of keys than the states and
// their join take: cut_saves and one for every cut_tiles tiles of rows (16 rows over 1016
// slots cut 16 us, whole 28; 1500 rows cut 61, whole 45; 64 x 64 rows over 2000 slots each 73
// and 61).  A tile of fp32 takes longer (300 rows cut 38 us, whole 56; 1000 rows of head_dim 64
// cut 88, whole 80).
constexpr int kItemsLog = 9, kLeastTiles = 4;
constexpr int cut_saves(bool fp32) { return fp32 ? 2 : 4; }
constexpr int cut_tiles(bool fp32) { return fp32 ? 24 : 16; }

// Tiles of keys of a work item at most, and of a sequence that is not cut.
struct PromptPlan {
  int per_item, whole;
  // Of how many chunks a sequence's longest tile has.
  PRISMKV_BOTH int chunks(int key_tiles) const {
    return key_tiles > whole ? (key_tiles + per_item - 1) / per_item : 1;
  }
};

// work: the sum of tiles of rows times tiles of keys of all sequences and KV heads, `tiles`
// those of rows.  (Sequences have fewer than 2^26 tiles of keys: an item of as many cuts
// nothing.  tiles < 2^24.)
PRISMKV_BOTH PromptPlan prompt_cuts(uint64_t work, int tiles, bool fp32) {
  const uint64_t share = (work >> kItemsLog) + 1;
  const int per_item = (int)(share < kLeastTiles ? kLeastTiles : share < (1u << 26) ? share : 1u << 26);
  return PromptPlan{per_item, per_item + cut_saves(fp32) + tiles / cut_tiles(fp32)};
}

// Tiles of rows of one KV head at most, however the rows are dealt to the sequences.
inline int64_t most_tiles(int64_t rows, int sequences, int group) {
  return rows * group / kTileRows + (sequences < rows ? sequences : rows);
}

// Work items, states and cut tiles of a launch at most; bytes of the states.
struct PromptLayout {
  int64_t items, states, cut_tiles;
  size_t bytes;
};

inline PromptLayout prompt_layout(int64_t rows, int sequences, int kv_heads, int group, int head_dim, int64_t slots,
                                  int row_bytes, bool fp32) {
  PromptLayout l;
  const int tokens = tile_tokens(row_bytes);
  const int64_t tiles = most_tiles(rows, sequences, group), key_tiles = (slots + tokens - 1) / tokens;
  const int64_t all = 1ll << kItemsLog;
  // A sequence that is cut has most = ceil(x) <= 2x chunks a tile, x > 1 its share of
  // an item: 2 all of them at most.
  const int64_t full = tiles * kv_heads * ((key_tiles + kLeastTiles - 1) / kLeastTiles);
  // Never cut: few slots; one sequence whose tiles are as many as the items are to be.
  const bool whole = key_tiles <= kLeastTiles + cut_saves(fp32) ||
                     (sequences == 1 && (rows * group + kTileRows - 1) / kTileRows * kv_heads >= all);
  l.items = (whole ? 0 : all) + tiles * kv_heads;
  // (powers of two, so that workspaces are of few sizes)
  l.states = whole || full < 1 ? 0 : 1;
  while (l.states && l.states < full && l.states < 2 * all) l.states *= 2;
  l.cut_tiles = whole ? 0 : tiles * kv_heads < all ? tiles * kv_heads : all;
  l.bytes = (size_t)l.states * kTileRows * (head_dim + 2) * sizeof(float);
  return l;
}

}  // namespace
}  // namespace prismkv
