// Host side of the prefill's entry points: the size of a launch and of its
// scratch.
#pragma once

#include "prefill_kernel.h"

namespace tmopt {
namespace {

// Work-groups of one level of the grid: HKV * items per head, rounded up to
// whole XCD rounds.
int64_t level_wgs(int HKV, int BQ, int S, int max_seqlen) {
  const int64_t items = (int64_t)S * ((max_seqlen + BQ - 1) / BQ);
  if (HKV <= 8 && 8 % HKV == 0) return 8 * ((items + 8 / HKV - 1) / (8 / HKV));
  return HKV * items;
}

// Levels of a launch (1: keys are not split): split where the items are at
// most half the compute units and a query may see `min_tiles` tiles of keys
// (`max_keys` keys at most). Between half and all of them the pieces' start
// and merge cost more than the idle units give (one 777-token prompt, 200
// items: 49.9 us per call in one launch, 67.5 us split); a larger grid fills
// the chip by itself, its heaviest items first. Without cached context the
// longest run's length is known and its blocks see half of it on average, so
// the line lies higher (2000 tokens, 16 query heads, 32 tiles: 46.4 us in one
// launch, 51.4 us split); with one, the row width of the block table is only a
// bound, and the device decides item by item.
int split_levels(int64_t n_base, int BQ, int64_t max_keys, int window,
                 int min_tiles) {
  const int cus = device_cus();
  if (2 * n_base > cus) return 1;
  int64_t keys = max_keys;
  if (window > 0 && keys > (int64_t)window + BQ + kBN) keys = window + BQ + kBN;
  const int64_t tiles = (keys + kBN - 1) / kBN;
  if (tiles < min_tiles) return 1;
  int64_t n = 2 * cus / n_base;
  if (n > 64) n = 64;
  if (n > tiles / kMinPiece + 1) n = tiles / kMinPiece + 1;
  return (int)n;
}

// The same from the arguments of a launch: keys a query may see, by the run's
// own length or the row width of a block table (with a ring, which is read
// under a window, the window bounds them).
int split_levels(int64_t n_base, int BQ, int max_seqlen, int64_t bt_stride,
                 int table_wrap, int window) {
  if (bt_stride <= 0)
    return split_levels(n_base, BQ, max_seqlen, window, 48);
  const int64_t keys =
      table_wrap > 0 ? 0x3fffffff : bt_stride * kPage + max_seqlen;
  return split_levels(n_base, BQ, keys, window, kMinSplit);
}

constexpr int64_t kSlotBytes = (256 * kD + 256) * sizeof(float);
int64_t workspace_bytes_of(int levels, int64_t n_base) {
  return levels * n_base * kSlotBytes + ((n_base * 4 + 15) & ~(int64_t)15);
}

// Query heads per work-group: the largest of 8, 4, 2, 1 dividing HQ/HKV; a
// ratio above it runs as several scheduled heads per stored KV head (its keys
// then load once per group of that many query heads).
int query_group(int ratio) {
  return ratio % 8 == 0 ? 8 : ratio % 4 == 0 ? 4 : ratio % 2 == 0 ? 2 : 1;
}

}  // namespace
}  // namespace tmopt
