// How the rows kernel of the paged attention (fa_paged_sm100.cuh) shares out its work: ONE list of key tiles over all (sequence, KV head,
// row tile) items, cut into equal runs.  The lengths are known on the device only, so every block works its run out from them.
// Shared by the kernels and a test on the CPU.
#pragma once

#include <stdint.h>

#include "fast_div.h"

namespace hb {

// Keys of a tile, what a warp works through at a time: 8 KB of codes either way.  us with 32 | 64 keys at D 64: B40 Hq12, one token, 900 to 1777 keys
// 30.6 | 25.7; B1 Hq32 Hkv8, 20000 keys 21.3 | 15.0; B24 Hq32 Hkv8, four tokens 27.6 | 26.4; B128 Hq16, 100 keys (two tiles that meet) 19.0 | 22.0.
HB_HD constexpr int paged_tile(int head_dim) { return head_dim == 128 ? 32 : 64; }
constexpr int kPagedWarps = 4;   // of a block; they take the tiles of its run in turn

// What a run pays for an item that it starts or goes on with, in tiles of the list: its queries, the meeting of the warps, the store
// (about 5000 cycles, and a tile takes a warp 3000).  An item has so many places in front of its tiles; a run that ends among
// them leaves the item to the next one.
constexpr int kPagedItemCost = 6;

// Key tiles of an item with `len` keys (an item without keys has a tile all the same: somebody has to write its rows).
HB_HD int paged_tiles(int len, int tile = 32) { return len <= 0 ? 1 : static_cast<int>((static_cast<unsigned>(len) + tile - 1) / tile); }
HB_HD int paged_places(int tiles) { return tiles + kPagedItemCost; }
HB_HD int paged_row_tiles(int n, int group, int rows) {
  return static_cast<int>((static_cast<long long>(n) * group + rows - 1) / rows);
}
// Of `blocks` blocks those that get a run: no run is shorter than a tile for every warp.
HB_HD int paged_runs(long long total, int blocks) {
  const long long most = (total + kPagedWarps - 1) / kPagedWarps;
  return static_cast<int>(most < blocks ? (most < 1 ? 1 : most) : blocks);
}
// a / b; 32-bit where both fit, which takes a fraction of the time
HB_HD long long paged_div(long long a, int b) {
  return (a >> 31) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
HB_HD long long paged_begin(long long total, int runs, int w) {  // total < 2^48, runs < 2^12
  const long long per = paged_div(total, runs);
  return per * w + paged_div((total - per * runs) * w, runs);
}
// a / b for any a and b that fit
HB_HD long long paged_div64(long long a, long long b) {
  return ((a | b) >> 31) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// The run of place t: the last w with begin(w) = floor(w total / runs) <= t.
HB_HD int paged_run_of(long long total, int runs, long long t) { return static_cast<int>(paged_div64((t + 1) * runs - 1, total)); }

}  // namespace hb
