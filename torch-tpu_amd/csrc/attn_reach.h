// Which keys a tile of attention's rows goes over, and which of them it reads.  Plain arithmetic, the same on the device and on the host, where a
// test compares it with what every row sees.
#pragma once

namespace moe {

// Without a window units 0 .. u of keys; with one the units that hold the first tokens and then those from the lowest key on that one of the
// tile's rows sees in its window.  Of these only first tokens and keys from the lowest on are read: in place of one between them the lowest, which
// is on its way anyway.  (64 single tokens in a window of 1024 with 4 first ones, units of 128: 37.2 us, 41.4 with all ten units read whole.)
struct AttnReach {
  int units, first, skip;              // in all; of the first tokens; left out behind them
  int every;                           // every row of the tile sees keys from here on (up to where the new tokens begin)
  int head, low;                       // first tokens, and the lowest key of a window
  constexpr int unit(int c) const { return c + (c >= first ? skip : 0); }
  constexpr int read(int key) const { return key < head ? key : key > low ? key : low; }
};

// Rows of tile m, `rows` of them, see keys below this.  A request's n tokens of G rows each stand behind prefix = kv - n cached ones; a token
// of a tree (masks) may see any new token.
constexpr int attn_tile_end(int rows, bool masks, int n, int G, int prefix, int kv, int m) {
  if (masks || n == 1) return kv;
  const int next = (m + 1) * rows < n * G ? (m + 1) * rows : n * G, tokens = (next - 1) / G + 1;
  return prefix + (tokens < n ? tokens : n);
}

// (The window may be 2^31 - 1: each sum's first term is a length.)  In a tree the lowest key is that of a token that sees no new one.
constexpr AttnReach attn_window_reach(int rows, int unit, bool masks, int n, int G, int prefix, int kv, int window, int sinks, int m) {
  const int end = attn_tile_end(rows, masks, n, G, prefix, kv, m), upto = (end + unit - 1) / unit;
  const int next = (m + 1) * rows < n * G ? (m + 1) * rows : n * G;
  const int j0 = masks ? -1 : m * rows / G, j1 = masks ? n - 1 : (next - 1) / G;
  const int below = prefix + j0 + 1 - window, low = below > 0 ? below : 0;
  const int head = sinks < end ? sinks : end, first = (head + unit - 1) / unit;
  const int behind = low / unit - first, skip = behind > 0 ? behind : 0;
  return {upto - skip, first, skip, prefix + j1 + 1 - window, head, low};
}

}  // namespace moe
