// Which keys attention with a window goes over and reads (csrc/attn_reach.h), against what every row sees, key by key.  Built and
// run without a GPU by tests/test_between_cpu.py; exits 0 when every check holds.
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "../torch-tpu_amd/csrc/attn_reach.h"

static int failures = 0;
#define CHECK(cond, ...)                                    \
  do {                                                      \
    if (!(cond) && failures++ < 20) {                       \
      std::printf("FAILED line %d: %s: ", __LINE__, #cond); \
      std::printf(__VA_ARGS__);                             \
      std::printf("\n");                                    \
    }                                                       \
  } while (0)

int main() {
  std::mt19937_64 rng(5);
  const auto pick = [&](std::initializer_list<int> of) { return of.begin()[rng() % of.size()]; };
  for (int turn = 0; turn < 6000; turn++) {
    const int rows = pick({16, 64, 128, 256}), unit = rows == 16 ? pick({64, 128}) : 64, G = pick({1, 2, 3, 8});
    const bool masks = rng() % 2;
    const int n = masks ? 1 + rng() % 64 : pick({1, 1, 2, 40, 150}), prefix = rng() % pick({1, 20, 300, 900}), kv = prefix + n;
    const int W = pick({1, 2, 31, 64, 65, 128, 300, 700, 2147483647}), S = pick({0, 1, 4, 63, 64, 65, 130, 500});
    // what each token sees: of the keys before it or in its mask the last W and the first S
    std::vector<std::vector<char>> sees(n, std::vector<char>(kv, 0));
    std::vector<char> seen(kv, 0);
    for (int j = 0; j < n; j++) {
      const uint64_t mask = rng() % 8 == 0 ? 0 : rng() & rng();
      std::vector<int> may;
      for (int k = 0; k < kv; k++)
        if (k < prefix || (masks ? mask >> (k - prefix) & 1 : k - prefix <= j)) may.push_back(k);
      for (int i = 0; i < (int)may.size(); i++)
        if (i >= (int64_t)may.size() - W || i < S) sees[j][may[i]] = seen[may[i]] = 1;
    }
    // (of a tree any new token may be read, and what one that sees no new token would see)
    if (masks)
      for (int k = 0; k < kv; k++)
        if (k >= (int64_t)prefix - W) seen[k] = 1;
    for (int m = 0; m * rows < n * G; m++) {
      const moe::AttnReach r = moe::attn_window_reach(rows, unit, masks, n, G, prefix, kv, W, S, m);
      const int clear = masks ? prefix : prefix + m * rows / G + 1;
      std::vector<char> read(kv, 0);
      CHECK(r.units > 0 && r.units <= (kv + unit - 1) / unit, "units %d of %d keys", r.units, kv);
      for (int c = 0; c < r.units; c++)
        for (int i = 0; i < unit; i++) {
          const int key = r.unit(c) * unit + i, from = r.read(key) < kv ? r.read(key) : kv - 1, size = rows == 16 ? 32 : unit, key0 = key - i % size;
          const bool edge = key0 + size > clear || key0 < r.every;
          CHECK(from >= 0 && seen[from], "key %d of %d read for %d, window %d, first %d, %s of %d", from, kv, key, W, S, masks ? "tree" : "chunk", n);
          if (key < kv && from == key) read[key]++;
          for (int row = m * rows; row < (m + 1) * rows && row < n * G; row++) {
            const bool here = key < kv && sees[row / G][key];
            CHECK(edge || here, "key %d of row %d is not looked at, window %d, first %d", key, row, W, S);
            CHECK(!here || from == key, "key %d of row %d, but %d is read", key, row, from);
          }
        }
      for (int row = m * rows; row < (m + 1) * rows && row < n * G; row++)
        for (int k = 0; k < kv; k++) CHECK(!sees[row / G][k] || read[k] == 1, "key %d of row %d is read %d times", k, row, read[k]);
    }
  }
  if (!failures) std::printf("reach checks passed\n");
  return failures != 0;
}
