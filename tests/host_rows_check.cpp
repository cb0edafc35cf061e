// Whether two sets of rows share memory (csrc/rows_clash.h), against a look at every byte.  Built and run without a GPU by
// tests/test_between_cpu.py; exits 0 when every check holds.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../torch-tpu_amd/csrc/rows_clash.h"

int main() {
  std::mt19937 rng(3);
  const auto upto = [&](int n) { return (int)(rng() % n); };
  static char memory[4096], marks[4096];
  int clashes = 0, between = 0;
  for (int turn = 0; turn < 300000; turn++) {
    const int a_rows = 1 + upto(5), b_rows = 1 + upto(5), a_bytes = 1 + upto(40), b_bytes = 1 + upto(40);
    const int a_stride = a_bytes + upto(60), b_stride = upto(2) ? b_bytes + upto(60) : a_stride < b_bytes ? b_bytes : a_stride;
    const int a0 = 1500 + upto(600), b0 = 1500 + upto(600);
    bool share = false;
    for (int r = 0; r < a_rows; r++)
      for (int i = 0; i < a_bytes; i++) marks[a0 + r * a_stride + i] = 1;
    for (int r = 0; r < b_rows; r++)
      for (int i = 0; i < b_bytes; i++) share |= marks[b0 + r * b_stride + i];
    for (int r = 0; r < a_rows; r++)
      for (int i = 0; i < a_bytes; i++) marks[a0 + r * a_stride + i] = 0;
    const bool said = moe::rows_clash(memory + a0, a_stride, a_bytes, a_rows, memory + b0, b_stride, b_bytes, b_rows);
    const bool other = moe::rows_clash(memory + b0, b_stride, b_bytes, b_rows, memory + a0, a_stride, a_bytes, a_rows);
    const bool apart = a0 + (a_rows - 1) * a_stride + a_bytes <= b0 || b0 + (b_rows - 1) * b_stride + b_bytes <= a0;
    // what shares memory is always told; what does not is told apart where the distances agree and the rows do not reach past each other's ends
    const bool alike = a_rows == b_rows && a_stride == b_stride;
    if (said != other || (share && !said) || (apart && said) || (alike && std::abs(a0 - b0) < a_stride && !share && said)) {
      std::printf("FAILED: %d rows of %d bytes, %d apart, at %d, and %d of %d, %d apart, at %d: %d\n", a_rows, a_bytes, a_stride, a0, b_rows, b_bytes, b_stride, b0, said);
      return 1;
    }
    clashes += share;
    between += !share && !apart && !said;
  }
  if (clashes < 1000 || between < 1000) return 1;
  std::printf("row checks passed\n");
  return 0;
}
