// kh::overlap (kaldi_amd/csrc/hip/overlap.h) against the sets of bytes themselves, on random small matrices.
// usage: overlap_check <cases>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../kaldi_amd/csrc/hip/overlap.h"

int main(int argc, char **argv) {
  const int cases = argc > 1 ? atoi(argv[1]) : 100000;
  srand(1);
  int yes = 0, within = 0;
  for (int n = 0; n < cases; ++n) {
    kh::Area m[2];
    std::vector<char> of[2];
    const int common = 1 + rand() % 12;
    for (int k = 0; k < 2; ++k) {
      const int rows = rand() % 9, cols = rand() % 7, ld = n % 2 ? std::max(cols, common) : cols + rand() % 6;
      // (byte addresses: an unaligned pair may share a part of an element)
      m[k] = {"", (const void *)(uintptr_t)(64 + (rand() % 3 ? 4 * (rand() % 60) : rand() % 240)), rows, cols, ld};
      of[k].assign(2048, 0);
      for (int r = 0; r < rows; ++r)
        for (int b = 0; b < 4 * cols; ++b) of[k][(uintptr_t)m[k].p + 4 * r * ld + b] = 1;
    }
    bool want = false;
    for (int i = 0; i < 2048; ++i) want |= of[0][i] && of[1][i];
    if (kh::overlap(m[0], m[1]) != want || kh::overlap(m[1], m[0]) != want) {
      printf("differs: %p %lld x %lld (%lld), %p %lld x %lld (%lld): %d\n", m[0].p, m[0].rows, m[0].cols, m[0].ld, m[1].p, m[1].rows,
             m[1].cols, m[1].ld, want);
      return 1;
    }
    yes += want;
    within += !want && !m[0].empty() && !m[1].empty() && m[0].begin() < m[1].end() && m[1].begin() < m[0].end();
  }
  printf("%d cases, %d overlap, %d lie between each other's rows\n", cases, yes, within);
  return yes > cases / 10 && within > cases / 100 ? 0 : 1;
}
