// The index arithmetic of paged attention (gdn_paged.h) on the host, over batches whose starts, lengths and
// block tables hold anything (tests/test_paged_host.py builds it with AddressSanitizer; every
// array is exactly as long as its batch says): each row a workgroup may touch lies in q, each key within the
// table's row, each place in the cache. Exit status: 0 if all do.
#include <cstdio>
#include <random>
#include <vector>

#include "../../tjev_amd/csrc/gdn_paged.h"

static long g_bad = 0;
static void check(bool ok, const char* what) {
  if (!ok && g_bad++ < 10) std::printf("out of bounds: %s\n", what);
}

template <int R, int KB>
static void walk(const gdn::Batch& A) {
  for (int b = 0; b < A.B; ++b) {
    const gdn::Request q = gdn::request<R, KB>(A, b);
    check(q.cost >= 0 && q.blocks >= 1 && q.tiles >= 0, "cost");
    check(q.keys >= 0 && q.keys <= (long)A.M * A.page, "keys");
    check(q.rows == 0 || (q.s0 >= 0 && q.s0 + (q.rows - 1) / A.g < A.N), "rows");
    check((long)q.tiles * R >= q.rows && (long)q.blocks * KB >= q.keys, "tiles");
    for (int r = 0; r < q.rows; ++r) {
      const int lim = gdn::row_limit(q, r, A.g);
      check(lim >= 0 && lim <= q.keys, "limit");
      check(r == 0 || lim >= gdn::row_limit(q, r - 1, A.g), "limits grow with the rows");
    }
    if (!q.rows) continue;
    const int hi = gdn::row_limit(q, q.rows - 1, A.g);
    for (int k0 = 0; k0 < hi; k0 += 32)  // a wave's steps (those of 16 keys are among them)
      for (int j = 0; j < 32; j += 16) {
        const int key0 = k0 + j;
        for (int r = 0; r < 16; ++r) {
          const gdn::Place p = gdn::place_of(A, A.table + (long)b * A.M, key0 + r, q.keys);
          check(p.page >= 0 && p.page < A.pages && p.in >= 0 && p.in < A.page, "place");
        }
        if (A.page % 16 == 0) {
          const gdn::Place p = gdn::place_of(A, A.table + (long)b * A.M, key0 < q.keys ? key0 : k0, q.keys);
          check(p.page >= 0 && p.page < A.pages && p.in >= 0 && p.in + 15 < A.page, "a group's page");
        }
      }
  }
}

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  const int pages[] = {1, 3, 8, 16, 24, 48, 64, 100};
  for (int it = 0; it < 4000; ++it) {
    gdn::Batch A{};
    A.B = pick(1, 6);
    A.M = pick(1, 9);
    A.page = pages[pick(0, 7)];
    A.pages = pick(1, 12);
    A.Hk = pick(1, 4);
    A.g = pick(1, 20);
    A.N = pick(0, 40);
    std::vector<int32_t> table(A.B * A.M), starts(A.B + 1), lengths(A.B);
    const int kind = it % 3;  // as a scheduler writes them; with bad pages and lengths; anything
    int at = 0;
    for (int b = 0; b <= A.B; ++b) {
      starts[b] = kind == 2 ? (int32_t)rng() : at;
      at += pick(0, 12);
    }
    for (auto& x : lengths) x = kind == 2 ? (int32_t)rng() : kind ? pick(-5, A.M * A.page + 50) : pick(0, A.M * A.page);
    for (auto& x : table) x = kind == 2 ? (int32_t)rng() : kind ? pick(-2, A.pages + 1) : pick(0, A.pages - 1);
    A.table = table.data();
    A.starts = starts.data();
    A.lengths = lengths.data();
    walk<16, 128>(A);
    walk<32, 64>(A);
  }
  std::printf("%ld out of bounds\n", g_bad);
  return g_bad != 0;
}
