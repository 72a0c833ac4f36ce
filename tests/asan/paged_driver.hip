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
    check(q.cost >= 0 && q.tiles >= 0 && q.cost == q.per_head * A.Hk, "cost");
    check(q.keys >= 0 && q.keys <= (long)A.M * A.page, "keys");
    check(q.rows == 0 || (q.s0 >= 0 && q.s0 + (q.rows - 1) / A.g < A.N), "rows");
    check((long)q.tiles * q.tile_rows >= q.rows, "tiles");
    for (int r = 0; r < q.rows; ++r) {
      const int lim = gdn::row_limit(A, q, r);
      check(lim >= 0 && lim <= q.keys, "limit");
      check(r == 0 || lim >= gdn::row_limit(A, q, r - 1), "limits grow with the rows");
      check((long)q.tile_blocks(r / q.tile_rows) * KB >= lim, "a tile's units hold its keys");
    }
    long sum = 0;  // every unit once, in order, and at least one to a tile
    for (int t = 0; t < q.tiles; ++t) {
      check(q.before_tile(t) == sum && q.tile_blocks(t) >= 1, "units before a tile");
      sum += q.extra + q.tile_blocks(t);
    }
    check(sum == q.per_head, "units of a head");
    long at = 0;
    for (int h = 0; h < A.Hk && q.cost < 3000; ++h)
      for (int t = 0; t < q.tiles; ++t)
        for (int k = 0; k < q.extra + q.tile_blocks(t); ++k, ++at) {
          const gdn::Unit u = gdn::unit_of(q, at);
          check(u.head == h && u.tile == t && u.at == k, "a unit's place");
        }
    if (!q.rows) continue;
    const int hi = gdn::row_limit(A, q, q.rows - 1);
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
  // a key's page: exact at the borders of pages of any size, up to the last key there can be
  for (int page = 1; page < 70000; page = page < 300 ? page + 1 : page * 5 / 4 + 1) {
    gdn::Batch A{};
    gdn::set_page(A, page);
    for (long i = 0; i < 2000; ++i) {
      const long top = 0x7fffffffl / page, n = i < 1000 ? i : top - (i - 1000);
      for (long k = n * page - 1; k <= n * page + 1; ++k)
        if (k >= 0 && k <= 0x7fffffffl) check(gdn::page_of(A, (int)k) == k / page, "a key's page");
      const long high = (1l << 50) / page * page + i * page;  // slots of a long cache
      for (long k = high - 1; k <= high + 1; ++k) check(gdn::div_by(page)(k) == k / page, "a slot's page");
    }
  }
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  const int pages[] = {1, 3, 8, 16, 24, 48, 64, 100};
  for (int it = 0; it < 4000; ++it) {
    gdn::Batch A{};
    A.B = pick(1, 6);
    A.M = pick(1, 9);
    gdn::set_page(A, pages[pick(0, 7)]);
    A.pages = pick(1, 12);
    A.Hk = pick(1, 4);
    gdn::set_group(A, it % 7 ? pick(1, 20) : pick(1, 300));
    A.N = pick(0, it % 5 ? 40 : 150);
    A.wide = it % 2 ? 1 << 30 : pick(0, 64);
    A.wide_extra = pick(1, 3);
    std::vector<int32_t> table(A.B * A.M), starts(A.B + 1), lengths(A.B);
    const int kind = it % 3;  // as a scheduler writes them; with bad pages and lengths; anything
    int at = 0;
    for (int b = 0; b <= A.B; ++b) {
      starts[b] = kind == 2 ? (int32_t)rng() : at;
      at += pick(0, it % 5 ? 12 : 40);
    }
    for (auto& x : lengths) x = kind == 2 ? (int32_t)rng() : kind ? pick(-5, A.M * A.page + 50) : pick(0, A.M * A.page);
    for (auto& x : table) x = kind == 2 ? (int32_t)rng() : kind ? pick(-2, A.pages + 1) : pick(0, A.pages - 1);
    A.table = table.data();
    A.starts = starts.data();
    A.lengths = lengths.data();
    walk<16, 128>(A);
    walk<32, 64>(A);
    walk<64, 128>(A);
  }
  std::printf("%ld out of bounds\n", g_bad);
  return g_bad != 0;
}
