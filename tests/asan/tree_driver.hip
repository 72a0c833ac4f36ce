// Which keys a row of a tree attends to (gdn_paged.h) on the host, against the definition key by key; rows' bits are exactly as long as
// they say (tests/test_drafts_host.py builds it with AddressSanitizer). Exit status: 0 if all are right.
#include <cstdio>
#include <random>
#include <vector>

#include "../../tjev_amd/csrc/gdn_paged.h"

int main() {
  std::mt19937_64 rng(5);
  long bad = 0;
  auto check = [&](const std::vector<uint64_t>& bits, long at, int left) {
    const uint64_t got = gdn::keys_of_bits(bits.data(), (long)bits.size(), at, left);
    for (int j = 0; j < 64; ++j) {
      const long t = at + j;
      const bool want = j < left && (t < 0 || (t < 64 * (long)bits.size() && (bits[t / 64] >> (t % 64) & 1)));
      bad += want != (bool)(got >> j & 1);
    }
  };
  for (long words = 1; words <= 4; ++words)
    for (long at = -140; at <= 64 * words + 140; ++at)
      for (int left : {-70, -1, 0, 1, 31, 63, 64, 65, 0x7fffffff}) {
        std::vector<uint64_t> bits(words);
        for (auto& b : bits) b = rng();
        check(bits, at, left);
      }
  for (long at : {-(1l << 40), -(1l << 31), (1l << 31), (1l << 40)}) check(std::vector<uint64_t>(3, ~0ull), at, 64);
  // requests of trees: every tile has all keys, and the units of a batch add up
  for (int it = 0; it < 2000; ++it) {
    gdn::Batch A{};
    A.B = 1;
    A.M = 1 + rng() % 9;
    gdn::set_page(A, 1 + rng() % 64);
    A.pages = 7;
    A.Hk = 1 + rng() % 3;
    gdn::set_group(A, 1 + rng() % 8);
    A.N = rng() % 300;
    A.wide = rng() % 2 ? 16 : 0x7fffffff;
    A.wide_extra = 2;
    const int32_t starts[2] = {(int32_t)(rng() % 400) - 50, (int32_t)(rng() % 400) - 50}, lengths[1] = {(int32_t)(rng() % 700) - 50};
    A.starts = starts;
    A.lengths = lengths;
    const bool pairs = rng() % 2;  // a streamed tile's unit is two blocks
    const gdn::Request q = pairs ? gdn::request<16, 128, true, 2>(A, 0) : gdn::request<16, 128, true>(A, 0);
    const long unit = pairs && q.tile_rows == 16 ? 256 : 128;
    bad += q.rows && !(q.s0 >= 0 && q.s0 + (q.rows - 1) / A.g < A.N);
    bad += q.keys < 0 || q.keys > (long)A.M * A.page;
    long sum = 0;
    for (int t = 0; t < q.tiles; ++t) {
      bad += q.before_tile(t) != sum || (long)q.tile_blocks(t) * unit < q.keys || (q.keys && (long)(q.tile_blocks(t) - 1) * unit >= q.keys) || q.tile_blocks(t) < 1;
      sum += q.extra + q.tile_blocks(t);
    }
    bad += sum != q.per_head || q.cost != q.per_head * A.Hk;
  }
  std::printf("%ld wrong\n", bad);
  return bad != 0;
}
