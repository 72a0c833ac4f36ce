// The index arithmetic of paged attention, for the kernels and for the host's test of its bounds
// (tests/asan/paged_driver.hip): which rows, keys and cache places a workgroup may touch, whatever the
// lengths, starts and block table on the GPU hold.
#pragma once

#include <stdint.h>

#include <hip/hip_runtime.h>

namespace gdn {

// Whole division by a number that stays the same, for 0 <= x < 2^52: the product with its reciprocal is off by less
// than one (about 10 instructions; a division of 64-bit integers is 150)
struct Div {
  double inv;
  long d;
  __host__ __device__ __forceinline__ long operator()(long x) const {
    const long q = (long)((double)x * inv), r = x - q * d;
    return r < 0 ? q - 1 : r >= d ? q + 1 : q;
  }
};
inline __host__ __device__ Div div_by(long d) { return {1.0 / (double)d, d}; }

// The same for 0 <= x < 2^31: the high word of x mul, shifted right. With 2^(L-1) < d <= 2^L and mul = ceil(2^(31+L) / d) <
// 2^32 the product is off by less than x d <= 2^(31+L): the quotient is exact. (d = 1: shift -1, x itself.)
struct Div32 {
  uint32_t mul;
  int shift;
  __host__ __device__ __forceinline__ int operator()(int x) const {
    return shift < 0 ? x : (int)(((uint64_t)(uint32_t)x * mul) >> 32 >> shift);
  }
};
inline __host__ __device__ Div32 div32_by(int d) {
  int L = 0;
  while ((1l << L) < d) ++L;
  return {(uint32_t)(((1ul << (31 + L)) + d - 1) / d), L - 1};
}

// The batch as the caller describes it
struct Batch {
  long N;                    // rows of q
  int B, M, page, pages;     // requests, table width, page size, pages of the cache
  int Hk, g;                 // key heads, query heads to each
  int wide, wide_extra;      // requests of more packed rows take wide tiles, which have so many units before their keys'
  Div32 by_page, by_g;       // a key's page, a packed row's token
  Div by_g_long;
  const int32_t *table, *starts, *lengths;
};

__host__ __device__ __forceinline__ void set_page(Batch& A, int page) {
  A.page = page;
  A.by_page = div32_by(page);
}
__host__ __device__ __forceinline__ void set_group(Batch& A, int g) {
  A.g = g;
  A.by_g = div32_by(g);
  A.by_g_long = div_by(g);
}
__host__ __device__ __forceinline__ int page_of(const Batch& A, int key) { return A.by_page(key); }

// The packed rows of a request and key head are its new tokens' query heads of that key head: row r
// is token r / g, head r % g. Requests of more than `wide` rows are worked on in tiles of kWideRows, the others
// in tiles of R. A unit of work is a tile's next KB keys, in the order key head, tile, keys; before its keys a tile has
// units for what it costs by itself (its queries, the first loads' latency, its results; a wide tile's gate). Measured with
// 0, 1, 2, 3, 4 of them for a wide tile: a prompt of 4096 tokens, 32 heads of 256 and 4 key heads, whose first tiles
// have one block of keys, without a gate -, 375, 337, 340, 341 us, with one 567, 447, 390, 354, 358; chunks of prompts
// beside decoding requests (32/4 heads of 128, no gate) 106, 92.5, 87.3, 90.5, 94.2. For a streamed tile: 0 to 2 alike but for
// ragged fp32 batches (22.2, 22.2, 24.4).
constexpr int kWideRows = 128, kWideExtra = 2, kGateExtra = 1, kExtra = 1;

struct Request {
  int s0, rows, tiles, tile_rows;  // first row of q; packed rows; tiles of them
  int keys;                        // keys that the table's row has pages for
  int extra;                       // units of a tile before its keys'
  int blocks;                      // blocks of keys of every tile, or 0: tile t has (y + t) / g of them
  long y;
  Div by_g;
  long first;                      // position of the first new token
  long per_head, cost;             // units of a key head, of the request

  // sum of (0 .. x - 1) / g
  __host__ __device__ __forceinline__ long below(long x) const {
    const long q = by_g(x);
    return by_g.d * (q * (q - 1) / 2) + q * (x - q * by_g.d);
  }
  __host__ __device__ __forceinline__ int tile_blocks(int t) const { return blocks ? blocks : (int)by_g(y + t); }
  // units of the tiles before it
  __host__ __device__ __forceinline__ long before_tile(int t) const {
    return (long)t * extra + (blocks ? (long)t * blocks : below(y + t) - below(y));
  }
};

template <int R, int KB>
__host__ __device__ __forceinline__ Request request(const Batch& A, int b) {
  Request q;
  const long n = A.N, a = A.starts[b], e = A.starts[b + 1], len = A.lengths[b];
  const long s0 = a < 0 ? 0 : a > n ? n : a, s1 = e < s0 ? s0 : e > n ? n : e;
  const long cap = (long)A.M * A.page, keys = len < 0 ? 0 : len < cap ? len : cap;
  q.s0 = (int)s0;
  q.rows = (int)(s1 - s0) * A.g;
  const bool wide = q.rows > A.wide;
  q.tile_rows = wide ? kWideRows : R;
  q.extra = wide ? A.wide_extra : kExtra;
  q.tiles = wide ? (q.rows + kWideRows - 1) / kWideRows : (q.rows + R - 1) / R;
  q.keys = (int)keys;
  q.first = len - (e - a);
  q.by_g = A.by_g_long;
  q.y = 0;
  q.blocks = keys ? (int)((keys + KB - 1) / KB) : 1;  // a row without keys is written too
  if (wide && q.first >= 0 && keys == len) {
    // Tile t's last row may attend to first + (kWideRows (t + 1) - 1) / g + 1 keys, which are
    // floor((first g + kWideRows (t + 1) - 1) / (KB g)) + 1 blocks, and with KB = kWideRows floor((y + t) / g)
    static_assert(KB == kWideRows || KB < kWideRows, "");
    if (KB == kWideRows) {
      q.blocks = 0;
      q.y = (q.first * A.g + KB * (long)A.g - 1) / KB + 1;
    }
  }
  q.per_head = q.before_tile(q.tiles);
  q.cost = q.per_head * A.Hk;
  return q;
}

// a unit of the request: its key head, tile and place in the tile
struct Unit {
  int head, tile, at;
};
__host__ __device__ __forceinline__ Unit unit_of(const Request& q, long local) {
  Unit u;
  u.head = (int)div_by(q.per_head)(local);  // (a division of 64-bit integers is 150 instructions)
  local -= (long)u.head * q.per_head;
  if (q.blocks) {
    u.tile = (int)div_by(q.blocks + q.extra)(local);
  } else {
    int lo = 0, hi = q.tiles;  // the last tile that begins at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (q.before_tile(mid) <= local) lo = mid; else hi = mid;
    }
    u.tile = lo;
  }
  u.at = (int)(local - q.before_tile(u.tile));
  return u;
}

// keys that the packed row may attend to: those up to its token's own, of the request's
__host__ __device__ __forceinline__ int row_limit(const Batch& A, const Request& q, int row) {
  const long last = q.first + A.by_g(row) + 1;
  return last < 0 ? 0 : last < q.keys ? (int)last : q.keys;
}

// A key's place. Keys behind the last are taken at the last (their weights are 0); an entry that is no page
// of the cache reads page 0 and is not good.
struct Place {
  int page, in;
  bool good;
};
__host__ __device__ __forceinline__ Place place_of(const Batch& A, const int32_t* row, int key, int keys) {
  const int k = key < keys ? key : keys - 1, i = page_of(A, k), p = row[i];
  const bool good = p >= 0 && p < A.pages;
  return {good ? p : 0, k - i * A.page, good};
}

// The paged attention's arguments, and how its rows are shared out
struct AttnArgs : Batch {
  int D, fill;
  float c;                          // scale * log2(e)
  const char *q, *k, *v, *gate;
  char* out;
  long qt, qh, gt, gh, ot, oh;      // bytes: token and head of q, gate, out
  long kp, ks, kh, vp, vs, vh;      // bytes: page, slot and head of the caches
  float* part;                      // the workgroups' unfinished rows, slots of `slot` floats
  long slot;
  int G;                            // workgroups, and the division by them
  Div by_G;
};

constexpr int kMostRanges = 768;
constexpr int kSplitBytes = 32;  // of the workspace, per range: the tile that goes on behind it

// How the parts of tiles are joined: a workgroup per range, several per tile, or as many as there are for the tiles found
enum Join : int { kJoinRanges, kJoinSliced, kJoinCounted };

struct AttnPlan {
  int nq;            // streamed tiles of 16 nq rows
  bool mixed;        // wide tiles too
  Join join;
  int tiles;         // the most there can be, up to 2^30
  int G;             // ranges
  long slot;         // floats of a workspace slot
  size_t bytes;      // workspace
};

// One unit of gdn_attn_inst.hip: attention in bf16 (bf = true) or fp32, head dims up to d
#define GDN_ATTENTION(t, d) hipError_t attention_##t##_##d(const AttnPlan& r, AttnArgs& A, hipStream_t st);
GDN_ATTENTION(bf16, 64)
GDN_ATTENTION(bf16, 128)
GDN_ATTENTION(bf16, 256)
GDN_ATTENTION(f32, 64)
GDN_ATTENTION(f32, 128)
GDN_ATTENTION(f32, 256)
#undef GDN_ATTENTION

}  // namespace gdn
