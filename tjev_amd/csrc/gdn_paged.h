// The index arithmetic of paged attention, for the kernels and for the host's test of its bounds
// (tests/asan/paged_driver.hip): which rows, keys and cache places a workgroup may touch, whatever the
// lengths, starts and block table on the GPU hold.
#pragma once

#include <stdint.h>

#include <hip/hip_runtime.h>

namespace gdn {

// The batch as the caller describes it
struct Batch {
  long N;                    // rows of q
  int B, M, page, pages;     // requests, table width, page size, pages of the cache
  int Hk, g;                 // key heads, query heads to each
  const int32_t *table, *starts, *lengths;
};

// The packed rows of a request and key head are its new tokens' query heads of that key head: row r
// is token r / g, head r % g; R of them are a tile. A unit of work is a tile's next KB keys.
struct Request {
  int s0, rows, tiles, blocks;  // first row of q; packed rows; tiles of them; key blocks
  int keys;                     // keys that the table's row has pages for
  long first;                   // position of the first new token
  long cost;                    // units
};

template <int R, int KB>
__host__ __device__ __forceinline__ Request request(const Batch& A, int b) {
  Request q;
  const long n = A.N, a = A.starts[b], e = A.starts[b + 1], len = A.lengths[b];
  const long s0 = a < 0 ? 0 : a > n ? n : a, s1 = e < s0 ? s0 : e > n ? n : e;
  const long cap = (long)A.M * A.page, keys = len < 0 ? 0 : len < cap ? len : cap;
  q.s0 = (int)s0;
  q.rows = (int)(s1 - s0) * A.g;
  q.tiles = (q.rows + R - 1) / R;
  q.keys = (int)keys;
  q.blocks = keys ? (int)((keys + KB - 1) / KB) : 1;  // a row without keys is written too
  q.first = len - (e - a);
  q.cost = (long)q.tiles * A.Hk * q.blocks;
  return q;
}

// keys that the packed row may attend to: those up to its token's own, of the request's
__host__ __device__ __forceinline__ int row_limit(const Request& q, int row, int g) {
  const long last = q.first + row / g + 1;
  return last < 0 ? 0 : last < q.keys ? (int)last : q.keys;
}

// A key's place. Keys behind the last are taken at the last (their weights are 0); an entry that is no page
// of the cache reads page 0 and is not good.
struct Place {
  int page, in;
  bool good;
};
__host__ __device__ __forceinline__ Place place_of(const Batch& A, const int32_t* row, int key, int keys) {
  const int k = key < keys ? key : keys - 1, i = k / A.page, p = row[i];
  const bool good = p >= 0 && p < A.pages;
  return {good ? p : 0, k - i * A.page, good};
}

}  // namespace gdn
