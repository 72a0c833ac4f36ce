// Who holds the pages of the paged key/value cache, for gfx950: the accepted ones of drafted tokens moved to their places
// (compaction), and requests that go on from others' pages, shortened, several times or not at all (forks).
//
// Compaction: token path[j] of a request's new ones becomes its j-th, path growing, so path[j] >= j and a place is read
// before it is written when the moves run in order. A workgroup moves some columns of 16 bytes of all tokens of one request, of
// one cache: a round of tokens is loaded, then (behind a barrier) stored. Bound by latency: lengths, path, table, keys, each
// behind the other; the bytes are few.
//
// Forks: place i of the new table holds the first pages of place sources[i] of the old one. What changes is counted per page
// with atomics on whole numbers (sums, minima: their order does not matter): `shared`, how many hold a page beside the first
// one, and of the last pages that are not full how many go on writing there. Pages that nobody holds go back on the free list
// in the order of the old table, copies of last pages are taken from it in the order of the new one.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/tjev_gdn.h"
#include "gdn_device.h"
#include "gdn_launch.h"
#include "gdn_paged.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kLayers = 16;  // of a launch

struct Caches {
  char *k[kLayers], *v[kLayers];
  long kp, ks, kh, vp, vs, vh;  // bytes: page, slot and head
  int chunks, per;              // vectors of a head, of a token
  int cols;                     // of them, a workgroup's
  int groups;                   // of columns
  // where a vector of a slot lies
  __device__ __forceinline__ char* at(int layer, bool values, long page, long in, int col, int bytes) const {
    const int h = col / chunks, c = col - h * chunks;
    return values ? v[layer] + page * vp + in * vs + h * vh + (long)c * bytes : k[layer] + page * kp + in * ks + h * kh + (long)c * bytes;
  }
};

// ---------------------------------------------------------------- compaction
struct CompactArgs {
  Caches c;
  int B, M, pages, layers;
  long most;
  Div page;
  const int32_t *table, *starts, *lengths, *path, *kept;
  int32_t* lengths_out;  // null: not this launch's
};

// a round's places: where a token is read and written, as page and slot (page -1: it is left out)
struct Move {
  int from, from_in, to, to_in;
};

// One tree of 16, 6 layers of 4 heads of 256: 5.0 us; 128 of up to 60, 8 layers of 8 heads of 128, 7.3 MB: 9.8.
template <class W>
__global__ __launch_bounds__(kThreads) void k_paged_compact(CompactArgs A) {
  constexpr int UN = 8;
  __shared__ Move smove[kThreads];
  GDN_POISON_LDS(smove);
  const int b = blockIdx.x, tid = threadIdx.x;
  const long n = max(0l, (long)A.starts[b + 1] - A.starts[b]), len = A.lengths[b], first = len - n;
  const long count = min(min((long)max(A.kept[b], 0), A.most), n);
  if (A.lengths_out && blockIdx.y == 0 && tid == 0) A.lengths_out[b] = (int)max(0l, first + count);
  if (!A.layers || first < 0) return;
  const int32_t* path = A.path + b * A.most;
  const int group = blockIdx.y % A.c.groups, cache = blockIdx.y / A.c.groups, layer = cache / 2;
  const bool values = cache % 2;
  const int cols = A.c.cols, step = kThreads / cols, mine = tid / cols, col = group * cols + tid % cols;
  const int round = min(UN * step, kThreads);
  for (long j0 = 0; j0 < count; j0 += round) {
    Move m{-1, 0, -1, 0};
    if (tid < round && j0 + tid < count) {
      const long j = j0 + tid, f = path[j];
      if (f > j && f < n) {
        const long pf = A.page(first + f), pt = A.page(first + j);
        if (pf < A.M) {  // (and pt, which is not behind it)
          const int from = A.table[(long)b * A.M + pf], to = A.table[(long)b * A.M + pt];
          if (from >= 0 && from < A.pages && to >= 0 && to < A.pages)
            m = {from, (int)(first + f - pf * A.page.d), to, (int)(first + j - pt * A.page.d)};
        }
      }
    }
    smove[tid] = m;
    // (none: everybody is at the same place, or before it)
    if (!__syncthreads_or(m.from >= 0)) continue;
    W x[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int t = i * step + mine;
      if (mine < step && col < A.c.per && t < round && smove[t].from >= 0)
        x[i] = *reinterpret_cast<const W*>(A.c.at(layer, values, smove[t].from, smove[t].from_in, col, sizeof(W)));
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): read by all before it is written by any
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int t = i * step + mine;
      if (mine < step && col < A.c.per && t < round && smove[t].from >= 0)
        *reinterpret_cast<W*>(A.c.at(layer, values, smove[t].to, smove[t].to_in, col, sizeof(W))) = x[i];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- forks
// What an old place loses: its pages from `kept` on, those that the first new place going on from it does not keep
struct ForkOld {
  int kept, held;
};
// What a new place goes on with: its source, pages, the page that it writes on in (or -1), and whether its pages are counted: the
// first new place of a source has them from it, and nothing is counted for that
struct ForkNew {
  int source, pages, last, counted;
};

struct ForkArgs {
  int B, B2, M, pages;  // places of the old and the new table
  long n_free;
  Div page;
  const int32_t *table, *lengths, *sources, *keep, *free, *taken, *shared;  // keep: null for all
  int32_t *table_out, *lengths_out, *free_out, *taken_out, *shared_out;
  ForkOld* old;
  ForkNew* fresh;
  // of each page: the new places that write on in it, and the first of them; the first of the old table's entries that leave it
  int32_t *writers, *writer, *entry;
  int32_t *freed, *copied;  // of each old place, the pages given back; of each new one, whether it takes a copy of its last page
  int32_t* where;           // and where that stands on the free list, or (k_fork_one) the page itself; -1: none
};

__device__ __forceinline__ int fork_pages(const ForkArgs& A, long n) {
  const long p = A.page(n + A.page.d - 1);
  return (int)(p < A.M ? p : A.M);
}
__device__ __forceinline__ bool is_page(const ForkArgs& A, int p) { return p >= 0 && p < A.pages; }

// What place r goes on with, and how many tokens; `counted` is not known yet
__device__ __forceinline__ ForkNew going(const ForkArgs& A, int r, long& keep) {
  ForkNew g{-1, 0, -1, 0};
  keep = 0;
  if (r >= A.B2) return g;
  const int s = A.sources[r];
  if (s < 0 || s >= A.B) return g;
  g.source = s;
  const long len = max(A.lengths[s], 0);
  keep = A.keep ? min((long)max(A.keep[r], 0), len) : len;
  g.pages = fork_pages(A, keep);
  const long j = A.page(keep);
  if (keep > j * A.page.d && j < A.M) {
    const int p = A.table[(long)s * A.M + j];
    if (is_page(A, p)) g.last = p;
  }
  return g;
}

// A workgroup per place: what the old place of that number loses, what the new one goes on with, and its row of the table. The
// list, the counts and the notes of all pages are shared out.
__global__ __launch_bounds__(kThreads) void k_fork_init(ForkArgs A) {
  __shared__ int sfirst[2];
  GDN_POISON_LDS(sfirst);
  const int r = blockIdx.x, tid = threadIdx.x;
  const long stride = (long)gridDim.x * kThreads, id = (long)r * kThreads + tid;
  for (long i = id; i < A.pages; i += stride) {
    A.shared_out[i] = A.shared[i];
    A.writers[i] = 0;
    A.writer[i] = A.entry[i] = 0x7fffffff;
  }
  for (long i = id; i < A.n_free; i += stride) A.free_out[i] = A.free[i];
  if (r >= max(A.B, A.B2)) return;
  long keep;
  ForkNew g = going(A, r, keep);
  if (tid < 2) sfirst[tid] = A.B2;
  __syncthreads();
  // the first new place that goes on from old place r, and the first that goes on from r's own source
  int heir = A.B2, mine = A.B2;
  for (int i = tid; i < A.B2; i += kThreads) {
    const int s = A.sources[i];
    if (s == r) heir = min(heir, i);
    if (s == g.source) mine = min(mine, i);
  }
  if (heir < A.B2) atomicMin(&sfirst[0], heir);
  if (mine < A.B2) atomicMin(&sfirst[1], mine);
  __syncthreads();
  heir = sfirst[0];
  if (r < A.B2) {
    for (int j = tid; j < A.M; j += kThreads) A.table_out[(long)r * A.M + j] = j < g.pages ? A.table[(long)g.source * A.M + j] : -1;
    if (tid == 0) {
      g.counted = g.source >= 0 && sfirst[1] != r;
      A.fresh[r] = g;
      A.lengths_out[r] = (int)keep;
    }
  }
  if (r < A.B && tid == 0) {
    const int kept = heir < A.B2 ? going(A, heir, keep).pages : 0;
    A.old[r] = {kept, max(kept, fork_pages(A, max(A.lengths[r], 0)))};
  }
}

// the old table's entry r, j loses its page; the new place's has one more holder
__device__ __forceinline__ void drop(const ForkArgs& A, int r, int j) {
  const int p = A.table[(long)r * A.M + j];
  if (!is_page(A, p)) return;
  atomicSub(&A.shared_out[p], 1);
  atomicMin(&A.entry[p], r * A.M + j);
}
__device__ __forceinline__ void add(const ForkArgs& A, int source, int j) {
  const int p = A.table[(long)source * A.M + j];
  if (is_page(A, p)) atomicAdd(&A.shared_out[p], 1);
}
// (k_fork_one reads what its own workgroup counted)
__device__ __forceinline__ int counted(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
// whether the old table's entry gives its page back
__device__ __forceinline__ bool gives_back(const ForkArgs& A, int r, int j, int& p) {
  p = A.table[(long)r * A.M + j];
  return is_page(A, p) && counted(&A.entry[p]) == r * A.M + j && counted(&A.shared_out[p]) == -1;
}
// A last page with room has one holder: the first of those that write on in it, if all of its holders do. The others take copies.
__device__ __forceinline__ bool takes_copy(const ForkArgs& A, int r, const ForkNew& g) {
  return g.last >= 0 && !(counted(&A.shared_out[g.last]) + 1 == counted(&A.writers[g.last]) && counted(&A.writer[g.last]) == r);
}
// the page at this place of the whole free list, or -1
__device__ __forceinline__ int page_at(const ForkArgs& A, long at) {
  const int got = at >= 0 && at < A.n_free ? counted(&A.free_out[at]) : -1;
  return is_page(A, got) ? got : -1;
}
__device__ __forceinline__ void take(const ForkArgs& A, int r, const ForkNew& g, int got) {
  A.table_out[(long)r * A.M + g.pages - 1] = got;
  if (got >= 0) A.shared_out[got] = 0;
}

// Few places and entries: the rest in one workgroup of a thread per place, whose barriers stand for the ends of three launches. An entry
// that loses its holder costs one CU 5 ns (two atomics, two loads and two stores, each lane's of a line of its own), so this is for calls
// that change few, which the host does not know and guesses. With lengths to keep (a step's roll back: most places go on, with
// what they had) tables of up to kOneTurns * kOne entries: 64 places of 512 pages, a page of each given back, 18.6 us a call, in
// launches of their own 26.7; with three whole rows 21.4 and 26.4, with twenty 70 and 26; all given back 178 and 26.5. Without (beams
// that go on from each other, samples) up to kFewTurns * kOne: 64 of 64, all given back, 26.2 and 26.4, a page of each 18.7 and 26.6; half
// of 64 of 512, the rest twice, would take 152 and 26.6. (Entries are the table's, not the requests': lengths are on the GPU.)
constexpr int kOne = 1024, kOneTurns = 64, kFewTurns = 4;
constexpr int kBatch = 4;  // entries that a thread has on their way at once

// running sums over the workgroup's threads of two numbers of 32 bits, and the whole
__device__ __forceinline__ long scan_one(long v, long* swave, long& total) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long t = __shfl_up(v, d);
    if (lane() >= d) v += t;
  }
  __syncthreads();
  if (lane() == 63) swave[wave()] = v;
  __syncthreads();
  total = 0;
  long before = 0;
#pragma unroll
  for (int w = 0; w < kOne / 64; ++w) {
    if (w < wave()) before += swave[w];
    total += swave[w];
  }
  return v + before;
}
__device__ __forceinline__ long pair(int hi, int lo) { return (long)hi << 32 | lo; }
__device__ __forceinline__ int hi_of(long v) { return (int)(v >> 32); }
__device__ __forceinline__ int lo_of(long v) { return (int)v; }
// of each of the entries e0, e0 + kOne, ... the place whose run of numbers holds it: the last of those that begin at or before it
__device__ __forceinline__ void runs_of(const int* begin, int n, int e0, int (&r)[kBatch]) {
#pragma unroll
  for (int u = 0; u < kBatch; ++u) r[u] = 0;
  for (int step = kOne / 2; step; step /= 2)
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (r[u] + step < n && begin[r[u] + step] <= e0 + u * kOne) r[u] += step;
}

// The entries that lose or gain a holder are numbered through, place by place, kOne to a turn. Each is a chain of latencies (its place, the
// table, the counts), so a thread has kBatch on their way at once; the entries' ranks among those given back come from one running
// sum over all turns' and waves' numbers of them.
__global__ __launch_bounds__(kOne) void k_fork_one(ForkArgs A) {
  __shared__ int sdrop[kOne], sadd[kOne];    // the first number of each place's entries
  __shared__ int sfrom[kOne], ssource[kOne];  // the table's index of an entry, less its number
  __shared__ int sback[kOneTurns][kOne / 64];
  __shared__ long swave[kOne / 64];
  static_assert(kOneTurns * (kOne / 64) == kOne && kOneTurns % kBatch == 0, "a thread per number");
  GDN_POISON_LDS(sdrop, sadd, sfrom, ssource, sback, swave);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(wave());
  const ForkOld o = tid < A.B ? A.old[tid] : ForkOld{0, 0};
  const ForkNew g = tid < A.B2 ? A.fresh[tid] : ForkNew{-1, 0, -1, 0};
  const long had = min((long)max(A.taken[0], 0), A.n_free);
  const int drops = o.held - o.kept, adds = g.counted ? g.pages : 0;
  long all;
  const long upto = scan_one(pair(drops, adds), swave, all);
  const int n_drop = hi_of(all), n_add = lo_of(all);
  int* const backs = &sback[0][0];
  sdrop[tid] = hi_of(upto) - drops;
  sadd[tid] = lo_of(upto) - adds;
  sfrom[tid] = tid * A.M + o.kept - sdrop[tid];
  ssource[tid] = g.source * A.M - sadd[tid];
  backs[tid] = 0;
  if (g.last >= 0) {
    atomicAdd(&A.writers[g.last], 1);
    atomicMin(&A.writer[g.last], tid);
  }
  __syncthreads();
  // the thread's entries of a batch: the index of each in the table, and its page (-1: none)
  auto entries = [&](const int* begin, const int* base, int places, int n, int e0, int (&at)[kBatch], int (&page)[kBatch]) {
    runs_of(begin, places, e0 + tid, at);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int e = e0 + u * kOne + tid;
      at[u] = e < n ? base[at[u]] + e : -1;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      page[u] = at[u] >= 0 ? A.table[at[u]] : -1;
      if (!is_page(A, page[u])) page[u] = -1;
    }
  };
  for (int e0 = 0; e0 < n_add; e0 += kBatch * kOne) {
    int at[kBatch], page[kBatch];
    entries(sadd, ssource, A.B2, n_add, e0, at, page);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (page[u] >= 0) atomicAdd(&A.shared_out[page[u]], 1);
  }
  int at0[kBatch], page0[kBatch];  // the first batch's, kept: most calls have no more
  entries(sdrop, sfrom, A.B, n_drop, 0, at0, page0);
  auto drop_all = [&](const int (&at)[kBatch], const int (&page)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (page[u] >= 0) {
        atomicSub(&A.shared_out[page[u]], 1);
        atomicMin(&A.entry[page[u]], at[u]);
      }
  };
  drop_all(at0, page0);
  for (int e0 = kBatch * kOne; e0 < n_drop; e0 += kBatch * kOne) {
    int at[kBatch], page[kBatch];
    entries(sdrop, sfrom, A.B, n_drop, e0, at, page);
    drop_all(at, page);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): all is counted
  __syncthreads();
  const bool copy = takes_copy(A, tid, g);
  uint64_t back_here = 0;  // of the thread's entries, by their turn
  auto look = [&](int e0, const int (&at)[kBatch], const int (&page)[kBatch]) {
    int first[kBatch], holders[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      first[u] = page[u] >= 0 ? counted(&A.entry[page[u]]) : -1;
      holders[u] = page[u] >= 0 ? counted(&A.shared_out[page[u]]) : 0;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int turn = e0 / kOne + u;
      const bool gone = page[u] >= 0 && first[u] == at[u] && holders[u] == -1;
      const uint64_t mask = __ballot(gone);
      if (gone) back_here |= 1ull << turn;
      if (mask && lane() == 0) sback[turn][w] = __builtin_popcountll(mask);
    }
  };
  look(0, at0, page0);
  for (int e0 = kBatch * kOne; e0 < n_drop; e0 += kBatch * kOne) {
    int at[kBatch], page[kBatch];
    entries(sdrop, sfrom, A.B, n_drop, e0, at, page);
    look(e0, at, page);
  }
  __syncthreads();
  const int mine = backs[tid];
  const long ranks = scan_one(pair(mine, copy), swave, all);
  const int n_back = hi_of(all), n_copy = lo_of(all), rank = lo_of(ranks) - copy;
  const long back = min((long)n_back, had);  // what the list has room for
  if (tid == 0) A.taken_out[0] = (int)min(had - back + n_copy, 0x7fffffffl);
  if (n_back) {
    backs[tid] = hi_of(ranks) - mine;
    __syncthreads();
    auto give = [&](int e0, const int (&page)[kBatch]) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int turn = e0 / kOne + u;
        const bool gone = back_here >> turn & 1;
        const uint64_t mask = __ballot(gone);
        if (gone) {
          const long place = sback[turn][w] + __builtin_popcountll(mask & ((1ull << lane()) - 1));
          A.shared_out[page[u]] = 0;
          if (place < back) A.free_out[had - back + place] = page[u];
        }
      }
    };
    give(0, page0);
    for (int e0 = kBatch * kOne; e0 < n_drop; e0 += kBatch * kOne) {
      int at[kBatch], page[kBatch];
      entries(sdrop, sfrom, A.B, n_drop, e0, at, page);
      give(e0, page);
    }
  }
  if (copy) atomicSub(&A.shared_out[g.last], 1);  // others hold it on: it is not given back
  if (n_copy) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // the list is whole
    __syncthreads();
  }
  if (tid < A.B2) {
    int got = -1;
    if (copy) {
      got = page_at(A, had - back + rank);
      take(A, tid, g, got);
    }
    A.where[tid] = got;
  }
}

// The same of many, each step a launch of a workgroup per place
__global__ __launch_bounds__(kThreads) void k_fork_count(ForkArgs A) {
  const int r = blockIdx.x, tid = threadIdx.x;
  if (r < A.B) {
    const ForkOld o = A.old[r];
    for (int j = o.kept + tid; j < o.held; j += kThreads) drop(A, r, j);
  }
  if (r >= A.B2) return;
  const ForkNew g = A.fresh[r];
  if (g.counted)
    for (int j = tid; j < g.pages; j += kThreads) add(A, g.source, j);
  if (tid == 0 && g.last >= 0) {
    atomicAdd(&A.writers[g.last], 1);
    atomicMin(&A.writer[g.last], r);
  }
}

__global__ __launch_bounds__(kThreads) void k_fork_decide(ForkArgs A) {
  __shared__ int scount;
  GDN_POISON_LDS(scount);
  const int r = blockIdx.x, tid = threadIdx.x;
  if (r < A.B2 && tid == 0) A.copied[r] = takes_copy(A, r, A.fresh[r]);
  if (r >= A.B) return;
  const ForkOld o = A.old[r];
  if (tid == 0) scount = 0;
  __syncthreads();
  int n = 0, p;
  for (int j = o.kept + tid; j < o.held; j += kThreads) n += gives_back(A, r, j, p);
#pragma unroll
  for (int d = 32; d; d /= 2) n += __shfl_xor(n, d);
  if (lane() == 0) atomicAdd(&scount, n);
  __syncthreads();
  if (tid == 0) A.freed[r] = scount;
}

// sums of freed and of copied before place r, and of all of them
struct Sums {
  int freed, copied, all_freed, all_copied;
};
__device__ __forceinline__ Sums sums_before(const ForkArgs& A, int r, int (*ssum)[4]) {
  int v[4] = {0, 0, 0, 0};
  for (int b = threadIdx.x; b < A.B; b += kThreads) {
    const int n = A.freed[b];
    v[2] += n;
    if (b < r) v[0] += n;
  }
  for (int i = threadIdx.x; i < A.B2; i += kThreads) {
    const int n = A.copied[i] != 0;
    v[3] += n;
    if (i < r) v[1] += n;
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
#pragma unroll
    for (int d = 32; d; d /= 2) v[x] += __shfl_xor(v[x], d);
    if (lane() == 0) ssum[wave()][x] = v[x];
  }
  __syncthreads();
  Sums s{0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    s.freed += ssum[w][0];
    s.copied += ssum[w][1];
    s.all_freed += ssum[w][2];
    s.all_copied += ssum[w][3];
  }
  return s;
}

__global__ __launch_bounds__(kThreads) void k_fork_push(ForkArgs A) {
  __shared__ int ssum[kThreads / 64][4], srank[kThreads / 64];
  GDN_POISON_LDS(ssum, srank);
  const int r = blockIdx.x, tid = threadIdx.x;
  const Sums s = sums_before(A, r, ssum);
  const long had = min((long)max(A.taken[0], 0), A.n_free);
  const long back = min((long)s.all_freed, had);  // what the list has room for
  if (r == 0 && tid == 0) A.taken_out[0] = (int)min(had - back + s.all_copied, 0x7fffffffl);
  if (r < A.B2 && tid == 0) {
    const bool copy = A.copied[r] != 0;
    A.where[r] = copy ? (int)min(had - back + s.copied, 0x7fffffffl) : -1;
    if (copy) atomicSub(&A.shared_out[A.fresh[r].last], 1);  // others hold it on: it is not given back
  }
  if (r >= A.B) return;
  const ForkOld o = A.old[r];
  long rank = s.freed;
  for (int j0 = o.kept; j0 < o.held; j0 += kThreads) {
    const int j = j0 + tid;
    int p = -1;
    const bool gone = j < o.held && gives_back(A, r, j, p);
    const uint64_t mask = __ballot(gone);
    if (lane() == 0) srank[wave()] = __builtin_popcountll(mask);
    __syncthreads();
    long at = rank + __builtin_popcountll(mask & ((1ull << lane()) - 1));
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < wave()) at += srank[w];
      rank += srank[w];
    }
    if (gone) {
      A.shared_out[p] = 0;  // (read by this entry alone from here on)
      if (at < back) A.free_out[had - back + at] = p;
    }
    __syncthreads();
  }
}

struct ForkCopyArgs {
  Caches c;
  ForkArgs f;
  int layers;
  bool known, first;  // where names pages; of the launches (the first takes them)
};

// Bound by memory: the last pages of 192 samples, 6 layers of 4 heads of 256 in pages of 64, 215 MB, 51 us, 4.2 TB/s (a large copy has 5.0).
// The copies: a workgroup per new place, cache, group of columns and kCopyTurns times the tokens that its threads have on their way at
// once. The free list is whole by now: a copy may take a page that
// was given back (which no copy is made of: what writers leave is held by others).
constexpr int kCopyTurns = 4, UN = 4;
template <class W>
__global__ __launch_bounds__(kThreads) void k_fork_copy(ForkCopyArgs A) {
  const ForkArgs& F = A.f;
  const int r = blockIdx.x, tid = threadIdx.x;
  const int at = F.where[r];
  if (at < 0) return;
  const ForkNew g = F.fresh[r];
  const int got = A.known ? at : page_at(F, at);
  if (!A.known && A.first && blockIdx.y == 0 && tid == 0) take(F, r, g, got);
  if (!A.layers || got < 0) return;
  const int group = blockIdx.y % A.c.groups, cache = blockIdx.y / A.c.groups, layer = cache / 2;
  const bool values = cache % 2;
  const int cols = A.c.cols, step = kThreads / cols, mine = tid / cols, col = group * cols + tid % cols;
  if (mine >= step || col >= A.c.per) return;
  const long keep = F.lengths_out[r];
  const int count = (int)(keep - (g.pages - 1) * F.page.d);
  const int z0 = blockIdx.z * kCopyTurns * UN * step, z1 = min(count, z0 + kCopyTurns * UN * step);
  for (int t0 = z0 + mine; t0 < z1; t0 += UN * step) {
    W x[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (t0 + i * step < z1) x[i] = *reinterpret_cast<const W*>(A.c.at(layer, values, g.last, t0 + i * step, col, sizeof(W)));
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (t0 + i * step < z1) *reinterpret_cast<W*>(A.c.at(layer, values, got, t0 + i * step, col, sizeof(W))) = x[i];
  }
}

// the workgroups that share out a page's tokens
long copy_parts(int page, int cols) {
  const long turn = kCopyTurns * UN * (kThreads / cols);
  return (page + turn - 1) / turn;
}

int check(const tjev_gdn_pages_params* p, void* const* k, void* const* v, bool caches) {
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->requests < 1 || p->table_width < 1 || p->page_size < 1 || p->pages < 1 || p->layers < 0)
    return fail(TJEV_GDN_EINVAL, "requests, table_width, pages and page_size must be positive, layers not negative");
  if (p->requests > TJEV_GDN_MAX_REQUESTS || p->new_requests > TJEV_GDN_MAX_REQUESTS)
    return fail(TJEV_GDN_EUNSUPPORTED, "block tables of up to 8192 requests");
  if (!caches || !p->layers) return 0;
  if ((p->dtype | 1) != 1) return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16");
  if (p->kv_heads < 1 || p->dim < 1) return fail(TJEV_GDN_EINVAL, "kv_heads and dim must be positive");
  if ((long)p->kv_heads * p->dim >= (1l << 24)) return fail(TJEV_GDN_EUNSUPPORTED, "kv_heads * dim too large");
  if (!k || !v) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  for (int l = 0; l < p->layers; ++l)
    if (!k[l] || !v[l]) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  return 0;
}

// The caches' addresses are given launch by launch; the width of a vector (16 bytes where every address and stride allows it), and
// how a token's are shared out
int fill(Caches& c, const tjev_gdn_pages_params* p, void* const* k, void* const* v) {
  const int bytes = p->dtype == TJEV_GDN_BF16 ? 2 : 4;
  c.kp = p->k_stride[0] * bytes, c.ks = p->k_stride[1] * bytes, c.kh = p->k_stride[2] * bytes;
  c.vp = p->v_stride[0] * bytes, c.vs = p->v_stride[1] * bytes, c.vh = p->v_stride[2] * bytes;
  long any = (long)p->dim * bytes | c.kp | c.ks | c.kh | c.vp | c.vs | c.vh;
  for (int l = 0; l < p->layers; ++l) any |= (long)reinterpret_cast<uintptr_t>(k[l]) | (long)reinterpret_cast<uintptr_t>(v[l]);
  if (any % bytes) return 0;
  const int w = any % 16 == 0 ? 16 : bytes;
  c.chunks = p->dim * bytes / w;
  c.per = c.chunks * p->kv_heads;
  c.cols = c.per < kThreads ? c.per : kThreads;
  c.groups = (c.per + c.cols - 1) / c.cols;
  return w;
}

// the same, refused before anything is launched; without layers there is one column of nothing
int layout(Caches& c, int& w, const tjev_gdn_pages_params* p, void* const* k, void* const* v) {
  c.groups = c.cols = 1;
  w = 16;
  if (p->layers && !(w = fill(c, p, k, v))) return fail(TJEV_GDN_EINVAL, "the caches must be aligned to their elements");
  if (2l * kLayers * c.groups > 65535) return fail(TJEV_GDN_EUNSUPPORTED, "kv_heads * dim too large");
  return 0;
}

// launch(W, caches of the launch, layers of the launch, whether it is the first) for every kLayers layers, once at least
template <class F>
int by_layers(const tjev_gdn_pages_params* p, Caches c, int w, void* const* k, void* const* v, F launch) {
  for (int l0 = 0; l0 == 0 || l0 < p->layers; l0 += kLayers) {
    const int n = p->layers - l0 < kLayers ? p->layers - l0 : kLayers;
    for (int l = 0; l < n; ++l) c.k[l] = static_cast<char*>(k[l0 + l]), c.v[l] = static_cast<char*>(v[l0 + l]);
    if (w == 16) {
      launch(uint4{}, c, n, l0 == 0);
    } else if (w == 4) {
      launch(uint32_t{}, c, n, l0 == 0);
    } else {
      launch(uint16_t{}, c, n, l0 == 0);
    }
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
}

}  // namespace
}  // namespace gdn

extern "C" {

int tjev_gdn_paged_compact(const tjev_gdn_pages_params* p, void* stream, void* const* k_caches, void* const* v_caches,
                           const int32_t* block_table, const int32_t* starts, const int32_t* lengths, const int32_t* path,
                           const int32_t* kept, int32_t* lengths_out) {
  using gdn::fail;
  if (int s = gdn::check(p, k_caches, v_caches, true)) return s;
  if (p->max_new < 1) return fail(TJEV_GDN_EINVAL, "max_new must be positive");
  if (p->max_new >= (1l << 31)) return fail(TJEV_GDN_EINVAL, "problem too large");
  if (!block_table || !starts || !lengths || !path || !kept || !lengths_out) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  if (lengths_out == lengths) return fail(TJEV_GDN_EINVAL, "lengths_out must not alias lengths (every workgroup reads it)");
  hipStream_t st = static_cast<hipStream_t>(stream);
  gdn::CompactArgs A{};
  A.B = p->requests, A.M = p->table_width, A.pages = p->pages, A.most = p->max_new;
  A.page = gdn::div_by(p->page_size);
  A.table = block_table, A.starts = starts, A.lengths = lengths, A.path = path, A.kept = kept;
  gdn::Caches caches{};
  int w = 0;
  if (int s = gdn::layout(caches, w, p, k_caches, v_caches)) return s;
  return gdn::by_layers(p, caches, w, k_caches, v_caches, [&](auto w, const gdn::Caches& c, int layers, bool first) {
    A.c = c;
    A.layers = layers;
    A.lengths_out = first ? lengths_out : nullptr;
    const int y = 2 * layers * c.groups;
    hipLaunchKernelGGL((gdn::k_paged_compact<decltype(w)>), dim3(A.B, y ? y : 1), dim3(gdn::kThreads), 0, st, A);
  });
}

size_t tjev_gdn_fork_workspace_bytes(const tjev_gdn_pages_params* p) {
  if (gdn::check(p, nullptr, nullptr, false) || p->new_requests < 1) return 0;
  return sizeof(gdn::ForkNew) * p->new_requests + sizeof(gdn::ForkOld) * p->requests +
         sizeof(int32_t) * (3 * (size_t)p->pages + p->requests + 2 * (size_t)p->new_requests);
}

int tjev_gdn_paged_fork(const tjev_gdn_pages_params* p, void* stream, void* const* k_caches, void* const* v_caches,
                        const int32_t* block_table, const int32_t* lengths, const int32_t* sources, const int32_t* keep,
                        const int32_t* free_pages, const int32_t* taken, const int32_t* shared, int32_t* table_out, int32_t* lengths_out,
                        int32_t* free_out, int32_t* taken_out, int32_t* shared_out, void* workspace, size_t workspace_bytes) {
  using gdn::fail;
  if (int s = gdn::check(p, k_caches, v_caches, true)) return s;
  if (p->new_requests < 1 || p->n_free < 0) return fail(TJEV_GDN_EINVAL, "new_requests must be positive, n_free not negative");
  if (p->n_free >= (1l << 31) || (long)p->requests * p->table_width >= (1l << 31) || (long)p->new_requests * p->table_width >= (1l << 31))
    return fail(TJEV_GDN_EINVAL, "problem too large");
  if (p->layers && p->page_size >= (1 << 20)) return fail(TJEV_GDN_EUNSUPPORTED, "forks copy last pages of less than 2^20 tokens");
  if (!block_table || !lengths || !sources || !taken || !shared || !table_out || !lengths_out || !taken_out || !shared_out ||
      (p->n_free && (!free_pages || !free_out)))
    return fail(TJEV_GDN_EINVAL, "null tensor argument");
  if (table_out == block_table || lengths_out == lengths || (p->n_free && free_out == free_pages) || taken_out == taken || shared_out == shared)
    return fail(TJEV_GDN_EINVAL, "the outputs must not alias the inputs");
  const size_t need = tjev_gdn_fork_workspace_bytes(p);
  if (!workspace || workspace_bytes < need) return fail(TJEV_GDN_EWORKSPACE, "forks need a workspace of tjev_gdn_fork_workspace_bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TJEV_GDN_EINVAL, "the workspace must be 256-byte aligned");
  gdn::Caches caches{};
  int w = 0;
  if (int s = gdn::layout(caches, w, p, k_caches, v_caches)) return s;
  const long parts = p->layers ? gdn::copy_parts(p->page_size, caches.cols) : 1;
  if (parts > 65535) return fail(TJEV_GDN_EUNSUPPORTED, "forks copy last pages of up to 2^20 - 16 tokens of more than 128 vectors each");
  if (int s = gdn::poison_workspace(workspace, need, stream)) return s;
  gdn::ForkCopyArgs C{};
  gdn::ForkArgs& A = C.f;
  A = {p->requests, p->new_requests, p->table_width, p->pages, p->n_free, gdn::div_by(p->page_size), block_table, lengths, sources, keep,
       free_pages, taken, shared, table_out, lengths_out, free_out, taken_out, shared_out};
  A.fresh = static_cast<gdn::ForkNew*>(workspace);
  A.old = reinterpret_cast<gdn::ForkOld*>(A.fresh + p->new_requests);
  A.writers = reinterpret_cast<int32_t*>(A.old + p->requests);
  A.writer = A.writers + p->pages;
  A.entry = A.writer + p->pages;
  A.freed = A.entry + p->pages;
  A.copied = A.freed + p->requests;
  A.where = A.copied + p->new_requests;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int places = A.B > A.B2 ? A.B : A.B2;
  const long most = p->pages > p->n_free ? p->pages : p->n_free, blocks = (most + 4 * gdn::kThreads - 1) / (4 * gdn::kThreads);
  const dim3 block(gdn::kThreads);
  hipLaunchKernelGGL(gdn::k_fork_init, dim3((unsigned)std::max((long)places, std::min(blocks, 1024l))), block, 0, st, A);
  const long entries = (long)std::max(A.B, A.B2) * A.M;
  C.known = places <= gdn::kOne && entries <= gdn::kOne * (keep ? gdn::kOneTurns : gdn::kFewTurns);
  if (C.known) {
    hipLaunchKernelGGL(gdn::k_fork_one, dim3(1), dim3(gdn::kOne), 0, st, A);
    if (!p->layers) {
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
    }
  } else {
    hipLaunchKernelGGL(gdn::k_fork_count, dim3(places), block, 0, st, A);
    hipLaunchKernelGGL(gdn::k_fork_decide, dim3(places), block, 0, st, A);
    hipLaunchKernelGGL(gdn::k_fork_push, dim3(places), block, 0, st, A);
  }
  return gdn::by_layers(p, caches, w, k_caches, v_caches, [&](auto w, const gdn::Caches& c, int layers, bool first) {
    C.c = c;
    C.layers = layers;
    C.first = first;
    const int y = 2 * layers * c.groups;
    hipLaunchKernelGGL((gdn::k_fork_copy<decltype(w)>), dim3(A.B2, y ? y : 1, (unsigned)parts), block, 0, st, C);
  });
}

}  // extern "C"
