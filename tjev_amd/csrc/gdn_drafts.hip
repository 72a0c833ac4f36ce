// Drafted tokens of a served batch for gfx950: the ancestors and positions of a tree of them, and their verification
// against the target model's probabilities.
//
// Tree: with A_i the tokens that token i attends to among its request's new ones, A_i = {i} + A_parent(i). A wave per
// request takes 64 tokens at a time; within them the sets are joined by doubling (after round r a token's bits hold
// its 2^r nearest ancestors), and what lies before them comes from the row of the last ancestor there.
//
// Verification: p_i is the target's distribution behind token i, x_i the token, u_i a uniform number. From the root on,
// the children c of the node r where the walk stands are looked at in order:
//   tokens that were chosen (trees, chains)   c is accepted if u_c R < p_r(x_c), R = 1 - what the siblings before it had
//   tokens drawn from q_c (chains)            c is accepted if u_c q_c(x_c) < p_r(x_c)
// and the walk goes on from the first accepted one. Where none is, one more token is drawn from what is left,
//   w(v) = p_r(v) without the rejected tokens   or   max(p_r(v) - q_c(v), 0)   (p_r(v) where no child was looked at),
// as the first v whose running sum of w is over u_root times the whole. Every emitted token is then distributed as the
// target's. The sums and products are taken in 64 bits: a choice among 100000 tokens must not depend on the order of a sum.
// The rows that the last tokens are drawn from are read by as many workgroups as there are slices of kSlice
// numbers (k_verify_sums; each finds the request's walk by itself), and the one slice that holds the token once more (k_verify_draw,
// which loads what it needs to find it at once).
#include <hip/hip_runtime.h>

#include "../../include/tjev_gdn.h"
#include "gdn_device.h"
#include "gdn_launch.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * l, (int)(uint32_t)v), hi = __builtin_amdgcn_ds_bpermute(4 * l, (int)(uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | lo;
}

// rows starts[b] .. starts[b + 1] - 1, within the batch whatever the starts hold
struct Rows {
  long s0, n;
};
__device__ __forceinline__ Rows rows_of(const int32_t* starts, int b, long N) {
  const long a = starts[b], e = starts[b + 1];
  const long s0 = a < 0 ? 0 : a > N ? N : a, s1 = e < s0 ? s0 : e > N ? N : e;
  return {s0, s1 - s0};
}

// ---------------------------------------------------------------- the tree
struct TreeArgs {
  long N, most;
  int B, W;
  const int32_t *parents, *starts, *lengths;
  uint64_t* bits;
  int32_t* positions;
};

// Bound by latency: the parents, then six rounds of two exchanges within the wave for each 64 tokens, then the rows. 64 trees of 16 tokens
// take 3.0 us, 256 of up to 250, whose later tokens wait for the rows of the earlier ones, 7.4.
__global__ __launch_bounds__(64) void k_draft_tree(TreeArgs A) {
  const int ln = lane();
  if ((int)blockIdx.x >= A.B) {  // rows of no request
    const long b0 = A.starts[0], b1 = A.starts[A.B];
    const long lo = b0 < 0 ? 0 : b0 > A.N ? A.N : b0, hi = b1 < lo ? lo : b1 > A.N ? A.N : b1;
    for (long i = (long)(blockIdx.x - A.B) * 64 + ln; i < lo + (A.N - hi); i += (long)(gridDim.x - A.B) * 64) {
      const long row = i < lo ? i : hi + (i - lo);
      for (int w = 0; w < A.W; ++w) A.bits[row * A.W + w] = 0;
      A.positions[row] = 0;
    }
    return;
  }
  const int b = blockIdx.x;
  const Rows r = rows_of(A.starts, b, A.N);
  const long before = (long)A.lengths[b] - ((long)A.starts[b + 1] - A.starts[b]), first = before < 0 ? 0 : before;
  for (long i0 = 0; i0 < r.n; i0 += 64) {
    const long i = i0 + ln;
    const bool here = i < r.n && i < A.most;
    const long up = here ? A.parents[r.s0 + i] : -1, p = up >= 0 && up < i ? up : -1;
    uint64_t m = 1ull << ln;
    int jump = p >= i0 ? (int)(p - i0) : -1;
    const int above = p >= 0 && p < i0 ? (int)p : -1;  // the parent, before these 64 tokens
    while (__any(jump >= 0)) {
      const int j = jump < 0 ? ln : jump;
      const uint64_t mj = from_lane(m, j);
      const int jj = __builtin_amdgcn_ds_bpermute(4 * j, jump);
      if (jump >= 0) m |= mj, jump = jj;
    }
    const int top = __builtin_amdgcn_ds_bpermute(4 * (int)__builtin_ctzll(m), above);  // the first ancestor here has it
    long depth = __builtin_popcountll(m) - 1;
    if (i < r.n) {
      uint64_t* row = A.bits + (r.s0 + i) * A.W;
      const uint64_t* from = A.bits + (r.s0 + (top < 0 ? 0 : top)) * A.W;
      if (here && top >= 0) depth += 1 + A.positions[r.s0 + top] - first;
      const long k = i0 / 64;
      for (int w = 0; w < A.W; ++w) row[w] = !here || w > k ? 0 : w == k ? m : top < 0 ? 0 : from[w];
      A.positions[r.s0 + i] = here ? (int)min(first + depth, 0x7fffffffl) : 0;
    }
    __threadfence_block();  // the next tokens' ancestors are read from here
  }
}

// ---------------------------------------------------------------- verification
constexpr int kSlice = 4096, kPart = kSlice / (kThreads / 64);  // numbers of a workgroup, of a wave

struct VerifyArgs {
  long N, most, pt, qt;  // tokens; the most of a request; elements from row to row
  int B, V, slices, parts;
  const int32_t *tokens, *parents, *starts;
  const float* u;
  const char *p, *q;     // q: null for chosen tokens
  int32_t *out, *path, *kept;
  // for the second launch: where each walk ends, the parts' sums; of each slice whether it has rejected tokens, and those as bits
  struct WalkEnd* ends;
  double* sums;
  int32_t* marked;
  uint32_t* bits;
  // the number of token i's parent within the request
  __device__ __forceinline__ int up(const Rows& r, long i) const { return parents ? parents[r.s0 + i] : (int)i - 1; }
};

template <class T>
__device__ __forceinline__ float number(const char* base, long at) {
  if constexpr (sizeof(T) == 2) return bf2f(reinterpret_cast<const uint16_t*>(base)[at]);
  return reinterpret_cast<const float*>(base)[at];
}
// what is no positive number counts as 0
__device__ __forceinline__ float clean(float x) { return __builtin_amdgcn_classf(x, 0x180) ? x : 0.f; }  // positive, finite

// What the second launch needs of a request: the rows that its token is drawn from (q's: -1 for none; p's: -1 for a request
// without tokens), its number, and the place for the token
struct WalkEnd {
  long prow, qrow, out;
  double u;
};

// The walk of a request, by one wave: the node it ends in, the child whose draft distribution is taken off (or -1), and how many
// tokens it has. write: its path, accepted tokens and their number too. Children that are looked at stand in a chain, and each behind the
// first 64 tokens reads the ones before its group again (one tree of 50257 tokens in bf16, all but the root rejected: 16 of them
// 13.7 us, 64 23, 128 51, 256 146, 512 495).
struct End {
  long node, off, count;
};
template <class T, bool CHOSEN>
__device__ __forceinline__ End walk(const VerifyArgs& A, int b, const Rows& r, bool write) {
  const int ln = lane();
  const long n = min(r.n, A.most);
  int32_t *path = A.path + b * A.most, *out = A.out + b * A.most;
  End end{0, -1, 0};
  long count = 1;
  if (write && ln == 0 && n > 0) path[0] = 0;
  if constexpr (!CHOSEN) {
    for (long i0 = 1; i0 < n; i0 += 64) {
      const long i = i0 + ln;
      bool ok = false;
      int x = -1;
      if (i < n) {
        x = A.tokens[r.s0 + i];
        if (x >= 0 && x < A.V) {
          const float p = clean(number<T>(A.p, (r.s0 + i - 1) * A.pt + x));
          const float q = clean(number<T>(A.q, (r.s0 + i) * A.qt + x));
          ok = p > 0.f && (double)A.u[r.s0 + i] * q < (double)p;
        }
      }
      const uint64_t no = ~__ballot(ok);
      const int good = no ? __builtin_ctzll(no) : 64;
      if (write && ln < good) path[i] = (int)i, out[i - 1] = x;
      count += good;
      end.node = count - 1;
      if (good < 64) {
        if (count < n) end.off = count;
        break;
      }
    }
  } else {
    double left = 1.0;
    for (long i0 = 0; i0 < n; i0 += 64) {
      const long i = i0 + ln;
      int x = -1, up = -1;
      float p = 0.f, u = 0.f;
      if (i < n && i > 0) {
        x = A.tokens[r.s0 + i];
        up = A.up(r, i);
        u = A.u[r.s0 + i];
        if (up >= 0 && up < i && x >= 0 && x < A.V) p = clean(number<T>(A.p, (r.s0 + up) * A.pt + x));
      }
      int from = -1;  // the last child looked at
      while (true) {
        const uint64_t left_here = from < 63 ? ~0ull << (from + 1) : 0;
        const uint64_t kids = __ballot(up == end.node && i > end.node) & left_here;
        if (!kids) break;
        from = __builtin_ctzll(kids);
        const int xc = __builtin_amdgcn_readlane(x, from);
        float pc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), from));
        const float uc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(u), from));
        // a token that a sibling before it had is rejected already
        bool again = __ballot(up == end.node && i > end.node && x == xc && ln < from) != 0;
        for (long j0 = (end.node + 1) / 64 * 64; j0 < i0 && !again; j0 += 64) {
          const long j = j0 + ln;
          again = __any(j > end.node && A.up(r, j) == end.node && A.tokens[r.s0 + j] == xc);
        }
        if (again) pc = 0.f;
        if (pc > 0.f && (double)uc * (left > 0.0 ? left : 0.0) < (double)pc) {
          end.node = i0 + from;
          if (write && ln == 0) path[count] = (int)end.node, out[count - 1] = xc;
          ++count;
          left = 1.0;
        } else {
          left -= (double)pc;
        }
      }
    }
  }
  if (write) {
    if (!n) count = 0;
    for (long j = count + ln; j < A.most; j += 64) path[j] = out[j] = -1;
    if (ln == 0) A.kept[b] = (int)count;
  }
  end.count = count;
  return end;
}

// The rejected ones of chosen tokens in the slice from v0 on, as bits: all children of the node that the walk ended in. Whether there
// are any.
__device__ __forceinline__ bool reject(const VerifyArgs& A, const Rows& r, long node, long v0, uint32_t* sbits) {
  const long n = min(r.n, A.most);
  bool any = false;
  for (long i = node + 1 + threadIdx.x; i < n; i += kThreads) {
    const long x = A.up(r, i) == node ? A.tokens[r.s0 + i] - v0 : -1;
    if (x >= 0 && x < kSlice) {
      atomicOr(&sbits[x / 32], 1u << (x % 32));
      any = true;
    }
  }
  return __syncthreads_or(any);
}

// 16 bytes that start on an element
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
  uint64_t lo, hi;
};

// The E numbers of a row from v on, 0 behind its end: the row's last piece, moved down, without a branch to each number
template <class T, int E>
__device__ __forceinline__ void numbers(const VerifyArgs& A, const char* row, long v, float (&x)[E]) {
  constexpr int BITS = 8 * sizeof(T);
  static_assert(E * BITS == 128, "");
  uint64_t lo = 0, hi = 0;
  if (A.V >= E) {
    const long at = min(v, (long)A.V - E);
    const Piece<T> a = *reinterpret_cast<const Piece<T>*>(row + at * (long)sizeof(T));
    lo = a.lo, hi = a.hi;
    if (v > at) {
      const int n = (int)min((v - at) * BITS, 128l);
      lo = n < 64 ? lo >> n | hi << (64 - n) : n < 128 ? hi >> (n - 64) : 0;
      hi = n < 64 ? hi >> n : 0;
    }
  } else {
    for (int e = 0; e < A.V; ++e) {
      const uint64_t y = v + e < A.V ? reinterpret_cast<const std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>*>(row)[v + e] : 0;
      (e * BITS < 64 ? lo : hi) |= y << (e * BITS % 64);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t y = (uint32_t)((e * BITS < 64 ? lo : hi) >> (e * BITS % 64));
    x[e] = clean(__uint_as_float(sizeof(T) == 2 ? y << 16 : y));
  }
}

// the weights of the E numbers from v on; sbits: the rejected tokens from v0 on, or null
template <class T, bool CHOSEN, int E>
__device__ __forceinline__ void weights(const VerifyArgs& A, const char* prow, const char* qrow, long v, const uint32_t* sbits, long v0,
                                        double (&w)[E]) {
  float p[E];
  numbers<T>(A, prow, v, p);
  if constexpr (CHOSEN) {
    static_assert(32 % E == 0, "E numbers lie in one word: v is a multiple of E");
    const uint32_t off = sbits && v < A.V ? sbits[(v - v0) / 32] >> ((v - v0) % 32) : 0;
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = off >> e & 1 ? 0.f : p[e];
  } else if (qrow) {
    float q[E];
    numbers<T>(A, qrow, v, q);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double x = (double)p[e] - (double)q[e];
      w[e] = x > 0.0 ? x : 0.0;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = p[e];
  }
}

// the lane's number moved by a row shift (or broadcast) within the wave, 0 where none comes
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// running sum over the wave's lanes: within rows of 16, then each row's last to the row behind it, then the first half's last to the
// second
__device__ __forceinline__ double scan_wave(double v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
// running sum over the workgroup's threads, the whole, and what stands before the thread: the sum of the thread before it
__device__ __forceinline__ double scan_block(double v, double* swave, double& total, double& until) {
  v = scan_wave(v);
  until = moved<0x138, 0xf>(v);  // the lane before, 0 in the first
  __syncthreads();
  if (lane() == 63) swave[wave()] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave()) before += swave[w];
    total += swave[w];
  }
  until += before;
  return v + before;
}

// The first of a wave's lanes whose running sum is over the goal, or (over: false) the last with a weight, or -1
__device__ __forceinline__ int pick_lane(double mine, double upto, double goal, bool& over) {
  const uint64_t some = __ballot(mine > 0.0), first = __ballot(mine > 0.0 && upto > goal);
  over = first != 0;
  return first ? __builtin_ctzll(first) : some ? 63 - __builtin_clzll(some) : -1;
}
// The same among the workgroup's waves: the first of all in `found`, the last in `last`. (One lane of a wave adds to each: left to
// the compiler, an atomic of many lanes on one address is a loop over them.)
__device__ __forceinline__ void note(double mine, double upto, double goal, int at, int& found, int& last) {
  const uint64_t some = __ballot(mine > 0.0), first = __ballot(mine > 0.0 && upto > goal);
  if (some && lane() == 63 - __builtin_clzll(some)) atomicMax(&last, at);
  if (first && lane() == __builtin_ctzll(first)) atomicMin(&found, at);
}
// The same of numbers in a row, of which one is positive; run: the sum before them, then the sum before the one picked
template <int N>
__device__ __forceinline__ int pick(const double (&x)[N], double goal, bool over, double& run) {
  int found = 0;
  bool done = false;
  double sum = run;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (x[i] > 0.0 && !done) {
      found = i;
      run = sum;
      done = over && sum + x[i] > goal;
    }
    sum += x[i];
  }
  return found;
}

// The sum of a part of the row, by one wave, in its last lane
template <class T, bool CHOSEN>
__device__ __forceinline__ double part_sum(const VerifyArgs& A, const char* prow, const char* qrow, long from, const uint32_t* sbits, long v0) {
  constexpr int E = 16 / sizeof(T), RUNS = kPart / (64 * E);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    double w[E];
    weights<T, CHOSEN, E>(A, prow, qrow, from + (i * 64 + lane()) * E, sbits, v0, w);
#pragma unroll
    for (int e = 0; e < E; ++e) s += w[e];
  }
  return scan_wave(s);
}

// Bound by memory where the rows are long and many: 64 chains of 6 drawn from 128000 in fp32, 65.5 MB, 13.0 to 13.9 us, 5.0 to 4.7 TB/s. The
// walk, a chain of latencies (starts, tokens, their numbers), is covered by the other workgroups of the CU.
template <class T, bool CHOSEN>
__global__ __launch_bounds__(kThreads) void k_verify_sums(VerifyArgs A) {
  __shared__ uint32_t sbits[kSlice / 32];
  __shared__ long send[2];
  GDN_POISON_LDS(sbits, send);
  const int b = blockIdx.y, slice = blockIdx.x;
  const Rows r = rows_of(A.starts, b, A.N);
  if (CHOSEN)
    for (int i = threadIdx.x; i < kSlice / 32; i += kThreads) sbits[i] = 0;
  if (uniform(wave()) == 0) {
    const End e = walk<T, CHOSEN>(A, b, r, slice == 0);
    if (lane() == 0) {
      send[0] = e.node;
      send[1] = e.off;
      if (slice == 0)
        A.ends[b] = {r.n ? r.s0 + e.node : -1, e.off >= 0 ? r.s0 + e.off : -1, b * A.most + e.count - 1, r.n ? (double)A.u[r.s0] : 0.0};
    }
  }
  __syncthreads();
  if (!r.n) return;
  const long node = send[0], off = send[1], v0 = (long)slice * kSlice, at = (long)b * A.slices + slice;
  bool any = false;
  if (CHOSEN) {
    any = reject(A, r, node, v0, sbits);
    if (threadIdx.x == 0) A.marked[at] = any;
    if (any)
      for (int i = threadIdx.x; i < kSlice / 32; i += kThreads) A.bits[at * (kSlice / 32) + i] = sbits[i];
  }
  const char* prow = A.p + (r.s0 + node) * A.pt * (long)sizeof(T);
  const char* qrow = off >= 0 ? A.q + (r.s0 + off) * A.qt * (long)sizeof(T) : nullptr;
  const int part = slice * (kSlice / kPart) + uniform(wave());
  if ((long)part * kPart >= A.V) return;
  const double s = part_sum<T, CHOSEN>(A, prow, qrow, (long)part * kPart, any ? sbits : nullptr, v0);
  if (lane() == 63) A.sums[(long)b * A.parts + part] = s;
}

// The first v whose running sum is over u times the whole: the part by the parts' sums, then the place in it. Where rounding
// leaves none (or u is 1 or more), the last token with a weight; a row without any gives -1. Bound by latency, 4 us: the sums and the
// end, two scans, then 1024 numbers.
template <class T, bool CHOSEN>
__global__ __launch_bounds__(kThreads) void k_verify_draw(VerifyArgs A) {
  constexpr int E = 16 / sizeof(T);
  static_assert(kPart % E == 0 && kPart / E <= kThreads, "a part is one load of the workgroup's");
  __shared__ double swave[kThreads / 64], sbefore;
  __shared__ int sfound, slast;
  GDN_POISON_LDS(swave, sbefore, sfound, slast);
  const int b = blockIdx.x, tid = threadIdx.x;
  const WalkEnd end = A.ends[b];
  double* sums = A.sums + (long)b * A.parts;
  double mine = tid < A.parts ? sums[tid] : 0.0;  // on its way with the end
  if (end.prow < 0) return;
  const char* prow = A.p + end.prow * A.pt * (long)sizeof(T);
  const char* qrow = end.qrow >= 0 ? A.q + end.qrow * A.qt * (long)sizeof(T) : nullptr;
  int32_t* out = A.out + end.out;
  if (tid == 0) sfound = 0x7fffffff, slast = -1;
  bool rest = CHOSEN || qrow;  // something is taken off the row
  double total, goal;
  while (true) {
    // the first part over the goal, kThreads of them at a time (their whole first, where there are more)
    double before = 0.0, until, upto;
    if (A.parts > kThreads) {
      for (int s = tid + kThreads; s < A.parts; s += kThreads) mine += sums[s];
      scan_block(mine, swave, total, until);
      goal = end.u > 0.0 ? end.u * total : 0.0;
    }
    for (int s0 = 0; s0 < A.parts; s0 += kThreads) {
      const int s = s0 + tid;
      if (A.parts > kThreads) mine = s < A.parts ? sums[s] : 0.0;
      double all;
      upto = before + scan_block(mine, swave, all, until);
      if (A.parts <= kThreads) {
        total = all;
        goal = end.u > 0.0 ? end.u * total : 0.0;
      }
      note(mine, upto, goal, s, sfound, slast);
      __syncthreads();
      if (sfound == s) sbefore = before + until;
      if (sfound != 0x7fffffff) break;
      before += all;
    }
    if (total > 0.0 || !rest) break;
    // nothing is left: from the row itself, whose parts are summed here
    rest = false;
    qrow = nullptr;
    for (int s = uniform(wave()); s < A.parts; s += kThreads / 64) {
      const double x = part_sum<T, false>(A, prow, nullptr, (long)s * kPart, nullptr, 0);
      if (lane() == 63) sums[s] = x;
    }
    __syncthreads();
    mine = tid < A.parts ? sums[tid] : 0.0;
  }
  __syncthreads();
  bool over = sfound != 0x7fffffff;
  const int part = uniform(over ? sfound : slast);
  const double start = sbefore;
  if (part < 0) {
    if (tid == 0) *out = -1;
    return;
  }
  __syncthreads();
  if (tid == 0) sfound = 0x7fffffff, slast = -1;
  // the numbers of the part, E to a thread, and whether the rejected ones are among them
  const long v = (long)part * kPart + tid * E, at = (long)b * A.slices + part / (kSlice / kPart);
  double x[E] = {};
  if (tid < kPart / E) weights<T, false, E>(A, prow, qrow, v, nullptr, 0, x);
  if (CHOSEN && rest && A.marked[at] && tid < kPart / E) {
    const uint32_t off = A.bits[at * (kSlice / 32) + v % kSlice / 32] >> (v % 32);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (off >> e & 1) x[e] = 0.0;
  }
  mine = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += x[e];
  double all, until;
  const double upto = start + scan_block(mine, swave, all, until);
  note(mine, upto, over ? goal : __builtin_inf(), tid, sfound, slast);
  __syncthreads();
  over = sfound != 0x7fffffff;
  if (tid == (over ? sfound : slast)) {
    double run = start + until;
    *out = (int)v + pick(x, goal, over, run);
  }
}

// The walk and both passes over the row in one launch, a request to a workgroup of kOne threads, whose numbers' sums LDS holds.
constexpr int kOne = 1024, kOneRow = 1 << 16;

// Bound by latency: one tree of 24 over 50257 tokens in bf16 10.0 us: the walk, the row's 100 KB on one CU,
// and the token's 16 bytes once more, each behind the other.
template <class T, bool CHOSEN>
__global__ __launch_bounds__(kOne) void k_verify_one(VerifyArgs A) {
  constexpr int E = 16 / sizeof(T), NW = kOne / 64, TURNS = kOneRow / (kOne * E), AT_ONCE = 16 / E;
  __shared__ double sturn[TURNS][kOne];  // the threads' sums of each turn
  __shared__ uint32_t sbits[CHOSEN ? kOneRow / 32 : 1];
  __shared__ double ssum[NW];
  __shared__ long send[3];
  __shared__ int smarked;
  GDN_POISON_LDS(sturn, sbits, ssum, send, smarked);
  const int b = blockIdx.x, tid = threadIdx.x, w = uniform(wave()), ln = lane();
  const Rows r = rows_of(A.starts, b, A.N);
  if (CHOSEN)
    for (int i = tid; i < (A.V + 31) / 32; i += kOne) sbits[i] = 0;
  if (tid == 0) smarked = 0;
  if (w == 0) {
    const End e = walk<T, CHOSEN>(A, b, r, true);
    if (ln == 0) send[0] = e.node, send[1] = e.off, send[2] = e.count;
  }
  __syncthreads();
  if (!r.n) return;
  const long node = send[0], off = send[1];
  const double u = A.u[r.s0];
  if (CHOSEN) {
    const long n = min(r.n, A.most);
    for (long i = node + 1 + tid; i < n; i += kOne) {
      const int x = A.up(r, i) == node ? A.tokens[r.s0 + i] : -1;
      if (x >= 0 && x < A.V) {
        atomicOr(&sbits[x / 32], 1u << (x % 32));
        smarked = 1;
      }
    }
    __syncthreads();
  }
  const char* prow = A.p + (r.s0 + node) * A.pt * (long)sizeof(T);
  const char* qrow = off >= 0 ? A.q + (r.s0 + off) * A.qt * (long)sizeof(T) : nullptr;
  int32_t* out = A.out + b * A.most + send[2] - 1;
  const uint32_t* bits = CHOSEN && smarked ? sbits : nullptr;
  // A wave has a part of the row to itself, `turns` times 64 E numbers side by side: its sum is one of 16
  const int turns = (A.V + kOne * E - 1) / (kOne * E);
  const long v0 = (long)w * turns * 64 * E + ln * E;
  while (true) {
    double mine = 0.0;
    for (int t0 = 0; t0 < turns; t0 += AT_ONCE) {
      double x[AT_ONCE][E];
#pragma unroll
      for (int t = 0; t < AT_ONCE; ++t)
        if (t0 + t < turns) weights<T, CHOSEN, E>(A, prow, qrow, v0 + (t0 + t) * 64 * E, bits, 0, x[t]);
#pragma unroll
      for (int t = 0; t < AT_ONCE; ++t)
        if (t0 + t < turns) {
          double s = 0.0;
#pragma unroll
          for (int e = 0; e < E; ++e) s += x[t][e];
          sturn[t0 + t][tid] = s;
          mine += s;
        }
    }
    mine = scan_wave(mine);
    if (ln == 63) ssum[w] = mine;
    __syncthreads();
    // every wave sums the 16, and knows whether the token is its own
    const double of = ln < NW ? ssum[ln] : 0.0;
    double upto = scan_wave(of), until = moved<0x138, 0xf>(upto);
    const double total = __shfl(upto, NW - 1), goal = u > 0.0 ? u * total : 0.0;
    bool over;
    const int at = pick_lane(of, upto, goal, over);
    if (at < 0 && (bits || qrow)) {  // nothing is left: from the row itself
      bits = nullptr;
      qrow = nullptr;
      __syncthreads();
      continue;
    }
    if (at < 0 && tid == 0) *out = -1;
    if (w != at) return;
    double before = __shfl(until, at);
    // the turn: the first that goes over the goal, or the last with a weight
    int turn = -1;
    double start = 0.0;
    for (int t = 0; t < turns && (turn < 0 || !over || !(before > goal)); ++t) {
      const double s = sturn[t][tid];
      if (!__any(s > 0.0)) continue;
      turn = t;
      start = before;
      before += __shfl(scan_wave(s), 63);
    }
    const long v = v0 + turn * 64 * E;
    double x[E];
    weights<T, CHOSEN, E>(A, prow, qrow, v, bits, 0, x);
    mine = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += x[e];
    upto = scan_wave(mine);
    double run = start + moved<0x138, 0xf>(upto);
    if (ln == pick_lane(mine, start + upto, over ? goal : __builtin_inf(), over)) *out = (int)v + pick(x, goal, over, run);
    return;
  }
}

int check(const tjev_gdn_draft_params* p) {
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->requests < 1 || p->tokens < 0 || p->max_new < 1)
    return fail(TJEV_GDN_EINVAL, "requests and max_new must be positive, tokens not negative");
  if (p->requests > (1 << 24)) return fail(TJEV_GDN_EUNSUPPORTED, "drafts of up to 2^24 requests");
  if (p->tokens >= (1l << 31) || p->max_new >= (1l << 31) || p->max_new * p->requests >= (1l << 40))
    return fail(TJEV_GDN_EINVAL, "problem too large");
  return 0;
}

int check_verify(const tjev_gdn_draft_params* p) {
  if (int s = check(p)) return s;
  if (p->requests > 65535) return fail(TJEV_GDN_EUNSUPPORTED, "drafts of up to 65535 requests are verified");
  if (p->vocab < 1) return fail(TJEV_GDN_EINVAL, "vocab must be positive");
  if ((p->dtype | 1) != 1) return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16");
  return 0;
}

// Whether a call's requests are verified by a workgroup each, in one launch: where a row is read in about the time that the second
// launch would take (chosen tokens of 50257 in bf16, 1 to 256 requests: 12.1 us, in two launches 14.1; of 65536 in fp32, 64: 13.4, 14.3; drawn
// ones, two rows of it, 16.6, 14.8), and every CU has one request at most, which is as many workgroups as its LDS holds (1024 requests of
// drawn ones of 32000 in bf16: 39.3, 29.5).
constexpr int kOneRequests = 256, kOneBytes = 1 << 18;
bool in_one(const tjev_gdn_draft_params* p, long row_bytes) {
  return p->vocab <= kOneRow && p->requests <= kOneRequests && row_bytes <= kOneBytes;
}

long slices_of(const tjev_gdn_draft_params* p) { return ((long)p->vocab + kSlice - 1) / kSlice; }
long parts_of(const tjev_gdn_draft_params* p) { return ((long)p->vocab + kPart - 1) / kPart; }
// the workspace: the ends, the parts' sums, the slices' bits and marks
size_t lay_out(const tjev_gdn_draft_params* p, VerifyArgs* A, char* ws) {
  const size_t n = (size_t)p->requests * slices_of(p), sums = p->requests * parts_of(p), ends = p->requests * sizeof(WalkEnd);
  if (A) {
    A->ends = reinterpret_cast<WalkEnd*>(ws);
    A->sums = reinterpret_cast<double*>(ws + ends);
    A->bits = reinterpret_cast<uint32_t*>(A->sums + sums);
    A->marked = reinterpret_cast<int32_t*>(A->bits + n * (kSlice / 32));
  }
  return ends + sums * sizeof(double) + n * (kSlice / 8 + sizeof(int32_t));
}

}  // namespace
}  // namespace gdn

extern "C" {

int tjev_gdn_draft_tree(const tjev_gdn_draft_params* p, void* stream, const int32_t* parents, const int32_t* starts,
                        const int32_t* lengths, int64_t* ancestors, int32_t* positions) {
  using gdn::fail;
  if (int s = gdn::check(p)) return s;
  if (!p->tokens) return 0;
  if (!parents || !starts || !lengths || !ancestors || !positions) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  const long words = (p->max_new + 63) / 64;
  if (words >= (1l << 24)) return fail(TJEV_GDN_EINVAL, "problem too large");
  const gdn::TreeArgs A{p->tokens, p->max_new, p->requests, (int)words, parents, starts, lengths, reinterpret_cast<uint64_t*>(ancestors),
                        positions};
  const long clear = (p->tokens + 63) / 64;
  hipLaunchKernelGGL(gdn::k_draft_tree, dim3((unsigned)(p->requests + (clear < 64 ? clear : 64))), dim3(64), 0,
                     static_cast<hipStream_t>(stream), A);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
}

size_t tjev_gdn_verify_workspace_bytes(const tjev_gdn_draft_params* p) {
  if (gdn::check_verify(p)) return 0;
  return gdn::lay_out(p, nullptr, nullptr);
}

int tjev_gdn_verify_drafts(const tjev_gdn_draft_params* p, void* stream, const int32_t* tokens, const int32_t* parents,
                           const int32_t* starts, const float* uniforms, const void* target, const void* draft, int32_t* tokens_out,
                           int32_t* path, int32_t* kept, void* workspace, size_t workspace_bytes) {
  using gdn::fail;
  if (int s = gdn::check_verify(p)) return s;
  if (!starts || !tokens_out || !path || !kept || (p->tokens && (!tokens || !uniforms || !target)))
    return fail(TJEV_GDN_EINVAL, "null tensor argument");
  if (parents && draft) return fail(TJEV_GDN_EINVAL, "draft probabilities are of chains: a tree's tokens are chosen, not drawn");
  const size_t need = tjev_gdn_verify_workspace_bytes(p);
  if (!workspace || workspace_bytes < need)
    return fail(TJEV_GDN_EWORKSPACE, "verification needs a workspace of tjev_gdn_verify_workspace_bytes");
  const long e = p->dtype == TJEV_GDN_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TJEV_GDN_EINVAL, "the workspace must be 256-byte aligned");
  if (reinterpret_cast<uintptr_t>(target) % e || reinterpret_cast<uintptr_t>(draft) % e)
    return fail(TJEV_GDN_EINVAL, "the probabilities must be aligned to their elements");
  if (int s = gdn::poison_workspace(workspace, need, stream)) return s;
  const long slices = gdn::slices_of(p);
  gdn::VerifyArgs A{p->tokens, p->max_new, p->target_stride, p->draft_stride, p->requests, p->vocab, (int)slices, (int)gdn::parts_of(p), tokens,
                    parents, starts, uniforms, static_cast<const char*>(target), static_cast<const char*>(draft), tokens_out, path, kept};
  gdn::lay_out(p, &A, static_cast<char*>(workspace));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 sums((unsigned)slices, (unsigned)p->requests), draw((unsigned)p->requests), block(gdn::kThreads);
  auto launch = [&](auto type, auto chosen) {
    using T = decltype(type);
    hipLaunchKernelGGL((gdn::k_verify_sums<T, chosen.value>), sums, block, 0, st, A);
    hipLaunchKernelGGL((gdn::k_verify_draw<T, chosen.value>), draw, block, 0, st, A);
  };
  auto one = [&](auto type, auto chosen) {
    hipLaunchKernelGGL((gdn::k_verify_one<decltype(type), chosen.value>), draw, dim3(gdn::kOne), 0, st, A);
  };
  if (gdn::in_one(p, p->vocab * e * (draft ? 2 : 1))) {
    if (e == 2) {
      draft ? one(uint16_t{}, std::false_type{}) : one(uint16_t{}, std::true_type{});
    } else {
      draft ? one(float{}, std::false_type{}) : one(float{}, std::true_type{});
    }
  } else if (e == 2) {
    draft ? launch(uint16_t{}, std::false_type{}) : launch(uint16_t{}, std::true_type{});
  } else {
    draft ? launch(float{}, std::false_type{}) : launch(float{}, std::true_type{});
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(err));
}

}  // extern "C"
