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
// numbers (k_verify_sums; each finds the request's walk by itself), and the one slice that holds the token once more (k_verify_draw).
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
constexpr int kSlice = 4096;

struct VerifyArgs {
  long N, most, pt, qt;  // tokens; the most of a request; elements from row to row
  int B, V, slices;
  const int32_t *tokens, *parents, *starts;
  const float* u;
  const char *p, *q;     // q: null for chosen tokens
  int32_t *out, *path, *kept;
  double* sums;          // [B, slices]
  int* ends;             // [B, 2]: the row that the walk ends in, q's row or -1
  // the number of token i's parent within the request
  __device__ __forceinline__ int up(const Rows& r, long i) const { return parents ? parents[r.s0 + i] : (int)i - 1; }
};

template <class T>
__device__ __forceinline__ float number(const char* base, long at) {
  if constexpr (sizeof(T) == 2) return bf2f(reinterpret_cast<const uint16_t*>(base)[at]);
  return reinterpret_cast<const float*>(base)[at];
}
// what is no positive number counts as 0
__device__ __forceinline__ float clean(float x) { return x > 0.f && x < __builtin_inff() ? x : 0.f; }

// The walk of a request, by one wave: the node it ends in, and the child whose draft distribution is taken off (or -1).
// write: its path, accepted tokens and their number too.
struct End {
  long node, off;
};
template <class T, bool CHOSEN>
__device__ __forceinline__ End walk(const VerifyArgs& A, int b, const Rows& r, bool write) {
  const int ln = lane();
  const long n = min(r.n, A.most);
  int32_t *path = A.path + b * A.most, *out = A.out + b * A.most;
  End end{0, -1};
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
  return end;
}

// The rejected ones of chosen tokens in the slice from v0 on, as bits: all children of the node that the walk ended in.
__device__ __forceinline__ void reject(const VerifyArgs& A, const Rows& r, long node, long v0, uint32_t* sbits) {
  for (int i = threadIdx.x; i < kSlice / 32; i += kThreads) sbits[i] = 0;
  __syncthreads();
  const long n = min(r.n, A.most);
  for (long i = node + 1 + threadIdx.x; i < n; i += kThreads) {
    const long x = A.up(r, i) == node ? A.tokens[r.s0 + i] - v0 : -1;
    if (x >= 0 && x < kSlice) atomicOr(&sbits[x / 32], 1u << (x % 32));
  }
  __syncthreads();
}

// 16 bytes that start on an element
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
  T x[16 / sizeof(T)];
};

// the weights of the E numbers from v on; behind the row's end 0
template <class T, bool CHOSEN, int E>
__device__ __forceinline__ void weights(const VerifyArgs& A, const char* prow, const char* qrow, long v, const uint32_t* sbits, long v0,
                                        double (&w)[E]) {
  static_assert(E * sizeof(T) == 16, "");
  float p[E], q[E];
  if (v + E <= A.V) {
    const Piece<T> a = *reinterpret_cast<const Piece<T>*>(prow + v * sizeof(T));
    const Piece<T> c = qrow ? *reinterpret_cast<const Piece<T>*>(qrow + v * sizeof(T)) : Piece<T>{};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (sizeof(T) == 2) {
        p[e] = bf2f(a.x[e]);
        q[e] = bf2f(c.x[e]);
      } else {
        p[e] = a.x[e];
        q[e] = c.x[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      p[e] = v + e < A.V ? number<T>(prow, v + e) : 0.f;
      q[e] = qrow && v + e < A.V ? number<T>(qrow, v + e) : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double x = (double)clean(p[e]) - (double)clean(q[e]);
    w[e] = x > 0.0 ? x : 0.0;
    if (CHOSEN && sbits && (sbits[(v - v0 + e) / 32] >> ((v - v0 + e) % 32) & 1)) w[e] = 0.0;
  }
}

__device__ __forceinline__ double sum_wave(double v) {
#pragma unroll
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ double sum_block(double v, double* swave) {
  v = sum_wave(v);
  __syncthreads();
  if (lane() == 0) swave[wave()] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += swave[w];
  return s;
}
// running sum over the workgroup's threads, the whole, and what stands before the thread: the sum of the thread before it, bit by bit
__device__ __forceinline__ double scan_block(double v, double* swave, double& total, double& until) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double t = __shfl_up(v, d);
    if (lane() >= d) v += t;
  }
  until = __shfl_up(v, 1);
  if (lane() == 0) until = 0.0;
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

template <class T, bool CHOSEN>
__device__ __forceinline__ double slice_sum(const VerifyArgs& A, const char* prow, const char* qrow, long v0, const uint32_t* sbits,
                                            double* swave) {
  constexpr int E = 16 / sizeof(T), RUNS = kSlice / (kThreads * E);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    double w[E];
    weights<T, CHOSEN, E>(A, prow, qrow, v0 + (i * kThreads + threadIdx.x) * E, sbits, v0, w);
#pragma unroll
    for (int e = 0; e < E; ++e) s += w[e];
  }
  return sum_block(s, swave);
}

template <class T, bool CHOSEN>
__global__ __launch_bounds__(kThreads) void k_verify_sums(VerifyArgs A) {
  __shared__ double swave[kThreads / 64];
  __shared__ uint32_t sbits[kSlice / 32];
  __shared__ long send[2];
  GDN_POISON_LDS(swave, sbits, send);
  const int b = blockIdx.y, slice = blockIdx.x;
  const Rows r = rows_of(A.starts, b, A.N);
  if (uniform(wave()) == 0) {
    const End e = walk<T, CHOSEN>(A, b, r, slice == 0);
    if (lane() == 0) {
      send[0] = e.node;
      send[1] = e.off;
      if (slice == 0) A.ends[2 * b] = (int)e.node, A.ends[2 * b + 1] = (int)send[1];
    }
  }
  __syncthreads();
  if (!r.n) return;
  const long node = send[0], off = send[1], v0 = (long)slice * kSlice;
  if (CHOSEN) reject(A, r, node, v0, sbits);
  const char* prow = A.p + (r.s0 + node) * A.pt * (long)sizeof(T);
  const char* qrow = off >= 0 ? A.q + (r.s0 + off) * A.qt * (long)sizeof(T) : nullptr;
  const double s = slice_sum<T, CHOSEN>(A, prow, qrow, v0, sbits, swave);
  if (threadIdx.x == 0) A.sums[(long)b * A.slices + slice] = s;
}

// The first v whose running sum is over u times the whole: the slice by the slices' sums, then the place in it. Where rounding
// leaves none (or u is 1 or more), the last token with a weight; a row without any gives -1.
template <class T, bool CHOSEN>
__global__ __launch_bounds__(kThreads) void k_verify_draw(VerifyArgs A) {
  constexpr int E = 16 / sizeof(T), PER = kSlice / kThreads;
  __shared__ double swave[kThreads / 64];
  __shared__ uint32_t sbits[kSlice / 32];
  __shared__ double sbefore;
  __shared__ int sfound, slast;
  GDN_POISON_LDS(swave, sbits, sbefore, sfound, slast);
  const int b = blockIdx.x, tid = threadIdx.x;
  const Rows r = rows_of(A.starts, b, A.N);
  if (!r.n) return;
  const long node = A.ends[2 * b], off = A.ends[2 * b + 1];
  const char* prow = A.p + (r.s0 + node) * A.pt * (long)sizeof(T);
  const char* qrow = off >= 0 ? A.q + (r.s0 + off) * A.qt * (long)sizeof(T) : nullptr;
  double* sums = A.sums + (long)b * A.slices;
  bool rest = CHOSEN || qrow;  // something is taken off the row
  double total = 0.0;
  for (int turn = 0; turn < 2; ++turn) {
    double mine = 0.0;
    for (int s = tid; s < A.slices; s += kThreads) mine += sums[s];
    total = sum_block(mine, swave);
    if (total > 0.0 || !rest) break;
    // nothing is left: from the row itself, whose slices are summed here
    rest = false;
    qrow = nullptr;
    for (int s = 0; s < A.slices; ++s) {
      const double x = slice_sum<T, false>(A, prow, nullptr, (long)s * kSlice, nullptr, swave);
      if (tid == 0) sums[s] = x;
    }
    __threadfence_block();
    __syncthreads();
  }
  if (tid == 0) sfound = -1, slast = -1;
  __syncthreads();
  const double u = A.u[r.s0], goal = u > 0.0 ? u * total : 0.0;
  double before = 0.0;  // of the turns
  for (int s0 = 0; s0 < A.slices; s0 += kThreads) {
    const int s = s0 + tid;
    const double v = s < A.slices ? sums[s] : 0.0;
    double all, until;
    const double upto = before + scan_block(v, swave, all, until);
    until += before;
    if (v > 0.0) atomicMax(&slast, s);
    if (until <= goal && upto > goal) sfound = s, sbefore = until;  // one thread's

    before += all;
    __syncthreads();
    if (sfound >= 0) break;
  }
  const int slice = sfound >= 0 ? sfound : slast;
  const double start = sfound >= 0 ? sbefore : -1.0;
  __syncthreads();
  int32_t* out = A.out + b * A.most + A.kept[b] - 1;
  if (slice < 0) {
    if (tid == 0) *out = -1;
    return;
  }
  const long v0 = (long)slice * kSlice;
  const uint32_t* bits = CHOSEN && rest ? sbits : nullptr;
  if (CHOSEN && rest) reject(A, r, node, v0, sbits);
  if (tid == 0) sfound = 0x7fffffff, slast = -1;
  double w[PER], sum = 0.0;
  int last = -1;
#pragma unroll
  for (int i = 0; i < PER; i += E) {
    double x[E];
    weights<T, CHOSEN, E>(A, prow, qrow, v0 + tid * PER + i, bits, v0, x);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[i + e] = x[e];
      sum += x[e];
      if (x[e] > 0.0) last = i + e;
    }
  }
  double all, until;
  const double upto = scan_block(sum, swave, all, until);
  if (last >= 0) atomicMax(&slast, tid * PER + last);
  if (start >= 0.0 && start + upto > goal) {
    double run = start + until;
    int at = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      run += w[i];
      if (at < 0 && w[i] > 0.0 && run > goal) at = i;
    }
    if (at >= 0) atomicMin(&sfound, tid * PER + at);
  }
  __syncthreads();
  if (tid == 0) *out = (int)v0 + (sfound != 0x7fffffff ? sfound : slast);
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

// the ends, on 256 bytes, then the slices' sums
long slices_of(const tjev_gdn_draft_params* p) { return ((long)p->vocab + kSlice - 1) / kSlice; }
size_t ends_bytes(const tjev_gdn_draft_params* p) { return ((size_t)p->requests * 2 * sizeof(int) + 255) / 256 * 256; }

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
  return gdn::ends_bytes(p) + (size_t)p->requests * gdn::slices_of(p) * sizeof(double);
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
  char* ws = static_cast<char*>(workspace);
  const gdn::VerifyArgs A{p->tokens, p->max_new, p->target_stride, p->draft_stride, p->requests, p->vocab, (int)slices, tokens, parents, starts,
                          uniforms, static_cast<const char*>(target), static_cast<const char*>(draft), tokens_out, path, kept,
                          reinterpret_cast<double*>(ws + gdn::ends_bytes(p)), reinterpret_cast<int*>(ws)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 sums((unsigned)slices, (unsigned)p->requests), draw((unsigned)p->requests), block(gdn::kThreads);
  auto launch = [&](auto type, auto chosen) {
    using T = decltype(type);
    hipLaunchKernelGGL((gdn::k_verify_sums<T, chosen.value>), sums, block, 0, st, A);
    hipLaunchKernelGGL((gdn::k_verify_draw<T, chosen.value>), draw, block, 0, st, A);
  };
  if (e == 2) {
    draft ? launch(uint16_t{}, std::false_type{}) : launch(uint16_t{}, std::true_type{});
  } else {
    draft ? launch(float{}, std::false_type{}) : launch(float{}, std::true_type{});
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(err));
}

}  // extern "C"
