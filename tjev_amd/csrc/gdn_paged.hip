// The bookkeeping of the paged key/value cache for gfx950: block tables and slot maps from the requests'
// lengths, and the write of new keys and values into their slots.
//
// Tables: with e_b the pages of request b's cached tokens and f_b those of all its tokens, its new
// pages are free[taken + sum_{i<b} (f_i - e_i) + ...]; the new tokens' rows start at the running sum of the
// new lengths. One launch: the two running sums over the requests are short (8 bytes a request), so
// every workgroup forms both in its LDS from the lengths, and then writes its share of the table and of the slots, a
// token's request found by bisection. What bounds it is the launch and that chain (load, scan, bisection);
// the bytes are few.
//
// Append: bound by memory, every vector of 16 bytes loaded and stored once, one at a time per lane and
// enough waves to cover it: 16000 tokens of 8 key heads of 128 (131 MB) take 21.7 us (6.0 TB/s, part of it from the last
// level cache). Two to eight vectors in flight per lane took 28 to 35 us (their addresses went to scratch memory).
#include <hip/hip_runtime.h>

#include "../../include/tjev_gdn.h"
#include "gdn_device.h"
#include "gdn_launch.h"
#include "gdn_paged.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;

struct TableArgs {
  int B, M;
  Div page, width;
  long N, n_free;
  const int32_t *cached, *fresh, *table, *free, *taken;
  int32_t* table_out;
  int64_t* slots;
  int32_t *starts, *lengths, *taken_out;
};

__device__ __forceinline__ int clamp_int(long v) { return (int)(v < 0 ? 0 : v > 0x7fffffffl ? 0x7fffffffl : v); }
// pages of n tokens, at most the table's width
__device__ __forceinline__ int pages_of(long n, const TableArgs& A) {
  const long p = A.page(n + A.page.d - 1);
  return (int)(p < A.M ? p : A.M);
}

template <int CAP>
__global__ __launch_bounds__(kThreads) void k_paged_tables(TableArgs A) {
  __shared__ int sstart[CAP + 1];  // first token of each request
  __shared__ int spage[CAP + 1];   // its first taken page, counted from `taken`
  __shared__ long swave[2][kThreads / 64];
  GDN_POISON_LDS(sstart, spage, swave);
  const int tid = threadIdx.x;
  // a thread sums a run of requests, the waves' sums are scanned by shuffles
  const int run = (A.B + kThreads - 1) / kThreads, b0 = tid * run, b1 = min(A.B, b0 + run);
  long tok = 0, pg = 0;
  for (int b = b0; b < b1; ++b) {
    const long c = clamp_int(A.cached[b]), n = clamp_int(A.fresh[b]);
    tok += n;
    pg += pages_of(c + n, A) - pages_of(c, A);
  }
  long it = tok, ip = pg;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long t = __shfl_up(it, d), p = __shfl_up(ip, d);
    if (lane() >= d) it += t, ip += p;
  }
  if (lane() == 63) swave[0][wave()] = it, swave[1][wave()] = ip;
  __syncthreads();
  for (int w = 0; w < wave(); ++w) it += swave[0][w], ip += swave[1][w];
  tok = it - tok;
  pg = ip - pg;
  for (int b = b0; b < b1; ++b) {
    sstart[b] = clamp_int(tok);
    spage[b] = clamp_int(pg);
    const long c = clamp_int(A.cached[b]), n = clamp_int(A.fresh[b]);
    tok += n;
    pg += pages_of(c + n, A) - pages_of(c, A);
  }
  if (tid == kThreads - 1) {  // the last thread's run ends the sums, empty or not
    sstart[A.B] = clamp_int(tok);
    spage[A.B] = clamp_int(pg);
  }
  __syncthreads();
  const long taken = A.taken ? clamp_int(A.taken[0]) : 0;
  auto fresh_page = [&](long at) { return at < A.n_free ? A.free[at] : -1; };
  if (blockIdx.x == 0) {
    for (int b = tid; b <= A.B; b += kThreads) {
      A.starts[b] = sstart[b];
      if (b < A.B) A.lengths[b] = clamp_int((long)clamp_int(A.cached[b]) + clamp_int(A.fresh[b]));
    }
    if (tid == 0) A.taken_out[0] = clamp_int(taken + spage[A.B]);
  }
  const long stride = (long)gridDim.x * kThreads, id = (long)blockIdx.x * kThreads + tid;
  const bool keep = A.table_out == A.table;
  for (long i = id; i < (long)A.B * A.M; i += stride) {
    const int b = (int)A.width(i), j = (int)(i - (long)b * A.M);
    const long c = clamp_int(A.cached[b]), n = clamp_int(A.fresh[b]);
    const int e = pages_of(c, A), f = pages_of(c + n, A);
    if (j >= e && j < f) {
      A.table_out[i] = fresh_page(taken + spage[b] + (j - e));
    } else if (!keep) {
      A.table_out[i] = j < e ? A.table[i] : -1;
    }
  }
  for (long t = id; t < A.N; t += stride) {
    long slot = -1;
    if (t < sstart[A.B]) {
      int lo = 0, hi = A.B;  // the last request that starts at t or before, and is not empty
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sstart[mid] <= t) lo = mid; else hi = mid;
      }
      const long c = clamp_int(A.cached[lo]), pos = c + (t - sstart[lo]), j = A.page(pos);
      if (j < A.M) {
        const int e = pages_of(c, A);
        const long p = j < e ? A.table[(long)lo * A.M + j] : fresh_page(taken + spage[lo] + (j - e));
        if (p >= 0) slot = p * A.page.d + (pos - j * A.page.d);
      }
    }
    A.slots[t] = slot;
  }
}

struct AppendArgs {
  long N, n_slots;
  Div page;
  int per, half, chunks, tile;  // vectors of a token: of k and v, of each; of a head; tokens per workgroup
  unsigned inv_per, inv_chunks;       // 2^32 / per, / chunks rounded up
  const void* src[2];
  void* dst[2];
  const int64_t* slots;
  long st[2], sh[2];                  // bytes: token and head of the new rows
  long dp[2], ds[2], dh[2];           // bytes: page, slot and head of the caches
};

// n / d for n d < 2^32, inv = ceil(2^32 / d)
__device__ __forceinline__ int divide(int n, unsigned inv, int d) { return d == 1 ? n : (int)__umulhi((unsigned)n, inv); }

template <class W>
__global__ __launch_bounds__(kThreads) void k_paged_append(AppendArgs A) {
  const long t0 = (long)blockIdx.x * A.tile;
  const int count = (int)min((long)A.tile, A.N - t0) * A.per;
  for (int u = threadIdx.x; u < count; u += kThreads) {
    const int tok = divide(u, A.inv_per, A.per), r = u - tok * A.per, which = r >= A.half, x = which ? r - A.half : r;
    const int h = divide(x, A.inv_chunks, A.chunks), c = x - h * A.chunks;
    // on its way while the slot is looked up
    const W v = *reinterpret_cast<const W*>(static_cast<const char*>(A.src[which]) + (t0 + tok) * A.st[which] + h * A.sh[which] +
                                            c * (long)sizeof(W));
    const long slot = A.slots[t0 + tok];
    if (slot >= 0 && slot < A.n_slots) {
      const long p = A.page(slot), o = slot - p * A.page.d;
      *reinterpret_cast<W*>(static_cast<char*>(A.dst[which]) + p * A.dp[which] + o * A.ds[which] + h * A.dh[which] + c * (long)sizeof(W)) = v;
    }
  }
}

}  // namespace
}  // namespace gdn

extern "C" {

int tjev_gdn_paged_tables(const tjev_gdn_paged_params* p, void* stream, const int32_t* cached, const int32_t* new_tokens,
                          const int32_t* block_table, const int32_t* free_pages, int64_t n_free, const int32_t* taken,
                          int32_t* table_out, int64_t* slots, int32_t* starts, int32_t* lengths, int32_t* taken_out) {
  using gdn::fail;
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->requests < 1 || p->table_width < 1 || p->page_size < 1 || p->tokens < 0 || n_free < 0)
    return fail(TJEV_GDN_EINVAL, "requests, table_width and page_size must be positive, tokens and n_free not negative");
  if (p->requests > TJEV_GDN_MAX_REQUESTS) return fail(TJEV_GDN_EUNSUPPORTED, "block tables of up to 8192 requests");
  if (p->tokens >= (1l << 31) || n_free >= (1l << 31)) return fail(TJEV_GDN_EINVAL, "problem too large");
  if (!cached || !new_tokens || !block_table || (n_free && !free_pages) || !table_out || (p->tokens && !slots) || !starts ||
      !lengths || !taken_out)
    return fail(TJEV_GDN_EINVAL, "null tensor argument");
  if (taken == taken_out) return fail(TJEV_GDN_EINVAL, "taken_out must not alias taken (every workgroup reads it)");
  const gdn::TableArgs A{p->requests, p->table_width, gdn::div_by(p->page_size), gdn::div_by(p->table_width), p->tokens, n_free,
                         cached, new_tokens, block_table, free_pages, taken, table_out, slots, starts, lengths, taken_out};
  const long work = (long)p->requests * p->table_width + p->tokens;
  const long blocks = (work + 2047) / 2048;
  const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024)), block(gdn::kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->requests <= 256) {
    hipLaunchKernelGGL((gdn::k_paged_tables<256>), grid, block, 0, st, A);
  } else {
    hipLaunchKernelGGL((gdn::k_paged_tables<TJEV_GDN_MAX_REQUESTS>), grid, block, 0, st, A);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
}

int tjev_gdn_paged_append(const tjev_gdn_paged_params* p, void* stream, const void* k, const void* v, void* k_cache, void* v_cache,
                          const int64_t* slots) {
  using gdn::fail;
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->tokens < 0 || p->pages < 1 || p->page_size < 1 || p->kv_heads < 1 || p->dim < 1)
    return fail(TJEV_GDN_EINVAL, "pages, page_size, kv_heads and dim must be positive, tokens not negative");
  if ((p->dtype | 1) != 1) return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16");
  if (p->tokens >= (1l << 31)) return fail(TJEV_GDN_EINVAL, "problem too large");
  if (!p->tokens) return 0;
  if (!k || !v || !k_cache || !v_cache || !slots) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  const int bytes = p->dtype == TJEV_GDN_BF16 ? 2 : 4;
  gdn::AppendArgs A{};
  A.N = p->tokens;
  A.n_slots = (long)p->pages * p->page_size;
  A.page = gdn::div_by(p->page_size);
  A.slots = slots;
  const void* src[2] = {k, v};
  void* dst[2] = {k_cache, v_cache};
  const int64_t* sn[2] = {p->k_new_stride, p->v_new_stride};
  const int64_t* sc[2] = {p->k_stride, p->v_stride};
  long any = (long)p->dim * bytes;  // a 16-byte vector where every address and stride allows one
  for (int i = 0; i < 2; ++i) {
    A.src[i] = src[i];
    A.dst[i] = dst[i];
    A.st[i] = sn[i][0] * bytes;
    A.sh[i] = sn[i][1] * bytes;
    A.dp[i] = sc[i][0] * bytes;
    A.ds[i] = sc[i][1] * bytes;
    A.dh[i] = sc[i][2] * bytes;
    any |= (long)reinterpret_cast<uintptr_t>(src[i]) | (long)reinterpret_cast<uintptr_t>(dst[i]) | A.st[i] | A.sh[i] | A.dp[i] | A.ds[i] | A.dh[i];
  }
  if (any % bytes) return fail(TJEV_GDN_EINVAL, "k, v and the caches must be aligned to their elements");
  const int w = any % 16 == 0 ? 16 : bytes;
  const long chunks = (long)p->dim * bytes / w, per = 2 * p->kv_heads * chunks;
  if (per >= (1l << 16)) return fail(TJEV_GDN_EUNSUPPORTED, "kv_heads * dim too large");
  A.chunks = (int)chunks;
  A.per = (int)per;
  A.half = A.per / 2;
  A.inv_per = (unsigned)(((1ul << 32) + per - 1) / per);
  A.inv_chunks = (unsigned)(((1ul << 32) + chunks - 1) / chunks);
  A.tile = per >= 512 ? 1 : (int)(512 / per);
  const long blocks = (A.N + A.tile - 1) / A.tile;
  if (blocks >= (1l << 32) / gdn::kThreads) return fail(TJEV_GDN_EINVAL, "problem too large");  // a launch's threads
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(gdn::kThreads);
  if (w == 16) {
    hipLaunchKernelGGL((gdn::k_paged_append<uint4>), grid, block, 0, st, A);
  } else if (w == 4) {
    hipLaunchKernelGGL((gdn::k_paged_append<uint32_t>), grid, block, 0, st, A);
  } else {
    hipLaunchKernelGGL((gdn::k_paged_append<uint16_t>), grid, block, 0, st, A);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
}

}  // extern "C"
