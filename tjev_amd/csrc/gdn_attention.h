// Causal attention of new tokens over the paged key/value cache for gfx950 (the full-attention layers
// that stand between the GDN layers), from one token per request to chunks of a prompt:
//   o_r = sum_k p_rk v_k / sum_k p_rk,  p_rk = 2^(c q_r k_k - m_r),  c = scale log2(e),
// one pass over the keys with the running maximum m_r and sum of each row in 32 bits.
//
// The query heads of a key head are rows of one tile beside its tokens, so a key is read once for all of them. Up to
// 16 or 32 rows a request (decoding) are bound by memory, and their keys and values stream straight into registers
// (stream_tile); more are bound by the products, and share tiles of 128 rows whose keys pass through LDS (wide_tile,
// bf16). All tiles of a batch are cut into as many equal ranges of work as workgroups fit the chip (gdn_paged.h); a
// tile that more than one range holds leaves its parts in the workspace for a second launch to join
// (k_attention_join). Two launches whatever the lengths, which only the GPU knows.
//
// Measured, bf16, with a gate but for the first, of several cards (beside the time that the cache and rows take at 5.12 TB/s, or the
// products at 1230 TFLOP/s: what a large copy and a large library product reach on the same card):
//   1 token over 4000, 16/4 heads of 256 (16 MB)                    16.5 us     3.2   two launches' latency
//   64 requests of up to 32768, 16/4 heads of 256 (1.57 GB)        300        307     memory, 5.2 TB/s
//   2048 tokens over 30000, 16/4 heads of 256 (1.04 TFLOP)        1100 to 1155  846   products, 900 to 945 TFLOP/s
//   a prompt of 4096, 32/4 heads of 256 (0.27 TFLOP)               344 to 366 224     products, 750 to 800 TFLOP/s, and the 1024
//                                                                                   tiles' starts and ends beside them
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "gdn_device.h"
#include "gdn_paged.h"

namespace gdn {

namespace {

constexpr int kThreads = 256;
constexpr float kNegInf = -__builtin_inff();

// ---------------------------------------------------------------- the stream's plan
// All units of a batch (gdn_paged.h) in a line (request, key head, tile, keys) are cut into G equal ranges, one
// per workgroup, so that requests of very different lengths keep every CU busy to the end, whatever
// the host knows of them.

// a value that is the same in all lanes, held once
__device__ __forceinline__ long uniform(long v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (long)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// one lane's value, held once
__device__ __forceinline__ int of_lane(int v, int from) { return __builtin_amdgcn_readlane(v, from); }
__device__ __forceinline__ long of_lane(long v, int from) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, from), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)v >> 32), from);
  return (long)((uint64_t)hi << 32 | lo);
}
// a request made of the values that f takes from q's
template <class F>
__device__ __forceinline__ Request each_of(const Request& q, F f) {
  return {f(q.s0), f(q.rows), f(q.tiles), f(q.tile_rows), f(q.keys), f(q.extra), f(q.blocks), f(q.y),
          {__builtin_bit_cast(double, f(__builtin_bit_cast(long, q.by_g.inv))), f(q.by_g.d)}, f(q.first), f(q.per_head), f(q.cost)};
}
__device__ __forceinline__ Request uniform(const Request& q) {
  return each_of(q, [](auto v) { return uniform(v); });
}

// The kernel's arguments read anew: what a tile needs of them is then held for the tile only, and not (spilled)
// across the whole kernel.
__device__ __forceinline__ const AttnArgs& arguments() {
  auto p = (const __attribute__((address_space(4))) AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttnArgs*)p;
}

// The lane, counted anew: values taken from it are not held (or spilled: a spilled value's load waits for all
// loads on their way) from before.
__device__ __forceinline__ int lane_anew() {
  int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(l));
  return l;
}

// the lane's value moved by a row shift (or broadcast) within the wave, 0 where none comes
template <int CTRL, int ROWS>
__device__ __forceinline__ long moved(long v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)v >> 32), CTRL, ROWS, 0xf, true);
  return (long)((uint64_t)hi << 32 | lo);
}
// inclusive running sum over the wave's lanes: within rows of 16, then each row's last to the row behind it, then
// the first half's last to the second (no LDS: a step is a few cycles, a shuffle's a hundred)
__device__ __forceinline__ long scan_wave(long v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

// inclusive running sum over the workgroup's threads (in order); total: the sum of all
__device__ __forceinline__ long scan_block(long v, long* swave, long& total) {
  v = scan_wave(v);
  __syncthreads();
  if (lane() == 63) swave[wave()] = v;
  __syncthreads();
  total = 0;
  long before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave()) before += swave[w];
    total += swave[w];
  }
  return v + before;
}

// What a workgroup finds out of the batch: the units of each range, the request that its range begins with and that
// request's first unit. b = -1: the range is empty.
struct Found {
  long total, each, unit;
  int b;
  Request q;
};
struct FoundLds {
  long swave[kThreads / 64], unit;
  int b;
  Request q;
};

// Up to 64 requests are read and summed by each wave for itself, more of them by the workgroup, in turns, twice.
template <int R, int KB>
__device__ __forceinline__ Found find_range(const AttnArgs& A, int range, FoundLds& f) {
  const int tid = threadIdx.x;
  Found r;
  auto load = [&](int b) { return b < A.B ? request<R, KB>(A, b) : Request{}; };
  if (A.B <= 64) {
    const Request q = load(lane());
    const long upto = scan_wave(q.cost);
    r.total = of_lane(upto, 63);
    r.each = r.total ? A.by_G(r.total + A.G - 1) : 1;
    const long place = range * r.each;
    const uint64_t here = __ballot(place >= upto - q.cost && place < upto);
    r.b = here ? __builtin_ctzll(here) : -1;
    if (here) {
      r.q = each_of(q, [&](auto v) { return of_lane(v, r.b); });
      r.unit = of_lane(upto, r.b) - r.q.cost;
    }
    return r;
  }
  if (tid == 0) f.b = -1;
  long mine = 0, sum = 0;
  for (int b0 = 0; b0 < A.B; b0 += kThreads) mine += load(b0 + tid).cost;
  scan_block(mine, f.swave, sum);
  r.total = sum;
  r.each = sum ? A.by_G(sum + A.G - 1) : 1;
  const long place = range * r.each;
  long before = 0;  // the turns' sum
  for (int b0 = 0; b0 < A.B && before <= place; b0 += kThreads) {
    const Request q = load(b0 + tid);
    const long upto = scan_block(q.cost, f.swave, sum) + before;
    before += sum;
    if (place >= upto - q.cost && place < upto) {
      f.b = b0 + tid;
      f.q = q;
      f.unit = upto - q.cost;
    }
  }
  __syncthreads();
  r.b = uniform(f.b);
  if (r.b >= 0) {
    r.q = uniform(f.q);
    r.unit = uniform(f.unit);
  }
  return r;
}

// ---------------------------------------------------------------- fragments
// Scores are computed transposed, 16 keys by 16 rows per MFMA, K from the first operand: a lane's four
// results are keys 4 (lane / 16) .. + 3 of row lane % 16, which is the layout of the second operand of
// out^T += V^T P^T when the contraction takes the keys in that order; V's fragments are read in the same
// order, straight from memory: a lane loads VE consecutive values of each of its keys, and value e of them
// is the first operand of the e-th MFMA (rows d = VE m + e). So neither P nor V passes through LDS; in bf16
// the 8 keys by 8 values of a lane are transposed by byte permutes.
template <class T, int DT>
struct Shape {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int KG = BF ? 2 : 1;                 // groups of 16 keys per step of a wave
  static constexpr int E = 16 / (int)sizeof(T);         // elements of a 16-byte piece
  static constexpr int KS = DT / (4 * E);               // pieces of a K or Q fragment row
  static constexpr int VE = BF && DT >= 128 ? 8 : 4;    // V's values per lane and key
  static constexpr int VH = DT / (16 * VE);
  static constexpr int KB = 64 * KG;                    // keys of a unit: a step of each of four waves
  using VVec = std::conditional_t<VE * sizeof(T) == 16, uint4, uint2>;
};

typedef uint32_t u32;
__device__ __forceinline__ u32 word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ u32 word(const uint2& v, int i) { return i == 0 ? v.x : v.y; }

template <class T, int DT>
__device__ __forceinline__ f32x4 dot_step(const uint4& k, const uint4& q, f32x4 acc) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(word(k, e)), __uint_as_float(word(q, e)), acc, 0, 0, 0);
    return acc;
  }
}

// f of the lane's value and that of the lane 32 (or 16) away: exchanged within the registers (through LDS a shuffle waits
// behind the fragments' reads)
template <class F>
__device__ __forceinline__ float with_far(float v, F f) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
template <class F>
__device__ __forceinline__ float with_near(float v, F f) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }
// max or sum over the four lanes that hold one row (lane % 16)
__device__ __forceinline__ float rows_max(float v) { return with_far(with_near(v, larger), larger); }
__device__ __forceinline__ float rows_sum(float v) { return with_far(with_near(v, sum_of), sum_of); }
// the base of the powers: 0 where a row has seen no key yet, so that its powers are 0 and not NaN
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.f : m; }

// Streamed rows' weights meet V, which is bf16, as two bf16 terms each, hi the first 8 bits and lo the rest (rounded:
// 2^-15 of the weight); the second product is free beside the loads. A weight's last bit is set first, so that lo is
// never 0 and an infinity of V stays one.
__device__ __forceinline__ Split2 split_weights(float a, float b) {
  const u32 x = __float_as_uint(a) | 1u, y = __float_as_uint(b) | 1u;
  return {__builtin_amdgcn_perm(y, x, 0x07060302u),
          pack2(__uint_as_float(x) - __uint_as_float(x & 0xffff0000u), __uint_as_float(y) - __uint_as_float(y & 0xffff0000u))};
}

// The wide tiles, bound by their products, round the weights to bf16; their sums, which stay in 32 bits, are of the rounded
// ones, so that a row's weights still add up to one.
__device__ __forceinline__ float sum_pair(u32 pair, float sum) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{(__bf16)1.f, (__bf16)1.f}, sum, false);
}

// out += P V for one step (KG groups of 16 keys). V [key group][r]: the lane's keys 4 (lane / 16) + r
template <class T, int DT, int NQ>
__device__ __forceinline__ void add_pv(const typename Shape<T, DT>::VVec (&v)[Shape<T, DT>::KG][4][Shape<T, DT>::VH],
                                       const f32x4 (&p)[Shape<T, DT>::KG][NQ],
                                       f32x4 (&o)[NQ][Shape<T, DT>::VH][Shape<T, DT>::VE]) {
  using S = Shape<T, DT>;
  if constexpr (S::BF) {
    bf16x8 hi[NQ], lo[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const Split2 a = split_weights(p[0][n][0], p[0][n][1]), b = split_weights(p[0][n][2], p[0][n][3]);
      const Split2 c = split_weights(p[1][n][0], p[1][n][1]), d = split_weights(p[1][n][2], p[1][n][3]);
      hi[n] = __builtin_bit_cast(bf16x8, make_uint4(a.hi, b.hi, c.hi, d.hi));
      lo[n] = __builtin_bit_cast(bf16x8, make_uint4(a.lo, b.lo, c.lo, d.lo));
    }
#pragma unroll
    for (int h = 0; h < S::VH; ++h)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) {
        const u32 sel = e % 2 ? 0x07060302u : 0x05040100u;
        u32 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(word(v[i / 2][2 * (i % 2) + 1][h], e / 2), word(v[i / 2][2 * (i % 2)][h], e / 2), sel);
        const bf16x8 a = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, lo[n], o[n][h][e], 0, 0, 0);
          o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, hi[n], o[n][h][e], 0, 0, 0);
        }
      }
  } else {
#pragma unroll
    for (int h = 0; h < S::VH; ++h)
#pragma unroll
      for (int e = 0; e < S::VE; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(word(v[0][r][h], e)), p[0][n][r], o[n][h][e], 0, 0, 0);
  }
}

template <class T, class W>
__device__ __forceinline__ bool not_finite(const W& v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(W) / 4); ++i) {
    const u32 w = word(v, i);
    if constexpr (sizeof(T) == 2) {
      bad = bad || (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
    } else {
      bad = bad || (w & 0x7f800000u) == 0x7f800000u;
    }
  }
  return bad;
}

// Infinities and NaN among values that some rows of a tile attend to and others do not: a product would
// give the others 0 * NaN. They are counted instead, by a product of marks (1 for infinity, 128 for minus infinity,
// 16384 for NaN; at most 64 of each, so the sum is exact) with ones for the keys a row attends to, and
// the counted values added to its result; the values themselves become 0.
__device__ __forceinline__ float special_of(float count) {
  const int n = (int)count;
  const float inf = __builtin_inff();
  const bool pos = n & 127, neg = (n >> 7) & 127, nan = n >> 14;
  return nan || (pos && neg) ? __builtin_nanf("") : pos ? inf : neg ? -inf : 0.f;
}
// the mark of one bf16 value (bits) as bf16 bits
__device__ __forceinline__ u32 mark_of(u32 h) {
  return (h & 0x7f80u) != 0x7f80u ? 0u : (h & 0x7fu) ? 0x4680u : (h & 0x8000u) ? 0x4300u : 0x3f80u;
}
__device__ __forceinline__ u32 marks_of(u32 w) { return mark_of(w & 0xffffu) | mark_of(w >> 16) << 16; }
__device__ __forceinline__ u32 finite_of(u32 w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

__device__ __forceinline__ void zero_word(uint4& v) { v = make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ void zero_word(uint2& v) { v = make_uint2(0, 0); }

__device__ __forceinline__ void set_word(uint4& v, int i, u32 w) { (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = w; }
__device__ __forceinline__ void set_word(uint2& v, int i, u32 w) { (i == 0 ? v.x : v.y) = w; }

template <class T, int DT>
using VStep = typename Shape<T, DT>::VVec[Shape<T, DT>::KG][4][Shape<T, DT>::VH];

template <class T, int DT, int NQ>
__device__ __forceinline__ void add_special(VStep<T, DT>& v,
                                            const bool (&on)[Shape<T, DT>::KG][4][NQ],
                                            f32x4 (&o)[NQ][Shape<T, DT>::VH][Shape<T, DT>::VE]) {
  using S = Shape<T, DT>;
#pragma unroll
  for (int h = 0; h < S::VH; ++h)
#pragma unroll
    for (int e = 0; e < S::VE; ++e)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if constexpr (S::BF) {
          u32 w[4], p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = i / 2, r = 2 * (i % 2), sh = 16 * (e % 2);
            w[i] = mark_of(word(v[j][r][h], e / 2) >> sh & 0xffffu) | mark_of(word(v[j][r + 1][h], e / 2) >> sh & 0xffffu) << 16;
            p[i] = (on[j][r][n] ? 0x3f80u : 0u) | (on[j][r + 1][n] ? 0x3f800000u : 0u);
          }
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3])),
                                                        __builtin_bit_cast(bf16x8, make_uint4(p[0], p[1], p[2], p[3])), acc, 0, 0, 0);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const u32 x = word(v[0][r][h], e);
            const float mark = (x & 0x7f800000u) != 0x7f800000u ? 0.f : (x & 0x7fffffu) ? 16384.f : (x >> 31) ? 128.f : 1.f;
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(mark, on[0][r][n] ? 1.f : 0.f, acc, 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][h][e][r] += special_of(acc[r]);
      }
#pragma unroll
  for (int j = 0; j < S::KG; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int h = 0; h < S::VH; ++h)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(typename S::VVec) / 4); ++i) {
          const u32 x = word(v[j][r][h], i);
          set_word(v[j][r][h], i, S::BF ? finite_of(x) : (x & 0x7f800000u) == 0x7f800000u ? 0u : x);
        }
}

// VE consecutive results of a row in every 16 VE of them, divided by the row's sum, gated, rounded once and stored
template <class T, int DT, bool PAD>
__device__ __forceinline__ void store_row(const AttnArgs& A, const float (&o)[Shape<T, DT>::VH][Shape<T, DT>::VE], float l, long token,
                                          int head, int d0) {
  using S = Shape<T, DT>;
  using G = std::conditional_t<S::VE == 8, Raw8<T>, Raw4<T>>;
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const T* gp = reinterpret_cast<const T*>(A.gate + token * A.gt + head * A.gh) + d0;
  T* op = reinterpret_cast<T*>(A.out + token * A.ot + head * A.oh) + d0;
  G gate[S::VH];  // all loaded before the first is used
  if (A.gate)
#pragma unroll
    for (int x = 0; x < S::VH; ++x)
      if (!PAD || d0 + x * 16 * S::VE < A.D) gate[x].load(gp + x * 16 * S::VE);
#pragma unroll
  for (int x = 0; x < S::VH; ++x) {
    if (PAD && d0 + x * 16 * S::VE >= A.D) continue;
    float y[S::VE];
#pragma unroll
    for (int e = 0; e < S::VE; ++e) y[e] = o[x][e] * inv;
    if (A.gate) {
      float gv[S::VE];
      gate[x].get(gv);
#pragma unroll
      for (int e = 0; e < S::VE; ++e) y[e] *= sigmoid_io<T>(gv[e]);
    }
    if constexpr (S::VE == 8) {
      st8_io(op + x * 16 * S::VE, y);
    } else {
      st4_io(op + x * 16 * S::VE, y);
    }
  }
}

// ---------------------------------------------------------------- the workgroups' ranges
// A range's first tile goes to slot 2 i of the workspace unless the range holds all its keys, its last, when it
// goes on behind the range's end, to slot 2 i + 1.
struct Part {
  float* p;       // where the tile's rows go, or null: they are finished here
  int tile, head;
};

template <int DT>
constexpr int slot_floats(int rows) { return rows * (DT + 2); }

// The tile that begins in a range and goes on behind it, for the kernel that joins its parts: the first lies in
// slot `first`, the others are the first ones of the next ranges. parts = 0: there is none.
struct Split {
  int parts, first, s0, rows, tile_rows, tile, head, pad;
};
static_assert(sizeof(Split) == kSplitBytes, "the workspace's last part");

__device__ __forceinline__ Split* split_of(const AttnArgs& A, int range) {
  return reinterpret_cast<Split*>(A.part + 2 * (size_t)A.G * A.slot) + range;
}

// the workgroup's i-th range: consecutive ranges stay on one XCD (its L2 holds the keys that they share)
__device__ __forceinline__ int range_of(int block, int G) { return G % 8 ? block : (block % 8) * (G / 8) + block / 8; }

// ---------------------------------------------------------------- few rows: keys streamed
// The four waves take steps of KG * 16 keys in turn, each with a running maximum, sum and result of its
// own, joined in LDS at the end. Bound by memory: the keys and values are read once, straight into registers (64 requests of
// up to 32768 tokens, 16/4 heads of 256, 128, 64: 5.2, 5.1, 4.7 TB/s), or by latency: one token over 4000 takes 11 us, of
// which its bytes are 3.
// WHOLE: pages hold whole groups of 16 keys, whose page is then one value per wave.
template <class T, int DT, int NQ>
struct StreamLds {
  static constexpr int NV = NQ * Shape<T, DT>::VH * Shape<T, DT>::VE;  // result registers of four
  static constexpr int Q = NQ * Shape<T, DT>::KS * 64, ACC = 2 * NV * 64;  // pieces of 16 bytes
};

template <class T, int DT, int NQ, bool PAD, bool WHOLE>
__device__ __forceinline__ void stream_tile(const Request& q, int b, const Part& part, int kb0, int seg, uint4* sq,
                                            f32x4* sacc, float (&sm)[4][16 * NQ], float (&sl)[4][16 * NQ]) {
  using S = Shape<T, DT>;
  constexpr int R = 16 * NQ, KB = S::KB, KG = S::KG, E = S::E;
  constexpr int NV = StreamLds<T, DT, NQ>::NV;
  const AttnArgs& A = arguments();
  const int w = __builtin_amdgcn_readfirstlane(wave()), ln = lane(), r16 = ln & 15, g4 = ln >> 4;
  const int row0 = part.tile * R, h = part.head;
  // The queries, staged once for the four waves in the order of the fragments: read first, stored (and waited for) when the
  // first keys and values are on their way
  constexpr int QN = (NQ * S::KS + 3) / 4;
  uint4 qv[QN];
#pragma unroll
  for (int y = 0; y < QN; ++y) {
    const int x = w + 4 * y, n = x / S::KS, i = x - n * S::KS, row = row0 + n * 16 + r16, e = (4 * i + g4) * E;
    qv[y] = make_uint4(0, 0, 0, 0);
    if (x < NQ * S::KS && row < q.rows && !(PAD && e >= A.D)) {
      const int t = A.by_g(row);
      qv[y] = *reinterpret_cast<const uint4*>(A.q + (long)(q.s0 + t) * A.qt + (h * A.g + (row - t * A.g)) * A.qh + e * (int)sizeof(T));
    }
  }
  bool staged = false;
  auto stage = [&]() {
#pragma unroll
    for (int y = 0; y < QN; ++y)
      if (w + 4 * y < NQ * S::KS) sq[(w + 4 * y) * 64 + ln] = qv[y];
    __syncthreads();
    staged = true;
  };
  int lim[NQ];  // the lane's row of each row tile: its last key + 1
  float m[NQ], l[NQ];
  f32x4 o[NQ][S::VH][S::VE];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + n * 16 + r16;
    lim[n] = row < q.rows ? row_limit(A, q, row) : 0;
    m[n] = kNegInf;
    l[n] = 0.f;
#pragma unroll
    for (int x = 0; x < S::VH; ++x)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) o[n][x][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int lo_lim = uniform(row_limit(A, q, row0)), hi_lim = uniform(row_limit(A, q, min(row0 + R, q.rows) - 1));
  const int32_t* table = A.table + (long)b * A.M;
  const char *kc = A.k + h * A.kh, *vc = A.v + h * A.vh;

  for (int kb = kb0; kb < kb0 + seg; ++kb) {
    const int k0 = kb * KB + w * 16 * KG;
    if (k0 >= hi_lim) break;
    uint4 kf[KG][S::KS];
    typename S::VVec vf[KG][4][S::VH];
    bool ok[KG][4];  // the lane's keys 4 g4 + r have a page
    bool all_ok = true;
#pragma unroll
    for (int j = 0; j < KG; ++j) {
      const int key0 = k0 + 16 * j;
      const char *krow, *vrow[4];
      if constexpr (WHOLE) {
        // the group lies in one page: its first key's, a group behind the last key the step's first one's
        const Place at = place_of(A, table, key0 < q.keys ? key0 : k0, q.keys);
        const long p = __builtin_amdgcn_readfirstlane(at.page), in = at.in;
        const bool good = __builtin_amdgcn_readfirstlane(at.good);
        all_ok = all_ok && good;
        krow = kc + p * A.kp + (in + r16) * A.ks;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          vrow[r] = vc + p * A.vp + (in + 4 * g4 + r) * A.vs;
          ok[j][r] = good;
        }
      } else {
        const Place at = place_of(A, table, key0 + r16, q.keys);
        krow = kc + at.page * A.kp + at.in * A.ks;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Place pv = place_of(A, table, key0 + 4 * g4 + r, q.keys);
          vrow[r] = vc + pv.page * A.vp + pv.in * A.vs;
          ok[j][r] = pv.good;
          all_ok = all_ok && pv.good;
        }
      }
#pragma unroll
      for (int i = 0; i < S::KS; ++i) {
        const int e = (4 * i + g4) * E;
        kf[j][i] = PAD && e >= A.D ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(krow + e * (int)sizeof(T));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < S::VH; ++x) {
          const int d = (16 * x + r16) * S::VE;
          if (PAD && d >= A.D) {
            zero_word(vf[j][r][x]);
          } else {
            vf[j][r][x] = *reinterpret_cast<const typename S::VVec*>(vrow[r] + d * (int)sizeof(T));
          }
        }
    }
    const bool bad_page = WHOLE ? !all_ok : __any(!all_ok);
    if (!staged) stage();

    f32x4 s[KG][NQ];
#pragma unroll
    for (int j = 0; j < KG; ++j)
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < S::KS; ++i)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const uint4 qf = sq[(n * S::KS + i) * 64 + ln];
#pragma unroll
        for (int j = 0; j < KG; ++j) s[j][n] = dot_step<T, DT>(kf[j][i], qf, s[j][n]);
      }
#pragma unroll
    for (int j = 0; j < KG; ++j)
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[j][n] *= A.c;
    const bool masked = k0 + 16 * KG > lo_lim || bad_page;
    bool careful = false;
    if (masked) {
#pragma unroll
      for (int j = 0; j < KG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k0 + 16 * j + 4 * g4 + r;
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[j][n][r] = key < lim[n] && ok[j][r] ? s[j][n][r] : kNegInf;
          // what no row attends to must not meet its zero weight: 0 * NaN
          if (key >= hi_lim || !ok[j][r])
#pragma unroll
            for (int x = 0; x < S::VH; ++x) zero_word(vf[j][r][x]);
        }
      if (lo_lim < hi_lim) {
#pragma unroll
        for (int j = 0; j < KG; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < S::VH; ++x) careful = careful || not_finite<T>(vf[j][r][x]);
        careful = __any(careful);
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float t = kNegInf;
#pragma unroll
      for (int j = 0; j < KG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) t = fmaxf(t, s[j][n][r]);
      const float mn = fmaxf(m[n], rows_max(t)), base = base_of(mn), a = __builtin_amdgcn_exp2f(m[n] - base);
      m[n] = mn;
      l[n] *= a;
#pragma unroll
      for (int j = 0; j < KG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[j][n][r] = __builtin_amdgcn_exp2f(s[j][n][r] - base);
#pragma unroll
      for (int j = 0; j < KG; ++j) l[n] += (s[j][n][0] + s[j][n][1]) + (s[j][n][2] + s[j][n][3]);
#pragma unroll
      for (int x = 0; x < S::VH; ++x)
#pragma unroll
        for (int e = 0; e < S::VE; ++e) o[n][x][e] *= a;
    }
    if (careful) {
      bool on[KG][4][NQ];
#pragma unroll
      for (int j = 0; j < KG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NQ; ++n) on[j][r][n] = k0 + 16 * j + 4 * g4 + r < lim[n];
      add_special<T, DT, NQ>(vf, on, o);
    }
    add_pv<T, DT, NQ>(vf, s, o);
  }

  if (!staged) stage();  // a wave without keys

  // The four waves' rows joined: of a lane's four results of each register, wave w ends with the w-th. Waves two
  // apart exchange halves (unscaled: their maxima are on their way too), then neighbours quarters, in the place
  // that only they have read; all four waves then store. (The halves added by waves 0 and 1, and by wave 0 alone:
  // five barriers instead of two, and one wave's stores.)
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = rows_sum(l[n]);
    if (g4 == 0) sm[w][n * 16 + r16] = m[n], sl[w][n * 16 + r16] = l[n];
  }
  const bool upper = w >> 1, odd = w & 1;
  float mj[NQ], lj[NQ], own[NQ], other[NQ], res[NQ][S::VH][S::VE];
  f32x4* const mine = sacc + w * (NV / 2) * 64 + ln;
  f32x4* const across = sacc + (w ^ 2) * (NV / 2) * 64 + ln;
  const f32x4* const beside = sacc + (w ^ 3) * (NV / 2) * 64 + ln;
  auto reg = [&](int v) -> f32x4& { return o[v / (S::VH * S::VE)][v / S::VE % S::VH][v % S::VE]; };
#pragma unroll
  for (int v = 0; v < NV; v += 2) {
    const f32x4 &x = reg(v), &y = reg(v + 1);
    mine[v / 2 * 64] = upper ? f32x4{x[0], x[1], y[0], y[1]} : f32x4{x[2], x[3], y[2], y[3]};
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    mj[n] = kNegInf;
#pragma unroll
    for (int i = 0; i < 4; ++i) mj[n] = fmaxf(mj[n], sm[i][n * 16 + r16]);
    const float base = base_of(mj[n]);
    lj[n] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) lj[n] += sl[i][n * 16 + r16] * __builtin_amdgcn_exp2f(sm[i][n * 16 + r16] - base);
    own[n] = __builtin_amdgcn_exp2f(m[n] - base);
    other[n] = __builtin_amdgcn_exp2f(sm[w ^ 2][n * 16 + r16] - base);
  }
  float keep[NV], send[NV];
#pragma unroll
  for (int v = 0; v < NV; v += 2) {
    const f32x4 t = across[v / 2 * 64];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = (v + j / 2) / (S::VH * S::VE);
      const f32x4& x = reg(v + j / 2);
      const float y = (upper ? x[2 + j % 2] : x[j % 2]) * own[n] + t[j] * other[n];
      if (j % 2 == 0) {
        keep[v + j / 2] = y;
      } else {
        const float z = keep[v + j / 2];
        keep[v + j / 2] = odd ? y : z;
        send[v + j / 2] = odd ? z : y;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < NV; v += 4) across[v / 4 * 64] = f32x4{send[v], send[v + 1], send[v + 2], send[v + 3]};
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NV; v += 4) {
    const f32x4 t = beside[v / 4 * 64];
#pragma unroll
    for (int j = 0; j < 4; ++j) res[(v + j) / (S::VH * S::VE)][(v + j) / S::VE % S::VH][(v + j) % S::VE] = keep[v + j] + t[j];
  }
  const int d0 = (4 * g4 + w) * S::VE;
  if (!part.p) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = row0 + n * 16 + r16, t = A.by_g(row);
      if (row < q.rows) store_row<T, DT, PAD>(A, res[n], lj[n], q.s0 + t, h * A.g + (row - t * A.g), d0);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int x = 0; x < S::VH; ++x)
#pragma unroll
        for (int e = 0; e < S::VE; e += 4)  // rows of DT values
          *reinterpret_cast<f32x4*>(part.p + (n * 16 + r16) * DT + d0 + x * 16 * S::VE + e) =
              f32x4{res[n][x][e], res[n][x][e + 1], res[n][x][e + 2], res[n][x][e + 3]};
      if (w == 0 && g4 == 0) {
        part.p[R * DT + n * 16 + r16] = mj[n];
        part.p[R * (DT + 1) + n * 16 + r16] = lj[n];
      }
    }
  }
}

// ---------------------------------------------------------------- many rows: tiles of 128 (bf16)
// Four waves of 32 rows each. K and V pass through LDS, TK keys at a time in two buffers, brought there by
// 16-byte loads that do not touch registers; scores are again transposed (32 keys by 32 rows per MFMA), so that a
// row's weights stay in its two lanes and are the second operand of out^T += V^T P^T as they come, V's
// fragments by transposing LDS reads. The pieces of a row of K or V lie in LDS in an order that depends on the row
// (swz), which spreads both kinds of read over the banks (no conflicts counted). Bound by the products and what
// stands between them: 2048 tokens over 30000 at head dims 256, 128, 64 run at 945, 944, 810 TFLOP/s (a
// warmer card 873, 877, 739), the matrix units busy for half of the cycles. The queries stay in registers (three fragments at 256 in LDS), the results too;
// two workgroups to a CU cover each other's softmax and barriers.
// The base of the powers follows the running maximum only when that has grown by more than 2^8: the rescaling
// of the results is skipped otherwise (a softmax does not depend on its base; weights up to 2^8 have bf16's
// relative precision like all others).
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

template <int DT>
struct Wide {
  static constexpr int TK = DT == 256 ? 32 : 64;  // keys per buffer
  static constexpr int NS = TK / 32, CPR = DT / 8, RW = TK / 4, RI = 64 / CPR, NI = RW / RI;
  static constexpr int QL = DT == 256 ? 3 : 0;  // fragments of a wave's queries kept in LDS: what the registers cannot hold
  static constexpr int SPAN = CPR >= 16 ? 256 : 128;  // bytes within which the pieces of a row are exchanged
  // the place of piece c of row r: c ^ swz(r)
  static constexpr __device__ __forceinline__ int swz(int r) {
    return CPR >= 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 1) << 2) | ((r >> 1) & 3);
  }
};

__device__ __forceinline__ i16x4 read_tr(const uint16_t* p) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
}

// the pieces of 16 bytes that a wave's lanes address, to consecutive places of LDS
__device__ __forceinline__ void load_to_lds(const char* from, uint16_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

template <int DT, bool PAD, bool WHOLE>
struct WideTile {
  using W = Wide<DT>;
  static constexpr int TK = W::TK, NS = W::NS;
  const AttnArgs& A;
  const Request& q;
  const int32_t* table;
  const char *kc, *vc;
  int w, k_first;
  u32 (*sbad)[4];  // [buffer][wave]: keys without a page

  // The table's entry for this wave's rows of the keys k0 .. k0 + TK - 1: of all of them (WHOLE: they lie in one
  // page; a group behind the last key stands for the range's first), or of the lane's. Loaded a buffer ahead of its use.
  __device__ __forceinline__ int first_key(int k0) const {
    const int key0 = k0 + w * W::RW;
    return key0 < q.keys ? key0 : k_first;
  }
  __device__ __forceinline__ int lane_key(int k0) const { return min(k0 + w * W::RW + lane_anew() % W::RW, q.keys - 1); }
  __device__ __forceinline__ int look(int k0) const { return table[page_of(A, WHOLE ? first_key(k0) : lane_key(k0))]; }

  // those rows on their way to LDS
  __device__ __forceinline__ void issue(int k0, int entry, int buf, uint16_t* sk, uint16_t* sv) const {
    const int ln = lane_anew(), rl = ln / W::CPR, pos = ln % W::CPR;
    const bool good = entry >= 0 && entry < A.pages;
    const int page = good ? entry : 0;
    const unsigned long bad = WHOLE ? (good ? 0ul : ~0ul) : __ballot(!good && ln < W::RW);
    if (ln == 0) sbad[buf][w] = (u32)bad;
    // a row's pieces are exchanged by swz(row): the lane's part of it, and below the part of i
    const u32 piece = (u32)(pos ^ W::swz(w * W::RW + rl)) << 4;
    if constexpr (WHOLE) {  // all rows lie in one page: a scalar base
      const int key = first_key(k0);
      const long p = __builtin_amdgcn_readfirstlane(page), in = uniform(key - page_of(A, key) * A.page);
      const char *kb = kc + p * A.kp + in * A.ks, *vb = vc + p * A.vp + in * A.vs;
      u32 kr = rl * (u32)A.ks, vr = rl * (u32)A.vs;
#pragma unroll
      for (int i = 0; i < W::NI; ++i, kb += W::RI * A.ks, vb += W::RI * A.vs) {
        const u32 c = piece ^ (u32)(W::swz(i * W::RI) << 4);
        if (!PAD || (int)c < 2 * A.D) {
          u32 ko = kr + c, vo = vr + c;
          asm volatile("" : "+v"(ko), "+v"(vo));  // 32 bits beside the scalar base, not 64 held for each row
          load_to_lds(kb + ko, sk + (w * W::RW + i * W::RI) * DT);
          load_to_lds(vb + vo, sv + (w * W::RW + i * W::RI) * DT);
        }
      }
    } else if (A.page % 8 == 0) {  // the rows of a load do
      const int in = lane_key(k0) - page_of(A, lane_key(k0)) * A.page;
#pragma unroll
      for (int i = 0; i < W::NI; ++i) {
        const long p = __builtin_amdgcn_readlane(page, i * W::RI), n = __builtin_amdgcn_readlane(in, i * W::RI);
        const u32 c = piece ^ (u32)(W::swz(i * W::RI) << 4);
        const u32 r = min(rl, (int)(A.page - 1 - n));  // rows behind the last key: none may lie past its page
        if (!PAD || (int)c < 2 * A.D) {
          u32 ko = r * (u32)A.ks + c, vo = r * (u32)A.vs + c;
          asm volatile("" : "+v"(ko), "+v"(vo));
          load_to_lds(kc + p * A.kp + n * A.ks + ko, sk + (w * W::RW + i * W::RI) * DT);
          load_to_lds(vc + p * A.vp + n * A.vs + vo, sv + (w * W::RW + i * W::RI) * DT);
        }
      }
    } else {
      const int key = lane_key(k0), in = key - page_of(A, key) * A.page;
#pragma unroll
      for (int i = 0; i < W::NI; ++i) {
        const u32 c = piece ^ (u32)(W::swz(i * W::RI) << 4);
        const long p = __shfl(page, i * W::RI + rl), n = __shfl(in, i * W::RI + rl);
        if (!PAD || (int)c < 2 * A.D) {
          load_to_lds(kc + p * A.kp + n * A.ks + c, sk + (w * W::RW + i * W::RI) * DT);
          load_to_lds(vc + p * A.vp + n * A.vs + c, sv + (w * W::RW + i * W::RI) * DT);
        }
      }
    }
  }
};

template <int DT, bool PAD, bool WHOLE>
__device__ __forceinline__ void wide_tile(const Request& q, int b, const Part& part, int kb0, int seg, uint16_t* sk0,
                                          uint16_t* sv0, uint16_t* sk1, uint16_t* sv1, uint4* sq, u32 (*sbad)[4]) {
  using W = Wide<DT>;
  using T = uint16_t;
  constexpr int TK = W::TK, NS = W::NS, KQ = DT / 16, ND = DT / 32, KB = 128, QL = W::QL;
  const AttnArgs& A = arguments();
  const int w = __builtin_amdgcn_readfirstlane(wave()), h = part.head, row0 = part.tile * kWideRows;
  // the lane's row: its token and head, the byte offset of its values (a row past the last: row 0's)
  auto place = [&](int l, bool& live, long& token, int& head) {
    const int row = row0 + w * 32 + l % 32, t = A.by_g(row);
    live = row < q.rows;
    token = q.s0 + (live ? t : 0);
    head = h * A.g + (live ? row - t * A.g : 0);
  };
  int lim;
  {
    const int row = row0 + w * 32 + lane_anew() % 32;
    lim = row < q.rows ? row_limit(A, q, row) : 0;
  }
  // limits of the wave's and of the workgroup's first and last rows
  const int wr = row0 + w * 32;
  const bool rows_w = wr < q.rows;  // a wave without rows only helps to bring K and V
  const int lo_w = uniform(rows_w ? row_limit(A, q, wr) : 0), hi_w = uniform(rows_w ? row_limit(A, q, min(wr + 32, q.rows) - 1) : 0);
  const int lo_g = uniform(row_limit(A, q, row0)), hi_g = uniform(row_limit(A, q, min(row0 + kWideRows, q.rows) - 1));
  const bool flip = A.c < 0.f;  // the scale's sign goes into q, which is exact
  const float c = flip ? -A.c : A.c;

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[d][x] = 0.f;
  float m = kNegInf, l = 0.f;

  const int k_first = kb0 * KB, k_end = min((kb0 + seg) * KB, hi_g);
  const WideTile<DT, PAD, WHOLE> tile{A, q, A.table + (long)b * A.M, A.k + h * A.kh, A.v + h * A.vh, w, k_first, sbad};
  if (PAD) {  // pieces past the head's dim are not loaded
    for (int x = threadIdx.x; x < TK * DT / 8; x += kThreads) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(sk0)[x] = reinterpret_cast<uint4*>(sk1)[x] = z;
      reinterpret_cast<uint4*>(sv0)[x] = reinterpret_cast<uint4*>(sv1)[x] = z;
    }
    __syncthreads();
  }

  int entry = 0;
  if (k_first < k_end) {  // the first keys are on their way while the queries are read
    tile.issue(k_first, tile.look(k_first), 0, sk0, sv0);
    entry = tile.look(k_first + TK);
  }
  bf16x8 qf[KQ - QL];
  {
  const int lq = lane_anew();
  bool live;
  long token;
  int head;
  place(lq, live, token, head);
#pragma unroll
  for (int i = 0; i < KQ; ++i) {
    const int e = i * 16 + lq / 32 * 8;
    uint4 v = make_uint4(0, 0, 0, 0);  // a row past the last reads row 0's: its results go nowhere
    if (!(PAD && e >= A.D)) v = *reinterpret_cast<const uint4*>(A.q + token * A.qt + head * A.qh + e * 2);
    if (flip) v.x ^= 0x80008000u, v.y ^= 0x80008000u, v.z ^= 0x80008000u, v.w ^= 0x80008000u;
    if (i < KQ - QL) {
      qf[i] = __builtin_bit_cast(bf16x8, v);
    } else {
      sq[(w * QL + i - (KQ - QL)) * 64 + lq] = v;  // read by this lane alone
    }
  }
  }
  // The lane's byte addresses in a buffer: its row of K's fragments, and of V's transposing reads. A piece's place is
  // then one exclusive or with a constant away (the buffers' rows are aligned to their length).
  static_assert(DT >= 64, "rows of 8 pieces and more");
  auto k_lane = [&](int l) { return (l % 32) * DT * 2 + (((l / 32) ^ W::swz(l % 32)) << 4); };
  auto v_lane = [&](int l) {
    const int r = 4 * (l / 32) + (l % 16) / 4, c = (l / 16 % 2) * 2 + (l & 3) / 2;
    return r * DT * 2 + ((c ^ W::swz(r)) << 4) + 8 * (l & 1);
  };

  int k_held = DT == 256 ? 0 : k_lane(lane_anew()), v_held = DT == 256 ? 0 : v_lane(lane_anew());
  // V's fragment: 32 values (d) by 16 keys, in the order of the weights' lanes
  auto v_frag = [&](const uint16_t* sv, int vl, int d, int n, int j) {
    i16x4 v[2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
      v[x] = read_tr(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(sv) +
                                                       (vl ^ ((d * 64) & (W::SPAN - 1)) ^ (W::swz(8 * x) << 4)) +
                                                       d * 64 / W::SPAN * W::SPAN + (n * 32 + 16 * j + 8 * x) * DT * 2));
    return __builtin_bit_cast(bf16x8, (i16x8){v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]});
  };
  // what no row attends to must not meet its zero weight (0 * NaN): values of keys behind the last row's last or
  // without a page become 0
  auto clear_unseen = [&](int k0, int buf, uint16_t* sv) {
    for (int x = threadIdx.x; x < TK * W::CPR; x += kThreads) {
      const int r = x / W::CPR;
      if (k0 + r >= hi_g || (sbad[buf][r / W::RW] >> (r % W::RW)) & 1) reinterpret_cast<uint4*>(sv)[x] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  };
  bool special = false;  // infinities or NaN where some rows attend and others do not

  auto compute = [&](int k0, int buf, uint16_t* sk, uint16_t* sv) {
    const bool live = k0 < hi_w;  // a wave without rows, or whose rows end before, only helps
    u32 any_bad = 0;  // read by now, looked at behind the scores
#pragma unroll
    for (int i = 0; i < 4; ++i) any_bad |= sbad[buf][i];
    // at head dim 256 taken anew for each buffer: what is held across the loop must fit the registers
    const int la = lane_anew(), kl = DT == 256 ? k_lane(la) : k_held, vl = DT == 256 ? v_lane(la) : v_held;
    f32x16 s[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int x = 0; x < 16; ++x) s[n][x] = 0.f;
    // Fragments are read AHEAD - 1 products before their own: left to itself the compiler reads them all first, which
    // runs it out of registers. At head dim 256 a fragment has one product, not two, to hide the next one's read
    // (2048 new tokens over 30000, 16/4 heads: 1192 us with AHEAD = 2, 1165 with 4, 1333 with 6, which spills).
    constexpr int AHEAD = DT == 256 ? 4 : 2;
    bf16x8 kf[AHEAD][NS];
    auto read_k = [&](int i) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
        kf[i % AHEAD][n] = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(sk) + (kl ^ ((i * 32) & (W::SPAN - 1))) +
                                                            i * 32 / W::SPAN * W::SPAN + n * 32 * DT * 2);
    };
    if (live) {
#pragma unroll
      for (int i = 0; i < AHEAD - 1; ++i) read_k(i);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        if (i + AHEAD - 1 < KQ) read_k(i + AHEAD - 1);
        const bf16x8 qi = i < KQ - QL ? qf[i < KQ - QL ? i : 0] : __builtin_bit_cast(bf16x8, sq[(w * QL + i - (KQ - QL)) * 64 + la]);
#pragma unroll
        for (int n = 0; n < NS; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % AHEAD][n], qi, s[n], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    any_bad = __builtin_amdgcn_readfirstlane(any_bad);
    const bool edge = k0 + TK > lo_g || any_bad;  // not all rows attend to all keys
    if (edge && (k0 + TK > hi_g || any_bad)) clear_unseen(k0, buf, sv);
    if (edge && k0 + TK > lo_g && lo_g < hi_g) {  // such values are left out here and counted at the end
      bool nf = false;
      for (int x = threadIdx.x; x < TK * W::CPR; x += kThreads) {
        uint4& v = reinterpret_cast<uint4*>(sv)[x];
        if (not_finite<T>(v)) {
          nf = true;
          v = make_uint4(finite_of(v.x), finite_of(v.y), finite_of(v.z), finite_of(v.w));
        }
      }
      special = __syncthreads_or(nf) || special;
    }
    if (!live) return;
    if (edge && k0 + TK > lo_w) {
      const int left = lim - k0 - 4 * (lane_anew() / 32);
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[n][x] = n * 32 + 8 * (x / 4) + x % 4 < left ? s[n][x] : kNegInf;
    }
    if (edge && any_bad) {
      const int hb = lane_anew() / 32;
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // 4 keys of one wave's rows
          const int r = n * 32 + 8 * x + 4 * hb;
          const u32 word = sbad[buf][r / W::RW] >> (r % W::RW);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][4 * x + i] = (word >> i) & 1 ? kNegInf : s[n][4 * x + i];
        }
    }
    // V's fragments in the order of the products: all of a run of 16 keys, then the next run's
    constexpr int F = 2 * NS, VA = 4;
    bf16x8 vf[VA];
    auto read_v = [&](int x) { vf[x % VA] = v_frag(sv, vl, x % ND, x / ND / 2, x / ND % 2); };
#pragma unroll
    for (int x = 0; x < VA - 1; ++x) read_v(x);  // on their way while the weights are computed
    __builtin_amdgcn_sched_barrier(0);
    float t = kNegInf;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int x = 0; x < 16; ++x) t = fmaxf(t, s[n][x]);
    t = with_far(t, larger) * c;
    if (__any(t > m + 8.f)) {
      const float mn = fmaxf(m, t), a = __builtin_amdgcn_exp2f(m - base_of(mn));
      m = mn;
      l *= a;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[d][x] *= a;
    }
    const float base = base_of(m);
    // the weights of a run of 16 keys are computed behind the products of the run before it, a pair at a time
    u32 pk[2][4];
    auto weights = [&](int f, int x) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[f / 2][8 * (f % 2) + 2 * x], c, -base));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[f / 2][8 * (f % 2) + 2 * x + 1], c, -base));
      pk[f % 2][x] = pack2(p0, p1);
      l = sum_pair(pk[f % 2][x], l);
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) weights(0, x);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const bf16x8 pf = __builtin_bit_cast(bf16x8, make_uint4(pk[f % 2][0], pk[f % 2][1], pk[f % 2][2], pk[f % 2][3]));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const int at = f * ND + d;
        if (at + VA - 1 < F * ND) read_v(at + VA - 1);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[at % VA], pf, o[d], 0, 0, 0);
        if (f + 1 < F)
#pragma unroll
          for (int x = (4 * d + ND - 1) / ND; x < (4 * d + 4 + ND - 1) / ND; ++x) weights(f + 1, x);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  // a buffer's loads are waited for and its readers of the step before joined by the one barrier of a step
  auto ready = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
  };
  for (int k0 = k_first; k0 < k_end; k0 += 2 * TK) {
    ready();
    if (k0 + TK < k_end) tile.issue(k0 + TK, entry, 1, sk1, sv1);
    entry = tile.look(k0 + 2 * TK);
    compute(k0, 0, sk0, sv0);
    if (k0 + TK >= k_end) break;
    ready();
    if (k0 + 2 * TK < k_end) tile.issue(k0 + 2 * TK, entry, 0, sk0, sv0);
    entry = tile.look(k0 + 3 * TK);
    compute(k0 + TK, 1, sk1, sv1);
  }
  const int ln = lane_anew(), r32 = ln % 32, hf = ln / 32;
  if (special) {  // the whole workgroup: counted per row (add_special), the values brought once more
    for (int k0 = k_first; k0 < k_end; k0 += TK) {
      if (k0 + TK <= lo_g) continue;
      __syncthreads();
      tile.issue(k0, tile.look(k0), 0, sk0, sv0);
      ready();
      clear_unseen(k0, 0, sv0);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x16 o1;
#pragma unroll
        for (int x = 0; x < 16; ++x) o1[x] = 0.f;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 v = __builtin_bit_cast(uint4, v_frag(sv0, v_lane(ln), d, n, j));
            u32 on[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = k0 + n * 32 + 16 * j + (x / 2) * 8 + 4 * hf + 2 * (x % 2);
              on[x] = (key < lim ? 0x3f80u : 0u) | (key + 1 < lim ? 0x3f800000u : 0u);
            }
            o1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(bf16x8, make_uint4(marks_of(v.x), marks_of(v.y), marks_of(v.z), marks_of(v.w))),
                __builtin_bit_cast(bf16x8, make_uint4(on[0], on[1], on[2], on[3])), o1, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          o[d][x] += special_of(o1[x]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  l = with_far(l, sum_of);
  // The lane's results: row r32, values 32 d + 8 x + 4 hf .. + 3. Finished rows are turned in the wave's own buffer (its
  // pieces of four exchanged by the row), so that gate and result move as 16-byte pieces of whole rows, all gates
  // of a turn on their way at once: taken as they lie, a lane's 8-byte pieces of the gate cost a memory round trip each
  // (a 4096-token prompt, 32 heads of 256 with a gate: 722 us; turned, and with the ranges counting each tile, 397).
  if (!part.p) {
    __syncthreads();  // the last buffers' readers
    if (rows_w) {
      constexpr int HD = DT == 64 ? 64 : 128, LPR = HD / 8, NI = 32 * LPR / 64;  // columns of a turn; lanes of a row
      float* sx = reinterpret_cast<float*>(w == 0 ? sk0 : w == 1 ? sv0 : w == 2 ? sk1 : sv1);
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      const int c8 = (ln % LPR) * 8;
#pragma unroll
      for (int p = 0; p < DT / HD; ++p) {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const f32x16& v = o[p * (HD / 32) + d];
            *reinterpret_cast<f32x4*>(sx + r32 * HD + (((8 * d + 2 * x + hf) ^ r32) & (HD / 4 - 1)) * 4) =
                f32x4{v[4 * x] * inv, v[4 * x + 1] * inv, v[4 * x + 2] * inv, v[4 * x + 3] * inv};
          }
        __builtin_amdgcn_wave_barrier();
        Raw8<T> gate[NI];
        T* op[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int r = i * (64 / LPR) + ln / LPR, row = row0 + w * 32 + r, t = A.by_g(row), e = p * HD + c8;
          op[i] = nullptr;
          if (row < q.rows && !(PAD && e >= A.D)) {
            const long token = q.s0 + t;
            const int head = h * A.g + (row - t * A.g);
            op[i] = reinterpret_cast<T*>(A.out + token * A.ot + head * A.oh) + e;
            if (A.gate) gate[i].load(reinterpret_cast<const T*>(A.gate + token * A.gt + head * A.gh) + e);
          }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int r = i * (64 / LPR) + ln / LPR;
          float y[8];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(sx + r * HD + (((c8 / 4 + x) ^ r) & (HD / 4 - 1)) * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[4 * x + j] = v[j];
          }
          if (A.gate && op[i]) {
            float gv[8];
            gate[i].get(gv);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= sigmoid_io<T>(gv[j]);
          }
          if (op[i]) st8_io(op[i], y);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  } else if (rows_w) {
    f32x4* po = reinterpret_cast<f32x4*>(part.p) + w * (ND * 4) * 64;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) po[(d * 4 + x) * 64 + ln] = f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
    if (hf == 0) {
      part.p[kWideRows * DT + w * 32 + r32] = m;
      part.p[kWideRows * DT + kWideRows + w * 32 + r32] = l;
    }
  }
}

// ---------------------------------------------------------------- the kernel
// the rows of no request, shared out to the workgroups
template <class T>
__device__ __forceinline__ void clear_rest(const AttnArgs& A) {
  const long b0 = A.starts[0], b1 = A.starts[A.B];
  const long lo = b0 < 0 ? 0 : b0 > A.N ? A.N : b0, hi = b1 < lo ? lo : b1 > A.N ? A.N : b1;
  const long rest = lo + (A.N - hi);
  const int heads = A.Hk * A.g;
  for (long i = blockIdx.x; i < rest; i += gridDim.x) {
    const long row = i < lo ? i : hi + (i - lo);
    for (int x = threadIdx.x; x < heads * (A.D / 4); x += kThreads) {
      T* o = reinterpret_cast<T*>(A.out + row * A.ot + (x / (A.D / 4)) * A.oh) + 4 * (x % (A.D / 4));
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      st4_io(o, z);
    }
  }
}

// MIXED: the batch may hold requests of more than A.wide packed rows, which take the wide tiles.
template <class T, int DT, int NQ, bool PAD, bool WHOLE, bool MIXED>
__global__ __launch_bounds__(kThreads, 2) void k_attention(AttnArgs A) {
  using S = Shape<T, DT>;
  using L = StreamLds<T, DT, NQ>;
  constexpr int R = 16 * NQ, KB = S::KB;
  constexpr int BUF = MIXED ? Wide<DT>::TK * DT / 8 : 0;  // pieces of 16 bytes
  constexpr int NA = L::ACC > 2 * BUF ? L::ACC : 2 * BUF, NB = L::Q > BUF ? L::Q : BUF;
  __shared__ FoundLds sfound;
  __shared__ float sm[4][R], sl[4][R];
  __shared__ u32 sbad[2][4];
  // the streamed tiles' sums and queries; the wide tiles' buffers
  __shared__ __align__(16) uint4 sa[NA];
  __shared__ __align__(16) uint4 sb[NB];
  __shared__ __align__(16) uint4 sc[MIXED ? BUF : 1];
  __shared__ __align__(16) uint4 sd[MIXED && Wide<DT>::QL ? 4 * Wide<DT>::QL * 64 : 1];
  // Where the range stands. In LDS while a tile is worked on: held in registers it would be spilled there.
  __shared__ struct {
    Request q;
    long u, u1, local, each;
    Unit at;
    int b, range, begun;
  } st;
  GDN_POISON_LDS(sfound, sm, sl, sbad, sa, sb, sc, sd, st);

  {
    const int range = range_of(blockIdx.x, A.G);
    const Found f = find_range<R, KB>(A, range, sfound);
    if (threadIdx.x == 0) split_of(A, range)->parts = 0;
    if (A.fill) clear_rest<T>(A);
    if (f.b < 0) return;
    if (threadIdx.x == 0) {
      const long u0 = range * f.each;
      st.q = f.q;
      st.u = u0;
      st.u1 = min(f.total, u0 + f.each);
      st.local = u0 - f.unit;
      st.each = f.each;
      st.at = unit_of(f.q, u0 - f.unit);
      st.b = f.b;
      st.range = range;
      st.begun = 0;
    }
    __syncthreads();
  }
  while (true) {
    {
      const Request q = uniform(st.q);
      const Unit at{uniform(st.at.head), uniform(st.at.tile), uniform(st.at.at)};
      const int b = uniform(st.b), range = uniform(st.range), begun = uniform(st.begun);
      const long u = uniform(st.u), u1 = uniform(st.u1);
      const int blocks = q.tile_blocks(at.tile), seg = (int)min((long)(q.extra + blocks - at.at), u1 - u);
      const int k0 = max(0, at.at - q.extra), keys = max(0, at.at + seg - q.extra) - k0;  // blocks of keys
      const int slot = 2 * range + begun;
      const Part part{keys == blocks ? nullptr : A.part + (size_t)slot * A.slot, at.tile, at.head};
      __syncthreads();
      if (threadIdx.x == 0) {
        if (keys > 0 && k0 == 0 && keys < blocks)  // the tile goes on in the next ranges
          *split_of(A, range) = {(int)div_by(st.each)(u - at.at + q.extra + blocks - 1) - range + 1, slot, q.s0, q.rows, q.tile_rows, at.tile,
                                 at.head};
        // the next tile, the next head's first, or the next request's (if that brings none, the next one's with rows is looked
        // for behind this tile)
        long local = st.local + seg;
        st.u = u + seg;
        st.begun = 1;
        if (local < q.cost) {
          st.at = at.tile + 1 < q.tiles ? Unit{at.head, at.tile + 1, 0} : Unit{at.head + 1, 0, 0};
        } else if (u + seg < u1) {
          const Request n = b + 1 < A.B ? request<R, KB>(A, b + 1) : Request{};
          local = 0;
          st.q = n;
          st.b = b + 1;
          st.at = {0, 0, 0};
        }
        st.local = local;
      }
      if (keys > 0) {
        if (MIXED && q.tile_rows == kWideRows) {
          uint16_t* pa = reinterpret_cast<uint16_t*>(sa);
          if constexpr (MIXED)
            wide_tile<DT, PAD, WHOLE>(q, b, part, k0, keys, pa, pa + Wide<DT>::TK * DT, reinterpret_cast<uint16_t*>(sb),
                                      reinterpret_cast<uint16_t*>(sc), sd, sbad);
        } else {
          stream_tile<T, DT, NQ, PAD, WHOLE>(q, b, part, k0, keys, sb, reinterpret_cast<f32x4*>(sa), sm, sl);
        }
      }
    }
    __syncthreads();
    if (uniform(st.u) >= uniform(st.u1)) break;
    if (uniform(st.q.cost) == 0) {  // 64 at once: thousands that bring nothing may lie between two requests
      __syncthreads();  // all waves have seen it
      if (uniform(wave()) == 0) {
        int b = uniform(st.b) + 1;
        for (; b < A.B; b += 64) {
          const Request n = b + lane() < A.B ? request<R, KB>(A, b + lane()) : Request{};
          const uint64_t here = __ballot(n.cost > 0);
          if (here) {
            const int first = __builtin_ctzll(here);
            if (lane() == first) st.q = n;
            b += first;
            break;
          }
        }
        if (threadIdx.x == 0) {
          st.b = b;
          if (b >= A.B) st.u = st.u1;
        }
      }
      __syncthreads();
      if (uniform(st.u) >= uniform(st.u1)) break;
    }
  }
}

// The tiles that more than one range holds: their parts joined, one workgroup per range. Bound by latency (few rows)
// or memory (wide tiles): the maxima and sums of all parts are read at once, the results as many at a time as the
// registers hold.
// Few tiles have many parts each (one request of 16000 tokens, 4 key heads: 126): kJoinSliced spreads a tile's results over
// gridDim.y workgroups and its parts over two halves of each, 16 at a time in each; gridDim.x is then the most tiles there can
// be, and a workgroup finds its one among the ranges' notes.
// Tiles of which the host does not know whether they are few (a table's unused places count as one each): the ranges' notes
// are counted (kJoinCounted), and each tile has an equal share of the workgroups where that is kShare or more (64 tokens over
// 30000 in one of 64 places, 16/4 heads of 256: 81 us, with one workgroup per range 136; with a share of 4 or more, which
// decoding requests' tiles have too, those of 20 requests take 66 us instead of 54).
constexpr int kSlice = 128;  // results of four per workgroup
constexpr int kShare = 32;
template <int DT, Join J>
constexpr int join_threads() { return DT == 64 || J == kJoinSliced ? 256 : 512; }
template <int DT, int ROWS>
constexpr int join_slices() { return ROWS * DT / 4 / kSlice; }

template <class T, int DT, int ROWS, bool WIDE, bool SLICED, int NT>
__device__ __forceinline__ void join_tile(const AttnArgs& A, const Split& q, const float* first, const float* next, int slice,
                                          float (*sm)[kWideRows], float (*sl)[kWideRows]) {
  constexpr int NG = NT / ROWS;
  constexpr int PG = SLICED ? NT / kSlice : 1, NE = SLICED ? 1 : ROWS * DT / 4 / NT;  // groups of parts; results of a thread
  static_assert(NG >= 1 && NE >= 1, "");
  // part p's slot: the range that the tile begins in holds part 0, the others follow two slots apart
  const int parts = q.parts, tile = q.tile, h = q.head;
  auto part = [&](int p) { return p ? next + (size_t)(p - 1) * 2 * A.slot : first; };
  const int tid = threadIdx.x, row = tid % ROWS, grp = tid / ROWS;
  const int live = min(ROWS, (q.rows - tile * ROWS + 31) / 32 * 32);  // rows that the parts hold
  // The thread's results of four, as they lie in a part (place i). Those of a wide tile, whole: NE pieces of one row, the
  // other half of each in the lane 32 on.
  constexpr bool ROW = WIDE && !SLICED;
  constexpr int NR = ROW ? 1 : NE;
  static_assert(!ROW || (DT / 8 % NE == 0 && NE % 2 == 0), "a wave's pieces are of 32 rows");
  const int x0 = SLICED ? slice * kSlice + tid % kSlice : ROW ? wave() * NE * 64 + lane() : tid;
  constexpr int STEP = ROW ? 64 : NT;
  f32x4 acc[NE];
  int er[NR];  // their rows
#pragma unroll
  for (int i = 0; i < NE; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int x = x0 + i * STEP;
    er[i] = WIDE ? x / (DT / 8 * 64) * 32 + x % 32 : x / (DT / 4);
  }
  constexpr int U = SLICED ? 16 : NE >= 8 ? 1 : 8 / NE;
  const int pg = SLICED ? tid / kSlice : 0;
  f32x4 v[U][NE];
  float pm[U][NR];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* s = part(min(p0 + u, parts - 1));
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        if (WIDE && er[i % NR] >= live) continue;
        v[u][i] = reinterpret_cast<const f32x4*>(s)[x0 + i * STEP];
        if (i < NR) pm[u][i] = s[ROWS * DT + er[i]];
      }
    }
  };
  fetch(pg * U);  // on their way while the maxima are read
  {
    float m = kNegInf, l = 0.f;
    constexpr int V = 8;  // parts at a time
    for (int p0 = grp; p0 < (row < live ? parts : 0); p0 += V * NG) {
      float pm[V], pl[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float* s = part(min(p0 + i * NG, parts - 1)) + ROWS * DT + row;
        pm[i] = s[0];
        pl[i] = s[ROWS];
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (p0 + i * NG < parts) {
          const float mn = fmaxf(m, pm[i]), base = base_of(mn);
          l = l * __builtin_amdgcn_exp2f(m - base) + pl[i] * __builtin_amdgcn_exp2f(pm[i] - base);
          m = mn;
        }
    }
    sm[grp][row] = m;
    sl[grp][row] = l;
  }
  __syncthreads();
  if (grp == 0) {
    float m = kNegInf, l = 0.f;
    for (int i = 0; i < NG; ++i) m = fmaxf(m, sm[i][row]);
    const float base = base_of(m);
    for (int i = 0; i < NG; ++i) l += sl[i][row] * __builtin_amdgcn_exp2f(sm[i][row] - base);
    sm[0][row] = base;
    sl[0][row] = l > 0.f || l != l ? 1.0f / l : 0.f;
  }
  __syncthreads();
  float eb[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) eb[i] = sm[0][er[i]];
  for (int p0 = pg * U; p0 < parts; p0 += PG * U) {
    if (p0 != pg * U) fetch(p0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) a[i] = __builtin_amdgcn_exp2f(pm[u][i] - eb[i]);
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (p0 + u < parts && !(WIDE && er[i % NR] >= live)) acc[i] += v[u][i] * a[i % NR];
    }
  }
  if constexpr (SLICED) {
    __shared__ __align__(16) f32x4 sacc[(PG - 1) * kSlice];
    GDN_POISON_LDS(sacc);
    if (pg) sacc[(pg - 1) * kSlice + tid % kSlice] = acc[0];
    __syncthreads();
    if (pg) return;
#pragma unroll
    for (int i = 0; i < PG - 1; ++i) acc[0] += sacc[i * kSlice + tid];
  }
  if constexpr (ROW) {
    // halves exchanged: a lane has 8 values side by side of every second piece, which move as 16 bytes (2048 tokens over
    // 30000, 135 MB of parts: 63 us with 8 bytes, 38 with 16)
    const int r = tile * ROWS + er[0], t = A.by_g(r);
    const float inv = sl[0][er[0]];
    const long token = q.s0 + t;
    const int head = h * A.g + (r - t * A.g), v0 = wave() * NE % (DT / 8) + lane() / 32;
    if (er[0] >= live) return;  // (both lanes of a row)
    const T* gp = reinterpret_cast<const T*>(A.gate + token * A.gt + head * A.gh) + 8 * v0;
    T* op = reinterpret_cast<T*>(A.out + token * A.ot + head * A.oh) + 8 * v0;
    Raw8<T> gate[NE / 2];
    const bool here = r < q.rows;
#pragma unroll
    for (int i = 0; i < NE; i += 2)
      if (A.gate && here && 8 * (v0 + i) < A.D) gate[i / 2].load(gp + 8 * i);
#pragma unroll
    for (int i = 0; i < NE; i += 2) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float lo = acc[i][j], hi = acc[i + 1][j];
        const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
        y[j] = __uint_as_float(z[0]) * inv;
        y[4 + j] = __uint_as_float(z[1]) * inv;
      }
      if (here && 8 * (v0 + i) < A.D) {
        if (A.gate) {
          float gf[8];
          gate[i / 2].get(gf);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= sigmoid_io<T>(gf[j]);
        }
        st8_io(op + 8 * i, y);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int x = x0 + i * STEP, r = tile * ROWS + er[i % NR], t = A.by_g(r), ln = x % 64, v = x / 64 % (DT / 8);
    const int d = WIDE ? 32 * (v / 4) + 8 * (v % 4) + 4 * (ln / 32) : x % (DT / 4) * 4;
    if (r >= q.rows || d >= A.D) continue;
    const long token = q.s0 + t;
    const int head = h * A.g + (r - t * A.g);
    const float inv = sl[0][er[i % NR]];
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = acc[i][j] * inv;
    if (A.gate) {
      Raw4<T> gt;
      gt.load(reinterpret_cast<const T*>(A.gate + token * A.gt + head * A.gh) + d);
      float gf[4];
      gt.get(gf);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] *= sigmoid_io<T>(gf[j]);
    }
    st4_io(reinterpret_cast<T*>(A.out + token * A.ot + head * A.oh) + d, y);
  }
}

template <class T, int DT, int NQ, bool MIXED, Join J>
__global__ __launch_bounds__((join_threads<DT, J>())) void k_attention_join(AttnArgs A) {
  constexpr int R = 16 * NQ, NT = join_threads<DT, J>(), RUN = (kMostRanges + NT - 1) / NT;
  __shared__ float sm[NT / R][kWideRows], sl[NT / R][kWideRows];
  GDN_POISON_LDS(sm, sl);
  int range = blockIdx.x;
  auto join = [&](const Split& q, auto sliced, int slice) {
    const float *first = A.part + (size_t)q.first * A.slot, *next = A.part + (size_t)(2 * (range + 1)) * A.slot;
    if constexpr (MIXED) {
      if (q.tile_rows == kWideRows) {
        join_tile<T, DT, kWideRows, true, sliced.value, NT>(A, q, first, next, slice, sm, sl);
        return;
      }
    }
    if (!sliced.value || slice < join_slices<DT, R>()) join_tile<T, DT, R, false, sliced.value, NT>(A, q, first, next, slice, sm, sl);
  };
  if constexpr (J == kJoinSliced) {  // the blockIdx.x-th of the ranges that left a note, all read at once
    __shared__ int scount[NT / 64], sfound;
    __shared__ __align__(16) i32x4 snote[2];
    GDN_POISON_LDS(scount, sfound, snote);
    i32x4 note[RUN][2];
    int n = 0;
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int r = i * NT + threadIdx.x;
      const i32x4* from = reinterpret_cast<const i32x4*>(split_of(A, r < A.G ? r : 0));
      note[i][0] = from[0];
      note[i][1] = from[1];
      if (r >= A.G) note[i][0].x = 0;
    }
#pragma unroll
    for (int i = 0; i < RUN; ++i) n += note[i][0].x > 1;  // Split::parts
    int upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int t = __shfl_up(upto, d);
      if (lane() >= d) upto += t;
    }
    if (lane() == 63) scount[wave()] = upto;
    if (threadIdx.x == 0) sfound = -1;
    __syncthreads();
    for (int w = 0; w < wave(); ++w) upto += scount[w];
    int k = upto - n;
#pragma unroll
    for (int i = 0; i < RUN; ++i)
      if (note[i][0].x > 1 && k++ == (int)blockIdx.x) {
        sfound = i * NT + threadIdx.x;
        snote[0] = note[i][0];
        snote[1] = note[i][1];
      }
    __syncthreads();
    range = uniform(sfound);
    if (range < 0) return;
    join(*reinterpret_cast<const Split*>(snote), std::true_type{}, blockIdx.y);
  } else if constexpr (J == kJoinCounted) {  // the ranges that left a note, in order, and how many workgroups each may have
    __shared__ int scount[RUN][NT / 64], swhere[kMostRanges];
    GDN_POISON_LDS(scount, swhere);
    uint64_t noted[RUN];
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      const int r = i * NT + threadIdx.x;
      const int parts = split_of(A, r < A.G ? r : 0)->parts;
      noted[i] = __ballot(r < A.G && parts > 1);
      if (lane() == 0) scount[i][wave()] = __builtin_popcountll(noted[i]);
    }
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int i = 0; i < RUN; ++i)
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) {
        if (w == wave() && (noted[i] >> lane() & 1)) swhere[n + __builtin_popcountll(noted[i] & ((1ull << lane()) - 1))] = i * NT + threadIdx.x;
        n += scount[i][w];
      }
    __syncthreads();
    n = uniform(n);
    const int share = n ? A.G / n : 0;
    const int k = share >= kShare ? (int)blockIdx.x / share : (int)blockIdx.x;
    if (k >= n) return;
    range = uniform(swhere[k]);
    const Split q = *split_of(A, range);
    if (share < kShare) {
      join(q, std::false_type{}, 0);
      return;
    }
    const int slices = MIXED && q.tile_rows == kWideRows ? join_slices<DT, kWideRows>() : join_slices<DT, R>();
    for (int slice = (int)blockIdx.x % share; slice < slices; slice += share) {
      join(q, std::true_type{}, slice);
      __syncthreads();
    }
  } else {
    const Split q = *split_of(A, range);
    if (q.parts < 2) return;
    join(q, std::false_type{}, 0);
  }
}

}  // namespace
}  // namespace gdn
