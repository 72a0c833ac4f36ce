// Causal attention of new tokens over the paged key/value cache for gfx950 (the full-attention layers
// that stand between the GDN layers), from one token per request to chunks of a prompt:
//   o_r = sum_k p_rk v_k / sum_k p_rk,  p_rk = 2^(c q_r k_k - m_r),  c = scale log2(e),
// one pass over the keys with the running maximum m_r and sum of each row in 32 bits.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/tjev_gdn.h"
#include "gdn_device.h"
#include "gdn_launch.h"
#include "gdn_paged.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr float kNegInf = -__builtin_inff();

struct AttnArgs : Batch {
  int D, fill;
  float c;                          // scale * log2(e)
  const char *q, *k, *v, *gate;
  char* out;
  long qt, qh, gt, gh, ot, oh;      // bytes: token and head of q, gate, out
  long kp, ks, kh, vp, vs, vh;      // bytes: page, slot and head of the caches
  float* part;                      // the workgroups' unfinished rows
  int G;                            // workgroups of the streaming kernel
};

// ---------------------------------------------------------------- the stream's plan
// All units of a batch (gdn_paged.h) in a line (request, tile, key head, keys) are cut into G equal ranges, one
// per workgroup, so that requests of very different lengths keep every CU busy to the end, whatever
// the host knows of them.

// inclusive running sum over the workgroup's threads (in order); total: the sum of all
__device__ __forceinline__ long scan_block(long v, long* swave, long& total) {
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
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave()) before += swave[w];
    total += swave[w];
  }
  return v + before;
}

template <int R, int KB>
__device__ __forceinline__ long total_units(const AttnArgs& A, long* swave) {
  long sum = 0, t;
  for (int b0 = 0; b0 < A.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    sum += b < A.B ? request<R, KB>(A, b).cost : 0;
  }
  scan_block(sum, swave, t);
  return t;
}

// units of one workgroup's range
__device__ __forceinline__ long units_each(long total, int G) { return total ? (total + G - 1) / G : 1; }

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

// max or sum over the four lanes that hold one row (lane % 16)
__device__ __forceinline__ float rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// the base of the powers: 0 where a row has seen no key yet, so that its powers are 0 and not NaN
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.f : m; }

// out += P V for one step (KG groups of 16 keys). V [key group][r]: the lane's keys 4 (lane / 16) + r
template <class T, int DT, int NQ>
__device__ __forceinline__ void add_pv(const typename Shape<T, DT>::VVec (&v)[Shape<T, DT>::KG][4][Shape<T, DT>::VH],
                                       const f32x4 (&p)[Shape<T, DT>::KG][NQ],
                                       f32x4 (&o)[NQ][Shape<T, DT>::VH][Shape<T, DT>::VE]) {
  using S = Shape<T, DT>;
  if constexpr (S::BF) {
    bf16x8 pb[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n)  // rounded to bf16 for the product, as V is: the sums stay in 32 bits
      pb[n] = __builtin_bit_cast(bf16x8, make_uint4(pack2(p[0][n][0], p[0][n][1]), pack2(p[0][n][2], p[0][n][3]),
                                                    pack2(p[1][n][0], p[1][n][1]), pack2(p[1][n][2], p[1][n][3])));
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
        for (int n = 0; n < NQ; ++n) o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[n], o[n][h][e], 0, 0, 0);
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

__device__ __forceinline__ void zero_word(uint4& v) { v = make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ void zero_word(uint2& v) { v = make_uint2(0, 0); }

// a row's 4 x VE consecutive results, divided by its sum, gated, rounded once and stored
template <class T, int DT, bool PAD>
__device__ __forceinline__ void store_row(const AttnArgs& A, const f32x4 (&o)[Shape<T, DT>::VH][Shape<T, DT>::VE], float l, long token,
                                          int head) {
  using S = Shape<T, DT>;
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
  for (int h = 0; h < S::VH; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = h * 16 * S::VE + (4 * (lane() / 16) + r) * S::VE;
      if (PAD && d >= A.D) continue;
      float x[S::VE];
#pragma unroll
      for (int e = 0; e < S::VE; ++e) x[e] = o[h][e][r] * inv;
      if (A.gate) {
        const T* gp = reinterpret_cast<const T*>(A.gate + token * A.gt + head * A.gh) + d;
#pragma unroll
        for (int e = 0; e < S::VE; ++e) x[e] *= sigmoidf_(ldf(gp + e));
      }
      T* op = reinterpret_cast<T*>(A.out + token * A.ot + head * A.oh) + d;
      if constexpr (S::VE == 8) {
        st8_io(op, x);
      } else {
        st4_io(op, x);
      }
    }
}

template <class T, int DT, int NQ>
constexpr int slot_floats() { return NQ * 16 * (DT + 2); }

// ---------------------------------------------------------------- the streaming kernel
// Four waves; each takes every fourth step of KG * 16 keys of the workgroup's range, with a running
// maximum, sum and result of its own, joined in LDS at a tile's end. A tile whose keys are all in the
// range is finished here; else its rows go to the workspace: slot 2 i for the tile that range i begins with,
// 2 i + 1 for one that begins inside it and goes on behind its end.
// WHOLE: pages hold whole groups of 16 keys, whose page is then one value per wave.
template <class T, int DT, int NQ, bool PAD, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_attn_stream(AttnArgs A) {
  using S = Shape<T, DT>;
  constexpr int R = 16 * NQ, KB = S::KB, KG = S::KG, E = S::E;
  constexpr int NV = NQ * S::VH * S::VE;  // result registers of four
  __shared__ long swave[kThreads / 64];
  __shared__ int sreq;
  __shared__ long sloc;
  __shared__ float sm[4][R], sl[4][R];
  __shared__ __align__(16) f32x4 sacc[2][NV * 64];
  GDN_POISON_LDS(swave, sreq, sloc, sm, sl, sacc);
  const int w = __builtin_amdgcn_readfirstlane(wave()), ln = lane(), r16 = ln & 15, g4 = ln >> 4;

  if (A.fill) {  // rows of no request
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

  const long total = total_units<R, KB>(A, swave), each = units_each(total, A.G);
  const long u0 = blockIdx.x * each, u1 = min(total, u0 + each);
  if (u0 >= u1) return;
  {  // the request and place that the range begins with
    long before = 0;
    for (int b0 = 0; b0 < A.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const long cost = b < A.B ? request<R, KB>(A, b).cost : 0;
      long sum;
      const long incl = before + scan_block(cost, swave, sum);
      if (u0 >= incl - cost && u0 < incl) {
        sreq = b;
        sloc = u0 - (incl - cost);
      }
      before += sum;
      if (before > u0) break;
    }
    __syncthreads();
  }
  int b = __builtin_amdgcn_readfirstlane(sreq);
  long local = sloc;
  Request q = request<R, KB>(A, b);
  for (long u = u0; u < u1;) {
    const int group = (int)(local / q.blocks), kb0 = (int)(local - (long)group * q.blocks);
    const int tile = group / A.Hk, h = group - tile * A.Hk;
    const int seg = (int)min((long)(q.blocks - kb0), u1 - u);

    // the lane's row of each row tile: its last key + 1, its query
    long tok[NQ];
    int head[NQ], lim[NQ];
    uint4 qf[NQ][S::KS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = tile * R + n * 16 + r16;
      const bool live = row < q.rows;
      const int t = live ? row / A.g : 0;
      tok[n] = q.s0 + t;
      head[n] = h * A.g + (live ? row - t * A.g : 0);
      lim[n] = live ? row_limit(q, row, A.g) : 0;
      const char* qp = A.q + tok[n] * A.qt + head[n] * A.qh;
#pragma unroll
      for (int i = 0; i < S::KS; ++i) {
        const int e = (4 * i + g4) * E;
        qf[n][i] = live && !(PAD && e >= A.D) ? *reinterpret_cast<const uint4*>(qp + e * (int)sizeof(T)) : make_uint4(0, 0, 0, 0);
      }
    }
    const int lo_lim = row_limit(q, tile * R, A.g), hi_lim = row_limit(q, min(tile * R + R, q.rows) - 1, A.g);

    float m[NQ], l[NQ];
    f32x4 o[NQ][S::VH][S::VE];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = kNegInf;
      l[n] = 0.f;
#pragma unroll
      for (int x = 0; x < S::VH; ++x)
#pragma unroll
        for (int e = 0; e < S::VE; ++e) o[n][x][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
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

      f32x4 s[KG][NQ];
#pragma unroll
      for (int j = 0; j < KG; ++j)
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < S::KS; ++i)
#pragma unroll
        for (int j = 0; j < KG; ++j)
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[j][n] = dot_step<T, DT>(kf[j][i], qf[n][i], s[j][n]);
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
          for (int r = 0; r < 4; ++r) {
            s[j][n][r] = __builtin_amdgcn_exp2f(s[j][n][r] - base);
            l[n] += s[j][n][r];
          }
#pragma unroll
        for (int x = 0; x < S::VH; ++x)
#pragma unroll
          for (int e = 0; e < S::VE; ++e) o[n][x][e] *= a;
      }
      if (!careful) {
        add_pv<T, DT, NQ>(vf, s, o);
      } else {
        // Infinities or NaN among values that some of the rows do not attend to: row by row, with the
        // values behind its last key set to 0
        for (int c = 0; c < 16; ++c) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const int cl = __shfl(lim[n], c);
            typename S::VVec vc2[KG][4][S::VH];
            f32x4 p1[KG][1], o1[1][S::VH][S::VE];
#pragma unroll
            for (int j = 0; j < KG; ++j) {
              p1[j][0] = s[j][n];
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < S::VH; ++x) {
                  vc2[j][r][x] = vf[j][r][x];
                  if (k0 + 16 * j + 4 * g4 + r >= cl) zero_word(vc2[j][r][x]);
                }
            }
#pragma unroll
            for (int x = 0; x < S::VH; ++x)
#pragma unroll
              for (int e = 0; e < S::VE; ++e) o1[0][x][e] = f32x4{0.f, 0.f, 0.f, 0.f};
            add_pv<T, DT, 1>(vc2, p1, o1);
            if (r16 == c)
#pragma unroll
              for (int x = 0; x < S::VH; ++x)
#pragma unroll
                for (int e = 0; e < S::VE; ++e) o[n][x][e] += o1[0][x][e];
          }
        }
      }
    }

    // the four waves' rows joined
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      l[n] = rows_sum(l[n]);
      if (g4 == 0) sm[w][n * 16 + r16] = m[n], sl[w][n * 16 + r16] = l[n];
    }
    __syncthreads();
    float mj[NQ], lj[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      mj[n] = kNegInf;
#pragma unroll
      for (int i = 0; i < 4; ++i) mj[n] = fmaxf(mj[n], sm[i][n * 16 + r16]);
      const float base = base_of(mj[n]);
      lj[n] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) lj[n] += sl[i][n * 16 + r16] * __builtin_amdgcn_exp2f(sm[i][n * 16 + r16] - base);
      const float a = __builtin_amdgcn_exp2f(m[n] - base);
#pragma unroll
      for (int x = 0; x < S::VH; ++x)
#pragma unroll
        for (int e = 0; e < S::VE; ++e) o[n][x][e] *= a;
    }
    auto each_reg = [&](auto f) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int x = 0; x < S::VH; ++x)
#pragma unroll
          for (int e = 0; e < S::VE; ++e) f(((n * S::VH + x) * S::VE + e) * 64 + ln, o[n][x][e]);
    };
    if (w >= 2) each_reg([&](int i, f32x4& x) { sacc[w - 2][i] = x; });
    __syncthreads();
    if (w < 2) each_reg([&](int i, f32x4& x) { x += sacc[w][i]; });
    __syncthreads();
    if (w == 1) each_reg([&](int i, f32x4& x) { sacc[0][i] = x; });
    __syncthreads();
    if (w == 0) {
      each_reg([&](int i, f32x4& x) { x += sacc[0][i]; });
      if (seg == q.blocks) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          if (tile * R + n * 16 + r16 < q.rows) store_row<T, DT, PAD>(A, o[n], lj[n], tok[n], head[n]);
      } else {
        float* p = A.part + (size_t)(2 * blockIdx.x + (u > u0 ? 1 : 0)) * slot_floats<T, DT, NQ>();
        f32x4* po = reinterpret_cast<f32x4*>(p);
        each_reg([&](int i, f32x4& x) { po[i] = x; });
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          if (g4 == 0) {
            p[NV * 256 + n * 16 + r16] = mj[n];
            p[NV * 256 + R + n * 16 + r16] = lj[n];
          }
      }
    }
    __syncthreads();

    u += seg;
    local += seg;
    while (u < u1 && local >= q.cost) {  // the next request with rows
      if (++b >= A.B) return;
      local -= q.cost;
      q = request<R, KB>(A, b);
    }
  }
}

// The tiles that more than one range holds: their parts joined. One workgroup per tile, its result
// registers spread over the waves.
template <class T, int DT, int NQ, bool PAD>
__global__ __launch_bounds__(kThreads) void k_attn_join(AttnArgs A) {
  using S = Shape<T, DT>;
  constexpr int R = 16 * NQ, KB = S::KB, NV = NQ * S::VH * S::VE, NW = kThreads / 64;
  __shared__ long swave[kThreads / 64];
  __shared__ int sreq, sgroup;
  __shared__ long sbegin;
  __shared__ __align__(16) f32x4 sacc[NV * 64];
  GDN_POISON_LDS(swave, sreq, sgroup, sbegin, sacc);
  const long total = total_units<R, KB>(A, swave), each = units_each(total, A.G);
  if (threadIdx.x == 0) sreq = -1;
  {  // the tile: request, place among the request's tiles, first unit
    long tiles = 0, units = 0;
    for (int b0 = 0; b0 < A.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      Request q{};
      if (b < A.B) q = request<R, KB>(A, b);
      const long n = (long)q.tiles * A.Hk;
      long sum_t, sum_u;
      const long t1 = tiles + scan_block(n, swave, sum_t), c1 = units + scan_block(q.cost, swave, sum_u);
      const long at = (long)blockIdx.x - (t1 - n);
      if (at >= 0 && at < n) {
        sreq = b;
        sgroup = (int)at;
        sbegin = c1 - q.cost + at * q.blocks;
      }
      tiles += sum_t;
      units += sum_u;
      if (tiles > blockIdx.x) break;
    }
    __syncthreads();
  }
  const int b = sreq;
  if (b < 0) return;
  const Request q = request<R, KB>(A, b);
  const long begin = sbegin, end = begin + q.blocks, i0 = begin / each, i1 = (end - 1) / each;
  if (i0 == i1) return;  // finished by its workgroup
  const int ln = lane(), r16 = ln & 15, g4 = ln >> 4;
  auto part = [&](long i) { return A.part + (size_t)(2 * i + (i == i0 && begin != i0 * each ? 1 : 0)) * slot_floats<T, DT, NQ>(); };
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kNegInf;
    l[n] = 0.f;
    for (long i = i0 + g4; i <= i1; i += 4) m[n] = fmaxf(m[n], part(i)[NV * 256 + n * 16 + r16]);
    m[n] = rows_max(m[n]);
    const float base = base_of(m[n]);
    for (long i = i0 + g4; i <= i1; i += 4) {
      const float* p = part(i) + NV * 256 + n * 16 + r16;
      l[n] += p[R] * __builtin_amdgcn_exp2f(p[0] - base);
    }
    l[n] = rows_sum(l[n]);
  }
  for (int v = wave(); v < NV; v += NW) {
    const int n = v / (S::VH * S::VE);
    float base = 0.f;
#pragma unroll
    for (int x = 0; x < NQ; ++x)
      if (x == n) base = base_of(m[x]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (long i = i0; i <= i1; ++i) {
      const float* p = part(i);
      acc += reinterpret_cast<const f32x4*>(p)[v * 64 + ln] * __builtin_amdgcn_exp2f(p[NV * 256 + n * 16 + r16] - base);
    }
    sacc[v * 64 + ln] = acc;
  }
  __syncthreads();
  const int tile = sgroup / A.Hk, h = sgroup - tile * A.Hk;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (n % NW != wave()) continue;
    const int row = tile * R + n * 16 + r16;
    f32x4 o[S::VH][S::VE];
#pragma unroll
    for (int x = 0; x < S::VH; ++x)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) o[x][e] = sacc[((n * S::VH + x) * S::VE + e) * 64 + ln];
    if (row < q.rows) store_row<T, DT, PAD>(A, o, l[n], q.s0 + row / A.g, h * A.g + row % A.g);
  }
}

// ---------------------------------------------------------------- launches
struct Plan {
  int G;             // ranges of the stream
  long joins;        // most tiles a stream may have
  size_t bytes;      // workspace
};

constexpr int kRanges = 512;

template <class T, int DT, int NQ>
Plan plan_of(const tjev_gdn_paged_params* p) {
  using S = Shape<T, DT>;
  const long g = p->heads / p->kv_heads, rows = p->tokens * g;
  const long tiles = (rows / (16 * NQ) + p->requests) * p->kv_heads;
  const long blocks = ((long)p->table_width * p->page_size + S::KB - 1) / S::KB;
  Plan r;
  r.G = tiles >= kRanges || blocks * tiles >= kRanges ? kRanges : (int)(blocks * tiles);
  r.joins = tiles;
  r.bytes = (size_t)2 * r.G * slot_floats<T, DT, NQ>() * sizeof(float);
  return r;
}

template <class T, int DT, int NQ, bool PAD>
hipError_t launch(const tjev_gdn_paged_params* p, AttnArgs& A, hipStream_t st) {
  const Plan r = plan_of<T, DT, NQ>(p);
  A.G = r.G;
  if (p->page_size % 16 == 0) {
    hipLaunchKernelGGL((k_attn_stream<T, DT, NQ, PAD, true>), dim3(r.G), dim3(kThreads), 0, st, A);
  } else {
    hipLaunchKernelGGL((k_attn_stream<T, DT, NQ, PAD, false>), dim3(r.G), dim3(kThreads), 0, st, A);
  }
  hipLaunchKernelGGL((k_attn_join<T, DT, NQ, PAD>), dim3((unsigned)r.joins), dim3(kThreads), 0, st, A);
  return hipGetLastError();
}

int dim_of(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <class F>
auto by_shape(const tjev_gdn_paged_params* p, F f) {
  if (p->dtype == TJEV_GDN_BF16) {
    switch (dim_of(p->dim)) {
      case 64: return f(uint16_t{}, std::integral_constant<int, 64>{});
      case 128: return f(uint16_t{}, std::integral_constant<int, 128>{});
      default: return f(uint16_t{}, std::integral_constant<int, 256>{});
    }
  }
  switch (dim_of(p->dim)) {
    case 64: return f(float{}, std::integral_constant<int, 64>{});
    case 128: return f(float{}, std::integral_constant<int, 128>{});
    default: return f(float{}, std::integral_constant<int, 256>{});
  }
}

int validate(const tjev_gdn_paged_params* p) {
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->requests < 1 || p->table_width < 1 || p->pages < 1 || p->page_size < 1 || p->tokens < 0)
    return fail(TJEV_GDN_EINVAL, "requests, table_width, pages and page_size must be positive, tokens not negative");
  if (p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads)
    return fail(TJEV_GDN_EINVAL, "the query heads must be groups of the key heads");
  if ((p->dtype | 1) != 1) return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16");
  if (p->dim < 8 || p->dim % 8 || p->dim > 256)
    return fail(TJEV_GDN_EUNSUPPORTED, "paged attention kernels hold head dims in multiples of 8 up to 256");
  if (!(p->scale - p->scale == 0.f)) return fail(TJEV_GDN_EINVAL, "scale must be finite");
  if ((long)p->table_width * p->page_size >= (1l << 31) || p->tokens * p->heads >= (1l << 31) ||
      ((p->tokens * (p->heads / p->kv_heads)) / 16 + p->requests) * p->kv_heads >= (1l << 31) / 256)
    return fail(TJEV_GDN_EINVAL, "problem too large");
  return 0;
}

}  // namespace
}  // namespace gdn

extern "C" {

size_t tjev_gdn_paged_workspace_bytes(const tjev_gdn_paged_params* p) {
  if (gdn::validate(p)) return 0;
  return gdn::by_shape(p, [&](auto t, auto d) { return gdn::plan_of<decltype(t), d.value, 1>(p).bytes; });
}

int tjev_gdn_paged_attention(const tjev_gdn_paged_params* p, void* stream, const void* q, const void* k_cache, const void* v_cache,
                             const int32_t* block_table, const int32_t* starts, const int32_t* lengths, const void* gate, void* out,
                             void* workspace, size_t workspace_bytes) {
  using gdn::fail;
  if (int s = gdn::validate(p)) return s;
  if (!p->tokens) return 0;
  if (!q || !k_cache || !v_cache || !block_table || !starts || !lengths || !out) return fail(TJEV_GDN_EINVAL, "null tensor argument");
  const size_t need = tjev_gdn_paged_workspace_bytes(p);
  if (!workspace || workspace_bytes < need)
    return fail(TJEV_GDN_EWORKSPACE, "paged attention needs a workspace of tjev_gdn_paged_workspace_bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TJEV_GDN_EINVAL, "the workspace must be 256-byte aligned");
  const long e = p->dtype == TJEV_GDN_BF16 ? 2 : 4;
  gdn::AttnArgs A{};
  A.N = p->tokens;
  A.B = p->requests;
  A.M = p->table_width;
  A.page = p->page_size;
  A.pages = p->pages;
  A.Hk = p->kv_heads;
  A.g = p->heads / p->kv_heads;
  A.D = p->dim;
  A.fill = p->fill;
  A.c = p->scale * 1.44269504088896341f;
  A.q = static_cast<const char*>(q);
  A.k = static_cast<const char*>(k_cache);
  A.v = static_cast<const char*>(v_cache);
  A.gate = static_cast<const char*>(gate);
  A.out = static_cast<char*>(out);
  A.table = block_table;
  A.starts = starts;
  A.lengths = lengths;
  A.qt = p->q_stride[0] * e, A.qh = p->q_stride[1] * e;
  A.gt = gate ? p->gate_stride[0] * e : 0, A.gh = gate ? p->gate_stride[1] * e : 0;
  A.ot = p->out_stride[0] * e, A.oh = p->out_stride[1] * e;
  A.kp = p->k_stride[0] * e, A.ks = p->k_stride[1] * e, A.kh = p->k_stride[2] * e;
  A.vp = p->v_stride[0] * e, A.vs = p->v_stride[1] * e, A.vh = p->v_stride[2] * e;
  A.part = static_cast<float*>(workspace);
  long any = A.qt | A.qh | A.gt | A.gh | A.ot | A.oh | A.kp | A.ks | A.kh | A.vp | A.vs | A.vh;
  for (const void* x : {q, k_cache, v_cache, gate, (const void*)out}) any |= (long)reinterpret_cast<uintptr_t>(x);
  if (any % 16) return fail(TJEV_GDN_EINVAL, "q, gate, out and the caches must be 16-byte aligned, with strides that keep their rows so");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t err = gdn::by_shape(p, [&](auto t, auto d) {
    using T = decltype(t);
    return p->dim == d.value ? gdn::launch<T, d.value, 1, false>(p, A, st) : gdn::launch<T, d.value, 1, true>(p, A, st);
  });
  return err == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(err));
}

}  // extern "C"
