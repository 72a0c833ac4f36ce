// Rotary positions with several axes (time, height, width) for gfx950: every pair of a head's first
// `rotary` lanes is turned by the angle position[axis of the pair] * inv_freq[pair],
//   (x, y) -> (x cos t - y sin t, y cos t + x sin t),
// the pairs being lanes i and i + rotary / 2 (or 2i and 2i + 1), the lanes behind them passed on. The
// gradient is the turn by -t: the same kernel, from the positions alone (no input is kept).
//
// Bound by memory: q and k read and written once. The angle is taken in 64 bits (a position of 10^6
// against a frequency near 1 leaves 32 bits an error of 0.03), reduced to a fraction of a turn there
// and only then given to the 32-bit sine and cosine. That is about 500 instructions for the 8 pairs of a
// lane, so a lane keeps its sines and cosines in registers and walks over the heads of its token, q's
// and then k's; few tokens spread the heads over lanes instead (each takes its angles anew), as
// the launch below decides.
#include <hip/hip_runtime.h>

#include "../../include/tjev_gdn.h"
#include "gdn_device.h"
#include "gdn_launch.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = TJEV_GDN_MAX_AXES;

struct RotaryArgs {
  long tokens, length;       // tokens = batch * length
  int heads[2], D, half;     // heads of q and of k; half = rotary / 2
  int axes, end[kMaxAxes];   // end[a]: one past axis a's pairs (sections in order) or its pairs' last turn
  int interleaved, wide_pos, wide_freq;
  int slots, groups;         // lanes per head row; head groups per token
  double sign;
  const void* x[2];
  void* y[2];
  long sb[2], st[2], sh[2];  // strides of x (elements): batch, token, head
  const void* pos;
  const void* freq;
};

// V consecutive elements, held as loaded
template <class T, int V>
struct Vec {
  float f[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 8) {
      ld8(p, f);
    } else if constexpr (V == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    } else {
      f[0] = ldf(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 8) {
      st8_io(p, f);
    } else if constexpr (V == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      stf(p, f[0]);
    }
  }
};

__device__ __forceinline__ int pair_axis(const RotaryArgs& A, int i) {
  int a = 0;
  if (A.interleaved) {
    const int r = i % A.axes;
#pragma unroll
    for (int j = 1; j < kMaxAxes; ++j)
      if (j == r && i < A.end[j]) a = j;
  } else {
#pragma unroll
    for (int j = 0; j < kMaxAxes - 1; ++j)
      if (j + 1 < A.axes && i >= A.end[j]) a = j + 1;
  }
  return a;
}

// A lane owns V pairs of a head row (or 2 V lanes behind the rotated ones) and every groups-th head.
template <class T, int V, bool ADJ>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs A) {
  const long u = (long)blockIdx.x * kThreads + threadIdx.x;
  const int s = (int)(u % A.slots);
  const long w = u / A.slots;
  const int hg = (int)(w % A.groups);
  const long token = w / A.groups;
  if (token >= A.tokens) return;
  const bool turns = s * V < A.half;
  // the lane's two runs of V elements; adjacent pairs lie in one run of 2 V
  const int e0 = turns && !ADJ ? s * V : 2 * s * V, e1 = turns && !ADJ ? A.half + s * V : e0 + V;
  float c[V], n[V];
  if (turns) {
    double p[kMaxAxes];
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a) {
      const long at = a * A.tokens + token;
      p[a] = a >= A.axes ? 0.0 : A.wide_pos ? (double)static_cast<const int64_t*>(A.pos)[at] : (double)static_cast<const int32_t*>(A.pos)[at];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = s * V + j, a = pair_axis(A, i);
      const double f = A.wide_freq ? static_cast<const double*>(A.freq)[i] : (double)static_cast<const float*>(A.freq)[i];
      double t = (a == 0 ? p[0] : a == 1 ? p[1] : a == 2 ? p[2] : p[3]) * f * (A.sign * 0.15915494309189533577);  // in turns
      t -= rint(t);
      sincospif((float)(2.0 * t), &n[j], &c[j]);
    }
  }
  const long row = token / A.length, col = token - row * A.length;
  const int total = A.heads[0] + A.heads[1];
  constexpr int U = 4;  // heads in flight
  for (int h0 = hg; h0 < total; h0 += U * A.groups) {
    Vec<T, V> x[U], y[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int h = h0 + k * A.groups;
      if (h < total) {
        const int which = h >= A.heads[0], hh = which ? h - A.heads[0] : h;
        const T* src = static_cast<const T*>(A.x[which]) + row * A.sb[which] + col * A.st[which] + hh * A.sh[which];
        x[k].load(src + e0);
        y[k].load(src + e1);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int h = h0 + k * A.groups;
      if (h < total) {
        const int which = h >= A.heads[0], hh = which ? h - A.heads[0] : h;
        if (turns) {
          if constexpr (ADJ) {
            float z[2 * V];
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = x[k].f[j], z[V + j] = y[k].f[j];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float a = z[2 * j], b = z[2 * j + 1];
              z[2 * j] = a * c[j] - b * n[j];
              z[2 * j + 1] = b * c[j] + a * n[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) x[k].f[j] = z[j], y[k].f[j] = z[V + j];
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float a = x[k].f[j], b = y[k].f[j];
              x[k].f[j] = a * c[j] - b * n[j];
              y[k].f[j] = b * c[j] + a * n[j];
            }
          }
        }
        T* dst = static_cast<T*>(A.y[which]) + (token * A.heads[which] + hh) * A.D;
        x[k].store(dst + e0);
        y[k].store(dst + e1);
      }
    }
  }
}

template <class T, int V>
void launch(const RotaryArgs& A, int adjacent, unsigned blocks, hipStream_t st) {
  if (adjacent) {
    hipLaunchKernelGGL((k_rotary<T, V, true>), dim3(blocks), dim3(kThreads), 0, st, A);
  } else {
    hipLaunchKernelGGL((k_rotary<T, V, false>), dim3(blocks), dim3(kThreads), 0, st, A);
  }
}

}  // namespace
}  // namespace gdn

extern "C" int tjev_gdn_rotary(const tjev_gdn_rotary_params* p, void* stream, const void* q, const void* k,
                               const void* positions, const void* inv_freq, void* q_out, void* k_out) {
  using gdn::fail;
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->batch < 0 || p->length < 0 || p->q_heads < 0 || p->k_heads < 0)
    return fail(TJEV_GDN_EINVAL, "batch, length and head counts must not be negative");
  if (p->dim < 2 || p->dim > 1024) return fail(TJEV_GDN_EUNSUPPORTED, "rotary positions: head dims of 2 to 1024");
  if (p->rotary < 2 || p->rotary % 2 || p->rotary > p->dim || (p->dim - p->rotary) % 2)
    return fail(TJEV_GDN_EINVAL, "the rotated lanes must be an even number of at most the head dim, and leave an even rest");
  if (p->axes < 1 || p->axes > TJEV_GDN_MAX_AXES) return fail(TJEV_GDN_EINVAL, "1 to 4 position axes");
  if ((p->dtype | 1) != 1 || (p->position_bits != 32 && p->position_bits != 64) || (p->freq_bits != 32 && p->freq_bits != 64))
    return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16, positions and frequencies of 32 or 64 bits");
  const int half = p->rotary / 2;
  gdn::RotaryArgs A{};
  long sum = 0;
  for (int a = 0; a < p->axes; ++a) {
    const int n = p->sections[a];
    if (n < 0 || n > half) return fail(TJEV_GDN_EINVAL, "the sections must add up to half the rotated lanes");
    sum += n;
    if (p->interleaved && a && n && a + p->axes * (n - 1) >= half)
      return fail(TJEV_GDN_EINVAL, "an interleaved section is too long: its axis runs out of pairs");
    A.end[a] = p->interleaved ? p->axes * n : (int)sum;
  }
  if (sum != half) return fail(TJEV_GDN_EINVAL, "the sections must add up to half the rotated lanes");
  const long tokens = (long)p->batch * p->length, total = (long)p->q_heads + p->k_heads;
  if (p->batch > (1l << 31) || p->length > (1l << 31) || total > (1 << 20) || tokens > (1l << 40) / (total * p->dim + 1))
    return fail(TJEV_GDN_EINVAL, "problem too large");
  if (!tokens || !total) return 0;
  if (!positions || !inv_freq || (p->q_heads && (!q || !q_out)) || (p->k_heads && (!k || !k_out)))
    return fail(TJEV_GDN_EINVAL, "null tensor argument");
  const int bytes = p->dtype == TJEV_GDN_BF16 ? 2 : 4, v = 16 / bytes;
  // 16-byte pieces where every run of a lane starts on one; one element at a time otherwise
  bool wide = half % v == 0 && (p->dim - p->rotary) % (2 * v) == 0 && p->dim % v == 0;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* strides[2] = {p->q_stride, p->k_stride};
  for (int i = 0; i < 2; ++i) {
    A.heads[i] = i ? p->k_heads : p->q_heads;
    A.x[i] = in[i];
    A.y[i] = out[i];
    A.sb[i] = strides[i][0];
    A.st[i] = strides[i][1];
    A.sh[i] = strides[i][2];
    if (!A.heads[i]) continue;
    if (reinterpret_cast<uintptr_t>(in[i]) % bytes || reinterpret_cast<uintptr_t>(out[i]) % bytes)
      return fail(TJEV_GDN_EINVAL, "q and k must be aligned to their elements");
    for (int j = 0; j < 3; ++j) wide = wide && strides[i][j] % v == 0;
    wide = wide && reinterpret_cast<uintptr_t>(in[i]) % 16 == 0 && reinterpret_cast<uintptr_t>(out[i]) % 16 == 0;
  }
  A.tokens = tokens;
  A.length = p->length;
  A.D = p->dim;
  A.half = half;
  A.axes = p->axes;
  A.interleaved = p->interleaved != 0;
  A.wide_pos = p->position_bits == 64;
  A.wide_freq = p->freq_bits == 64;
  A.sign = p->inverse ? -1.0 : 1.0;
  A.pos = positions;
  A.freq = inv_freq;
  A.slots = p->dim / 2 / (wide ? v : 1);
  // 16 waves to a CU, then a lane takes further heads: a training step's 16384 tokens of 20 heads of 256 take 71 us forward
  // (4.74 TB/s), with half as many lanes 74, with four times as many 78
  const long fill = 262144 / (tokens * A.slots) + 1;
  A.groups = (int)(fill < total ? fill : total);
  const long blocks = (tokens * A.slots * A.groups + gdn::kThreads - 1) / gdn::kThreads;
  if (blocks >= (1l << 32) / gdn::kThreads) return fail(TJEV_GDN_EINVAL, "problem too large");  // a launch's threads
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == TJEV_GDN_BF16) {
    wide ? gdn::launch<uint16_t, 8>(A, p->adjacent, (unsigned)blocks, st) : gdn::launch<uint16_t, 1>(A, p->adjacent, (unsigned)blocks, st);
  } else {
    wide ? gdn::launch<float, 4>(A, p->adjacent, (unsigned)blocks, st) : gdn::launch<float, 1>(A, p->adjacent, (unsigned)blocks, st);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(e));
}
