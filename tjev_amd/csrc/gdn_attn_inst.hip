// One unit of paged attention: the kernels of one type (GDN_T: bf16 or f32) and head dims up to GDN_D, with GDN_TREE those for
// trees of new tokens.
#include "gdn_attention.h"

namespace gdn {
namespace {

#ifdef GDN_TREE
constexpr bool kTree = true;
#else
constexpr bool kTree = false;
#endif

template <class T, int DT, int NQ, bool PAD, bool WHOLE, bool MIXED>
hipError_t launch(const AttnPlan& r, AttnArgs& A, hipStream_t st) {
  A.G = r.G;
  A.by_G = div_by(r.G);
  A.slot = r.slot;
  A.wide = MIXED ? 16 * NQ : 0x7fffffff;
  A.wide_extra = kWideExtra + (A.gate ? kGateExtra : 0);
  hipLaunchKernelGGL((k_attention<T, DT, NQ, PAD, WHOLE, MIXED, kTree>), dim3(r.G), dim3(kThreads), 0, st, A);
  constexpr int slices = join_slices<DT, MIXED ? kWideRows : 16 * NQ>();
  if (r.join == kJoinSliced) {
    hipLaunchKernelGGL((k_attention_join<T, DT, NQ, MIXED, kJoinSliced>), dim3(r.tiles, slices), dim3(join_threads<DT, kJoinSliced>()), 0, st, A);
  } else if (MIXED && r.join == kJoinCounted) {
    if constexpr (MIXED)
      hipLaunchKernelGGL((k_attention_join<T, DT, NQ, MIXED, kJoinCounted>), dim3(r.G), dim3(join_threads<DT, kJoinCounted>()), 0, st, A);
  } else {
    hipLaunchKernelGGL((k_attention_join<T, DT, NQ, MIXED, kJoinRanges>), dim3(r.G), dim3(join_threads<DT, kJoinRanges>()), 0, st, A);
  }
  return hipGetLastError();
}

template <class T, int DT, int NQ>
hipError_t dispatch(const AttnPlan& r, AttnArgs& A, hipStream_t st) {
  auto with = [&](auto pad, auto whole) {
    if constexpr (sizeof(T) == 2)
      if (r.mixed) return launch<T, DT, NQ, pad.value, whole.value, true>(r, A, st);
    return launch<T, DT, NQ, pad.value, whole.value, false>(r, A, st);
  };
  const std::true_type yes;
  const std::false_type no;
  const bool pad = A.D != DT, whole = A.page % 16 == 0;
  return pad ? whole ? with(yes, yes) : with(yes, no) : whole ? with(no, yes) : with(no, no);
}

// bf16: requests of more rows than a streamed tile has take the wide tiles. fp32 streams all. Streamed tiles have 16 rows or
// 32 (more are spilled: in fp32 64 at head dim 128 and 32 at 256 take twice the time).
template <class T, int DT>
hipError_t by_rows(const AttnPlan& r, AttnArgs& A, hipStream_t st) {
  if constexpr (DT <= (sizeof(T) == 4 ? 128 : 64))
    if (r.nq > 1) return dispatch<T, DT, 2>(r, A, st);
  return dispatch<T, DT, 1>(r, A, st);
}

using bf16 = uint16_t;
using f32 = float;

}  // namespace

#ifdef GDN_TREE
#define GDN_NAME_(t, d) attention_tree_##t##_##d
#else
#define GDN_NAME_(t, d) attention_##t##_##d
#endif
#define GDN_NAME(t, d) GDN_NAME_(t, d)
hipError_t GDN_NAME(GDN_T, GDN_D)(const AttnPlan& r, AttnArgs& A, hipStream_t st) { return by_rows<GDN_T, GDN_D>(r, A, st); }

}  // namespace gdn
