// The C entry of paged attention: what the host decides, and the checks before a launch. The kernels are in
// gdn_attention.h, their units in gdn_attn_inst.hip.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/tjev_gdn.h"
#include "gdn_launch.h"
#include "gdn_paged.h"

namespace gdn {
namespace {

// Workgroups of the attention kernel, all on the chip at once: two to a CU by their registers, three at head dims up to
// 64 in bf16 (2048 new tokens over 30000, 16/4 heads of 64: 412 us with two, 362 with three; at 128, where the streaming
// kernel alone would fit three times: 64 decoding requests 158 with two, 166 with three).
int ranges_of(const tjev_gdn_paged_params* p) { return p->dtype == TJEV_GDN_BF16 && p->dim <= 64 ? kMostRanges : 512; }

// What the host knows: the rows and requests of the call, not how they are shared out.
AttnPlan plan_of(const tjev_gdn_paged_params* p) {
  const bool bf = p->dtype == TJEV_GDN_BF16;
  const int dt = p->dim <= 64 ? 64 : p->dim <= 128 ? 128 : 256;
  const long g = p->heads / p->kv_heads, rows = p->tokens * g;
  // Requests that bring a token, at most: a table may have places for many more. The most rows of one request: the caller's
  // bound, or what is left when the others bring one token each (a batch with fewer tokens than that would bring is taken for
  // decoding requests alone, which the streaming kernel serves 1 to 3% faster at head dims up to 128, 5 to 15% at 256; the
  // bound tells 64 tokens of one request of 64 from them: over 30000, 16/4 heads of 256, 81 us instead of 283).
  const long active = std::max<long>(1, std::min<long>(p->tokens, p->requests)), mean = (rows + active - 1) / active;
  const long top = (p->max_new ? std::min<long>(p->max_new, p->tokens) : p->tokens - active + 1) * g;
  AttnPlan r;
  // Streamed tiles of 32 rows instead of 16 where the registers hold them without a loss. In bf16 at head dims up to 64 for
  // requests of 17 to 32 on average (or at most, where the caller says so), which would else take a tile of 128 (32 requests of
  // 5 tokens over 8192, 32/8 heads of 64: 33.7 us, with that 39.0; one request 18.2, 21.8; at 128 the tile of 128 is the
  // faster one, 63 against 69). In fp32 up to 128 where there are enough of them (2 requests of 910 tokens after 858, 4/1 heads
  // of 128: 50.5 us, with 16 rows 55.0; 20 of 6 after 1858, 8/1 heads: 22.4, with 16 rows 17.6).
  auto few = [](long n) { return n > 16 && n <= 32; };
  r.nq = (bf ? dt == 64 && (few(mean) || (p->max_new && few(top))) : mean > 16 && dt <= 128 && rows / 32 * p->kv_heads >= 128) ? 2 : 1;
  r.mixed = bf && top > 16 * r.nq;
  const int kb = bf ? 128 : 64;
  // a request's rows are one streamed tile (mixed) or tiles of one kind, of which its last may be short
  const long tiles = (rows / (r.mixed ? kWideRows : 16 * r.nq) + active) * p->kv_heads;
  const long blocks = ((long)p->table_width * p->page_size + kb - 1) / kb + kWideExtra + kGateExtra;
  const int most = ranges_of(p);
  r.G = tiles >= most || blocks * tiles >= most ? most : (int)(blocks * tiles);
  // so few tiles that a workgroup each would leave most CUs idle, and take parts by the dozen; or rows for so few, in a batch
  // whose other requests may bring none
  r.join = tiles <= (r.mixed ? 16 : 64) ? kJoinSliced : r.mixed && p->max_new && rows / kWideRows * p->kv_heads <= 16 ? kJoinCounted : kJoinRanges;
  r.tiles = (int)(tiles < (1l << 30) ? tiles : 1l << 30);
  r.slot = (long)(r.mixed ? kWideRows : 16 * r.nq) * (dt + 2);
  r.bytes = (size_t)r.G * (2 * r.slot * sizeof(float) + kSplitBytes);
  return r;
}

int validate(const tjev_gdn_paged_params* p) {
  if (!p) return fail(TJEV_GDN_EINVAL, "null params");
  if (p->requests < 1 || p->table_width < 1 || p->pages < 1 || p->page_size < 1 || p->tokens < 0 || p->max_new < 0)
    return fail(TJEV_GDN_EINVAL, "requests, table_width, pages and page_size must be positive, tokens and max_new not negative");
  if (p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads)
    return fail(TJEV_GDN_EINVAL, "the query heads must be groups of the key heads");
  if ((p->dtype | 1) != 1) return fail(TJEV_GDN_EINVAL, "dtype must be TJEV_GDN_F32 or TJEV_GDN_BF16");
  if (p->dim < 8 || p->dim % 8 || p->dim > 256)
    return fail(TJEV_GDN_EUNSUPPORTED, "paged attention kernels hold head dims in multiples of 8 up to 256");
  if (!(p->scale - p->scale == 0.f)) return fail(TJEV_GDN_EINVAL, "scale must be finite");
  // (keys are 32-bit numbers, and a tile looks some blocks past the last)
  if ((long)p->table_width * p->page_size > TJEV_GDN_MAX_KEYS || p->tokens * p->heads >= (1l << 31) ||
      ((p->tokens * (p->heads / p->kv_heads)) / 16 + p->requests) * p->kv_heads >= (1l << 31) / 256)
    return fail(TJEV_GDN_EINVAL, "problem too large");
  return 0;
}

}  // namespace
}  // namespace gdn

extern "C" {

size_t tjev_gdn_paged_workspace_bytes(const tjev_gdn_paged_params* p) {
  if (gdn::validate(p)) return 0;
  return gdn::plan_of(p).bytes;
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
  gdn::set_page(A, p->page_size);
  A.pages = p->pages;
  A.Hk = p->kv_heads;
  gdn::set_group(A, p->heads / p->kv_heads);
  A.D = p->dim;
  A.fill = p->fill;
  // a scale of 0 as the smallest number, so that a masked score stays at minus infinity
  A.c = (p->scale == 0.f ? 1.17549435e-38f : p->scale) * 1.44269504088896341f;
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
  // a wave's rows of a page are addressed by 32-bit offsets from its first
  if (A.ks > (1l << 26) || A.vs > (1l << 26)) return fail(TJEV_GDN_EUNSUPPORTED, "cache slots more than 64 MB apart");
  if (any % 16) return fail(TJEV_GDN_EINVAL, "q, gate, out and the caches must be 16-byte aligned, with strides that keep their rows so");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const gdn::AttnPlan plan = gdn::plan_of(p);
  // (the parts: the ranges' notes behind them, which say how many there are, are never NaN)
  if (int s = gdn::poison_workspace(workspace, plan.bytes - (size_t)plan.G * gdn::kSplitBytes, stream)) return s;
  using gdn::AttnArgs;
  hipError_t (*const unit[2][3])(const gdn::AttnPlan&, AttnArgs&, hipStream_t) = {
      {gdn::attention_f32_64, gdn::attention_f32_128, gdn::attention_f32_256},
      {gdn::attention_bf16_64, gdn::attention_bf16_128, gdn::attention_bf16_256}};
  const hipError_t err = unit[p->dtype == TJEV_GDN_BF16][p->dim <= 64 ? 0 : p->dim <= 128 ? 1 : 2](plan, A, st);
  return err == hipSuccess ? 0 : fail(TJEV_GDN_EHIP, hipGetErrorString(err));
}

}  // extern "C"
