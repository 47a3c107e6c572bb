// Attention of new tokens over a paged key/value cache: one a sequence (decode) or a packed chunk of
// each (prefill), causal, with groups of query heads that share a key/value head.
//
// Query head h of a token at position p reads key/value head h / (nh / nkv):
//   s_j = scale q . k_j  for j <= p, page mapped;  m = max s,  l = sum e^{s_j - m}
//   O = sum e^{s_j - m} v_j / l,  L = m + ln l;  without a key O = 0 and L = -inf.
#include "paged.hpp"

namespace cta {

int check_paged(const PagedArgs& a, int elem, PagedPlan& plan) {
  if (a.B < 0 || a.nh < 0 || a.nkv < 0 || a.num_pages < 0 || a.pages_per_seq < 0)
    return fail(CTA_ERR_INVALID_ARGUMENT, "negative size");
  if (a.hs != 32 && a.hs != 64 && a.hs != 128)
    return fail(CTA_ERR_UNSUPPORTED_HEAD_DIM,
                "Unsupported head dimension! Only hs=32, hs=64, and hs=128 are supported.");
  if (a.nkv == 0 || a.nh % a.nkv != 0)
    return fail(CTA_ERR_INVALID_ARGUMENT, "nh must be a multiple of nkv");
  if (a.page_size < 1) return fail(CTA_ERR_INVALID_ARGUMENT, "page_size must be at least 1");
  if (a.B > (int64_t)1 << 20 || a.nh > (int64_t)1 << 16 || a.num_pages >= (int64_t)1 << 31 ||
      a.page_size > (int64_t)1 << 30 || a.pages_per_seq > (int64_t)1 << 30 ||
      a.pages_per_seq * a.page_size > (int64_t)1 << 30)
    return fail(CTA_ERR_INVALID_ARGUMENT,
                "size too large (a sequence has at most 2^30 positions in its pages)");
  if (a.B > 0 && (!a.seq_lens || (!a.page_table && a.pages_per_seq > 0)))
    return fail(CTA_ERR_INVALID_ARGUMENT, "null page table or sequence lengths");
  const int64_t vec = 16 / elem;
  for (const int64_t* s : {a.ks, a.vs})
    if (!s || s[3] != 1 || s[0] % vec || s[1] % vec || s[2] % vec || s[0] < 0 || s[1] < 0 ||
        s[2] < 0 || s[2] >= (int64_t)1 << 24)
      return fail(CTA_ERR_LAYOUT,
                  "the caches need a unit last stride, 16-byte rows and row strides below 2^24");
  if (a.num_pages > 0 && (!a.k_cache || !a.v_cache || !aligned16(a.k_cache) || !aligned16(a.v_cache)))
    return fail(CTA_ERR_LAYOUT, "the caches need 16-byte aligned bases");
  plan.table = a.page_table;
  plan.table_stride = a.table_stride;
  plan.lens = a.seq_lens;
  plan.cu_q = a.cu_q;
  plan.B = (int)a.B;
  plan.num_pages = (int)a.num_pages;
  plan.capacity = a.num_pages == 0 ? 0 : (int)(a.pages_per_seq * a.page_size);
  plan.ps = FastDiv((uint32_t)a.page_size);
  return CTA_OK;
}

bool tokens_layout_ok(const void* p, const int64_t* s, int elem) {
  const int64_t vec = 16 / elem;
  return p != nullptr && s != nullptr && aligned16(p) && s[2] == 1 && s[0] % vec == 0 &&
         s[1] % vec == 0;
}

int check_paged_rows(const void* q, const int64_t* qs, int64_t rows, const PagedArgs& a, float scale,
                     const void* o, const float* l, int elem, const char* what) {
  if (rows < 0 || rows > (int64_t)1 << 24 || rows * a.nh > (int64_t)1 << 30)
    return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (!std::isfinite(scale)) return fail(CTA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (rows * a.nh == 0) return CTA_OK;
  if (!o || !l) return fail(CTA_ERR_INVALID_ARGUMENT, "null output pointer");
  if (!tokens_layout_ok(q, qs, elem) || !aligned16(o))
    return fail(CTA_ERR_LAYOUT,
                std::string(what) + " needs dense heads in 16-byte aligned rows (q, o)");
  return CTA_OK;
}

namespace {

template <class E>
struct AttnArgs {
  const E *q, *k, *v;
  int64_t qt, qh;
  Strides3 sk, sv;
  int rows, nh, group;
  float scale_log2;
  E* o;
  float* l;
};

// One wave per token and query head.  A lane takes one key of 64 for the scores, and HS / 64 (or
// one) elements of the output row for the products with V.
template <class E, int HS>
__global__ __launch_bounds__(256) void paged_attention_rows_kernel(AttnArgs<E> a, PagedPlan plan) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + wave_index();
  if (id >= (int64_t)a.rows * a.nh) return;
  const int t = (int)(id / a.nh), h = (int)(id - (int64_t)t * a.nh);
  const int kvh = h / a.group;
  const int b = plan.find_seq(t);
  const int keys = b < plan.B ? plan.keys_to(plan.position(b, t)) : 0;

  float qf[HS];
  const E* qp = a.q + t * a.qt + h * a.qh;
#pragma unroll
  for (int d = 0; d < HS; ++d) qf[d] = (float)qp[d];
  constexpr int DL = HS <= 64 ? 1 : HS / 64;
  float acc[DL] = {};
  float m = -INFINITY, l = 0.0f;
  for (int j0 = 0; j0 < keys; j0 += 64) {
    const int j = j0 + lane;
    int row = 0, page = -1;
    if (j < keys) page = plan.page(b, j, row);
    float s = -INFINITY;
    if (page >= 0) {
      const E* kp = a.k + page * a.sk.a + kvh * a.sk.h + row * a.sk.r;
      float dot = 0.0f;
#pragma unroll
      for (int d = 0; d < HS; ++d) dot = fmaf(qf[d], (float)kp[d], dot);
      s = dot * a.scale_log2;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float off = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = fast_exp2(m - off);
    const float p = page >= 0 ? fast_exp2(s - off) : 0.0f;
    l = l * alpha + wave_sum(p);
    m = m_new;
#pragma unroll
    for (int e = 0; e < DL; ++e) acc[e] *= alpha;
    for (int i = 0; i < min(64, keys - j0); ++i) {
      const int pg = __shfl(page, i), rw = __shfl(row, i);
      const float pi = __shfl(p, i);
      if (pg < 0) continue;
      const E* vp = a.v + pg * a.sv.a + kvh * a.sv.h + rw * a.sv.r;
#pragma unroll
      for (int e = 0; e < DL; ++e)
        if (lane + 64 * e < HS) acc[e] = fmaf(pi, (float)vp[lane + 64 * e], acc[e]);
    }
  }
  E* op = a.o + id * HS;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < DL; ++e)
    if (lane + 64 * e < HS) op[lane + 64 * e] = (E)(acc[e] * inv);
  if (lane == 0) a.l[id] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

template <class E, class P>
int attention(const P* q, const int64_t* qs, int64_t rows, float scale, P* o, float* l,
              const PagedArgs& pa, void* stream, const char* what) {
  PagedPlan plan;
  if (int rc = check_paged(pa, sizeof(E), plan)) return rc;
  if (int rc = check_paged_rows(q, qs, rows, pa, scale, o, l, sizeof(E), what)) return rc;
  if (rows * pa.nh == 0) return CTA_OK;
  AttnArgs<E> a;
  a.q = reinterpret_cast<const E*>(q);
  a.k = static_cast<const E*>(pa.k_cache); a.v = static_cast<const E*>(pa.v_cache);
  a.qt = qs[0]; a.qh = qs[1];
  a.sk = {pa.ks[0], pa.ks[1], pa.ks[2]};
  a.sv = {pa.vs[0], pa.vs[1], pa.vs[2]};
  a.rows = (int)rows; a.nh = (int)pa.nh; a.group = (int)(pa.nh / pa.nkv);
  a.scale_log2 = scale * kLog2e;
  a.o = reinterpret_cast<E*>(o); a.l = l;
  const hipStream_t st = as_stream(stream);
  const dim3 grid((unsigned)((rows * pa.nh + 3) / 4));
  if (pa.hs == 32) hipLaunchKernelGGL((paged_attention_rows_kernel<E, 32>), grid, dim3(256), 0, st, a, plan);
  else if (pa.hs == 64) hipLaunchKernelGGL((paged_attention_rows_kernel<E, 64>), grid, dim3(256), 0, st, a, plan);
  else hipLaunchKernelGGL((paged_attention_rows_kernel<E, 128>), grid, dim3(256), 0, st, a, plan);
  return check_launch(what);
}

}  // namespace
}  // namespace cta

using namespace cta;

#define CTA_PAGED_ATTENTION(NAME_SUFFIX, TYPE, PTR)                                               \
  extern "C" int cta_paged_attention_prefill##NAME_SUFFIX(                                        \
      const PTR* q, const int64_t* q_strides, const PTR* k_cache, const int64_t* k_cache_strides, \
      const PTR* v_cache, const int64_t* v_cache_strides, int64_t num_pages, int64_t page_size,   \
      const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,                     \
      const int32_t* seq_lens, const int32_t* cu_q, int64_t B, int64_t N, int64_t nh,             \
      int64_t nkv, int64_t hs, float scale, PTR* o, float* l, void* workspace,                    \
      int64_t workspace_bytes, void* stream) {                                                    \
    if (!cu_q) return fail(CTA_ERR_INVALID_ARGUMENT, "null cu_q");                                \
    return attention<TYPE>(q, q_strides, N, scale, o, l,                                          \
                           {k_cache_strides, v_cache_strides, num_pages, page_size, table_stride, \
                            pages_per_seq, B, nh, nkv, hs, page_table, seq_lens, cu_q, k_cache,   \
                            v_cache},                                                             \
                           stream, "paged_attention_prefill");                                    \
  }
CTA_PAGED_ATTENTION(, float, float)
CTA_PAGED_ATTENTION(_bf16, __bf16, uint16_t)
CTA_PAGED_ATTENTION(_f16, _Float16, uint16_t)
#undef CTA_PAGED_ATTENTION

extern "C" int64_t cta_paged_attention_prefill_workspace(int64_t, int64_t, int64_t, int64_t, int64_t,
                                                         int64_t, int64_t) {
  return 0;
}
