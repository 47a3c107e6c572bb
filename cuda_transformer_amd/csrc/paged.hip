// Argument checks that the entries of the paged key/value cache share.
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
  if (!std::isfinite(scale * kLog2e)) return fail(CTA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (rows * a.nh == 0) return CTA_OK;
  if (!o || !l) return fail(CTA_ERR_INVALID_ARGUMENT, "null output pointer");
  if (!tokens_layout_ok(q, qs, elem) || !aligned16(o))
    return fail(CTA_ERR_LAYOUT,
                std::string(what) + " needs dense heads in 16-byte aligned rows (q, o)");
  return CTA_OK;
}

}  // namespace cta
