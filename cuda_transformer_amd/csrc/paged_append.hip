// Appends the keys and values of new tokens to a paged cache, rotating queries and keys by their
// position on the way.
//
// The rotation takes the first `rot` elements of a head in pairs (x, y): elements i and i + rot/2,
// or 2i and 2i + 1 (interleaved).  With c = cos[pos][i] and s = sin[pos][i] from the caller's
// tables the pair becomes (x c - y s, y c + x s), formed in FP32 and rounded once to the tensor's
// type; what lies behind `rot`, and the values, are copied.
//
// Bandwidth bound: every element is read once and written once.  A thread takes 32 bytes of a
// head: two 16-byte chunks, rot/2 apart where they are rotated as pairs and adjacent elsewhere, so
// both members of each pair are in its registers and every access is 16 bytes wide.  It takes the
// same chunks of up to kHeadsPerThread heads of one token, for which the angle's 64 bytes are
// loaded once.  18013 tokens of 32 + 2 x 8 heads of 128 in BF16 (452 MB): 83 us, 5.45 TB/s (two
// heads a thread 88, eight 86; stores through the caches 89, loads through them too 92).
#include "paged.hpp"

namespace cta {
namespace {

template <class E>
struct AppendArgs {
  const E *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // token and head strides
  const float *cos, *sin;
  int half;  // rot / 2
  E *k_cache, *v_cache, *q_out;
  Strides3 sk, sv;
  int N, nh, nkv, groups;  // groups of heads a token: group g takes heads g, g + groups, ...
  FastDiv per_token;       // threads a token: groups x 32-byte units a head
};

template <class E>
struct Chunk {  // 16 bytes
  static constexpr int N = 16 / sizeof(E);
  E e[N] __attribute__((aligned(16)));
};
// Loads go past the caches: what is loaded is not needed again, what is stored is, by attention.
template <class E>
__device__ __forceinline__ Chunk<E> ld_chunk(const E* p) {
  return __builtin_bit_cast(Chunk<E>, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
}
// PAST: so do stores.
template <bool PAST, class E>
__device__ __forceinline__ void st_chunk(E* p, const Chunk<E>& c) {
  if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, c), reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, c);
}

// (x, y) -> (x c - y s, y c + x s)
template <class E>
__device__ __forceinline__ void rotate(E& x, E& y, float c, float s) {
  const float a = (float)x, b = (float)y;
  x = (E)fmaf(a, c, -(b * s));
  y = (E)fmaf(b, c, a * s);
}

constexpr int kHeadsPerThread = 4;

template <class E, int HS, int HEADS, bool PAST>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs<E> a, PagedPlan plan,
                                                           bool interleaved) {
  constexpr int N = Chunk<E>::N;
  constexpr int UNITS = HS / (2 * N);  // 32-byte units a head
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t last = (int64_t)a.N * a.per_token.d - 1;
  const bool live = id <= last;
  const int idc = (int)(live ? id : last);
  const int t = a.per_token.div(idc);
  const int in_token = idc - t * (int)a.per_token.d;
  const int g = in_token / UNITS, u = in_token % UNITS;
  // the unit's two chunks, in elements; rotated as pairs across rot/2, or adjacent
  const bool split = !interleaved && u * N < a.half;
  const bool turned = interleaved ? 2 * u * N < 2 * a.half : split;
  const int d0 = split ? u * N : 2 * u * N, d1 = split ? d0 + a.half : d0 + N;
  const int heads = a.nh + 2 * a.nkv;

  Chunk<E> x[HEADS], y[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = min(g + i * a.groups, heads - 1);
    const E* src = h < a.nh            ? a.q + t * a.qt + h * a.qh
                   : h < a.nh + a.nkv ? a.k + t * a.kt + (h - a.nh) * a.kh
                                      : a.v + t * a.vt + (h - a.nh - a.nkv) * a.vh;
    x[i] = ld_chunk(src + d0);
    y[i] = ld_chunk(src + d1);
  }

  // the tokens of a wave are neighbours, mostly one or two: find each one's sequence in turn
  int b = plan.B;
  if (plan.cu_q == nullptr) {
    b = t;
  } else {
    const int t0 = __builtin_amdgcn_readfirstlane(t);
    const int t1 = __builtin_amdgcn_readlane(t, 63);
    for (int w = t0; w <= t1; ++w) {
      const int s = plan.find_seq(w);
      b = t == w ? s : b;
    }
  }
  const int64_t at_pos = b < plan.B ? plan.position(b, t) : -1;
  const int pos = at_pos >= 0 && at_pos < plan.capacity ? (int)at_pos : -1;
  int row = 0;
  const int page = pos >= 0 ? plan.page(b, pos, row) : -1;
  if (!live) return;

  float c[N], s[N];  // of the N pairs: chunk against chunk, or inside the two
  const bool turn = turned && pos >= 0;
  if (turn) {
    const int64_t at = (int64_t)pos * a.half + (interleaved ? d0 / 2 : d0);
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 cv = ld4(a.cos + at + j), sv = ld4(a.sin + at + j);
      c[j] = cv.x; c[j + 1] = cv.y; c[j + 2] = cv.z; c[j + 3] = cv.w;
      s[j] = sv.x; s[j + 1] = sv.y; s[j + 2] = sv.z; s[j + 3] = sv.w;
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = g + i * a.groups;
    if (h >= heads) break;
    if (turn && h < a.nh + a.nkv) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (split) {
          rotate(x[i].e[j], y[i].e[j], c[j], s[j]);
        } else {
          Chunk<E>& z = j < N / 2 ? x[i] : y[i];
          rotate(z.e[2 * j % N], z.e[2 * j % N + 1], c[j], s[j]);
        }
      }
    }
    E* dst;
    if (h < a.nh) {
      dst = a.q_out + ((int64_t)t * a.nh + h) * HS;
    } else {
      if (page < 0) continue;
      dst = h < a.nh + a.nkv
                ? a.k_cache + page * a.sk.a + (h - a.nh) * a.sk.h + row * a.sk.r
                : a.v_cache + page * a.sv.a + (h - a.nh - a.nkv) * a.sv.h + row * a.sv.r;
    }
    st_chunk<PAST>(dst + d0, x[i]);
    st_chunk<PAST>(dst + d1, y[i]);
  }
}

template <class E, int HS>
void launch_append(AppendArgs<E> a, const PagedPlan& plan, bool interleaved, hipStream_t st) {
  constexpr int UNITS = HS / (2 * Chunk<E>::N);
  const int heads = a.nh + 2 * a.nkv;
  auto go = [&]<int HEADS, bool PAST>() {
    a.groups = (heads + HEADS - 1) / HEADS;
    a.per_token = FastDiv((uint32_t)(a.groups * UNITS));
    const int64_t threads = (int64_t)a.N * a.groups * UNITS;
    hipLaunchKernelGGL((paged_append_kernel<E, HS, HEADS, PAST>), dim3((unsigned)((threads + 255) / 256)),
                       dim3(256), 0, st, a, plan, interleaved);
  };
  const int64_t units = (int64_t)a.N * heads * UNITS;
  // several heads a thread once that still leaves every SIMD a few waves; stores past the caches
  // where reads and writes together exceed the last-level one (256 MB): it would keep none of them
  if (units < (int64_t)kNumSimds * 64 * 4 * kHeadsPerThread) go.template operator()<1, false>();
  else if (units * 64 < (int64_t)256 << 20) go.template operator()<kHeadsPerThread, false>();
  else go.template operator()<kHeadsPerThread, true>();
}

template <class E, class P>
int append(const P* q, const int64_t* qs, const P* k, const int64_t* ks, const P* v,
           const int64_t* vs, int64_t N, const float* cos, const float* sin, int64_t rot,
           int interleaved, P* q_out, const PagedArgs& pa, void* stream) {
  PagedPlan plan;
  if (int rc = check_paged(pa, sizeof(E), plan)) return rc;
  if (N < 0 || N > (int64_t)1 << 24) return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (!pa.cu_q && N != pa.B)
    return fail(CTA_ERR_INVALID_ARGUMENT, "without cu_q there is one token a sequence");
  if (rot < 0 || rot > pa.hs || rot % 16 != 0)
    return fail(CTA_ERR_INVALID_ARGUMENT, "the rotated size must be a multiple of 16 up to hs");
  if (rot > 0 && (!cos || !sin || !aligned16(cos) || !aligned16(sin)))
    return fail(CTA_ERR_LAYOUT, "cos and sin must be 16-byte aligned");
  if (N * (pa.nh + 2 * pa.nkv) * pa.hs * (int64_t)sizeof(E) / 32 >= (int64_t)1 << 31)  // threads
    return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (N == 0) return CTA_OK;
  if (!tokens_layout_ok(k, ks, sizeof(E)) || !tokens_layout_ok(v, vs, sizeof(E)) ||
      (pa.nh > 0 && (!tokens_layout_ok(q, qs, sizeof(E)) || !q_out || !aligned16(q_out))))
    return fail(CTA_ERR_LAYOUT,
                "paged_kv_append needs dense heads in 16-byte aligned rows (q, k, v, q_out)");
  AppendArgs<E> a{};
  a.q = reinterpret_cast<const E*>(q); a.k = reinterpret_cast<const E*>(k);
  a.v = reinterpret_cast<const E*>(v);
  if (pa.nh > 0) { a.qt = qs[0]; a.qh = qs[1]; }
  a.kt = ks[0]; a.kh = ks[1]; a.vt = vs[0]; a.vh = vs[1];
  a.cos = cos; a.sin = sin; a.half = (int)rot / 2;
  a.k_cache = (E*)pa.k_cache; a.v_cache = (E*)pa.v_cache; a.q_out = reinterpret_cast<E*>(q_out);
  a.sk = {pa.ks[0], pa.ks[1], pa.ks[2]};
  a.sv = {pa.vs[0], pa.vs[1], pa.vs[2]};
  a.N = (int)N; a.nh = (int)pa.nh; a.nkv = (int)pa.nkv;
  const hipStream_t st = as_stream(stream);
  if (pa.hs == 32) launch_append<E, 32>(a, plan, interleaved != 0, st);
  else if (pa.hs == 64) launch_append<E, 64>(a, plan, interleaved != 0, st);
  else launch_append<E, 128>(a, plan, interleaved != 0, st);
  return check_launch("paged_kv_append");
}

}  // namespace
}  // namespace cta

using namespace cta;

extern "C" int cta_paged_kv_append(
    const float* q, const int64_t* q_strides, const float* k, const int64_t* k_strides,
    const float* v, const int64_t* v_strides, int64_t N, int64_t nh, int64_t nkv, int64_t hs,
    const float* cos, const float* sin, int64_t rot, int interleaved, float* k_cache,
    const int64_t* k_cache_strides, float* v_cache, const int64_t* v_cache_strides,
    int64_t num_pages, int64_t page_size, const int32_t* page_table, int64_t table_stride,
    int64_t pages_per_seq, const int32_t* seq_lens, const int32_t* cu_q, int64_t B, float* q_out,
    void* stream) {
  return append<float>(q, q_strides, k, k_strides, v, v_strides, N, cos, sin, rot, interleaved,
                       q_out,
                       {k_cache_strides, v_cache_strides, num_pages, page_size, table_stride,
                        pages_per_seq, B, nh, nkv, hs, page_table, seq_lens, cu_q, k_cache,
                        v_cache},
                       stream);
}

#define CTA_APPEND_HALF(SUFFIX, TYPE)                                                             \
  extern "C" int cta_paged_kv_append_##SUFFIX(                                                    \
      const uint16_t* q, const int64_t* q_strides, const uint16_t* k, const int64_t* k_strides,   \
      const uint16_t* v, const int64_t* v_strides, int64_t N, int64_t nh, int64_t nkv,            \
      int64_t hs, const float* cos, const float* sin, int64_t rot, int interleaved,               \
      uint16_t* k_cache, const int64_t* k_cache_strides, uint16_t* v_cache,                       \
      const int64_t* v_cache_strides, int64_t num_pages, int64_t page_size,                       \
      const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,                     \
      const int32_t* seq_lens, const int32_t* cu_q, int64_t B, uint16_t* q_out, void* stream) {   \
    return append<TYPE>(q, q_strides, k, k_strides, v, v_strides, N, cos, sin, rot, interleaved,  \
                        q_out,                                                                    \
                        {k_cache_strides, v_cache_strides, num_pages, page_size, table_stride,    \
                         pages_per_seq, B, nh, nkv, hs, page_table, seq_lens, cu_q, k_cache,      \
                         v_cache},                                                                \
                        stream);                                                                  \
  }
CTA_APPEND_HALF(bf16, __bf16)
CTA_APPEND_HALF(f16, _Float16)
#undef CTA_APPEND_HALF
