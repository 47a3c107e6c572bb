// Attention of packed new tokens over a paged key/value cache: prompts, chunks of prompts behind a
// cached context, drafts.  Causal: a token at position p sees the positions up to p.
//
// Formulas as in paged_decode.hip.  The work is matrix products (4 hs operations a visible pair),
// but for few rows on a long cache, whose bytes then count.
//  * The query heads that share a key/value head are rows of one product: row r of a sequence is
//    token r / group, head r % group, so a stage of K and V serves 128 rows whatever the group.  A
//    workgroup has 128 rows (4 waves x 32) and walks their keys in stages, global -> registers ->
//    LDS, double buffered, one barrier a stage.
//  * Pages may end anywhere: for each stage 128 threads look the rows' addresses up two stages
//    ahead and leave them in LDS, -1 for a row that holds no key.  Any page size takes this path.
//  * Both products are laid out as in the dense forward: S^T = K Q^T with a row's scores in one lane
//    (lane l, register r: key R(r, l / 32) of row l % 32), so the maximum and sum of a row need one
//    exchange, and P^T is the B operand of O^T += V^T P^T as it lies.  16-bit types: 32x32x16 MFMA, V
//    transposed in LDS with bits 2 and 3 of the key swapped (kt_pos), probabilities rounded once to
//    the type; FP32: 32x32x2 MFMA, V by rows.
//  * Workgroups are ordered by head first (neighbours go to different XCDs, so an XCD's L2 holds few
//    heads' keys), then from each sequence's last, longest tile to its first.
//  * Few rows on a long cache: `splits` workgroups share the stages of a tile and leave partial
//    results in the workspace, which a second kernel joins in order.
#include "paged.hpp"

namespace cta {
namespace {

template <class E>
struct PrefillArgs {
  const E *q, *k, *v;
  int64_t qt, qh;
  Strides3 sk, sv;
  int N, nh, nkv;
  FastDiv group;
  float scale_log2;
  int tiles, splits;  // tiles of 128 rows there may be; workgroups that share a tile's keys
  E* o;
  float* l;
  float* ws;          // splits > 1: O (splits, N nh, HS), then (m, l) (splits, N nh, 2)
};

// Tokens of sequence b: first row and count, inside [0, N) whatever cu_q holds.
__device__ __forceinline__ int tokens_of(const PagedPlan& plan, int N, int b, int& first) {
  first = max(plan.cu_q[b], 0);
  return max(min(plan.cu_q[b + 1], N) - first, 0);
}

template <class E, int HS>
__global__ __launch_bounds__(256, 2) void paged_prefill_kernel(PrefillArgs<E> a, PagedPlan plan) {
  constexpr bool F32 = sizeof(E) == 4;
  constexpr float kRescaleGap = 8.0f;  // log2 units: probabilities stay below 2^8
  constexpr int BM = 128;              // rows
  constexpr int BN = F32 ? 32 : 64;    // keys a stage
  constexpr int V16 = 16 / sizeof(E);  // elements of 16 bytes
  constexpr int KP = HS + V16;         // pitch of a K row
  constexpr int VP = F32 ? HS + 8 : BN + 8;  // pitch of a V row, or of a V^T row (16-bit)
  constexpr int KTILE = BN * KP, VTILE = F32 ? BN * VP : HS * VP;
  constexpr int CH = HS / V16;         // 16-byte chunks a row
  constexpr int LOADS = BN * CH / 256;
  constexpr int VPAIRS = 32 * CH;      // row pairs of V chunks (16-bit)
  constexpr int VL = F32 ? LOADS : 2 * ((VPAIRS + 255) / 256);
  static_assert(LOADS >= 1 && BN * CH % 256 == 0, "a stage splits evenly over the threads");
  __shared__ __attribute__((aligned(16))) E smem[2 * (KTILE + VTILE)];
  __shared__ int64_t offs[2][2][BN];   // element offsets of a stage's K and V rows, -1: no key

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  const int half = lane >> 5, col = lane & 31;
  const int G = (int)a.group.d;
  const int kvh = blockIdx.x % a.nkv, rest = blockIdx.x / a.nkv;
  const int split = rest / a.tiles, x = rest - split * a.tiles;

  auto tiles_of = [&](int i) {
    int first;
    return ((int64_t)tokens_of(plan, a.N, i, first) * G + BM - 1) / BM;
  };
  int64_t before;
  const int b = find_tile(plan.B, x, before, tiles_of);
  if (b == plan.B) {  // no tile: rows of no sequence count as empty (the join writes them if split)
    if (a.splits > 1) return;
    const int spare = a.tiles - (int)min(before, (int64_t)a.tiles - 1);
    const int lo = min(max(plan.cu_q[0], 0), a.N), hi = min(max(plan.cu_q[plan.B], lo), a.N);
    const int64_t n = (int64_t)(a.N - (hi - lo)) * G;  // padding tokens x heads
    for (int64_t i = x - before; i < n; i += spare) {
      const int j = (int)(i / G), t = j < lo ? j : j - lo + hi;
      const int64_t row = (int64_t)t * a.nh + kvh * G + (i - (int64_t)j * G);
      if (tid < HS) a.o[row * HS + tid] = (E)0.0f;
      if (tid == 0) a.l[row] = -INFINITY;
    }
    return;
  }
  int first;
  const int R = tokens_of(plan, a.N, b, first) * G;
  const int tile = (int)(tiles_of(b) - 1 - (x - before));
  auto keys_at = [&](int r) {  // keys that row r sees
    return plan.keys_to(plan.position(b, first + a.group.div(min(r, R - 1))));
  };
  const int r0 = tile * BM + wave * 32, my_r = r0 + col;
  const bool live = my_r < R;
  const int my_tok = first + a.group.div(min(my_r, R - 1));
  const int my_head = kvh * G + min(my_r, R - 1) - (my_tok - first) * G;
  const int my_keys = plan.keys_to(plan.position(b, my_tok));
  const int wave_lo = keys_at(r0), wave_hi = r0 < R ? keys_at(r0 + 31) : 0;
  const int n_keys = keys_at(tile * BM + BM - 1);
  const int n_all = (n_keys + BN - 1) / BN;
  const int s_begin = (int)((int64_t)n_all * split / a.splits);
  const int s_end = (int)((int64_t)n_all * (split + 1) / a.splits);

  // This lane's query row: the chunks of d that its half takes of each MFMA step
  constexpr int QC = HS / (2 * V16);
  u32x4 qf[QC];
  {
    const E* qp = a.q + my_tok * a.qt + my_head * a.qh + V16 * half;
#pragma unroll
    for (int s = 0; s < QC; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + 2 * V16 * s);
  }

  f32x16 oacc[HS / 32];
#pragma unroll
  for (int d = 0; d < HS / 32; ++d) oacc[d] = zero16();
  float mb = -INFINITY, l_run = 0.0f;  // exponent offset, and this lane's part of the row's sum

  // Page of row `lane` of a stage, -1 for none: threads 0 .. BN - 1 for K, BN .. 2 BN - 1 for V.
  const int32_t* table = plan.table + b * plan.table_stride;
  auto look_up = [&](int stage) -> int64_t {
    const int which = tid / BN, j = stage * BN + tid % BN;
    if (which > 1 || stage >= s_end || j >= n_keys) return -1;
    const int i = plan.ps.div(j), row = j - i * (int)plan.ps.d;
    const int page = table[i];
    if ((uint32_t)page >= (uint32_t)plan.num_pages) return -1;
    return which == 0 ? page * a.sk.a + row * a.sk.r : page * a.sv.a + row * a.sv.r;
  };
  auto put = [&](int stage, int64_t off) {
    if (tid < 2 * BN) offs[stage & 1][tid / BN][tid % BN] = off;
  };

  const E* kb = a.k + kvh * a.sk.h;
  const E* vb = a.v + kvh * a.sv.h;
  u32x4 kst[LOADS], vst[VL];
  auto vtask = [&](int u2, int& rp, int& ch) {  // 16-bit: rows 2 rp, 2 rp + 1 of chunk ch
    rp = lane & 31;
    ch = 2 * (wave + 4 * u2) + (lane >> 5);
    return VPAIRS % 256 == 0 || ch < CH;
  };
  // bit j: row j of the stage holds a key.  Rows that hold none read the first page's first row;
  // their scores are masked, and their V counts as zeros.
  auto gload = [&](int stage) -> uint64_t {
    const int64_t(*of)[BN] = offs[stage & 1];
    const uint64_t ok = __ballot(of[0][lane % BN] >= 0);
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = tid + 256 * u;
      kst[u] = *reinterpret_cast<const u32x4*>(kb + max(of[0][c / CH], (int64_t)0) + V16 * (c % CH));
    }
    if constexpr (F32) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int c = tid + 256 * u;
        const int64_t at = of[1][c / CH];
        vst[u] = *reinterpret_cast<const u32x4*>(vb + max(at, (int64_t)0) + V16 * (c % CH));
        if (at < 0) vst[u] = u32x4{0, 0, 0, 0};
      }
    } else {
#pragma unroll
      for (int u2 = 0; u2 < VL / 2; ++u2) {
        int rp, ch;
        if (!vtask(u2, rp, ch)) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t at = of[1][2 * rp + e];
          vst[2 * u2 + e] = *reinterpret_cast<const u32x4*>(vb + max(at, (int64_t)0) + V16 * ch);
          if (at < 0) vst[2 * u2 + e] = u32x4{0, 0, 0, 0};
        }
      }
    }
    return ok;
  };
  auto lstore = [&](int buf) {
    E* ks = smem + buf * (KTILE + VTILE);
    E* vt = ks + KTILE;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = tid + 256 * u;
      *reinterpret_cast<u32x4*>(ks + (c / CH) * KP + V16 * (c % CH)) = kst[u];
      if constexpr (F32)
        *reinterpret_cast<u32x4*>(vt + (c / CH) * VP + V16 * (c % CH)) = vst[u];
    }
    if constexpr (!F32) {
#pragma unroll
      for (int u2 = 0; u2 < VL / 2; ++u2) {
        int rp, ch;
        if (!vtask(u2, rp, ch)) continue;
        const u32x4 e0 = vst[2 * u2], e1 = vst[2 * u2 + 1];
        uint32_t* col2 = reinterpret_cast<uint32_t*>(vt + kt_pos(2 * rp));
#pragma unroll
        for (int t = 0; t < 4; ++t) {  // d = 8 ch + 2 t and 8 ch + 2 t + 1 of both rows
          col2[(8 * ch + 2 * t) * (VP / 2)] = pack_lo16(e0[t], e1[t]);
          col2[(8 * ch + 2 * t + 1) * (VP / 2)] = pack_hi16(e0[t], e1[t]);
        }
      }
    }
  };

  // Scaled scores of one 32-key tile -> probabilities against the row's offset, which moves only
  // when some row of the wave sees a score more than kRescaleGap above it.
  auto softmax_step = [&](f32x16& s) {
    const float mb0 = mb == -INFINITY ? 0.0f : mb;
    float t[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __fsub_rn(s[r], mb0);
      t[r] = s[r];
    }
    const float my = max_halves(max3_tree(t));
    if (__any(mb == -INFINITY || my > kRescaleGap)) {
      const float mb_new = fmaxf(mb, mb0 + my);
      const float to = mb_new == -INFINITY ? 0.0f : mb_new;
      const float alpha = fast_exp2(mb - to);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < HS / 32; ++d) oacc[d] *= alpha;
      const float shift = to - mb0;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] -= shift;
      mb = mb_new;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(s[r]);
      t[r] = s[r];
    }
#pragma unroll
    for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
      for (int r = 0; r < w; ++r) t[r] += t[r + w];
    l_run += t[0];
  };

  uint64_t mask = 0, mask_next = 0;
  if (s_begin < s_end) {  // workgroup-uniform
    put(s_begin, look_up(s_begin));
    put(s_begin + 1, look_up(s_begin + 1));
    __syncthreads();
    mask = gload(s_begin);
    lstore(s_begin & 1);
    __syncthreads();
  }
  for (int st = s_begin; st < s_end; ++st) {
    const int64_t off2 = look_up(st + 2);
    if (st + 1 < s_end) mask_next = gload(st + 1);
    const E* ks = smem + (st & 1) * (KTILE + VTILE);
    const E* vt = ks + KTILE;
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int j0 = st * BN + 32 * sub;
      if (j0 >= wave_hi) continue;  // no row of this wave sees the tile
      const uint32_t ok = (uint32_t)(mask >> (32 * sub));
      f32x16 s = zero16();
      const E* krow = ks + (32 * sub + col) * KP + V16 * half;
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const u32x4 kk = *reinterpret_cast<const u32x4*>(krow + 2 * V16 * c);
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s = mfma32(__uint_as_float(kk[i]), __uint_as_float(qf[c][i]), s);
        } else {
          s = Half16<E>::mfma(__builtin_bit_cast(vec8_t<E>, kk), __builtin_bit_cast(vec8_t<E>, qf[c]), s);
        }
      }
      // rounded before the offset is taken off: equal scores of any size have equal exponents
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __fmul_rn(s[r], a.scale_log2);
      if (j0 + 32 > wave_lo || ok != 0xffffffffu) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = mfma_row(r, half);
          if (j0 + j >= my_keys || !(ok >> j & 1)) s[r] = -INFINITY;
        }
      }
      softmax_step(s);
      if constexpr (F32) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const E* vrow = vt + (32 * sub + mfma_row(r, half)) * VP + col;
#pragma unroll
          for (int d = 0; d < HS / 32; ++d) oacc[d] = mfma32(vrow[32 * d], s[r], oacc[d]);
        }
      } else {
        vec8_t<E> pf[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) pf[r >> 3][r & 7] = (E)s[r];
#pragma unroll
        for (int d = 0; d < HS / 32; ++d) {
          const E* vrow = vt + (d * 32 + col) * VP + sub * 32 + 8 * half;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            oacc[d] = Half16<E>::mfma(ld8<E>(vrow + 16 * i), pf[i], oacc[d]);
        }
      }
    }
    mask = mask_next;
    if (st + 1 < s_end) lstore((st + 1) & 1);
    put(st + 2, off2);
    __syncthreads();
  }

  const float l_tot = sum_halves(l_run);
  if (!live) return;
  const int64_t row = (int64_t)my_tok * a.nh + my_head;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)split * a.N * a.nh) + row;
    float* op = a.ws + at * HS;
#pragma unroll
    for (int d = 0; d < HS / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        st4(op + d * 32 + 8 * g + 4 * half, make_float4(oacc[d][4 * g], oacc[d][4 * g + 1],
                                                        oacc[d][4 * g + 2], oacc[d][4 * g + 3]));
    if (half == 0)
      *reinterpret_cast<float2*>(a.ws + (int64_t)a.splits * a.N * a.nh * HS + at * 2) = make_float2(mb, l_tot);
    return;
  }
  E* op = a.o + row * HS;
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
#pragma unroll
  for (int d = 0; d < HS / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      struct alignas(4 * sizeof(E)) { E e[4]; } o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) o4.e[e] = (E)(oacc[d][4 * g + e] * inv);
      *reinterpret_cast<decltype(o4)*>(op + d * 32 + 8 * g + 4 * half) = o4;
    }
  if (half == 0) a.l[row] = l_tot == 0.0f ? -INFINITY : mb * kLn2 + logf(l_tot);
}

// Joins the splits' parts of each row in order; padding rows.  A thread takes four elements.
template <class E, int HS>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(PrefillArgs<E> a, PagedPlan plan) {
  const int64_t rows = (int64_t)a.N * a.nh;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / (HS / 4);
  const int d = 4 * (int)(id % (HS / 4));
  if (row >= rows) return;
  const int t = (int)(row / a.nh);
  const bool padding = t < plan.cu_q[0] || t >= plan.cu_q[plan.B];
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.splits * rows * HS);
  float m = -INFINITY, l = 0.0f;
  float4 o = zero4();
  if (!padding) {
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[s * rows + row].x);
    const float off = m == -INFINITY ? 0.0f : m;
    for (int s = 0; s < a.splits; ++s) {
      const float2 p = ml[s * rows + row];
      const float f = fast_exp2(p.x - off);
      const float4 v = ld4(a.ws + (s * rows + row) * HS + d);
      l = fmaf(f, p.y, l);
      o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  E* op = a.o + row * HS + d;
  op[0] = (E)(o.x * inv); op[1] = (E)(o.y * inv);
  op[2] = (E)(o.z * inv); op[3] = (E)(o.w * inv);
  if (d == 0) a.l[row] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

// Tiles of 128 rows a key/value head may have (each sequence may end inside one), one more than
// that so that some workgroup is left for padding rows; and how many workgroups share a tile's keys:
// as many as fill the GPU's 512 places, eight stages of 64 keys or more each.
struct PrefillGrid {
  int64_t tiles;
  int splits;
};
PrefillGrid prefill_grid(int64_t B, int64_t N, int64_t nh, int64_t nkv, int64_t capacity) {
  PrefillGrid g;
  g.tiles = N * (nh / nkv) / 128 + std::min(B, N) + 1;
  const int64_t fill = 512 / (std::max<int64_t>(g.tiles - 1, 1) * nkv);
  g.splits = (int)std::max<int64_t>(1, std::min<int64_t>({fill, capacity / 512, 16}));
  return g;
}

template <class E, int HS>
void launch_prefill(const PrefillArgs<E>& a, const PagedPlan& plan, hipStream_t st) {
  hipLaunchKernelGGL((paged_prefill_kernel<E, HS>), dim3((unsigned)((int64_t)a.tiles * a.nkv * a.splits)),
                     dim3(256), 0, st, a, plan);
  if (a.splits > 1)
    hipLaunchKernelGGL((paged_prefill_join_kernel<E, HS>),
                       dim3((unsigned)(((int64_t)a.N * a.nh * (HS / 4) + 255) / 256)), dim3(256), 0,
                       st, a, plan);
}

template <class E, class P>
int prefill(const P* q, const int64_t* qs, int64_t N, float scale, P* o, float* l, void* ws,
            int64_t ws_bytes, const PagedArgs& pa, void* stream) {
  PagedPlan plan;
  if (int rc = check_paged(pa, sizeof(E), plan)) return rc;
  if (!pa.cu_q) return fail(CTA_ERR_INVALID_ARGUMENT, "null cu_q");
  if (int rc = check_paged_rows(q, qs, N, pa, scale, o, l, sizeof(E), "paged_attention_prefill"))
    return rc;
  if (N * pa.nh == 0) return CTA_OK;
  const PrefillGrid g = prefill_grid(pa.B, N, pa.nh, pa.nkv, plan.capacity);
  if (g.tiles * pa.nkv * g.splits >= (int64_t)1 << 31)
    return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (g.splits > 1 && (!ws || !aligned16(ws) ||
                       ws_bytes < cta_paged_attention_prefill_workspace(
                                      pa.B, N, pa.nh, pa.nkv, pa.hs, pa.pages_per_seq, pa.page_size)))
    return fail(CTA_ERR_INVALID_ARGUMENT, "paged_attention_prefill needs its workspace");
  PrefillArgs<E> a;
  a.q = reinterpret_cast<const E*>(q);
  a.k = static_cast<const E*>(pa.k_cache); a.v = static_cast<const E*>(pa.v_cache);
  a.qt = qs[0]; a.qh = qs[1];
  a.sk = {pa.ks[0], pa.ks[1], pa.ks[2]};
  a.sv = {pa.vs[0], pa.vs[1], pa.vs[2]};
  a.N = (int)N; a.nh = (int)pa.nh; a.nkv = (int)pa.nkv;
  a.group = FastDiv((uint32_t)(pa.nh / pa.nkv));
  a.scale_log2 = scale * kLog2e;
  a.tiles = (int)g.tiles; a.splits = g.splits;
  a.o = reinterpret_cast<E*>(o); a.l = l; a.ws = static_cast<float*>(ws);
  const hipStream_t st = as_stream(stream);
  if (pa.hs == 32) launch_prefill<E, 32>(a, plan, st);
  else if (pa.hs == 64) launch_prefill<E, 64>(a, plan, st);
  else launch_prefill<E, 128>(a, plan, st);
  return check_launch("paged_attention_prefill");
}

}  // namespace
}  // namespace cta

using namespace cta;

extern "C" int64_t cta_paged_attention_prefill_workspace(int64_t B, int64_t N, int64_t nh,
                                                         int64_t nkv, int64_t hs,
                                                         int64_t pages_per_seq, int64_t page_size) {
  if (B <= 0 || N <= 0 || nh <= 0 || nkv <= 0 || pages_per_seq <= 0 || page_size <= 0 ||
      (hs != 32 && hs != 64 && hs != 128) || pages_per_seq > ((int64_t)1 << 30) / page_size)
    return 0;
  const PrefillGrid g = prefill_grid(B, N, nh, nkv, pages_per_seq * page_size);
  return g.splits > 1 ? (int64_t)g.splits * N * nh * (hs + 2) * 4 : 0;
}

#define CTA_PAGED_PREFILL(SUFFIX, TYPE, PTR)                                                      \
  extern "C" int cta_paged_attention_prefill##SUFFIX(                                             \
      const PTR* q, const int64_t* q_strides, const PTR* k_cache, const int64_t* k_cache_strides, \
      const PTR* v_cache, const int64_t* v_cache_strides, int64_t num_pages, int64_t page_size,   \
      const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,                     \
      const int32_t* seq_lens, const int32_t* cu_q, int64_t B, int64_t N, int64_t nh,             \
      int64_t nkv, int64_t hs, float scale, PTR* o, float* l, void* workspace,                    \
      int64_t workspace_bytes, void* stream) {                                                    \
    return prefill<TYPE>(q, q_strides, N, scale, o, l, workspace, workspace_bytes,                \
                         {k_cache_strides, v_cache_strides, num_pages, page_size, table_stride,   \
                          pages_per_seq, B, nh, nkv, hs, page_table, seq_lens, cu_q, k_cache,     \
                          v_cache},                                                               \
                         stream);                                                                 \
  }
CTA_PAGED_PREFILL(, float, float)
CTA_PAGED_PREFILL(_bf16, __bf16, uint16_t)
CTA_PAGED_PREFILL(_f16, _Float16, uint16_t)
#undef CTA_PAGED_PREFILL
