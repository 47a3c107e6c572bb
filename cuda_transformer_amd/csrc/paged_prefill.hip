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
//    ahead and leave them in LDS, that of a row of zeros for a row that holds no key.  Any page
//    size takes this path.
//  * Both products are laid out as in the dense forward: S^T = K Q^T with a row's scores in one lane
//    (lane l, register r: key R(r, l / 32) of row l % 32), so the maximum and sum of a row need one
//    exchange, and P^T is the B operand of O^T += V^T P^T as it lies.
//  * 16-bit types: 32x32x16 MFMA, probabilities rounded once to the type.  K and V stages go straight
//    from memory to LDS, by rows, and V's operand is read transposed (ds_read_b64_tr_b16: the 16
//    lanes of a group read 16 d of 4 keys and get 4 keys of one d).  A row's 16-byte chunks are
//    swapped by its number (row_swap), so that neither read meets a bank twice.
//  * FP32: 32x32x2 MFMA, stages through registers.
//  * Workgroups are ordered by head and split first (neighbours go to different XCDs, so an XCD's L2
//    holds few heads' keys), then from each sequence's last, longest tile to its first.
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

constexpr int BM = 128;              // rows a workgroup
constexpr float kRescaleGap = 8.0f;  // log2 units: probabilities stay below 2^8

// A workgroup's tile of rows: rows tile BM .. of the R that sequence b has for key/value head kvh.
struct RowTile {
  int b, first, R, tile, kvh, split;
};
// Finds it, or fills this workgroup's share of the padding rows and returns false.
template <class E, int HS>
__device__ __forceinline__ bool find_rows(const PrefillArgs<E>& a, const PagedPlan& plan, RowTile& w) {
  const int G = (int)a.group.d, tid = threadIdx.x;
  const int x = blockIdx.x / (a.nkv * a.splits), rest = blockIdx.x - x * (a.nkv * a.splits);
  w.split = rest / a.nkv;
  w.kvh = rest - w.split * a.nkv;
  auto tiles_of = [&](int i) {
    int first;
    return ((int64_t)tokens_of(plan, a.N, i, first) * G + BM - 1) / BM;
  };
  int64_t before;
  w.b = find_tile(plan.B, x, before, tiles_of);
  if (w.b < plan.B) {
    int first;
    w.R = uniform(tokens_of(plan, a.N, w.b, first)) * G;
    w.first = uniform(first);
    w.tile = (w.R + BM - 1) / BM - 1 - (int)(x - before);
    return true;
  }
  // no tile: rows of no sequence count as empty (the join writes them if split)
  if (a.splits > 1) return false;
  const int spare = a.tiles - (int)min(before, (int64_t)a.tiles - 1);
  const int lo = min(max(plan.cu_q[0], 0), a.N), hi = min(max(plan.cu_q[plan.B], lo), a.N);
  const int64_t n = (int64_t)(a.N - (hi - lo)) * G;  // padding tokens x heads
  for (int64_t i = x - before; i < n; i += spare) {
    const int j = (int)(i / G), t = j < lo ? j : j - lo + hi;
    const int64_t row = (int64_t)t * a.nh + w.kvh * G + (i - (int64_t)j * G);
    if (tid < HS) a.o[row * HS + tid] = (E)0.0f;
    if (tid == 0) a.l[row] = -INFINITY;
  }
  return false;
}

// The rows of one wave, one a lane (both halves): which they are and which keys they see.
struct WaveRows {
  bool live;
  int token, head, keys;   // of this lane's row (the sequence's last one behind the end)
  int lo, hi;              // the fewest and the most keys that a row of the wave sees
  int n_keys;              // ... a row of the workgroup
};
template <class E>
__device__ __forceinline__ WaveRows wave_rows(const PrefillArgs<E>& a, const PagedPlan& plan,
                                              const RowTile& w, int wave, int col) {
  auto token = [&](int r) { return w.first + a.group.div(min(r, w.R - 1)); };
  const int64_t p0 = uniform(plan.position(w.b, 0));  // of packed token 0, were it the sequence's
  auto keys = [&](int r) { return plan.keys_to(p0 + token(r)); };
  const int r0 = w.tile * BM + wave * 32, r = r0 + col;
  WaveRows v;
  v.live = r < w.R;
  v.token = token(r);
  v.head = w.kvh * (int)a.group.d + min(r, w.R - 1) - (v.token - w.first) * (int)a.group.d;
  v.keys = keys(r);
  v.lo = uniform(keys(r0));
  v.hi = r0 < w.R ? uniform(keys(r0 + 31)) : 0;
  v.n_keys = uniform(keys(w.tile * BM + BM - 1));
  return v;
}

// The first half of an online-softmax step: scores s (N of this lane's row) become exponents against
// the row's offset mb, which moves only when some row of the wave sees one more than kRescaleGap
// above it; `mask` sets those that do not count to -inf, `rescale` scales the output and the sum.
// The exponent of score x is x c - mb in one rounding while offsets are small.  Beyond 2^20, where
// the offset's own rounding would show, x c is rounded first: equal scores of any size then have
// equal exponents.
template <int N, class M, class F>
__device__ __forceinline__ void exponents(float (&s)[N], float c, float& mb, M&& mask, F&& rescale) {
  const float mb0 = mb == -INFINITY ? 0.0f : mb;
  if (__all(fabsf(mb0) <= 0x1p20f)) {
#pragma unroll
    for (int r = 0; r < N; ++r) s[r] = fmaf(s[r], c, -mb0);
  } else {
#pragma unroll
    for (int r = 0; r < N; ++r) s[r] = __fsub_rn(__fmul_rn(s[r], c), mb0);
  }
  mask();
  float t[N];
#pragma unroll
  for (int r = 0; r < N; ++r) t[r] = s[r];
  const float my = max_halves(max3_tree(t));
  if (__any(mb == -INFINITY || my > kRescaleGap)) {
    const float mb_new = fmaxf(mb, mb0 + my);
    const float to = mb_new == -INFINITY ? 0.0f : mb_new;
    rescale(fast_exp2(mb - to));
    const float shift = to - mb0;
#pragma unroll
    for (int r = 0; r < N; ++r) s[r] -= shift;
    mb = mb_new;
  }
}
// 2^s in place, and their sum.
template <int N>
__device__ __forceinline__ float exp2_sum(float* s) {
  float t[N];
#pragma unroll
  for (int r = 0; r < N; ++r) t[r] = s[r] = fast_exp2(s[r]);
#pragma unroll
  for (int w = N / 2; w >= 1; w >>= 1)
#pragma unroll
    for (int r = 0; r < w; ++r) t[r] += t[r + w];
  return t[0];
}

// Writes a lane's part of its row: the result, or the split's part of it.
template <class E, int HS>
__device__ __forceinline__ void store_rows(const PrefillArgs<E>& a, const RowTile& w, const WaveRows& v,
                                           const f32x16 (&oacc)[HS / 32], float mb, float l_run, int half) {
  const float l_tot = sum_halves(l_run);
  if (!v.live) return;
  const int64_t row = (int64_t)v.token * a.nh + v.head;
  if (a.splits > 1) {
    const int64_t at = (int64_t)w.split * a.N * a.nh + row;
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

// What a row that holds no key reads.
__device__ const float kZeroRow[128] = {};

// Chunk c (16 bytes) of a row of RB bytes goes to chunk c ^ row_swap(row).  LDS serves 256 bytes a
// cycle from 64 banks: 16 lanes of a 16-byte read (one chunk of 16 rows: the swap takes each value
// of the chunks that share a row's banks once), 32 lanes of an 8-byte one (four chunks of 4 rows: the
// swap's upper bits are those of the row that do not choose the bank yet).
template <int RB>
__device__ __forceinline__ constexpr int row_swap(int row) {
  const int low = row >> 2 & 3;
  return RB == 256 ? (row & 3) << 2 | low : RB == 128 ? (row >> 1 & 1) << 2 | low : low;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// Four keys (rows) of this lane's d: lane i of a group of 16 reads 4 d of row i / 4 at p.
__device__ __forceinline__ s16x4 ld_transposed(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
}

template <class E, int HS>
__global__ __launch_bounds__(256, HS == 32 ? 3 : 2) void paged_prefill_half_kernel(PrefillArgs<E> a, PagedPlan plan) {
  constexpr int BN = 64;           // keys a stage, one step of the softmax
  constexpr int RB = 2 * HS;       // bytes of a row
  constexpr int STAGE = BN * RB;   // bytes of K (or V) a stage
  constexpr int COPIES = STAGE / 4096;      // 1 KiB copies a wave makes of each
  constexpr int ROWS = 1024 / RB;  // rows a copy
  constexpr int QC = HS / 16;      // MFMA steps of S over d
  constexpr int ND = HS / 32;
  constexpr int kAhead = QC < 3 ? 2 * QC : 6;
  constexpr int kDsRead = 0x100, kMfma = 0x8;  // instruction classes of sched_group_barrier
  // two buffers, apart so that reads of one are known not to meet the copies into the other
  __shared__ __attribute__((aligned(16))) char buf0[2 * STAGE], buf1[2 * STAGE];
  __shared__ uint64_t row_at[2][2][BN];  // addresses of a stage's K and V rows
  __shared__ uint64_t holds[4];          // bit j: row j holds a key; four stages, as a slow wave
                                         // may still look at a stage while the third is put

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  const int half = lane >> 5, col = lane & 31;
  RowTile w;
  if (!find_rows<E, HS>(a, plan, w)) return;
  const WaveRows v = wave_rows(a, plan, w, wave, col);
  const int n_all = (v.n_keys + BN - 1) / BN;
  const int s_begin = (int)((int64_t)n_all * w.split / a.splits);
  const int s_end = (int)((int64_t)n_all * (w.split + 1) / a.splits);

  // This lane's query row, d = 16 s + 8 half .. of step s
  vec8_t<E> qf[QC];
  {
    const E* qp = a.q + v.token * a.qt + v.head * a.qh + 8 * half;
#pragma unroll
    for (int s = 0; s < QC; ++s) qf[s] = ld8<E>(qp + 16 * s);
  }
  f32x16 oacc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) oacc[d] = zero16();
  float mb = -INFINITY, l_run = 0.0f;  // exponent offset, and this lane's part of the row's sum

  // Page of key `lane` of a stage, by waves 0 (K) and 1 (V); -1: none.
  const int32_t* table = plan.table + w.b * plan.table_stride;
  auto look_up = [&](int stage) {
    const int j = stage * BN + lane;
    return wave < 2 && stage < s_end && j < v.n_keys ? table[plan.ps.div(j)] : -1;
  };
  const E* kb = a.k + w.kvh * a.sk.h;
  const E* vb = a.v + w.kvh * a.sv.h;
  auto put = [&](int stage, int page) {
    if (wave >= 2) return;
    const int j = stage * BN + lane, row = j - plan.ps.div(j) * (int)plan.ps.d;
    const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
    const E* p = wave == 0 ? kb + page * a.sk.a + row * a.sk.r : vb + page * a.sv.a + row * a.sv.r;
    row_at[stage & 1][wave][lane] = ok ? (uint64_t)p : (uint64_t)kZeroRow;
    const uint64_t all = __ballot(ok);
    if (tid == 0) holds[stage & 3] = all;
  };
  // Copy c of a stage: rows ROWS (4 c + wave) .., 16 bytes a lane, chunks swapped at the source.
  const int c_row = ROWS * wave + lane / (RB / 16);
  const int c_at = ((lane % (RB / 16)) ^ row_swap<RB>(c_row)) * 16;
  auto copy = [&](int stage, char* to) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        const char* p = reinterpret_cast<const char*>(row_at[stage & 1][kv][4 * ROWS * c + c_row]) + c_at;
        async_copy16(reinterpret_cast<const float*>(p),
                     reinterpret_cast<float*>(to + kv * STAGE + 1024 * (4 * c + wave)));
      }
  };

  // K operand: row col (+ 32), chunk 2 s + half of step s.  V operand: rows 4 half + lane % 16 / 4
  // (+ 16 i), 4 d from 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) on; then 8 rows on, where the swap
  // differs by 2 chunks.
  int k_at[QC], v_at[2][ND];
#pragma unroll
  for (int s = 0; s < QC; ++s) k_at[s] = col * RB + ((2 * s + half) ^ row_swap<RB>(col)) * 16;
  const int v_row = 4 * half + lane % 16 / 4;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int chunk = 4 * d + 2 * (lane / 16 % 2) + lane % 4 / 2;
    v_at[0][d] = v_row * RB + (chunk ^ row_swap<RB>(v_row)) * 16 + lane % 2 * 8;
    v_at[1][d] = v_at[0][d] ^ 32;
  }

  auto compute = [&](int st, const char* from) {
    const int j0 = st * BN;
    if (j0 >= v.hi) return;  // no row of this wave sees the stage
    const uint64_t ok = holds[st & 3];
    f32x16 s2[2] = {zero16(), zero16()};
#pragma unroll
    for (int c = 0; c < QC; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s2[i] = Half16<E>::mfma(*reinterpret_cast<const vec8_t<E>*>(from + k_at[c] + 32 * RB * i), qf[c], s2[i]);
    // the reads run ahead of the products by up to kAhead operands (LDS answers after about 100
    // cycles, a product takes 32)
    __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
    for (int i = 0; i < 2 * QC; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      if (i + kAhead < 2 * QC) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
    }
    float s[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) s[r] = s2[r >> 4][r & 15];
    exponents(
        s, a.scale_log2, mb,
        [&] {
          if (j0 + BN <= v.lo && ~ok == 0) return;
#pragma unroll
          for (int r = 0; r < 32; ++r) {
            const int j = 32 * (r >> 4) + mfma_row(r & 15, half);
            if (j0 + j >= v.keys || !(ok >> j & 1)) s[r] = -INFINITY;
          }
        },
        [&](float alpha) {
          l_run *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) oacc[d] *= alpha;
        });
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 16 keys: the lane's 4 half + 0 .. 3 and 8 more
      l_run += exp2_sum<8>(s + 8 * i);
      vec8_t<E> pf;
#pragma unroll
      for (int r = 0; r < 8; ++r) pf[r] = (E)s[8 * i + r];
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const char* p = from + STAGE + 16 * RB * i;
        struct { s16x4 a, b; } t = {ld_transposed(p + v_at[0][d]), ld_transposed(p + v_at[1][d] + 8 * RB)};
        oacc[d] = Half16<E>::mfma(__builtin_bit_cast(vec8_t<E>, t), pf, oacc[d]);
      }
    }
  };
  auto step = [&](int st, const char* from, char* to) {
    const int page = look_up(st + 2);
    if (st + 1 < s_end) copy(st + 1, to);
    compute(st, from);
    put(st + 2, page);
    vm_wait_all();
    __syncthreads();
  };

  if (s_begin < s_end) {  // workgroup-uniform
    put(s_begin, look_up(s_begin));
    put(s_begin + 1, look_up(s_begin + 1));
    __syncthreads();
    copy(s_begin, buf0);
    vm_wait_all();
    __syncthreads();
  }
  for (int st = s_begin; st < s_end; st += 2) {
    step(st, buf0, buf1);
    if (st + 1 < s_end) step(st + 1, buf1, buf0);
  }
  store_rows<E, HS>(a, w, v, oacc, mb, l_run, half);
}

template <int HS>
__global__ __launch_bounds__(256, 2) void paged_prefill_f32_kernel(PrefillArgs<float> a, PagedPlan plan) {
  constexpr int BN = 32;            // keys a stage
  constexpr int KP = HS + 4;        // pitch of a K row
  constexpr int VP = HS + 8;        // pitch of a V row
  constexpr int CH = HS / 4;        // 16-byte chunks a row
  constexpr int LOADS = BN * CH / 256;
  __shared__ __attribute__((aligned(16))) float smem[2][BN * (KP + VP)];
  __shared__ uint64_t row_at[2][2][BN];  // addresses of a stage's K and V rows
  __shared__ uint32_t holds[4];          // bit j: row j holds a key (four stages, as above)

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  const int half = lane >> 5, col = lane & 31;
  RowTile w;
  if (!find_rows<float, HS>(a, plan, w)) return;
  const WaveRows v = wave_rows(a, plan, w, wave, col);
  const int n_all = (v.n_keys + BN - 1) / BN;
  const int s_begin = (int)((int64_t)n_all * w.split / a.splits);
  const int s_end = (int)((int64_t)n_all * (w.split + 1) / a.splits);

  float4 qf[HS / 8];  // d = 8 s + 4 half ..
  {
    const float* qp = a.q + v.token * a.qt + v.head * a.qh + 4 * half;
#pragma unroll
    for (int s = 0; s < HS / 8; ++s) qf[s] = ld4(qp + 8 * s);
  }
  f32x16 oacc[HS / 32];
#pragma unroll
  for (int d = 0; d < HS / 32; ++d) oacc[d] = zero16();
  float mb = -INFINITY, l_run = 0.0f;

  // Page of a stage's key lane % 32, in wave 0: lanes 0 .. 31 for K, 32 .. 63 for V.
  const int32_t* table = plan.table + w.b * plan.table_stride;
  auto look_up = [&](int stage) {
    const int j = stage * BN + col;
    return wave == 0 && stage < s_end && j < v.n_keys ? table[plan.ps.div(j)] : -1;
  };
  const float* kb = a.k + w.kvh * a.sk.h;
  const float* vb = a.v + w.kvh * a.sv.h;
  auto put = [&](int stage, int page) {
    if (wave != 0) return;
    const int j = stage * BN + col, row = j - plan.ps.div(j) * (int)plan.ps.d;
    const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
    const float* p = half == 0 ? kb + page * a.sk.a + row * a.sk.r : vb + page * a.sv.a + row * a.sv.r;
    row_at[stage & 1][half][col] = ok ? (uint64_t)p : (uint64_t)kZeroRow;
    const uint64_t all = __ballot(ok);
    if (tid == 0) holds[stage & 3] = (uint32_t)all;
  };
  float4 kst[LOADS], vst[LOADS];
  auto gload = [&](int stage) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = tid + 256 * u;
      kst[u] = ld4(reinterpret_cast<const float*>(row_at[stage & 1][0][c / CH]) + 4 * (c % CH));
      vst[u] = ld4(reinterpret_cast<const float*>(row_at[stage & 1][1][c / CH]) + 4 * (c % CH));
    }
  };
  auto lstore = [&](int stage) {
    float* ks = smem[stage & 1];
    float* vs = ks + BN * KP;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = tid + 256 * u;
      st4(ks + (c / CH) * KP + 4 * (c % CH), kst[u]);
      st4(vs + (c / CH) * VP + 4 * (c % CH), vst[u]);
    }
  };
  if (s_begin < s_end) {  // workgroup-uniform
    put(s_begin, look_up(s_begin));
    put(s_begin + 1, look_up(s_begin + 1));
    __syncthreads();
    gload(s_begin);
    lstore(s_begin);
    __syncthreads();
  }
  for (int st = s_begin; st < s_end; ++st) {
    const int page = look_up(st + 2);
    if (st + 1 < s_end) gload(st + 1);
    const float* ks = smem[st & 1];
    const float* vs = ks + BN * KP;
    const int j0 = st * BN;
    if (j0 < v.hi) {  // else no row of this wave sees the stage
      const uint32_t ok = holds[st & 3];
      f32x16 acc = zero16();
#pragma unroll
      for (int c = 0; c < HS / 8; ++c) {
        const float4 k4 = ld4(ks + col * KP + 4 * half + 8 * c);
        acc = mfma32(k4.x, qf[c].x, acc);
        acc = mfma32(k4.y, qf[c].y, acc);
        acc = mfma32(k4.z, qf[c].z, acc);
        acc = mfma32(k4.w, qf[c].w, acc);
      }
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc[r];
      exponents(
          s, a.scale_log2, mb,
          [&] {
            if (j0 + BN <= v.lo && ~ok == 0) return;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int j = mfma_row(r, half);
              if (j0 + j >= v.keys || !(ok >> j & 1)) s[r] = -INFINITY;
            }
          },
          [&](float alpha) {
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < HS / 32; ++d) oacc[d] *= alpha;
          });
      l_run += exp2_sum<16>(s);
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < HS / 32; ++d)
          oacc[d] = mfma32(vs[mfma_row(r, half) * VP + col + 32 * d], s[r], oacc[d]);
    }
    if (st + 1 < s_end) lstore(st + 1);
    put(st + 2, page);
    __syncthreads();
  }
  store_rows<float, HS>(a, w, v, oacc, mb, l_run, half);
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
  const int64_t about = std::max<int64_t>(1, (N * (nh / nkv) + 64 * std::min(B, N)) / 128);
  const int64_t fill = 512 / (about * nkv);
  g.splits = (int)std::max<int64_t>(1, std::min<int64_t>({fill, capacity / 512, 16}));
  return g;
}

template <class E, int HS>
void launch_prefill(const PrefillArgs<E>& a, const PagedPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.tiles * a.nkv * a.splits));
  if constexpr (sizeof(E) == 4)
    hipLaunchKernelGGL((paged_prefill_f32_kernel<HS>), grid, dim3(256), 0, st, a, plan);
  else
    hipLaunchKernelGGL((paged_prefill_half_kernel<E, HS>), grid, dim3(256), 0, st, a, plan);
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
