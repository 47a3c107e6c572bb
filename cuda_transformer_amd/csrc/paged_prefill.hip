// Attention of packed new tokens over a paged key/value cache: prompts, chunks of prompts behind a
// cached context, drafts.  Causal: a token at position p sees the positions up to p.
//
// Formulas as in paged_decode.hip.  The work is matrix products (4 hs operations a visible pair),
// but for few rows on a long cache, whose bytes then count.
//  * The query heads that share a key/value head are rows of one product: row r of a sequence is
//    token r / group, head r % group, so a stage of K and V serves 128 rows whatever the group.  A
//    workgroup has 128 rows (4 waves x 32) and walks their keys in stages, global -> registers ->
//    LDS, double buffered, one barrier a stage.
//  * Pages may end anywhere: for each stage the rows' addresses are looked up two stages ahead and
//    left in LDS, that of a row of zeros for a row that holds no key.  In the 16-bit types, where a
//    page holds whole groups of 16 keys, a lane keeps where a group begins, for 16 stages at a time,
//    and stages need no LDS for addresses (ragged prompts of 11883 tokens 300 -> 294 us).
//  * Both products are laid out as in the dense forward: S^T = K Q^T with a row's scores in one lane
//    (lane l, register r: key R(r, l / 32) of row l % 32), so the maximum and sum of a row need one
//    exchange, and P^T is the B operand of O^T += V^T P^T as it lies.
//  * 16-bit types: 32x32x16 MFMA, probabilities rounded once to the type.  K and V stages go straight
//    from memory to LDS, by rows, and V's operand is read transposed (ds_read_b64_tr_b16: the 16
//    lanes of a group read 16 d of 4 keys and get 4 keys of one d).  A row's 16-byte chunks are
//    swapped by its number (row_swap), so that neither read meets a bank twice.
//  * FP32: six BF16 products for one FP32 product, stages split on their way through registers.
//  * Tiles differ in cost by any factor.  Many tiles: a workgroup each, heads side by side
//    (neighbours go to different XCDs, so an XCD's L2 holds few heads' keys), each sequence's last,
//    longest tile first.  Fewer: their cost is dealt evenly to as many workgroups as the GPU holds
//    at once; the parts of a tile that several of them share go to the workspace, which a second
//    kernel joins in order.  Both kernels compute the deal from cu_q and seq_lens.
// Measured, 32 over 8 heads of 128: six BF16 prompts of 11883 tokens (255 GFLOP) 290 us, 880 TFLOP/s; 32
// over 4, 256 FP16 tokens behind 60000 (252 GFLOP) 300 us; five FP32 prompts of 4349 tokens, 12 heads of
// 64 (12.6 GFLOP) 104 us.  Bound by exponentials and dependencies at two waves a SIMD, the matrix pipe
// 38% busy, at 2.0 of 2.4 GHz where calls follow each other.
#include "paged.hpp"
#include "split_bf16.hpp"

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
  int tiles;  // tiles of 128 rows that a key/value head may have
  int W;      // workgroups that the tiles' cost is dealt to; 0: a workgroup a tile
  int set_up;  // cost of beginning a tile
  E* o;
  float* l;
  float* ws;  // W > 0: O (2 W, 128, HS), then (m, l) (2 W, 128): a workgroup's first and last part
};

// Tokens of sequence b: first row and count, inside [0, N) whatever cu_q holds.
__device__ __forceinline__ int tokens_of(const PagedPlan& plan, int N, int b, int& first) {
  first = min(max(plan.cu_q[b], 0), N);
  return max(min(max(plan.cu_q[b + 1], 0), N) - first, 0);
}

constexpr int BM = 128;              // rows a workgroup
constexpr float kRescaleGap = 8.0f;  // log2 units: probabilities stay below 2^8

// What a workgroup works on: rows tile BM .. of the R that sequence b has for key/value head kvh,
// and the share [lo, hi) of their `cost` units of work.
struct RowTile {
  int b, first, R, tile, kvh;
  int64_t lo, hi, cost;
  __device__ __forceinline__ bool whole() const { return lo == 0 && hi == cost; }
  // The share of n stages.
  __device__ __forceinline__ int stage(int64_t at, int n) const {
    return at == 0 ? 0 : at == cost ? n : (int)(n * at / cost);
  }
};
// Work of a sequence's tiles: tile q costs base + 128 (q + 1).  That is the keys that its last row
// would see were the tile full, times group, and as much as kSetUp stages for beginning a tile.
// Every cost is positive, and the sum of the first q has a closed form.
struct SeqCost {
  int first, R;
  int64_t base;
  __device__ __forceinline__ int tiles() const { return (R + BM - 1) / BM; }
  __device__ __forceinline__ int64_t upto(int64_t q) const { return q * base + BM / 2 * q * (q + 1); }
};
template <class E>
__device__ __forceinline__ SeqCost seq_cost(const PrefillArgs<E>& a, const PagedPlan& plan, int b) {
  SeqCost c;
  c.R = tokens_of(plan, a.N, b, c.first) * (int)a.group.d;
  c.base = (int64_t)plan.keys_to(plan.position(b, c.first) - 1) * a.group.d + a.set_up;
  return c;
}
// Tile x of a head, all sequences' tiles in a row; false: there are fewer (then before is their
// number).
template <class E>
__device__ __forceinline__ bool find_rows(const PrefillArgs<E>& a, const PagedPlan& plan, int x,
                                          RowTile& w, int64_t& before) {
  w.b = find_unit(plan.B, (int64_t)x, before, [&](int i) { return seq_cost(a, plan, i).tiles(); });
  if (w.b == plan.B) return false;
  const SeqCost c = seq_cost(a, plan, w.b);
  w.first = uniform(c.first);
  w.R = uniform(c.R);
  w.tile = x - (int)before;
  w.cost = uniform(c.base) + BM * (int64_t)(w.tile + 1);
  w.lo = 0;
  w.hi = w.cost;
  return true;
}
// How the work of all heads' tiles, units in a row, is dealt to W workgroups: about units / W each.
// A cut that would fall within `slack` of a tile's end is made there: small pieces cost more than
// they balance.
struct Deal {
  int64_t head, units, slack;  // units of one head, of all of them
  int W;
  __device__ __forceinline__ int64_t cut(int n) const { return units * n / W; }
  // The last workgroup whose cut is at or before u.
  __device__ __forceinline__ int owner(int64_t u) const { return (int)(((u + 1) * W - 1) / units); }
  // Distance from its ends within which a tile is not cut.
  __device__ __forceinline__ int64_t edge(int64_t cost) const { return min(slack, cost / 4); }
};
template <class E>
__device__ __forceinline__ Deal make_deal(const PrefillArgs<E>& a, const PagedPlan& plan, int b,
                                          int64_t& before) {
  Deal d;
  d.head = count_units(plan.B, b, before, [&](int i) {
    const SeqCost c = seq_cost(a, plan, i);
    return c.upto(c.tiles());
  });
  d.units = d.head * a.nkv;
  // Shares are as long as it takes to begin them, in FP32 twice: 8 tokens of 32 over 8 heads of 128 behind
  // 2791 in BF16 23.5 us twice, 22.5 once; 11 of FP32 heads of 64 29.5 and 30.4.
  const int least = sizeof(E) == 4 ? 2 : 1;
  d.W = (int)max((int64_t)1, min((int64_t)a.W, d.units / (least * a.set_up)));
  d.slack = d.units / d.W / 8;
  return d;
}
// The tile that holds unit u, which is made relative to the tile's begin.
template <class E>
__device__ __forceinline__ void find_share(const PrefillArgs<E>& a, const PagedPlan& plan,
                                           const Deal& d, int64_t& u, RowTile& w) {
  w.kvh = (int)(u / d.head);
  u -= w.kvh * d.head;
  int64_t before;
  w.b = find_unit(plan.B, u, before, [&](int i) {
    const SeqCost c = seq_cost(a, plan, i);
    return c.upto(c.tiles());
  });
  SeqCost c = seq_cost(a, plan, w.b);
  w.first = c.first = uniform(c.first);
  w.R = c.R = uniform(c.R);
  c.base = uniform(c.base);
  u -= before;
  int q = 0;  // the last tile that begins at or before u
  for (int n = c.tiles(); n > 1;) {
    const int h = n / 2;
    if (c.upto(q + h) <= u) { q += h; n -= h; }
    else n = h;
  }
  u -= c.upto(q);
  w.tile = q;
  w.cost = c.base + BM * (int64_t)(q + 1);
}
// The next tile of the deal (there is one).
template <class E>
__device__ __forceinline__ void next_tile(const PrefillArgs<E>& a, const PagedPlan& plan, RowTile& w) {
  if ((w.tile + 1) * BM < w.R) {
    ++w.tile;
    w.cost += BM;
    return;
  }
  SeqCost c;
  do {
    if (++w.b == plan.B) { w.b = 0; ++w.kvh; }
    c = seq_cost(a, plan, w.b);
    w.R = uniform(c.R);
  } while (w.R == 0);
  w.first = uniform(c.first);
  w.tile = 0;
  w.cost = uniform(c.base) + BM;
}
// Rows of no sequence count as empty: share i of n of them, for head kvh.
template <class E, int HS>
__device__ __forceinline__ void fill_padding(const PrefillArgs<E>& a, const PagedPlan& plan, int kvh,
                                             int i, int n) {
  const int G = (int)a.group.d, tid = threadIdx.x;
  const int lo = min(max(plan.cu_q[0], 0), a.N), hi = min(max(plan.cu_q[plan.B], lo), a.N);
  const int64_t rows = (int64_t)(a.N - (hi - lo)) * G;  // padding tokens x heads
  for (int64_t r = i; r < rows; r += n) {
    const int j = (int)(r / G), t = j < lo ? j : j - lo + hi;
    const int64_t row = (int64_t)t * a.nh + kvh * G + (r - (int64_t)j * G);
    if (tid < HS) a.o[row * HS + tid] = (E)0.0f;
    if (tid == 0) a.l[row] = -INFINITY;
  }
}
// Calls body(tile, slot of the workspace for a part of it) for each of this workgroup's tiles: one, or
// (DEAL) those of its share.
template <class E, int HS, bool DEAL, class F>
__device__ __forceinline__ void each_tile(const PrefillArgs<E>& a, const PagedPlan& plan, F&& body) {
  RowTile w;
  int64_t before;
  if constexpr (!DEAL) {
    // longest first: x counts a sequence's tiles from the last
    const int x = blockIdx.x / a.nkv;
    w.kvh = blockIdx.x - x * a.nkv;
    if (!find_rows(a, plan, x, w, before)) {
      const int base = (int)min(before, (int64_t)a.tiles - 1);
      fill_padding<E, HS>(a, plan, w.kvh, x - base, a.tiles - base);
      return;
    }
    w.tile = (w.R + BM - 1) / BM - 1 - w.tile;
    body(w, 0);
  } else {
    const Deal deal = make_deal(a, plan, 0, before);
    const int n = xcd_work_item(blockIdx.x, deal.W);  // an XCD has neighbouring shares: few heads
    if ((int)blockIdx.x / kNumXcds >= (deal.W + kNumXcds - 1) / kNumXcds) return;
    if (n >= deal.W) return;
    int64_t u = deal.cut(n);
    int64_t left = deal.cut(n + 1) - u;  // units from the tile's begin to this workgroup's end
    if (left == 0) return;
    find_share(a, plan, deal, u, w);
    left += u;
    w.lo = u <= deal.edge(w.cost) ? 0 : u;
    if (u >= w.cost - deal.edge(w.cost)) {  // the share begins at the next tile
      left -= w.cost;
      w.lo = 0;
      if (left <= 0) return;
      next_tile(a, plan, w);
    }
    for (;;) {
      const int64_t edge = deal.edge(w.cost);
      if (w.lo == 0 && left <= edge) return;  // the tile is the next workgroup's
      w.hi = left >= w.cost - edge ? w.cost : left;
      // a tile that began in an earlier workgroup goes to this one's first slot, else to its second
      body(w, 2 * n + (w.lo == 0));
      left -= w.cost;
      if (left <= 0) return;
      w.lo = 0;
      next_tile(a, plan, w);
    }
  }
}

// Token and query head of row r of a tile's sequence (its last row behind the end).
template <class E>
__device__ __forceinline__ void row_of(const PrefillArgs<E>& a, const RowTile& w, int r, int& token, int& head) {
  r = min(r, w.R - 1);
  const int i = a.group.div(r);
  token = w.first + i;
  head = w.kvh * (int)a.group.d + r - i * (int)a.group.d;
}
// Which keys the rows of one wave see, one row a lane (both halves).
struct WaveRows {
  int keys;    // this lane's row
  int lo, hi;  // the fewest and the most of the wave's rows
  int n_keys;  // the most of the workgroup's rows
};
template <class E>
__device__ __forceinline__ WaveRows wave_rows(const PrefillArgs<E>& a, const PagedPlan& plan,
                                              const RowTile& w, int wave, int col) {
  const int64_t p0 = uniform(plan.position(w.b, w.first));
  auto keys = [&](int r) { return plan.keys_to(p0 + a.group.div(min(r, w.R - 1))); };
  const int r0 = w.tile * BM + wave * 32;
  WaveRows v;
  v.keys = keys(r0 + col);
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
#pragma clang fp contract(off)
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const float x = s[r] * c;
      s[r] = x - mb0;
    }
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
// Exponents of a 32-key tile (register r: key R(r, half)) that do not count -> -inf: bit j of `ok` says
// whether key j holds one, of which the row sees the first `seen`.  Two instructions a value.
__device__ __forceinline__ void mask_tile(float* s, uint32_t ok, int seen, int half) {
  ok = seen >= 32 ? ok : seen <= 0 ? 0 : ok & ((1u << seen) - 1);
  ok >>= 4 * half;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)ok, mfma_row(r, 0), 1);  // 0 or all ones
    s[r] = __uint_as_float((keep & __float_as_uint(s[r])) | (~keep & 0xff800000u));
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

// Where a part of a tile keeps the four elements d 32 + 8 g + 4 (lane / 32) .. of row
// 32 wave + lane % 32.
template <int HS>
__device__ __forceinline__ int64_t part_at(int slot, int wave, int d, int g, int lane) {
  return (int64_t)slot * BM * HS + (((wave * (HS / 32) + d) * 4 + g) * 64 + lane) * 4;
}

// Writes a lane's part of its row: the result, or the share's part of it (`any`: it had stages).
template <class E, int HS>
__device__ __forceinline__ void store_rows(const PrefillArgs<E>& a, const RowTile& w, int slot,
                                           const f32x16 (&oacc)[HS / 32], float mb, float l_run, bool any) {
  const int lane = threadIdx.x & 63, half = lane >> 5, in_tile = wave_index() * 32 + (lane & 31);
  const float l_tot = sum_halves(l_run);
  if (w.tile * BM + in_tile >= w.R) return;
  if (!w.whole()) {
    // in the order of the registers: a wave's store is 1 KiB in a row
    if (any) {
#pragma unroll
      for (int d = 0; d < HS / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          st4(a.ws + part_at<HS>(slot, wave_index(), d, g, lane),
              make_float4(oacc[d][4 * g], oacc[d][4 * g + 1], oacc[d][4 * g + 2], oacc[d][4 * g + 3]));
    }
    if (half == 0)
      *reinterpret_cast<float2*>(a.ws + (int64_t)2 * a.W * BM * HS + ((int64_t)slot * BM + in_tile) * 2) =
          make_float2(mb, l_tot);
    return;
  }
  int token, head;
  row_of(a, w, w.tile * BM + in_tile, token, head);
  const int64_t row = (int64_t)token * a.nh + head;
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

// UNIFORM: a group of 16 keys lies in one page (the page size is a multiple of 16).
// Three waves a SIMD at hs 32, two else: registers would allow more, but fewer workgroups walk the
// same keys closer together (4 x 2000 tokens of 16 heads: hs 32 50.6 us with three and 59.8 with
// four, hs 64 65.5 with two and 66.2 with three).
template <class E, int HS, bool DEAL, bool UNIFORM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HS == 32 ? 3 : 2, HS == 32 ? 3 : 2)))
void paged_prefill_half_kernel(PrefillArgs<E> a, PagedPlan plan) {
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
  // any page size: addresses of a stage's K and V rows, and the rows that hold a key (four stages, as
  // a slow wave may still look at a stage while the third is put)
  __shared__ uint64_t row_at[2][2][UNIFORM ? 1 : BN];
  __shared__ uint64_t holds[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  const int half = lane >> 5, col = lane & 31;
  each_tile<E, HS, DEAL>(a, plan, [&](const RowTile& w, int slot) {
  const WaveRows v = wave_rows(a, plan, w, wave, col);
  const int n_all = (v.n_keys + BN - 1) / BN;
  const int s_begin = w.stage(w.lo, n_all);
  const int s_end = w.stage(w.hi, n_all);

  // This lane's query row, d = 16 s + 8 half .. of step s
  vec8_t<E> qf[QC];
  {
    int token, head;
    row_of(a, w, w.tile * BM + wave * 32 + col, token, head);
    const E* qp = a.q + token * a.qt + head * a.qh + 8 * half;
#pragma unroll
    for (int s = 0; s < QC; ++s) qf[s] = ld8<E>(qp + 16 * s);
  }
  f32x16 oacc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) oacc[d] = zero16();
  float mb = -INFINITY, l_run = 0.0f;  // exponent offset, and this lane's part of the row's sum

  const int32_t* table = plan.table + w.b * plan.table_stride;
  const E* kb = a.k + w.kvh * a.sk.h;
  const E* vb = a.v + w.kvh * a.sv.h;

  // Any page size.  Page of key `lane` of a stage, by waves 2 (K) and 3 (V), which idle where a tile
  // has few rows; -1: none.
  auto look_up = [&](int stage) {
    const int j = stage * BN + lane;
    return wave >= 2 && stage < s_end && j < v.n_keys ? table[plan.ps.div(j)] : -1;
  };
  auto put = [&](int stage, int page) {
    if (wave < 2) return;
    const int j = stage * BN + lane, row = j - plan.ps.div(j) * (int)plan.ps.d;
    const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
    const E* p = wave == 2 ? kb + page * a.sk.a + row * a.sk.r : vb + page * a.sv.a + row * a.sv.r;
    row_at[stage & 1][wave - 2][lane] = ok ? (uint64_t)p : (uint64_t)kZeroRow;
    const uint64_t all = __ballot(ok);
    if (tid == 128) holds[stage & 3] = all;
  };
  // UNIFORM.  Where 64 groups of 16 keys begin in the pools, a group a lane, from stage tp on
  // (`mapped`: those with a page), and the pages of the next 64.
  auto load_pages = [&](int stage) {
    const int j = stage * BN + 16 * lane;
    return stage + lane / 4 < s_end && j < v.n_keys ? table[plan.ps.div(j)] : -1;
  };
  int tp = s_begin, pages_next = -1;
  const E *k_group = kb, *v_group = vb;
  uint64_t mapped = 0;
  auto next_groups = [&](int stage, int page) {
    tp = stage;
    pages_next = load_pages(tp + 16);
    const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
    const int j = tp * BN + 16 * lane, row = j - plan.ps.div(j) * (int)plan.ps.d;
    k_group = kb + (ok ? page * a.sk.a + row * a.sk.r : 0);
    v_group = vb + (ok ? page * a.sv.a + row * a.sv.r : 0);
    mapped = __ballot(ok);
  };
  if constexpr (UNIFORM) next_groups(s_begin, load_pages(s_begin));

  // Copy c of a stage: rows ROWS (4 c + wave) .., 16 bytes a lane, chunks swapped at the source.
  // Returns which rows hold a key.
  const int c_row = ROWS * wave + lane / (RB / 16);
  const int c_at = ((lane % (RB / 16)) ^ row_swap<RB>(c_row)) * 16;
  const uint32_t k_off = (uint32_t)(c_row % 16 * (int)a.sk.r * 2 + c_at);
  const uint32_t v_off = (uint32_t)(c_row % 16 * (int)a.sv.r * 2 + c_at);
  auto copy = [&](int stage, char* to) -> uint64_t {
    if constexpr (!UNIFORM) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const char* p = reinterpret_cast<const char*>(row_at[stage & 1][kv][4 * ROWS * c + c_row]) + c_at;
          async_copy16(reinterpret_cast<const float*>(p),
                       reinterpret_cast<float*>(to + kv * STAGE + 1024 * (4 * c + wave)));
        }
      return holds[stage & 3];
    } else {
      if (stage - tp >= 16) next_groups(tp + 16, pages_next);
      const int first = 4 * (stage - tp), groups = (int)(mapped >> first) & 15;
      const int left = v.n_keys - stage * BN;
      auto at = [&](const E* group, int g) {  // group g's, the same for the wave
        const uint64_t p = (uint64_t)group;
        return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), first + g) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)p, first + g));
      };
      if (groups == 15 && left >= BN) {
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const int g = ROWS * (4 * c + wave) / 16;  // a copy's rows lie in one group
          async_copy16(reinterpret_cast<const float*>(at(k_group, g) + k_off),
                       reinterpret_cast<float*>(to + 1024 * (4 * c + wave)));
          async_copy16(reinterpret_cast<const float*>(at(v_group, g) + v_off),
                       reinterpret_cast<float*>(to + STAGE + 1024 * (4 * c + wave)));
        }
        return ~(uint64_t)0;
      }
      uint64_t ok = 0;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (groups >> g & 1) ok |= (uint64_t)0xffff << 16 * g;
      if (left < BN) ok &= ((uint64_t)1 << left) - 1;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        const int g = ROWS * (4 * c + wave) / 16;
        const bool mine = ok >> (4 * ROWS * c + c_row) & 1;
        const char* const zero = reinterpret_cast<const char*>(kZeroRow) + c_at;
        async_copy16(reinterpret_cast<const float*>(mine ? at(k_group, g) + k_off : zero),
                     reinterpret_cast<float*>(to + 1024 * (4 * c + wave)));
        async_copy16(reinterpret_cast<const float*>(mine ? at(v_group, g) + v_off : zero),
                     reinterpret_cast<float*>(to + STAGE + 1024 * (4 * c + wave)));
      }
      return ok;
    }
  };

  // K operand: row col (+ 32), chunk 2 s + half of step s.  V operand: rows 4 half + lane % 16 / 4
  // (+ 16 i), 4 d from 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) on; then 8 rows on, where the swap
  // differs by 2 chunks.  Steps and blocks differ by the bits 32 s and 64 d of the address.
  const int v_row = 4 * half + lane % 16 / 4;
  const int k_lane = col * RB + (half ^ row_swap<RB>(col)) * 16;
  const int v_lane = v_row * RB + ((2 * (lane / 16 % 2) + lane % 4 / 2) ^ row_swap<RB>(v_row)) * 16 + lane % 2 * 8;

  uint64_t ok_next = 0;  // of the stage copied last
  auto compute = [&](int st, const char* from, uint64_t ok) {
    const int j0 = st * BN;
    if (j0 >= v.hi) return;  // no row of this wave sees the stage
    // made anew each stage: fourteen registers less to keep
    int k_at = k_lane, v_at = v_lane;
    asm volatile("" : "+v"(k_at), "+v"(v_at));
    f32x16 s2[2] = {zero16(), zero16()};
#pragma unroll
    for (int c = 0; c < QC; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s2[i] = Half16<E>::mfma(
            *reinterpret_cast<const vec8_t<E>*>(from + (k_at ^ 32 * c) + 32 * RB * i), qf[c], s2[i]);
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
          mask_tile(s, (uint32_t)ok, v.keys - j0, half);
          mask_tile(s + 16, (uint32_t)(ok >> 32), v.keys - j0 - 32, half);
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
        struct { s16x4 a, b; } t = {ld_transposed(p + (v_at ^ 64 * d)),
                                    ld_transposed(p + (v_at ^ 64 * d ^ 32) + 8 * RB)};
        oacc[d] = Half16<E>::mfma(__builtin_bit_cast(vec8_t<E>, t), pf, oacc[d]);
      }
    }
  };
  auto step = [&](int st, const char* from, char* to) {
    int page = -1;
    if constexpr (!UNIFORM) page = look_up(st + 2);
    const uint64_t ok = ok_next;
    if (st + 1 < s_end) ok_next = copy(st + 1, to);
    compute(st, from, ok);
    if constexpr (!UNIFORM) put(st + 2, page);
    vm_wait_all();
    __syncthreads();
  };

  if (s_begin < s_end) {  // workgroup-uniform
    if constexpr (!UNIFORM) {
      put(s_begin, look_up(s_begin));
      put(s_begin + 1, look_up(s_begin + 1));
      __syncthreads();
    }
    ok_next = copy(s_begin, buf0);
    vm_wait_all();
    __syncthreads();
  }
  for (int st = s_begin; st < s_end; st += 2) {
    step(st, buf0, buf1);
    if (st + 1 < s_end) step(st + 1, buf1, buf0);
  }
  store_rows<E, HS>(a, w, slot, oacc, mb, l_run, s_begin < s_end);
  });
}

// FP32.  Both products run as six BF16 products of three-part operands (split_bf16.hpp), laid out
// and scaled as in the dense forward: Q, P and V by 2^24, sums of the first parts and of the smaller
// ones apart.  A workgroup that meets a query beyond the parts' range, or whose sums are not finite,
// walks its keys again on the FP32 MFMA.
template <int HS, bool DEAL>
__global__ __launch_bounds__(256, HS == 128 ? 1 : 2) void paged_prefill_f32_kernel(
    PrefillArgs<float> a, PagedPlan plan) {
  constexpr int BN = 32;               // keys a stage
  constexpr int PART = BN * HS * 2;    // bytes of one part of a stage's K (or V)
  constexpr int STAGE = 6 * PART;
  constexpr int UNITS = BN * HS / 8;   // 16-byte units of a part
  constexpr int NU = (UNITS + 255) / 256;
  constexpr int KP = HS + 4, VP = HS + 8;  // row pitches of an FP32 stage
  static_assert(BN * (KP + VP) * 4 <= 2 * STAGE, "an FP32 stage fits");
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  __shared__ uint64_t row_at[2][2][BN];  // addresses of a stage's K and V rows
  __shared__ uint32_t holds[4];          // bit j: row j holds a key (four stages, as above)

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
  const int half = lane >> 5, col = lane & 31;
  each_tile<float, HS, DEAL>(a, plan, [&](const RowTile& w, int slot) {
  const WaveRows v = wave_rows(a, plan, w, wave, col);
  const int n_all = (v.n_keys + BN - 1) / BN;
  const int s_begin = w.stage(w.lo, n_all);
  const int s_end = w.stage(w.hi, n_all);

  // Parts of this lane's query row, d = 16 s + 8 half .. of step s
  int token, head;
  row_of(a, w, w.tile * BM + wave * 32 + col, token, head);
  const float* qrow = a.q + token * a.qt + head * a.qh;
  bf16x8 qp[HS / 16][3];
  float qmax = 0.0f;
#pragma unroll
  for (int s = 0; s < HS / 16; ++s) {
    float x[8];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float4 q4 = ld4(qrow + 16 * s + 8 * half + 4 * c);
      x[4 * c] = q4.x; x[4 * c + 1] = q4.y; x[4 * c + 2] = q4.z; x[4 * c + 3] = q4.w;
    }
    split_bf16<true>(x, qp[s]);
#pragma unroll
    for (int e = 0; e < 8; e += 2) qmax = fmaxf(fmaxf(qmax, fabsf(x[e])), fabsf(x[e + 1]));
  }
  bool odd = __any(qmax >= kMaxScoreFactor);

  f32x16 oacc[HS / 32], olow[HS / 32];
#pragma unroll
  for (int d = 0; d < HS / 32; ++d) { oacc[d] = zero16(); olow[d] = zero16(); }
  float mb = -INFINITY, l_run = 0.0f;

  // Page of a stage's key lane % 32, in wave 3, which idles where a tile has few rows: lanes 0 .. 31
  // for K, 32 .. 63 for V.
  const int32_t* table = plan.table + w.b * plan.table_stride;
  auto look_up = [&](int stage) {
    const int j = stage * BN + col;
    return wave == 3 && stage < s_end && j < v.n_keys ? table[plan.ps.div(j)] : -1;
  };
  const float* kb = a.k + w.kvh * a.sk.h;
  const float* vb = a.v + w.kvh * a.sv.h;
  auto put = [&](int stage, int page) {
    if (wave != 3) return;
    const int j = stage * BN + col, row = j - plan.ps.div(j) * (int)plan.ps.d;
    const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
    const float* p = half == 0 ? kb + page * a.sk.a + row * a.sk.r : vb + page * a.sv.a + row * a.sv.r;
    row_at[stage & 1][half][col] = ok ? (uint64_t)p : (uint64_t)kZeroRow;
    const uint64_t all = __ballot(ok);
    if (tid == 192) holds[stage & 3] = (uint32_t)all;
  };
  auto mask = [&](float (&s)[16], int j0, uint32_t ok) {
    if (j0 + BN <= v.lo && ~ok == 0) return;
    mask_tile(s, ok, v.keys - j0, half);
  };

  // K unit (d8, key), d 8 d8 .. of a key, lies at d8 * 32 + (key ^ (d8 & 7)); V unit (d, sh), the
  // eight keys that half sh & 1 of the product's step sh >> 1 takes, at (d / 32, sh, d % 32).
  float kst[NU][8], vst[NU][8];
  auto gload = [&](int stage) {
    const uint64_t(*at)[BN] = row_at[stage & 1];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int f = tid + 256 * u;
      if (UNITS % 256 != 0 && f >= UNITS) continue;  // wave-uniform
      const float* kp = reinterpret_cast<const float*>(at[0][f / (HS / 8)]) + 8 * (f % (HS / 8));
      const float4 x = ld4(kp), y = ld4(kp + 4);
      kst[u][0] = x.x; kst[u][1] = x.y; kst[u][2] = x.z; kst[u][3] = x.w;
      kst[u][4] = y.x; kst[u][5] = y.y; kst[u][6] = y.z; kst[u][7] = y.w;
      const int d = f % HS, sh = f / HS, key = 16 * (sh >> 1) + 4 * (sh & 1);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        vst[u][j] = reinterpret_cast<const float*>(at[1][key + 8 * (j >> 2) + (j & 3)])[d];
    }
  };
  auto lstore = [&](int stage) {
    char* ks = smem + (stage & 1) * STAGE;
    char* vs = ks + 3 * PART;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int f = tid + 256 * u;
      if (UNITS % 256 != 0 && f >= UNITS) continue;
      const int key = f / (HS / 8), d8 = f % (HS / 8);
      const int d = f % HS, sh = f / HS;
      bf16x8 p[3];
      split_bf16(kst[u], p);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<bf16x8*>(ks + q * PART + (d8 * 32 + (key ^ (d8 & 7))) * 16) = p[q];
      split_bf16<true>(vst[u], p);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<bf16x8*>(vs + q * PART + ((d >> 5) * 128 + sh * 32 + (d & 31)) * 16) = p[q];
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
    const char* ks = smem + (st & 1) * STAGE;
    const char* vs = ks + 3 * PART;
    const int j0 = st * BN;
    if (j0 < v.hi) {  // else no row of this wave sees the stage
      f32x16 acc = zero16(), acc2 = zero16();  // even and odd steps
#pragma unroll
      for (int c = 0; c < HS / 16; c += 2) {
        bf16x8 ka[2][3];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int d8 = 2 * (c + o) + half;
          const char* at = ks + (d8 * 32 + (col ^ (d8 & 7))) * 16;
#pragma unroll
          for (int q = 2; q >= 0; --q) ka[o][q] = *reinterpret_cast<const bf16x8*>(at + q * PART);
        }
#pragma unroll
        for (int p = 0; p < 6; ++p) {
          acc = mfma_bf16(ka[0][kSplitA[p]], qp[c][kSplitB[p]], acc);
          acc2 = mfma_bf16(ka[1][kSplitA[p]], qp[c + 1][kSplitB[p]], acc2);
        }
      }
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc[r] + acc2[r];
      exponents(s, a.scale_log2 * kSplitUnscale, mb, [&] { mask(s, j0, holds[st & 3]); },
                [&](float alpha) {
                  l_run *= alpha;
#pragma unroll
                  for (int d = 0; d < HS / 32; ++d) { oacc[d] *= alpha; olow[d] *= alpha; }
                });
      l_run += exp2_sum<16>(s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // 16 keys
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[8 * i + e];
        bf16x8 pp[3], va[HS / 32][3];
#pragma unroll
        for (int d = 0; d < HS / 32; ++d)
#pragma unroll
          for (int q = 2; q >= 0; --q)
            va[d][q] = *reinterpret_cast<const bf16x8*>(
                vs + q * PART + (d * 128 + (2 * i + half) * 32 + col) * 16);
        split_bf16<true>(x, pp);
#pragma unroll
        for (int p = 0; p < 6; ++p)
#pragma unroll
          for (int d = 0; d < HS / 32; ++d) {
            f32x16& c = p == 5 ? oacc[d] : olow[d];
            c = mfma_bf16(va[d][kSplitA[p]], pp[kSplitB[p]], c);
          }
      }
    }
    if (st + 1 < s_end) lstore(st + 1);
    put(st + 2, page);
    __syncthreads();
  }

  odd |= !(l_run < INFINITY);
#pragma unroll
  for (int d = 0; d < HS / 32; ++d) {
    oacc[d] += olow[d];
    odd |= not_finite(oacc[d]);
    oacc[d] *= kSplitUnscale * kSplitUnscale;
  }
  if (__syncthreads_or(odd)) {
    float* const ks = reinterpret_cast<float*>(smem);
    float* const vs = ks + BN * KP;
    mb = -INFINITY;
    l_run = 0.0f;
#pragma unroll
    for (int d = 0; d < HS / 32; ++d) oacc[d] = zero16();
    for (int st = s_begin; st < s_end; ++st) {
      put(st, look_up(st));
      __syncthreads();
      for (int f = tid; f < BN * HS / 4; f += 256) {
        const int r = f / (HS / 4), c = f % (HS / 4) * 4;
        st4(ks + r * KP + c, ld4(reinterpret_cast<const float*>(row_at[st & 1][0][r]) + c));
        st4(vs + r * VP + c, ld4(reinterpret_cast<const float*>(row_at[st & 1][1][r]) + c));
      }
      __syncthreads();
      const int j0 = st * BN;
      if (j0 < v.hi) {
        f32x16 acc = zero16();
#pragma unroll 2
        for (int c = 0; c < HS / 8; ++c) {
          const float4 x = ld4(qrow + 8 * c + 4 * half), y = ld4(ks + col * KP + 8 * c + 4 * half);
          acc = mfma32(y.x, x.x, acc);
          acc = mfma32(y.y, x.y, acc);
          acc = mfma32(y.z, x.z, acc);
          acc = mfma32(y.w, x.w, acc);
        }
        float s[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = acc[r];
        exponents(s, a.scale_log2, mb, [&] { mask(s, j0, holds[st & 3]); }, [&](float alpha) {
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
      __syncthreads();
    }
  }
  store_rows<float, HS>(a, w, slot, oacc, mb, l_run, s_begin < s_end);
  });
}

// Joins the parts of the tiles that several workgroups share, in order, and fills padding rows.  A part
// consists of 1 KiB stores; a wave has SETS of them that share their rows, a thread four elements of a
// row from each, and the loads of FLIGHT parts at a time in flight.  Few parts a tile: SETS = 4, as the
// deal costs a wave more than its loads (a prompt of 2000 tokens, 32 over 8 heads of 128: 77 us with
// one, 66 with four).  Many: SETS = 1 and more waves walk them (two drafts of 4 tokens behind 60000:
// 109 us with four, 103 with one).
template <class E, int HS, int SETS>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(PrefillArgs<E> a, PagedPlan plan) {
  constexpr int BLOCKS = BM * HS / (1024 * SETS);  // a tile
  constexpr int FLIGHT = SETS == 4 ? 2 : 4;
  const int x = blockIdx.x / (BLOCKS * a.nkv), rest = blockIdx.x - x * BLOCKS * a.nkv;
  RowTile w;
  w.kvh = rest / BLOCKS;
  int64_t before;
  if (!find_rows(a, plan, x, w, before)) {
    const int base = (int)min(before, (int64_t)a.tiles - 1);
    fill_padding<E, HS>(a, plan, w.kvh, BLOCKS * (x - base) + rest % BLOCKS, BLOCKS * (a.tiles - base));
    return;
  }
  int64_t front;
  const Deal deal = make_deal(a, plan, w.b, front);
  const int64_t begin = w.kvh * deal.head + front + (w.cost - BM * (int64_t)(w.tile + 1)) * w.tile +
                        BM / 2 * (int64_t)w.tile * (w.tile + 1);
  const int64_t edge = deal.edge(w.cost);
  const int w0 = deal.owner(begin + edge), w1 = deal.owner(begin + w.cost - edge - 1);
  if (w0 == w1) return;  // written whole
  const int lane = threadIdx.x & 63, set = rest % BLOCKS * 4 + wave_index();
  const int g0 = set * SETS % 4, d32 = set * SETS / 4 % (HS / 32), wave = set * SETS / (HS / 8);
  const int r = wave * 32 + lane % 32;
  if (w.tile * BM + r >= w.R) return;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + (int64_t)2 * a.W * BM * HS);
  auto slot = [&](int i) { return 2 * i + (i == w0); };
  float m = -INFINITY;
  for (int i = w0; i <= w1; i += 4) {
    float x4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x4[j] = ml[(int64_t)slot(min(i + j, w1)) * BM + r].x;
    m = fmaxf(m, max3_tree(x4));
  }
  const float off = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4 o[SETS];
#pragma unroll
  for (int g = 0; g < SETS; ++g) o[g] = zero4();
  for (int i = w0; i <= w1; i += FLIGHT) {
    float2 p[FLIGHT];
    float4 v[FLIGHT][SETS];
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      const int at = slot(min(i + j, w1));
      p[j] = ml[(int64_t)at * BM + r];
#pragma unroll
      for (int g = 0; g < SETS; ++g) v[j][g] = ld4(a.ws + part_at<HS>(at, wave, d32, g0 + g, lane));
    }
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      // a share without stages has written no O
      if (i + j > w1 || (p[j].x == -INFINITY && p[j].y == 0.0f)) continue;
      const float f = fast_exp2(p[j].x - off);
      l = fmaf(f, p[j].y, l);
#pragma unroll
      for (int g = 0; g < SETS; ++g) {
        const float4 x = v[j][g];
        o[g].x = fmaf(f, x.x, o[g].x); o[g].y = fmaf(f, x.y, o[g].y);
        o[g].z = fmaf(f, x.z, o[g].z); o[g].w = fmaf(f, x.w, o[g].w);
      }
    }
  }
  int token, head;
  row_of(a, w, w.tile * BM + r, token, head);
  const int64_t to = (int64_t)token * a.nh + head;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int g = 0; g < SETS; ++g) {
    E* op = a.o + to * HS + 32 * d32 + 8 * (g0 + g) + 4 * (lane / 32);
    op[0] = (E)(o[g].x * inv); op[1] = (E)(o[g].y * inv);
    op[2] = (E)(o[g].z * inv); op[3] = (E)(o[g].w * inv);
  }
  if (g0 == 0 && d32 == 0 && lane < 32) a.l[to] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

// Tiles of 128 rows that a key/value head may have (each sequence may end inside one; one more, so
// that some workgroup is left for padding rows), and the workgroups that their cost is dealt to: as
// many as the GPU holds at once.  Dealing costs a second kernel, parts written and read, and more
// tiles begun, so a workgroup takes a whole tile (W = 0) where
//  * there is a tile or more for each of these places.  Whole and dealt, us: 4 x 2000 tokens of 16
//    heads of 64 in BF16 (two tiles a place) 70 and 99; 8 x 50 to 1500 of 32 over 8 heads of 128 behind
//    up to 2000 (1.1) 108 and 159; but 5 x 200 to 2000 FP32 tokens of 12 heads of 64 (0.9) 155 and 104;
//  * or the longest tile, by the table's width, has few stages: 8 in FP32; in the 16-bit types 14, and
//    up to 20 more as the places fill.  One BF16 sequence of 32 over 8 heads of 128: 700 tokens (11
//    stages, 0.34) 22 and 34, 2000 (32, 0.98) 55 and 66, 128 behind 900 (17, 0.06) 28.9 and 28.2, 1000
//    behind 4000 (79, 0.48) 110 and 105, 500 behind 4000 (71, 0.25) 99 and 61; 16 x up to 150 behind
//    up to 2000 (34, 0.7) 52 and 36.  FP32: 2 x 128 behind 300 (14, 0.1) 33 and 30.
// 256 tokens behind 60000 cannot be whole tiles: 64 places of 512.
constexpr int kSetUp = 3;  // stages' time that a tile's lookups, queries and stores take
struct PrefillGrid {
  int64_t tiles;
  int W, stage;
};
PrefillGrid prefill_grid(int64_t B, int64_t N, int64_t nh, int64_t nkv, int64_t hs, int64_t capacity,
                         int elem) {
  PrefillGrid g;
  g.tiles = N * (nh / nkv) / 128 + std::min(B, N) + 1;
  g.stage = elem == 4 ? 32 : 64;
  const int64_t places = 256 * (elem == 4 ? (hs == 128 ? 1 : 2) : (hs == 32 ? 3 : 2));
  const int64_t group = nh / nkv;
  const int64_t about = std::max<int64_t>(1, (N * group + 64 * std::min(B, N)) / 128) * nkv;
  const int64_t stages = (capacity + g.stage - 1) / g.stage;
  // Units of work, whatever cu_q holds: a deal needs them in 53 bits, and a tile's times its stages
  // in 63.
  const double most = (double)N * group / 128 + 1;
  const double units = (double)B * most * nkv * ((double)group * (capacity + kSetUp * g.stage) + 128 * most);
  const int64_t few = elem == 4 ? 8 : 14 + 20 * about / places;
  g.W = about >= places || stages <= few || units >= 0x1p53 || units * stages >= 0x1p62 * (B * most * nkv)
            ? 0
            : (int)std::min(places, (g.tiles - 1) * nkv * stages / 2);
  return g;
}

template <class E, int HS>
void launch_prefill(const PrefillArgs<E>& a, const PagedPlan& plan, hipStream_t st) {
  const dim3 grid(a.W > 0 ? xcd_grid(a.W) : (unsigned)((int64_t)a.tiles * a.nkv));
  auto go = [&]<bool DEAL>() {
    if constexpr (sizeof(E) == 4)
      hipLaunchKernelGGL((paged_prefill_f32_kernel<HS, DEAL>), grid, dim3(256), 0, st, a, plan);
    else if (plan.ps.d % 16 == 0)
      hipLaunchKernelGGL((paged_prefill_half_kernel<E, HS, DEAL, true>), grid, dim3(256), 0, st, a, plan);
    else
      hipLaunchKernelGGL((paged_prefill_half_kernel<E, HS, DEAL, false>), grid, dim3(256), 0, st, a, plan);
  };
  if (a.W > 0) go.template operator()<true>();
  else go.template operator()<false>();
  if (a.W == 0) return;
  auto join = [&]<int SETS>() {
    const int64_t blocks = (int64_t)a.tiles * a.nkv * (BM * HS / (1024 * SETS));
    hipLaunchKernelGGL((paged_prefill_join_kernel<E, HS, SETS>), dim3((unsigned)blocks), dim3(256), 0, st, a, plan);
  };
  // more than eight workgroups a tile, at least: many parts
  if (a.W > 8 * (int64_t)a.tiles * a.nkv) join.template operator()<1>();
  else join.template operator()<4>();
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
  const PrefillGrid g = prefill_grid(pa.B, N, pa.nh, pa.nkv, pa.hs, plan.capacity, sizeof(E));
  if (g.tiles * pa.nkv >= (int64_t)1 << 31) return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (g.W > 0 && (!ws || !aligned16(ws) ||
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
  a.tiles = (int)g.tiles; a.W = g.W; a.set_up = kSetUp * g.stage * (int)a.group.d;
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
  int64_t bytes = 0;  // the most that a type needs
  for (int elem : {2, 4})
    bytes = std::max(bytes, (int64_t)prefill_grid(B, N, nh, nkv, hs, pages_per_seq * page_size, elem).W * 2 *
                                128 * (hs + 2) * 4);
  return bytes;
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
