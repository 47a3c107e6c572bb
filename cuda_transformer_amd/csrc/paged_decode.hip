// Attention of one new token a sequence over a paged key/value cache, its length split over the GPU.
//
// Query head h of sequence b reads key/value head h / group; over the sequence's keys j < seq_lens[b]
// whose page is mapped, in exponents of 2 (t_j = scale log2(e) q . k_j):
//   m = max t,  l = sum 2^{t_j - m},  O = sum 2^{t_j - m} v_j / l,  L = (m + log2 l) ln 2;
// without a key O = 0, L = -inf.  Any cut of the keys gives parts (m_i, l_i, O_i l_i) that add up
// against the largest m_i.
//
// What bounds it: every key and value is read once, 2 group to 4 group operations a byte.  So the
// products run on the matrix pipe, whose idle columns cost nothing (16 query heads a pass, or 32 for
// groups above 16), and everything else serves the loads.
//  * A job is one sequence's keys for one key/value head (and 16 or 32 of its query heads).  Jobs are cut
//    into tiles of 4 x WK keys and all tiles of all jobs are dealt evenly, in order, to a fixed
//    number of workgroups: lengths that differ by any factor load the GPU evenly.  A workgroup
//    writes the jobs it has whole, and partial results (at most two: the job it enters in the
//    middle, and the job it leaves) to the workspace, which a second kernel joins in tile order.
//    Both recompute the deal from seq_lens, so the host never looks at the lengths.
//  * A wave takes WK keys of each tile.  K goes from memory to registers in the order of the MFMA's
//    A operand (row = key): lane l, key l % 16, 16 bytes at 64 s + 16 (l / 16) for step s.  The
//    scores come back with four keys of one head in a lane: S[key 4 (l / 16) + r][head l % 16].
//  * V: lane l reads, for the keys whose scores it holds, elements (HS / 16) (l % 16) .. of the row
//    (16 lanes read a whole row), and turns them in registers (one v_perm a pair of values) into the
//    A operand of O^T += V^T P^T: MFMA e has rows d = (HS / 16) c + e.  The lane's probabilities are
//    the B operand as they are.  No LDS, no shuffle of K, V or P, and both products' loads are
//    issued a tile ahead.
//  * Probabilities are kept to two 16-bit parts for the 16-bit types (the second product is free
//    beside the loads): rounding them once would add as much error as the output's own rounding.
//  * FP32 runs on the FP32 MFMA (16x16x4).
// Measured: 64 sequences of 500 to 8000 tokens, 32 over 8 heads of 128 in BF16 (743 MB) 124 us, 6.1 TB/s
// (a plain copy reaches 5.8); two of 60000 and 130000, 32 over 4 in FP16 (424 MB) 71 us and 5 for the
// join; 33 FP32 sequences of up to 4000, 12 over 4 heads of 32 (19 MB) 12.5 us and 8 of up to 251, 6
// heads of 64, 7.3 us: chains of dependent steps.
#include "paged.hpp"

namespace cta {
namespace {

template <class E>
struct DecodeArgs {
  const E *q, *k, *v;
  int64_t qt, qh;
  Strides3 sk, sv;
  int nh, nkv, group, chunks;  // chunks of 16 M query heads a key/value head
  float scale_log2;
  E* o;
  float* l;
  float* ws;
};

// Geometry of a type, head size and number M of 16 query heads a pass: 16 KB of K and V a wave and
// tile.
template <class E, int HS, int M = 1>
struct DecodeTile {
  static constexpr int KG = sizeof(E) == 2 ? 256 / HS : 128 / HS;  // groups of 16 keys a wave
  static constexpr int WK = 16 * KG;                               // keys a wave
  static constexpr int TILE = 4 * WK;
  static constexpr int CK = HS * (int)sizeof(E) / 64;  // 16-byte chunks a lane has of a K row
  static constexpr int DW = HS * (int)sizeof(E) / 64;  // dwords a lane has of a V row
  static constexpr int NE = HS / 16;                   // output elements of a lane and register
  static constexpr int HEADS = 16 * M;
  static constexpr int PART = HEADS * (HS + 2);        // floats of a partial result: O, m, l
};

// Largest of the values that lanes l, l ^ 16, l ^ 32, l ^ 48 hold, and their sum.
__device__ __forceinline__ float max_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ f32x4 mfma16(vec8_t<__bf16> a, vec8_t<__bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(vec8_t<_Float16> a, vec8_t<_Float16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// The deal of all sequences' tiles, `jobs` times over, to W workgroups: units / W each, the first
// `more` workgroups one more.
struct Deal {
  int units, W, each, more;
  __device__ __forceinline__ Deal(int units_, int grid) : units(units_), W(max(1, min(units_, grid))) {
    each = (int)((unsigned)units / (unsigned)W);
    more = units - each * W;
  }
  __device__ __forceinline__ int start(int w) const { return w * each + min(w, more); }
  __device__ __forceinline__ int owner(int u) const {  // the workgroup that has unit u
    const int cut = more * (each + 1);
    return u < cut ? (int)((unsigned)u / (unsigned)(each + 1)) : more + (int)((unsigned)(u - cut) / (unsigned)each);
  }
};
// Keys of the sequences.  Up to 64 of them are looked up once, a sequence a lane.
struct SeqKeys {
  int lane_keys;
  bool few;
  __device__ __forceinline__ explicit SeqKeys(const PagedPlan& plan) : few(plan.B <= 64) {
    const int lane = threadIdx.x & 63;
    lane_keys = few && lane < plan.B ? keys(plan, lane) : 0;
  }
  static __device__ __forceinline__ int keys(const PagedPlan& plan, int b) {
    return plan.keys_to((int64_t)plan.lens[b] - 1);
  }
  __device__ __forceinline__ int of(const PagedPlan& plan, int b) const {
    return few ? __builtin_amdgcn_readlane(lane_keys, b) : uniform(keys(plan, b));
  }
  // Tiles of all sequences, and of those in front of b.
  template <int TILE>
  __device__ __forceinline__ int count(const PagedPlan& plan, int b, int& before) const {
    if (!few)
      return count_units(plan.B, b, before, [&](int i) { return (keys(plan, i) + TILE - 1) / TILE; });
    const int end = wave_scan((lane_keys + TILE - 1) / TILE);
    before = b == 0 ? 0 : __builtin_amdgcn_readlane(end, b - 1);
    return __builtin_amdgcn_readlane(end, 63);
  }
  // Sequence of tile x, and the tiles before it.
  template <int TILE>
  __device__ __forceinline__ int find(const PagedPlan& plan, int x, int& before) const {
    if (!few)
      return find_unit(plan.B, x, before, [&](int i) { return (keys(plan, i) + TILE - 1) / TILE; });
    const int n = (lane_keys + TILE - 1) / TILE, end = wave_scan(n);
    const int w = __builtin_ctzll(__ballot(end > x));
    before = __builtin_amdgcn_readlane(end - n, w);
    return w;
  }
};

// UNIFORM: a group of 16 keys lies in one page (the page size is a multiple of 16).  STREAM: K and V
// are read past the caches.
template <class E, int HS, int M, bool UNIFORM, bool STREAM>
__global__ __launch_bounds__(256, 2) void paged_decode_kernel(DecodeArgs<E> a, PagedPlan plan,
                                                              bool direct) {
  using D = DecodeTile<E, HS, M>;
  constexpr int KG = D::KG, WK = D::WK, TILE = D::TILE, CK = D::CK, DW = D::DW, NE = D::NE;
  constexpr bool F32 = sizeof(E) == 4;
  constexpr int OP = HS + 4;  // pitch of a head's row in the exchange
  __shared__ __attribute__((aligned(16))) float xo[4][D::HEADS][OP];
  __shared__ float xm[4][D::HEADS], xl[4][D::HEADS];
  __shared__ int64_t rows_at[UNIFORM ? 1 : 4][2][UNIFORM ? 1 : WK];

  const int lane = threadIdx.x & 63, wave = wave_index();
  const int col = lane & 15, quarter = lane >> 4;
  const int jobs = a.nkv * a.chunks;  // jobs a sequence

  const SeqKeys seqs(plan);
  int u = 0, u_end, b, job, t, keys, n_tiles;
  if (direct) {
    b = blockIdx.x / jobs;
    job = blockIdx.x - b * jobs;
    t = 0;
    keys = uniform(SeqKeys::keys(plan, b));
    u_end = n_tiles = (keys + TILE - 1) / TILE;
  } else {
    int before;
    const Deal deal(seqs.count<TILE>(plan, 0, before) * jobs, gridDim.x);
    if ((int)blockIdx.x >= deal.W || deal.units == 0) return;
    u = deal.start(blockIdx.x);
    u_end = deal.start(blockIdx.x + 1);
    b = seqs.find<TILE>(plan, (int)((unsigned)u / (unsigned)jobs), before);
    keys = seqs.of(plan, b);
    n_tiles = (keys + TILE - 1) / TILE;
    const int in_seq = u - before * jobs;
    job = (int)((unsigned)in_seq / (unsigned)n_tiles);
    t = in_seq - job * n_tiles;
  }

  for (;;) {
    // ---- one job, tiles [t, t_end)
    const int t_end = min(n_tiles, t + (u_end - u));
    const int kvh = job / a.chunks, chunk = job - kvh * a.chunks;
    const int head0 = kvh * a.group + D::HEADS * chunk, heads = min(D::HEADS, a.group - D::HEADS * chunk);
    const int32_t* table = plan.table + b * plan.table_stride;
    const E* kb = a.k + kvh * a.sk.h;
    const E* vb = a.v + kvh * a.sv.h;

    // Q in the order of the B operand: column = head, the chunk of d of the K operand
    u32x4 qf[M][CK];
    f32x4 acc[M][NE];
    float m[M], l[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
#pragma unroll
      for (int s = 0; s < CK; ++s) {
        qf[i][s] = u32x4{0, 0, 0, 0};
        if (16 * i + col < heads)
          qf[i][s] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(
                         a.q + b * a.qt + (head0 + 16 * i + col) * a.qh) + 64 * s + 16 * quarter);
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) acc[i][e] = f32x4{0, 0, 0, 0};
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }

    // Page of this wave's group of 16 keys (UNIFORM): lane i has group i % KG of the i / KG-th tile
    // from tp on.  Entries behind the last key are not read.
    constexpr int TP = 64 / KG;  // tiles that a load of pages covers
    auto load_pages = [&](int tp) {
      const int key = (tp + lane / KG) * TILE + wave * WK + 16 * (lane % KG);
      int page = -1;
      if (key < keys && tp + lane / KG < t_end) {
        page = table[plan.ps.div(key)];
        page = (uint32_t)page < (uint32_t)plan.num_pages ? page : -1;
      }
      return page;
    };
    int tp = t, pages = -1, pages_next = -1;
    if constexpr (UNIFORM) {
      pages = load_pages(tp);
      pages_next = load_pages(tp + TP);
    }

    u32x4 kr[KG][CK];
    uint32_t vr[4 * KG][DW];
    uint32_t valid_k = 0, valid_v = 0;  // bit 4 g + r: key 16 g + 4 quarter + r of the tile in kr, vr
    bool full_k = false, full_v = false;
    int page_of[KG];  // of the tile whose K was loaded last (UNIFORM)

    auto load = []<class T>(const char* p) {
      if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
      else return *reinterpret_cast<const T*>(p);
    };
    auto load_k = [&](int tile) {
      const int k0 = tile * TILE + wave * WK;
      if constexpr (UNIFORM) {
        if (tile - tp >= TP) {
          tp += TP;
          pages = pages_next;
          pages_next = load_pages(tp + TP);
        }
        full_k = k0 + WK <= keys;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          page_of[g] = __builtin_amdgcn_readlane(pages, (tile - tp) * KG + g);
          full_k = full_k && page_of[g] >= 0;
        }
        valid_k = 0;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const int key = k0 + 16 * g;
          const int row = key - plan.ps.div(key) * (int)plan.ps.d;
          // an unmapped group reads page 0; nothing of it is used
          const E* p = kb + max(page_of[g], 0) * a.sk.a + row * a.sk.r;
          const int at = col * (int)a.sk.r * (int)sizeof(E) + 16 * quarter;
#pragma unroll
          for (int s = 0; s < CK; ++s)
            kr[g][s] = load.template operator()<u32x4>(reinterpret_cast<const char*>(p) + (uint32_t)(at + 64 * s));
          if (page_of[g] >= 0)
            valid_k |= (0xfu >> (4 - min(max(keys - key - 4 * quarter, 0), 4))) << (4 * g);
        }
      } else {
        // offsets of the tile's rows, one a lane, through this wave's part of LDS; -1: no key
        wave_lds_fence();
#pragma unroll
        for (int i = 0; i < (WK + 63) / 64; ++i) {
          const int j = lane + 64 * i, key = k0 + j;
          int page = -1, row = 0;
          if (key < keys) {
            const int at = plan.ps.div(key);
            row = key - at * (int)plan.ps.d;
            page = table[at];
          }
          const bool ok = (uint32_t)page < (uint32_t)plan.num_pages;
          if (j < WK) {
            rows_at[wave][0][j] = ok ? page * a.sk.a + row * a.sk.r : -1;
            rows_at[wave][1][j] = ok ? page * a.sv.a + row * a.sv.r : -1;
          }
        }
        wave_lds_fence();
        valid_k = 0;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const int64_t at = max(rows_at[wave][0][16 * g + col], (int64_t)0);
#pragma unroll
          for (int s = 0; s < CK; ++s)
            kr[g][s] = load.template operator()<u32x4>(reinterpret_cast<const char*>(kb + at) + 64 * s + 16 * quarter);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            valid_k |= (uint32_t)(rows_at[wave][0][16 * g + 4 * quarter + r] >= 0) << (4 * g + r);
        }
        full_k = __all(valid_k == (uint32_t)((1ull << (4 * KG)) - 1));
      }
    };
    auto load_v = [&](int tile) {  // of the tile whose K was loaded last
      valid_v = valid_k;
      full_v = full_k;
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const E* p = vb;
        if constexpr (UNIFORM) {
          const int key = tile * TILE + wave * WK + 16 * g;
          const int row = key - plan.ps.div(key) * (int)plan.ps.d;
          p = vb + max(page_of[g], 0) * a.sv.a + row * a.sv.r;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char* src;
          if constexpr (UNIFORM) {
            src = reinterpret_cast<const char*>(p) +
                  (uint32_t)((4 * quarter + r) * (int)a.sv.r * (int)sizeof(E) + col * DW * 4);
          } else {
            const int64_t at = max(rows_at[wave][1][16 * g + 4 * quarter + r], (int64_t)0);
            src = reinterpret_cast<const char*>(vb + at) + col * DW * 4;
          }
          uint32_t(&x)[DW] = vr[4 * g + r];
          if constexpr (DW >= 4) {
#pragma unroll
            for (int c = 0; c < DW / 4; ++c) {
              const u32x4 w = load.template operator()<u32x4>(src + 16 * c);
#pragma unroll
              for (int i = 0; i < 4; ++i) x[4 * c + i] = w[i];
            }
          } else if constexpr (DW == 2) {
            const u32x2 w = load.template operator()<u32x2>(src);
            x[0] = w[0]; x[1] = w[1];
          } else {
            x[0] = load.template operator()<uint32_t>(src);
          }
        }
      }
    };

    if (t < t_end) {
      load_k(t);
      load_v(t);
    }
    for (int tile = t; tile < t_end; ++tile) {
      // no contraction: scaled scores are rounded before the offset is taken off, so that equal
      // scores of any size have equal exponents
#pragma clang fp contract(off)
      // ---- scores of 16 KG keys: lane, register r of group g: key 16 g + 4 quarter + r, head col
      f32x4 s[M][KG];
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int g = 0; g < KG; ++g) s[i][g] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < CK; ++c)
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int i = 0; i < M; ++i) {
            if constexpr (F32) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                s[i][g] = mfma16(__uint_as_float(kr[g][c][j]), __uint_as_float(qf[i][c][j]), s[i][g]);
            } else {
              s[i][g] = mfma16(__builtin_bit_cast(vec8_t<E>, kr[g][c]),
                               __builtin_bit_cast(vec8_t<E>, qf[i][c]), s[i][g]);
            }
          }
      if (tile + 1 < t_end) load_k(tile + 1);
#pragma unroll
      for (int i = 0; i < M; ++i) {
        float mt = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[i][g][r] *= a.scale_log2;
            if (!full_v && !(valid_v >> (4 * g + r) & 1)) s[i][g][r] = -INFINITY;
            mt = fmaxf(mt, s[i][g][r]);
          }
        mt = max_quarters(mt);
        if (__any(mt > m[i])) {
          const float m_new = fmaxf(m[i], mt);
          const float alpha = fast_exp2(m[i] - (m_new == -INFINITY ? 0.0f : m_new));
          l[i] *= alpha;
#pragma unroll
          for (int e = 0; e < NE; ++e) acc[i][e] *= alpha;
          m[i] = m_new;
        }
        const float off = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[i][g][r] = fast_exp2(s[i][g][r] - off);
            l[i] += s[i][g][r];
          }
      }
      // rows without a key count as zeros: what lies there may be anything
      if (!full_v) {
#pragma unroll
        for (int i = 0; i < 4 * KG; ++i)
          if (!(valid_v >> i & 1)) {
#pragma unroll
            for (int w = 0; w < DW; ++w) vr[i][w] = 0;
          }
      }
      // ---- O^T += V^T P^T
      if constexpr (F32) {
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
              for (int i = 0; i < M; ++i)
                acc[i][e] = mfma16(__uint_as_float(vr[4 * g + r][e]), s[i][g][r], acc[i][e]);
      } else {
#pragma unroll
        for (int g = 0; g < KG; g += 2) {  // 32 keys: the lane's 8 are its k-slots
          vec8_t<E> hi[M], lo[M];
#pragma unroll
          for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float p = s[i][g + (j >> 2)][j & 3];
              hi[i][j] = (E)p;
              lo[i][j] = (E)(p - (float)hi[i][j]);
            }
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = vr[4 * g + 2 * i][e / 2], y = vr[4 * g + 2 * i + 1][e / 2];
              w[i] = e % 2 ? pack_hi16(x, y) : pack_lo16(x, y);
            }
            const auto va = __builtin_bit_cast(vec8_t<E>, w);
#pragma unroll
            for (int i = 0; i < M; ++i) {
              acc[i][e] = mfma16(va, lo[i], acc[i][e]);
              acc[i][e] = mfma16(va, hi[i], acc[i][e]);
            }
          }
        }
      }
      if (tile + 1 < t_end) load_v(tile + 1);
    }

    // ---- the four waves' parts, against the largest offset
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const float sum = sum_quarters(l[i]);
      if (quarter == 0) { xm[wave][16 * i + col] = m[i]; xl[wave][16 * i + col] = sum; }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < NE; ++e) xo[wave][16 * i + col][NE * (4 * quarter + r) + e] = acc[i][e][r];
    }
    __syncthreads();
    const bool whole = t == 0 && t_end == n_tiles;
    // a job that began in an earlier workgroup goes to this one's first slot, else to its second
    float* part = a.ws + ((int64_t)blockIdx.x * 2 + (t == 0)) * D::PART;
    constexpr int TPH = HS / 4;  // threads a head
    for (int h = threadIdx.x / TPH; h < heads; h += 256 / TPH) {
      const int d = 4 * (threadIdx.x % TPH);
      float mj = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mj = fmaxf(mj, xm[w][h]);
      const float off = mj == -INFINITY ? 0.0f : mj;
      float lj = 0.0f;
      float4 o = zero4();
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = fast_exp2(xm[w][h] - off);
        const float4 x = ld4(&xo[w][h][d]);
        lj = fmaf(f, xl[w][h], lj);
        o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y);
        o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
      }
      if (whole) {
        const float inv = lj == 0.0f ? 0.0f : 1.0f / lj;
        const int64_t at = (int64_t)b * a.nh + head0 + h;
        E* op = a.o + at * HS + d;
        op[0] = (E)(o.x * inv); op[1] = (E)(o.y * inv);
        op[2] = (E)(o.z * inv); op[3] = (E)(o.w * inv);
        if (d == 0) a.l[at] = lj == 0.0f ? -INFINITY : off * kLn2 + logf(lj);
      } else {
        st4(part + h * HS + d, o);
        if (d == 0) { part[D::HEADS * HS + h] = mj; part[D::HEADS * (HS + 1) + h] = lj; }
      }
    }

    u += t_end - t;
    if (direct || u >= u_end) return;
    __syncthreads();  // the exchange is read: the next job may write it
    t = 0;
    if (++job == jobs) {
      job = 0;
      do keys = seqs.of(plan, ++b); while (keys == 0);
      n_tiles = (keys + TILE - 1) / TILE;
    }
  }
}

// Joins the parts of the jobs that several workgroups share, in order of groups of parts; rows without
// a key.  WAVES waves have a row of O (a sequence and query head), HS / 4 lanes a part of it.
template <class E, int HS, int M, int WAVES>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(DecodeArgs<E> a, PagedPlan plan,
                                                                int grid) {
  using D = DecodeTile<E, HS, M>;
  constexpr int LP = HS / 4, PG = 64 / LP;  // lanes a part; parts a wave takes at a time
  __shared__ __attribute__((aligned(16))) float xo[WAVES][HS];
  __shared__ float xm[WAVES], xl[WAVES];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int id = blockIdx.x * (4 / WAVES) + wave / WAVES;
  const bool live = id < plan.B * a.nh;  // idle waves of the last workgroup stay for the barrier
  const int b = live ? id / a.nh : 0, h = live ? id - b * a.nh : 0;
  const int kvh = h / a.group, in_group = h - kvh * a.group;
  const int job = kvh * a.chunks + in_group / D::HEADS, row = in_group % D::HEADS;
  const int jobs = a.nkv * a.chunks;
  const SeqKeys seqs(plan);
  int before;
  const Deal deal(seqs.count<D::TILE>(plan, b, before) * jobs, grid);
  const int n = (seqs.of(plan, b) + D::TILE - 1) / D::TILE;
  int w0 = 0, w1 = -1;
  if (n > 0) {
    const int first = before * jobs + job * n;
    w0 = deal.owner(first);
    w1 = deal.owner(first + n - 1);
    if (w0 == w1) return;  // written whole (all waves of the row agree)
  }
  if (!live) return;
  const int d = 4 * (lane % LP);
  constexpr int STEP = PG * WAVES;
  float m = -INFINITY, l = 0.0f;
  float4 o = zero4();
  for (int w = w0 + lane / LP + PG * (wave % WAVES); w <= w1; w += 2 * STEP) {
    // two parts' loads in flight
    float pm[2], pl[2];
    float4 v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = w + j * STEP <= w1 ? w + j * STEP : w;
      const float* p = a.ws + ((int64_t)i * 2 + (i == w0)) * D::PART;
      pm[j] = w + j * STEP <= w1 ? p[D::HEADS * HS + row] : -INFINITY;
      pl[j] = p[D::HEADS * (HS + 1) + row];
      v[j] = ld4(p + row * HS + d);
    }
    const float m_new = fmaxf(m, fmaxf(pm[0], pm[1])), off = m_new == -INFINITY ? 0.0f : m_new;
    const float f = fast_exp2(m - off), f0 = fast_exp2(pm[0] - off), f1 = fast_exp2(pm[1] - off);
    l = l * f + (pl[0] * f0 + pl[1] * f1);
    o.x = o.x * f + (v[0].x * f0 + v[1].x * f1);
    o.y = o.y * f + (v[0].y * f0 + v[1].y * f1);
    o.z = o.z * f + (v[0].z * f0 + v[1].z * f1);
    o.w = o.w * f + (v[0].w * f0 + v[1].w * f1);
    m = m_new;
  }
  auto join = [&](float m2, float l2, float4 o2) {
    const float m_new = fmaxf(m, m2), off = m_new == -INFINITY ? 0.0f : m_new;
    const float f = fast_exp2(m - off), f2 = fast_exp2(m2 - off);
    l = l * f + l2 * f2;
    o.x = o.x * f + o2.x * f2; o.y = o.y * f + o2.y * f2;
    o.z = o.z * f + o2.z * f2; o.w = o.w * f + o2.w * f2;
    m = m_new;
  };
#pragma unroll
  for (int x = LP; x < 64; x <<= 1)
    join(__shfl_xor(m, x), __shfl_xor(l, x),
         make_float4(__shfl_xor(o.x, x), __shfl_xor(o.y, x), __shfl_xor(o.z, x), __shfl_xor(o.w, x)));
  if constexpr (WAVES > 1) {
    if (lane < LP) st4(&xo[wave][d], o);
    if (lane == 0) { xm[wave] = m; xl[wave] = l; }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int x = 1; x < WAVES; ++x) join(xm[x], xl[x], ld4(&xo[x][d]));
  }
  if (lane >= LP) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = (int64_t)b * a.nh + h;
  E* op = a.o + at * HS + d;
  op[0] = (E)(o.x * inv); op[1] = (E)(o.y * inv);
  op[2] = (E)(o.z * inv); op[3] = (E)(o.w * inv);
  if (lane == 0) a.l[at] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

// How a call is laid out.  pass: query heads that a pass over K and V serves (16 M).  W: workgroups
// that the tiles are dealt to, two a CU, or 0 where every job is one workgroup's (direct): up to five
// tiles a job are walked in the time that the deal and the second kernel take, and up to eight where
// the jobs alone fill the GPU.  Dealt and direct, us, BF16, 32 over 8 heads of 128 (128 keys a tile): 8
// sequences of 600 (5 tiles) 12.5 and 11.3, 4 of 750 (6) 10.7 and 12.6; 64 of 1000 (8) 46.1 and 43.6, of
// 50 to 1000 25.0 and 23.5, of 50 to 2000 (16) 36.2 and 39.4.
struct DecodeGrid {
  int64_t chunks, jobs;
  int pass, W;
};
int tile_keys(int64_t hs, int elem) { return (int)(4 * 16 * (elem == 2 ? 256 / hs : 128 / hs)); }
DecodeGrid decode_grid(int64_t B, int64_t nh, int64_t nkv, int64_t hs, int64_t capacity, int elem) {
  DecodeGrid g;
  g.pass = nh / nkv > 16 ? 32 : 16;
  g.chunks = (nh / nkv + g.pass - 1) / g.pass;
  g.jobs = B * nkv * g.chunks;
  const int64_t tiles = (capacity + tile_keys(hs, elem) - 1) / tile_keys(hs, elem);
  const int64_t places = 512;
  g.W = tiles <= (g.jobs < places ? 5 : 8) ? 0 : (int)std::min<int64_t>(g.jobs * tiles, places);
  return g;
}

// Pools from this size on are read past the caches, unless several chunks of heads read the same
// keys: four layers of them exceed the 256 MB last-level cache, so nothing is left of a layer's keys
// when the next token reads them.  64 sequences of 500 to 8000 tokens (743 MB): 140 us through the
// caches, 124 past them; 16 of 200 to 1000 (37 MB, read again while still cached): 15.1 and 15.9.
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

template <class E, int HS, int M>
void launch_decode(const DecodeArgs<E>& a, const PagedPlan& plan, const DecodeGrid& g, bool stream,
                   hipStream_t st) {
  const dim3 grid((unsigned)(g.W > 0 ? g.W : g.jobs));
  auto go = [&]<bool UNIFORM>() {
    if (stream)
      hipLaunchKernelGGL((paged_decode_kernel<E, HS, M, UNIFORM, true>), grid, dim3(256), 0, st, a, plan, g.W == 0);
    else
      hipLaunchKernelGGL((paged_decode_kernel<E, HS, M, UNIFORM, false>), grid, dim3(256), 0, st, a, plan, g.W == 0);
  };
  if (plan.ps.d % 16 == 0) go.template operator()<true>();
  else go.template operator()<false>();
  if (g.W == 0) return;
  const int64_t rows = (int64_t)plan.B * a.nh;
  // four waves a row where a job has eight parts or more on average
  if (g.W >= 8 * g.jobs)
    hipLaunchKernelGGL((paged_decode_join_kernel<E, HS, M, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, plan, g.W);
  else
    hipLaunchKernelGGL((paged_decode_join_kernel<E, HS, M, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, plan, g.W);
}

template <class E, class P>
int decode(const P* q, const int64_t* qs, float scale, P* o, float* l, void* ws, int64_t ws_bytes,
           const PagedArgs& pa, void* stream) {
  PagedPlan plan;
  if (int rc = check_paged(pa, sizeof(E), plan)) return rc;
  if (int rc = check_paged_rows(q, qs, pa.B, pa, scale, o, l, sizeof(E), "paged_attention_decode"))
    return rc;
  if (pa.B * pa.nh == 0) return CTA_OK;
  const DecodeGrid g = decode_grid(pa.B, pa.nh, pa.nkv, pa.hs, plan.capacity, sizeof(E));
  if ((double)g.jobs * (plan.capacity / tile_keys(pa.hs, sizeof(E)) + 1) >= 0x1p31)  // tiles dealt
    return fail(CTA_ERR_INVALID_ARGUMENT, "size too large");
  if (g.W > 0 && (!ws || !aligned16(ws) ||
                  ws_bytes < cta_paged_attention_decode_workspace(pa.B, pa.nh, pa.nkv, pa.hs,
                                                                  pa.pages_per_seq, pa.page_size)))
    return fail(CTA_ERR_INVALID_ARGUMENT, "paged_attention_decode needs its workspace");
  DecodeArgs<E> a;
  a.q = reinterpret_cast<const E*>(q);
  a.k = static_cast<const E*>(pa.k_cache); a.v = static_cast<const E*>(pa.v_cache);
  a.qt = qs[0]; a.qh = qs[1];
  a.sk = {pa.ks[0], pa.ks[1], pa.ks[2]};
  a.sv = {pa.vs[0], pa.vs[1], pa.vs[2]};
  a.nh = (int)pa.nh; a.nkv = (int)pa.nkv; a.group = (int)(pa.nh / pa.nkv);
  a.chunks = (int)g.chunks;
  a.scale_log2 = scale * kLog2e;
  a.o = reinterpret_cast<E*>(o); a.l = l; a.ws = static_cast<float*>(ws);
  const hipStream_t st = as_stream(stream);
  const bool past = g.chunks == 1 &&
                    pa.num_pages * pa.page_size * pa.nkv * pa.hs * 2 * (int64_t)sizeof(E) >= kStreamBytes;
  auto go = [&]<int HS>() {
    if (g.pass == 32) launch_decode<E, HS, 2>(a, plan, g, past, st);
    else launch_decode<E, HS, 1>(a, plan, g, past, st);
  };
  if (pa.hs == 32) go.template operator()<32>();
  else if (pa.hs == 64) go.template operator()<64>();
  else go.template operator()<128>();
  return check_launch("paged_attention_decode");
}

}  // namespace
}  // namespace cta

using namespace cta;

// The larger of what the types need: 16-bit tiles are the longer ones, FP32 has more of them.
extern "C" int64_t cta_paged_attention_decode_workspace(int64_t B, int64_t nh, int64_t nkv,
                                                        int64_t hs, int64_t pages_per_seq,
                                                        int64_t page_size) {
  if (B <= 0 || nh <= 0 || nkv <= 0 || pages_per_seq <= 0 || page_size <= 0 ||
      (hs != 32 && hs != 64 && hs != 128) || pages_per_seq > ((int64_t)1 << 30) / page_size)
    return 0;
  const DecodeGrid g = decode_grid(B, nh, nkv, hs, pages_per_seq * page_size, 4);
  return (int64_t)g.W * 2 * g.pass * (hs + 2) * 4;
}

#define CTA_PAGED_DECODE(SUFFIX, TYPE, PTR)                                                       \
  extern "C" int cta_paged_attention_decode##SUFFIX(                                              \
      const PTR* q, const int64_t* q_strides, const PTR* k_cache, const int64_t* k_cache_strides, \
      const PTR* v_cache, const int64_t* v_cache_strides, int64_t num_pages, int64_t page_size,   \
      const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,                     \
      const int32_t* seq_lens, int64_t B, int64_t nh, int64_t nkv, int64_t hs, float scale,       \
      PTR* o, float* l, void* workspace, int64_t workspace_bytes, void* stream) {                 \
    return decode<TYPE>(q, q_strides, scale, o, l, workspace, workspace_bytes,                    \
                        {k_cache_strides, v_cache_strides, num_pages, page_size, table_stride,    \
                         pages_per_seq, B, nh, nkv, hs, page_table, seq_lens, nullptr, k_cache,   \
                         v_cache},                                                                \
                        stream);                                                                  \
  }
CTA_PAGED_DECODE(, float, float)
CTA_PAGED_DECODE(_bf16, __bf16, uint16_t)
CTA_PAGED_DECODE(_f16, _Float16, uint16_t)
#undef CTA_PAGED_DECODE
