// The paged key/value cache as its kernels see it: what is appended to it (paged_append.hip), and
// the attention over it (paged_decode.hip, paged_prefill.hip).
//
// A cache is a pool of pages, (pages, kv heads, page size, hs).  Row b of the page table lists the
// pages of sequence b in order: position p lies in page table[b][p / page size], row p % page size.
// seq_lens[b] counts the sequence's tokens, new ones included.  Packed tokens cu_q[b] ..
// cu_q[b + 1] - 1 are the new ones of sequence b, its last n_b = cu_q[b + 1] - cu_q[b] positions.
//
// The plan (table, lengths, cu_q) lives on the device, so the host cannot look at it without a
// synchronisation.  Every kernel therefore takes any values in it: an entry of the table outside
// [0, pages) maps no page, and positions outside [0, pages per sequence x page size) have none:
// they hold no key and store nothing.
#pragma once

#include "cta_common.hpp"

namespace cta {

// n / d for 0 <= n < 2^31 by one 64-bit product: m = ceil(2^(31 + s) / d) with s = ceil(log2 d)
// overshoots by less than 2^s, so n m / 2^(31 + s) exceeds n / d by less than n 2^-31 / d < 1 / d.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t den) : d(den), m(0), s(0) {
    while (((uint64_t)1 << s) < den) ++s;
    m = (uint32_t)((((uint64_t)1 << (31 + s)) + den - 1) / den);
    s += 31;
  }
  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> s); }
};

// Page table, lengths and geometry.
struct PagedPlan {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* cu_q;  // null: one new token a sequence
  int B;
  int num_pages;
  int capacity;  // positions a sequence can have: pages per sequence x page size
  FastDiv ps;

  // Page of a position in [0, capacity), or -1.
  __device__ __forceinline__ int page(int b, int pos, int& row) const {
    const int i = ps.div(pos);
    row = pos - i * (int)ps.d;
    const int p = table[b * table_stride + i];
    return (uint32_t)p < (uint32_t)num_pages ? p : -1;
  }
  // Sequence of packed token t, the same for the whole wave: the number of sequences that end at
  // or before t, B for the rows behind the last sequence (or in front of the first).  64 ends a
  // step, so that up to 64 sequences cost one load's latency where a binary search costs six.
  __device__ __forceinline__ int find_seq(int t) const {
    if (cu_q == nullptr) return t;
    const int lane = threadIdx.x & 63;
    int n = t < cu_q[0] ? B : 0;
    for (int i = lane; i - lane < B; i += 64)
      n += __popcll(__ballot(i < B && cu_q[min(i, B - 1) + 1] <= t));
    return min(n, B);
  }
  // Position of packed token t of sequence b; any value, where the plan holds any.
  __device__ __forceinline__ int64_t position(int b, int t) const {
    return cu_q == nullptr ? (int64_t)lens[b] - 1 : (int64_t)lens[b] - cu_q[b + 1] + t;
  }
  // How many positions in front of position p, and p, can hold keys.
  __device__ __forceinline__ int keys_to(int64_t p) const {
    return (int)min(max(p + 1, (int64_t)0), (int64_t)capacity);
  }
};

// A value that is the same in every lane, marked so: branches on it are scalar ones.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// Value of one lane (the same lane for all).
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)lane_of((int)(v >> 32), lane) << 32 | (uint32_t)lane_of((int)v, lane));
}
// The value that a data-parallel-primitive control brings from another lane; 0 where it brings none.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)dpp<CTRL, ROWS>((int)(v >> 32)) << 32 | (uint32_t)dpp<CTRL, ROWS>((int)v));
}
// Sums of the lanes' values up to and with each lane, all 64 active: shifts by 1, 2, 4 and 8 inside rows
// of 16, then the last lane of row 0 into row 1 and of row 2 into row 3, and lane 31 into the upper rows.
// (33 FP32 sequences of up to 4000 tokens, decode: 13.3 us with shuffles, 12.8 so; a prompt of 128 tokens
// behind 900: 28.1 and 26.9.)
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
  v += dpp<0x111, 0xf>(v);
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);
  v += dpp<0x143, 0xc>(v);
  return v;
}

// Work counted in units, units(b) for sequence b, in integers T: the host does not know the lengths,
// so a kernel that shares it out counts them itself, 64 sequences a step, a whole wave at a time.
//
// Units of all B sequences; before: those of the sequences in front of b.
template <class T, class F>
__device__ __forceinline__ T count_units(int B, int b, T& before, F&& units) {
  const int lane = threadIdx.x & 63;
  T total = 0, front = 0;
  for (int i = lane; i < B; i += 64) {
    const T n = units(i);
    total += n;
    if (i < b) front += n;
  }
  before = lane_of(wave_scan(front), 63);
  return lane_of(wave_scan(total), 63);
}
// Sequence that holds unit x of all units in a row, and the units before it; B, and all units, if
// there are no more than x.
template <class T, class F>
__device__ __forceinline__ int find_unit(int B, T x, T& before, F&& units) {
  const int lane = threadIdx.x & 63;
  before = 0;
  for (int i0 = 0; i0 < B; i0 += 64) {
    const int i = i0 + lane;
    const T n = i < B ? (T)units(i) : (T)0;
    const T end = wave_scan(n);
    const uint64_t past = __ballot(before + end > x);
    if (past) {
      const int w = __builtin_ctzll(past);
      before += lane_of(end - n, w);
      return i0 + w;
    }
    before += lane_of(end, 63);
  }
  return B;
}

// Element strides of a cache or of packed tokens (the last dimension is dense).
struct Strides3 {
  int64_t a, h, r;  // cache: page, head, row;  tokens: token, head, unused
};

// Host side: the arguments that every entry point takes.
struct PagedArgs {
  const int64_t *ks, *vs;  // cache strides, 4 entries (page, head, row, d)
  int64_t num_pages, page_size, table_stride, pages_per_seq, B, nh, nkv, hs;
  const int32_t *page_table, *seq_lens, *cu_q;
  const void *k_cache, *v_cache;
};
// Validates them (elem: bytes of an element) and fills the plan.
int check_paged(const PagedArgs& a, int elem, PagedPlan& plan);
// Packed tokens: strides (token, head, d) with 16-byte rows.
bool tokens_layout_ok(const void* p, const int64_t* s, int elem);
// Validates what the attention entries take besides: queries, results, the scale.
int check_paged_rows(const void* q, const int64_t* qs, int64_t rows, const PagedArgs& a, float scale,
                     const void* o, const float* l, int elem, const char* what);

}  // namespace cta
