// Geometry and masks of causal sliding-window attention with sink tokens, shared by the forward kernel (contiguous
// and paged keys) and the two backward kernels.
//
// Keys sit at positions 0..len-1 of their sequence, query row i at position base + i (base = Sk - Sq, or the
// sequence's length minus the number of new tokens over a cache).  Key j is visible to a row at position p iff
//     0 <= p < len,   j <= p,   (j > p - window  or  j < sinks).
// Rows of a tree of drafts hold a 64-bit mask: bit u = draft u (the key at base + u) is visible; the row's position
// is base + popcount - 1 (its depth), and it sees the keys before base by the rule above.  In a sequence shorter than the
// tree base is negative: drafts with base + u < 0 have no key but count for the positions.
//
// The kernels work on 128-token key tiles.  The tiles a query tile needs are those its rows' windows touch, walked
// from the diagonal downwards (so the running maximum is set by visible scores from the first tile on), and then
// tile 0 once more for the sinks if no window reaches it: sinks <= 128, so that is one tile.  A tile that every row of
// the query tile sees entirely takes an unmasked path; in the others each thread builds one visibility bit per column
// of its row.
//
// Times in the comments of the windowed kernels: "measured" ones are whole calls on inputs that change from call to call, in a
// captured graph (no host time).  Pairs "a -> b" or "a against b" compare two builds of one moment, kernels alone on one
// state, ten launches at a time: at the clock of a short burst, 5 to 15 % below the former.
#pragma once

#include "bsa_common.cuh"

namespace bsa {

constexpr int kMaxSinks = 128;
constexpr int kWindowAll = 1 << 29;  // "no window": no length is larger, and its sums with positions stay inside 32 bits
constexpr int kMaxTreeNodes = 64;
constexpr long long kGroupBytes = 48ll << 20;

// Bits [0, n) of a 32-bit word; n is clamped to [0, 32].
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : ((1u << n) - 1u));
}
// Word w (bits 32w .. 32w+31) of the bit range [lo, hi).
__device__ __forceinline__ uint32_t range_word(int lo, int hi, int w) {
  return low_bits(hi - 32 * w) & ~low_bits(lo - 32 * w);
}

// The key tiles of one query tile whose rows have positions in [p_lo, p_hi].
struct TileList {
  int n_win;  // window tiles t_hi, t_hi - 1, ..., t_hi - n_win + 1
  int n;      // n_win, plus one when tile 0 follows for the sinks
  int t_hi;
  int k_lo;   // first key any window reaches
  __device__ __forceinline__ int tile(int it) const { return it < n_win ? t_hi - it : 0; }
};

__device__ __forceinline__ TileList window_tiles(int p_lo, int p_hi, int len, int window, int sinks) {
  TileList t;
  p_lo = max(p_lo, 0);
  p_hi = min(p_hi, len - 1);
  t.n = t.n_win = 0;
  t.t_hi = 0;
  t.k_lo = 0;
  if (p_lo > p_hi) return t;
  t.k_lo = max(0, p_lo - window + 1);
  t.t_hi = p_hi >> 7;
  const int t_lo = t.k_lo >> 7;
  t.n_win = t.t_hi - t_lo + 1;
  t.n = t.n_win + ((sinks > 0 && t_lo > 0) ? 1 : 0);
  return t;
}

// The order in which whole tiles are dealt to the CTAs: `group` columns (heads of sequences) at a time, for each of their
// tiles in turn all columns of the group.  CTAs that run side by side then work on different heads instead of asking L2 for
// the same keys at the same time, and the last items are the short ones if the ranks go from long lists to short ones.
// Against one head after the other (forward / backward, us): 16 heads of 16384 tokens, window 1024, 202 / 646 -> 182 / 620;
// 80 heads of 5000, window 700, 329 / 990 -> 240 / 860; 256 causal heads of 2048, 450 / 1460 -> 365 / 1200.
struct Dealt {
  int column, rank;
};
__device__ __forceinline__ Dealt deal_item(int w, int columns, int tiles, int group) {
  const int g = w / (group * tiles), first = g * group;
  const int width = min(group, columns - first);
  w -= first * tiles;
  Dealt d;
  d.rank = w / width;
  d.column = first + w - d.rank * width;
  return d;
}
// The group's width: as many columns as keep what they re-read (`span` keys and values each, shared by `share` columns) in
// L2.  64 heads of 16384 tokens, window 8192: 16, 48, 96 MB and all heads at once 3.11, 3.05, 3.20 and 3.19 ms forward, 10.2,
// 10.3, 10.5 and 11.0 backward; 80 heads of 5000, window 700, 250, 240, 249 and 252 us.
inline int head_group(long long columns, long long span, int D, int share) {
  const long long bytes = span * 4 * D, most = kGroupBytes * share / (bytes > 0 ? bytes : 1);
  const long long g = most < 1 ? 1 : most;
  return (int)(g < columns ? g : columns);
}

// Stores 64 bytes of each thread's row, u[chunk][word], at `dst` = (lane's chunk in the rows of its group of four lanes):
// four lanes exchange their chunks, so that a store covers 64 bytes of eight rows instead of 16 of 32, each of which takes
// a cycle of its own.  `rows_ok` = bits of the group's rows that exist.  Called by whole warps.
__device__ __forceinline__ void store_exchanged(uint4* const* dst, int at, uint32_t (*u)[4], uint32_t rows_ok) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int bit = 1; bit < 4; bit <<= 1) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s & bit) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (lane & bit) ? u[s][e] : u[s | bit][e], bit);
        if (lane & bit) u[s][e] = got;
        else u[s | bit][e] = got;
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
    if ((rows_ok >> s) & 1u) dst[s][at] = make_uint4(u[s][0], u[s][1], u[s][2], u[s][3]);
}
// The addresses for it: those of the group's rows, at the lane's chunk.
__device__ __forceinline__ void exchange_rows(void* row, uint4** dst) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
    dst[s] = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), s, 4)) + (threadIdx.x & 3);
}

// Equal runs of a list: CTA c of the n that have work gets all / n entries, and one of the all % n that are left over.
struct Runs {
  int q, r;
  __device__ __forceinline__ int begin(int c) const { return c * q + min(c, r); }
  __device__ __forceinline__ int holder(int x) const { return x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q; }
};

// Finds entry `lo` of a list of `items` items with cost(i) >= 1 entries each: its item, and `lo` becomes its place in
// the item.  Called by whole warps.
template <typename Cost>
__device__ __forceinline__ int find_item(int items, int& lo, Cost cost) {
  const int lane = threadIdx.x & 31;
  for (int i0 = 0; i0 < items; i0 += 32) {
    const int mine = i0 + lane < items ? cost(i0 + lane) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, upto > lo);
    if (over) {
      const int holder = __ffs(over) - 1;
      lo -= __shfl_sync(0xffffffffu, upto - mine, holder);
      return i0 + holder;
    }
    lo -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return 0;
}
template <typename Cost>
__device__ __forceinline__ int total_cost(int items, Cost cost) {
  int all = 0;
  for (int i = threadIdx.x & 31; i < items; i += 32) all += cost(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}

}  // namespace bsa
