// Causal sliding-window attention with sink tokens, backward, for sm_100a (contiguous keys, grouped heads).
//
//   delta_i = sum_d O_id dO_id,  P_ij = exp(scale q_i k_j - lse_i) on the visible pairs,  dS = P o (dO V^T - delta)
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO     (dK, dV of a KV head sum over its G query heads)
//
// Four launches, no atomics, every sum in a fixed order:
//   1. preprocess: -delta and -lse log2(e) per query row, padded to whole 128-row tiles
//   2. dQ kernel: one item per query tile, over the key tiles its windows touch (and tile 0 for the sinks)
//   3. dK/dV kernel: one item per key tile, over the (query head, query tile) pairs that see it.  Tile 0 holds the
//      sinks, which every later query tile sees: those tiles beyond the windows' reach are dealt to further items of
//      about the length of an ordinary one (G * n pairs of tiles against G * (W / 128 + 1): without the split, one CTA
//      would work on tile 0 while the others have finished).  They and tile 0's own item leave fp32 sums of the sink
//      rows in the workspace,
//   4. which the reduce kernel adds up in order.
// With few key tiles the list of each is cut into parts instead (tile 0's with all that see its sinks), whose fp32 sums
// a last pass adds up.
// The structure of the two main kernels is the one that measured best for the block-sparse backward: warps 0-7 compute
// (two groups of 128 threads, thread = tensor-memory lane, group g owns columns [64g, 64g + 64) of the score tiles),
// warps 8-10 (dQ) or 8-9 (dK/dV) issue the MMAs of one dependency chain each, the last warp loads by TMA.
// P and dS are rounded to 16 bits for the tensor cores (all sums are fp32), and delta is that of the 16-bit `out` that the
// forward call returned: relative to the gradients' own rounding the three give errors of 1.4 to 1.6 times in all (rows of a
// few keys, where delta nearly cancels dP, get a delta of their own).  With fp16, small gradients need the loss scaling that
// fp16 training uses anyway.
// What rows that take no part hold - padding, keys before every window, NaN included - reaches no sum: P is replaced by 0 on
// masked pairs, dP too where a tile holds such rows, the statistics of such queries are those of a row that sees nothing, and
// the rows are zeroed in shared memory where an MMA contracts over them.
//
// Bound by the instructions of the compute warps between two MMAs of a chain, like the block-sparse backward.  Measured: 16
// heads of 16384 tokens, window 1024, 4 sinks, bf16: 685 us for the four launches, 680 TFLOP/s of the operations that they execute
// on the visible pairs (14 D each, where the formula has 10 D).
#include "bsa_b200.h"
#include "bsa_common.cuh"
#include "bsa_host.h"
#include "bsa_window.cuh"

#include <type_traits>

namespace bsa {
namespace winbwd {

constexpr int kMmaWarp = 8;
constexpr int kDqThreads = 384;
constexpr int kDqLoadWarp = 11;
constexpr int kDkvThreads = 352;
constexpr int kDkvLoadWarp = 10;
constexpr int kTile = 128 * 128 * 2;
constexpr int kSlab = 128 * 128;
constexpr int kBarBytes = 256 + 16;  // 32 mbarriers, tensor-memory base, abort flag
constexpr int kSmsForParts = 148;    // (a constant, so that the workspace's size does not depend on the device)

struct Params {
  const int32_t* __restrict__ kv_lens;
  const float* __restrict__ lse_log2;  // [B, Hq, Nq * 128]  -lse * log2(e)
  const float* __restrict__ delta;     // [B, Hq, Nq * 128]  -sum_d O dO
  float* partial;                      // [B * Hkv, slots, 2 (dK, dV), sinks, D]
  uint8_t* dq;
  uint8_t* dk;
  uint8_t* dv;
  int* status;
  long long dq_stride[3], dk_stride[3], dv_stride[3];  // elements
  int B, Hq, Hkv, G, Sq, Sk, Nq, Nkv, D;
  int window, sinks;
  int sink_items;  // further items of tile 0 per (batch, KV head); the workspace holds sink_items + 1 slots
  int sink_m0;     // first query tile beyond the reach of tile 0's windows
  int parts;       // few key tiles: parts that each one's list is cut into (partial [B * Hkv * Nkv][parts][2][128][D]); else 0
  int dq_group, dkv_group;  // of deal_item
  int unseen_hi;   // keys [sinks, unseen_hi) lie before every window: no query of the call sees them
  float scale_log2, softmax_scale;
  __device__ __forceinline__ bool holds_unseen(int j0) const { return j0 < unseen_hi && j0 + 128 > sinks; }  // of a key tile
  __device__ __forceinline__ bool unseen(int j) const { return j >= sinks && j < unseen_hi; }
};

template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t u) {
  float2 f;
  if (F16) unpack_f16x2(u, f.x, f.y);
  else {
    f.x = __uint_as_float(u << 16);
    f.y = __uint_as_float(u & 0xffff0000u);
  }
  return f;
}
__device__ __forceinline__ int seq_len(const Params& p, int b) {
  return p.kv_lens ? max(0, min(p.kv_lens[b], p.Sk)) : p.Sk;
}

__device__ __forceinline__ void bulk_load_1d(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}

// Up to 64 fp32 accumulator columns of a row -> 16 bits, scaled -> global.
template <bool F16>
__device__ __forceinline__ void store_half(uint8_t* row, bool valid, const uint32_t* acc, float scale, int cols) {
  const uint32_t all_ok = __ballot_sync(0xffffffffu, valid);
  if (all_ok == 0) return;
  uint4* dst[4];
  exchange_rows(row, dst);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h * 32 < cols) {
      uint32_t u[4][4];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        u[e >> 2][e & 3] = pack16<F16>(__uint_as_float(acc[h * 32 + 2 * e]) * scale, __uint_as_float(acc[h * 32 + 2 * e + 1]) * scale);
      store_exchanged(dst, h * 4, u, all_ok >> (threadIdx.x & 28));
    }
  }
}
__device__ __forceinline__ void store_half_f32(float* dst, const uint32_t* acc, int cols) {
#pragma unroll
  for (int ch = 0; ch < 16; ++ch)
    if (ch * 4 < cols) reinterpret_cast<uint4*>(dst)[ch] = make_uint4(acc[4 * ch], acc[4 * ch + 1], acc[4 * ch + 2], acc[4 * ch + 3]);
}

template <bool F16>
struct Idesc {
  static constexpr uint32_t kFmt = F16 ? 0u : 1u;
  static constexpr uint32_t kKK = umma_idesc(kFmt, kFmt, 0, 0, 128, 128);
  static __device__ __forceinline__ uint32_t kmn(int n) { return umma_idesc(kFmt, kFmt, 0, 1, 128, (uint32_t)n); }
};
__device__ __forceinline__ uint64_t desc_k_major(uint32_t saddr) { return umma_desc_sw128(saddr, 0, 1024); }
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t saddr) { return umma_desc_sw128(saddr, kSlab, 1024); }
constexpr uint64_t kTileStep = kTile >> 4;

// D = A(smem, K-major) * B(smem, K-major)^T, contracting over the head dimension in `ksteps` = D / 16 steps.
template <bool F16>
__device__ __forceinline__ void mma_ss_kk(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t led, int ksteps) {
  auto steps = [&](int k0, int k1) {
#pragma unroll
    for (int k = k0; k < k1; ++k) {
      const uint64_t off = (uint64_t)((k >> 2) * (kSlab >> 4) + (k & 3) * 2);
      umma_f16_ss_led(d, a_desc + off, b_desc + off, Idesc<F16>::kKK, k > 0 ? 1u : 0u, led);
    }
  };
  steps(0, 4);
  if (ksteps > 4) steps(4, 6);  // (an MMA that is predicated off takes as long to issue as one that runs)
  if (ksteps > 6) steps(6, 8);
}
// D (+)= A(tmem, 16 bits, two 32-column halves) * B(smem, MN-major), contracting over 128 tokens.
__device__ __forceinline__ void mma_ts_kmn(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint64_t b_desc, bool acc, uint32_t led, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t a = (k < 4) ? (a_lo + (uint32_t)k * 8u) : (a_hi + (uint32_t)(k - 4) * 8u);
    umma_f16_ts_led(d, a, b_desc + (uint64_t)(k * 128), idesc, (acc || k > 0) ? 1u : 0u, led);
  }
}

// ------------------------------------------------------------------------------------------------
// 1. preprocess: HBM-bound, reads O and dO once.  A warp handles eight consecutive padded rows: sixteen lanes per row
//    with 16 bytes each, all loads of a thread in flight before the first use.
//    Rows that see at most kFewKeys keys take delta = sum_j P_ij dO_i v_j instead, from q, k, v and the LSE: the rounding of
//    O to 16 bits is not small against dP - delta there.  Error of dQ and dK in half steps of the type, from the rounded O: 0.94
//    for rows of two keys, 0.81, 0.74, 0.70 for three to five, 0.68 for eight; this way 0.61.  Those are the first rows of any
//    sequence (blocks of their own, in front of the others: dQ of the rows at positions 0 to 4 0.81 -> 0.61, the whole
//    backward of 8 heads of 300 tokens 15.7 -> 16.0 us, of 16 heads of 16384 equal), and every row of a window that holds no more,
//    which has a kernel of its own (16 heads of 16384 tokens, window 2: the whole backward 227 -> 296 us).
// ------------------------------------------------------------------------------------------------
constexpr int kFewKeys = 5;
struct PreParams {
  const uint8_t *o, *d_o, *q, *k, *v;
  const float* __restrict__ lse;
  float* __restrict__ lse_log2;
  float* __restrict__ delta;
  const int32_t* __restrict__ kv_lens;
  long long o_stride[3], do_stride[3], q_stride[3], k_stride[3], v_stride[3];  // elements
  long long rows_pad;
  int H, G, Sq, SqPad, D, base, window, sinks;
  int first_blocks;  // blocks of the first rows: B * H, or none
  float scale_log2;

  // Rows [first, behind) of a sequence take part; the others may hold anything: their statistics are those of a row that sees
  // nothing.
  __device__ __forceinline__ int first() const { return max(0, -base); }
  __device__ __forceinline__ int behind(long long b) const {
    return kv_lens == nullptr ? Sq : max(0, max(0, min(kv_lens[b], base + Sq)) - base);
  }
};
__device__ __forceinline__ uint4 load16(const uint8_t* p, const long long* stride, long long b, long long h, long long s, int chunk) {
  return *reinterpret_cast<const uint4*>(p + (b * stride[0] + h * stride[1] + s * stride[2] + chunk * 8) * 2);
}
template <bool F16>
__device__ __forceinline__ float dot16(uint4 x, uint4 y) {
  const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
  float acc = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 u = unpack16<F16>(a[e]), w = unpack16<F16>(b[e]);
    acc = fmaf(u.x, w.x, acc);
    acc = fmaf(u.y, w.y, acc);
  }
  return acc;
}
__device__ __forceinline__ float sum16(float x) {  // over sixteen lanes
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// The first rows of a head, at positions below kFewKeys of a wider window: row p sees keys 0..p.  A block takes a head, a
// half-warp one of the 15 pairs of row and key (one round of loads), then a thread each row.
template <bool F16>
__device__ __forceinline__ void first_rows(const PreParams& p) {
  __shared__ float s_qk[16], s_dov[16];
  const long long bh = blockIdx.x, b = bh / p.H;
  const int h = (int)(bh % p.H), pair = threadIdx.x >> 4, chunk = threadIdx.x & 15;
  int pos = 0;
  while ((pos + 1) * (pos + 2) / 2 <= pair) ++pos;
  const int j = pair - pos * (pos + 1) / 2, behind = p.behind(b);
  float qk = 0.f, dov = 0.f;
  if (pos < kFewKeys && pos >= p.base && pos - p.base < behind && chunk * 8 < p.D) {
    qk = dot16<F16>(load16(p.q, p.q_stride, b, h, pos - p.base, chunk), load16(p.k, p.k_stride, b, h / p.G, j, chunk));
    dov = dot16<F16>(load16(p.d_o, p.do_stride, b, h, pos - p.base, chunk), load16(p.v, p.v_stride, b, h / p.G, j, chunk));
  }
  qk = sum16(qk);
  dov = sum16(dov);
  if (chunk == 0) {
    s_qk[pair] = qk;
    s_dov[pair] = dov;
  }
  __syncthreads();
  pos = threadIdx.x;
  const int s = pos - p.base;
  if (pos >= kFewKeys || s < 0 || s >= p.SqPad) return;
  float acc = 0.f, l = -INFINITY;
  if (s < behind) {
    l = p.lse[bh * p.Sq + s] * kLog2e;
    for (int key = 0; key <= pos; ++key) {
      const int e = pos * (pos + 1) / 2 + key;
      if (l != -INFINITY) acc = fmaf(ex2_approx(fmaf(s_qk[e], p.scale_log2, -l)), s_dov[e], acc);
    }
  }
  p.delta[bh * p.SqPad + s] = -acc;
  p.lse_log2[bh * p.SqPad + s] = l == -INFINITY ? -INFINITY : -l;
}

template <bool F16>
__global__ void __launch_bounds__(256)
window_bwd_pre_kernel(const PreParams p) {
  if ((int)blockIdx.x < p.first_blocks) {
    first_rows<F16>(p);
    return;
  }
  const long long row0 = ((long long)(blockIdx.x - p.first_blocks) * 8 + (threadIdx.x >> 5)) * 8;
  if (row0 >= p.rows_pad) return;
  const int lane = threadIdx.x & 31;
  const int sub = lane >> 4, chunk = lane & 15;
  const long long bh = row0 / p.SqPad;  // the eight rows lie in one (batch, head) plane: SqPad is a multiple of 128
  const int s0 = (int)(row0 - bh * p.SqPad);
  const int h = (int)(bh % p.H);
  const long long b = bh / p.H;
  const int first = p.first(), behind = p.behind(b), done = p.first_blocks > 0 ? kFewKeys - p.base : 0;
  uint4 ov[4], dv[4];
  float lv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = s0 + 2 * i + sub;
    const bool live = s >= first && s < behind;
    lv[i] = (live && chunk == 0) ? p.lse[bh * p.Sq + s] : -INFINITY;
    ov[i] = make_uint4(0, 0, 0, 0);
    dv[i] = make_uint4(0, 0, 0, 0);
    if (live && chunk * 8 < p.D) {
      ov[i] = load16(p.o, p.o_stride, b, h, s, chunk);
      dv[i] = load16(p.d_o, p.do_stride, b, h, s, chunk);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = s0 + 2 * i + sub;
    const float acc = sum16(dot16<F16>(ov[i], dv[i]));
    if (chunk == 0 && (s >= done || s < first)) {
      const float l = lv[i] == -INFINITY ? INFINITY : lv[i] * kLog2e;
      p.delta[bh * p.SqPad + s] = -acc;
      p.lse_log2[bh * p.SqPad + s] = -l;
    }
  }
}

// Every row, for windows that hold at most kFewKeys keys together with the sinks.
template <bool F16>
__global__ void __launch_bounds__(256)
window_bwd_pre_few_kernel(const PreParams p) {
  const long long row0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * 8;
  if (row0 >= p.rows_pad) return;
  const int lane = threadIdx.x & 31;
  const int sub = lane >> 4, chunk = lane & 15;
  const long long bh = row0 / p.SqPad;
  const int s0 = (int)(row0 - bh * p.SqPad);
  const int h = (int)(bh % p.H);
  const long long b = bh / p.H;
  const int first = p.first(), behind = p.behind(b);
  uint4 qv[4], dv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = s0 + 2 * i + sub;
    qv[i] = make_uint4(0, 0, 0, 0);
    dv[i] = make_uint4(0, 0, 0, 0);
    if (s >= first && s < behind && chunk * 8 < p.D) {
      qv[i] = load16(p.q, p.q_stride, b, h, s, chunk);
      dv[i] = load16(p.d_o, p.do_stride, b, h, s, chunk);
    }
  }
  // The dot products of four rows are summed over the sixteen lanes together, each exchange halving the values a lane
  // carries: q k and dO v of row `own` end at the lanes whose chunk has its bits 3 and 2.
  const int own = chunk >> 2, s_own = s0 + 2 * own + sub, p_own = p.base + s_own;
  const float l_own = s_own >= first && s_own < behind ? p.lse[bh * p.Sq + s_own] * kLog2e : -INFINITY;
  auto key = [&](int pos, int t) { return t < p.window ? pos - t : t - p.window; };
  auto sees = [&](int pos, int t, int j) { return j >= 0 && (t < p.window || j <= pos - p.window); };
  float acc = 0.f;
#pragma unroll 1
  for (int t = 0; t < p.window + p.sinks; ++t) {
    float d[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = s0 + 2 * i + sub, j = key(p.base + row, t);
      d[2 * i] = d[2 * i + 1] = 0.f;
      if (row < behind && sees(p.base + row, t, j) && chunk * 8 < p.D) {
        d[2 * i] = dot16<F16>(qv[i], load16(p.k, p.k_stride, b, h / p.G, j, chunk));
        d[2 * i + 1] = dot16<F16>(dv[i], load16(p.v, p.v_stride, b, h / p.G, j, chunk));
      }
    }
#pragma unroll
    for (int n = 4; n > 0; n >>= 1) {  // n values are left; lanes whose bit 2n is set keep the upper ones
      const bool upper = (chunk & (2 * n)) != 0;
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const float got = __shfl_xor_sync(0xffffffffu, upper ? d[e] : d[e + n], 2 * n);
        d[e] = (upper ? d[e + n] : d[e]) + got;
      }
    }
    d[0] += __shfl_xor_sync(0xffffffffu, d[0], 1);
    const float other = __shfl_xor_sync(0xffffffffu, d[0], 2);
    const float qk = (chunk & 2) ? other : d[0], dov = (chunk & 2) ? d[0] : other;
    if (l_own != -INFINITY && sees(p_own, t, key(p_own, t))) acc = fmaf(ex2_approx(fmaf(qk, p.scale_log2, -l_own)), dov, acc);
  }
  if ((chunk & 3) == 0) {
    p.delta[bh * p.SqPad + s_own] = -acc;
    p.lse_log2[bh * p.SqPad + s_own] = l_own == -INFINITY ? -INFINITY : -l_own;
  }
}

// ------------------------------------------------------------------------------------------------
// 2. dQ kernel
// ------------------------------------------------------------------------------------------------
// smem: Q | dO | ring of 5 tiles (K_0, V_0, K_1, V_1, ...) | barriers.  Tensor memory: S @0, dP / dS buffers @128 and
// @256 (dS overwrites the head of each group's half), dQ @384.  S_{j+1} is issued once every compute thread holds S_j
// in registers and dP_{j+1} goes to the buffer that dQ_{j-1} has finished reading, so both run under the arithmetic of
// iteration j.
constexpr int kDqStages = 5;
constexpr int kDqSmem = (2 + kDqStages) * kTile + kBarBytes;

struct DqItem {
  int b, h, m, len, base, p_lo, p_hi;
  TileList tiles;
};
__device__ __forceinline__ DqItem dq_item(const Params& p, int w) {
  DqItem t;
  const Dealt d = deal_item(w, p.B * p.Hq, p.Nq, p.dq_group);
  t.m = p.Nq - 1 - d.rank;  // (the last ones have the longest lists)
  t.h = d.column % p.Hq;
  t.b = d.column / p.Hq;
  t.len = seq_len(p, t.b);
  t.base = p.Sk - p.Sq;
  t.p_lo = t.base + t.m * 128;
  t.p_hi = t.base + min(p.Sq, t.m * 128 + 128) - 1;
  t.tiles = window_tiles(t.p_lo, t.p_hi, t.len, p.window, p.sinks);
  return t;
}

template <bool F16>
__global__ void __launch_bounds__(kDqThreads, 1)
window_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  constexpr int NS = kDqStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sQ = smem_raw;
  uint8_t* sdO = sQ + kTile;
  uint8_t* sRing = sdO + kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRing + NS * kTile);
  uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(bars + 32);
  volatile int& s_abort = *reinterpret_cast<volatile int*>(bars + 33);
  if ((smem_u32(smem_raw) & 1023u) != 0) {
    if (threadIdx.x == 0 && atomicCAS(p.status, 0, (int)kStatusBadIndex) == 0) p.status[2] = 995;
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the dK/dV kernel may start where an SM is free
  const uint32_t bar_base = smem_u32(bars);
  auto BAR = [&](int i) { return bar_base + (uint32_t)i * 8u; };
  constexpr int kRFull = 0, kREmpty = NS, kQFull = 2 * NS, kQEmpty = kQFull + 1, kDoFull = kQEmpty + 1,
                kDoEmpty = kDoFull + 1, kSFull = kDoEmpty + 1, kSFree = kSFull + 1, kDpFull = kSFree + 1,
                kDsFull = kDpFull + 2, kDsUsed = kDsFull + 2, kDqFinal = kDsUsed + 2, kDqFree = kDqFinal + 1,
                kNumBars = kDqFree + 1;
  static_assert(kNumBars <= 32, "barrier slots");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WaitCtx wctx{&s_abort, p.status};
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < NS; ++i) {
      mbar_init(BAR(kRFull + i), 1);
      mbar_init(BAR(kREmpty + i), 3);  // released once by each issuing warp
    }
    mbar_init(BAR(kQFull), 1);
    mbar_init(BAR(kQEmpty), 1);
    mbar_init(BAR(kDoFull), 1);
    mbar_init(BAR(kDoEmpty), 1);
    mbar_init(BAR(kSFull), 1);
    mbar_init(BAR(kSFree), 8);  // (one arrival a warp: those of its lanes are taken in turn)
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(kDpFull + i), 1);
      mbar_init(BAR(kDsFull + i), 8);
      mbar_init(BAR(kDsUsed + i), 1);
    }
    mbar_init(BAR(kDqFinal), 1);
    mbar_init(BAR(kDqFree), 8);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  const uint32_t tS = tmem, tdP = tmem + 128u, tdQ = tmem + 384u;
  const int num_work = p.B * p.Hq * p.Nq;

  if (warp == kDqLoadWarp) {
    uint32_t r_cnt = 0, tile_cnt = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const DqItem t = dq_item(p, w);
      const int n = t.tiles.n;
      if (n == 0) continue;
      for (int which = 0; which < 2 && ok; ++which) {  // Q, dO
        const int full = which ? kDoFull : kQFull, empty = which ? kDoEmpty : kQEmpty;
        ok = mbar_wait(BAR(empty), (tile_cnt & 1) ^ 1, wctx, 400);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(BAR(full), kTile);
          const CUtensorMap* tm = which ? &tm_do : &tm_q;
          for (int sl = 0; sl < 2; ++sl)
            tma_load_4d(smem_u32((which ? sdO : sQ) + sl * kSlab), tm, BAR(full), sl * 64, t.m * 128, t.h, t.b);
        }
      }
      ++tile_cnt;
      for (int j = 0; j < n && ok; ++j) {
        const int row = t.tiles.tile(j) * 128;
        for (int which = 0; which < 2 && ok; ++which) {
          const uint32_t stage = r_cnt % NS, ph = (r_cnt / NS) & 1;
          ok = mbar_wait(BAR(kREmpty + stage), ph ^ 1, wctx, 401);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(BAR(kRFull + stage), kTile);
            const CUtensorMap* tm = which ? &tm_v : &tm_k;
            for (int sl = 0; sl < 2; ++sl)
              tma_load_4d(smem_u32(sRing + stage * kTile + sl * kSlab), tm, BAR(kRFull + stage), sl * 64, row,
                          t.h / p.G, t.b);
          }
          ++r_cnt;
        }
      }
    }
  } else if (warp >= kMmaWarp && warp < kMmaWarp + 3) {
    // issuer 0: S_j = Q K_j^T;  issuer 1: dQ += dS_j K_j;  issuer 2: dP_j = dO V_j^T.  All three visit every ring
    // position in order and release every stage once.
    const int who = warp - kMmaWarp;
    uint32_t r_cnt = 0, free_cnt = 0, s_issued = 0, dp_issued = 0, ds_seen = 0, tile_cnt = 0;
    bool ok = true;
    bool first_tile = true;
    const uint32_t led = lane == 0;
    const uint64_t ring_k = desc_k_major(smem_u32(sRing)), ring_mn = desc_mn_major(smem_u32(sRing));
    const int ksteps = p.D / 16;
    const uint32_t idesc_n = Idesc<F16>::kmn(p.D);
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const int n = dq_item(p, w).tiles.n;
      if (n == 0) continue;
      const uint32_t base = r_cnt;  // K_j at base + 2j, V_j at base + 2j + 1
      auto stage_of = [&](uint32_t pos) { return pos % NS; };
      auto wait_full = [&](uint32_t pos) { return mbar_wait(BAR(kRFull + stage_of(pos)), (pos / NS) & 1, wctx, 411); };
      auto pass = [&](uint32_t pos) {  // a tile this issuer does not read
        if (!wait_full(pos)) return false;
        if (led) mbar_arrive(BAR(kREmpty + stage_of(pos)));
        __syncwarp();
        return true;
      };
      if (who == 0) {
        ok = mbar_wait(BAR(kQFull), tile_cnt & 1, wctx, 410);
        const uint64_t q_desc = desc_k_major(smem_u32(sQ));
        for (int j = 0; j < n && ok; ++j) {
          ok = wait_full(base + 2 * j);
          if (!ok) break;
          if (s_issued > 0) {  // the previous S is in the registers of every compute thread
            ok = mbar_wait(BAR(kSFree), (s_issued - 1) & 1, wctx, 414);
            if (!ok) break;
          }
          ++s_issued;
          tc_fence_after();
          const uint32_t sk = stage_of(base + 2 * j);
          mma_ss_kk<F16>(tS, q_desc, ring_k + sk * kTileStep, led, ksteps);
          umma_commit_led(BAR(kSFull), led);
          umma_commit_led(BAR(kREmpty + sk), led);
          if (j == n - 1) umma_commit_led(BAR(kQEmpty), led);
          __syncwarp();
          ok = pass(base + 2 * j + 1);
        }
        if (!ok) break;
      } else if (who == 2) {
        ok = mbar_wait(BAR(kDoFull), tile_cnt & 1, wctx, 416);
        const uint64_t do_desc = desc_k_major(smem_u32(sdO));
        for (int j = 0; j < n && ok; ++j) {
          ok = pass(base + 2 * j);
          if (ok) ok = wait_full(base + 2 * j + 1);
          if (!ok) break;
          const uint32_t buf = dp_issued & 1;
          if (dp_issued >= 2) {  // dS of two iterations back has been read from this buffer
            ok = mbar_wait(BAR(kDsUsed + buf), ((dp_issued >> 1) - 1) & 1, wctx, 415);
            if (!ok) break;
          }
          ++dp_issued;
          tc_fence_after();
          const uint32_t sv = stage_of(base + 2 * j + 1);
          mma_ss_kk<F16>(tdP + buf * 128u, do_desc, ring_k + sv * kTileStep, led, ksteps);
          umma_commit_led(BAR(kDpFull + buf), led);
          umma_commit_led(BAR(kREmpty + sv), led);
          if (j == n - 1) umma_commit_led(BAR(kDoEmpty), led);
          __syncwarp();
        }
        if (!ok) break;
      } else {
        for (int j = 0; j < n && ok; ++j) {
          ok = wait_full(base + 2 * j);
          if (ok) ok = pass(base + 2 * j + 1);
          if (!ok) break;
          const uint32_t buf = ds_seen & 1;
          ok = mbar_wait(BAR(kDsFull + buf), (ds_seen >> 1) & 1, wctx, 412);
          if (!ok) break;
          ++ds_seen;
          if (j == 0 && !first_tile) {  // the previous tile's epilogue has drained dQ
            ok = mbar_wait(BAR(kDqFree), free_cnt & 1, wctx, 413);
            if (!ok) break;
            ++free_cnt;
          }
          tc_fence_after();
          const uint32_t sk = stage_of(base + 2 * j);
          const uint32_t t = tdP + buf * 128u;
          mma_ts_kmn(tdQ, t, t + 64u, ring_mn + sk * kTileStep, j > 0, led, idesc_n);
          umma_commit_led(BAR(kDsUsed + buf), led);
          umma_commit_led(BAR(kREmpty + sk), led);
          __syncwarp();
        }
        if (!ok) break;
        umma_commit_led(BAR(kDqFinal), led);
        __syncwarp();
      }
      r_cnt += 2 * n;
      ++tile_cnt;
      first_tile = false;
    }
  } else if (warp < 8) {
    const int grp = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s_cnt = 0, dp_cnt = 0, fin_cnt = 0, r_cnt = 0;
    bool ok = true;
    const int cols = p.D - grp * 64;  // output columns of this group (<= 0: none)
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const DqItem t = dq_item(p, w);
      const int n = t.tiles.n;
      const int seq = t.m * 128 + row, pos = t.base + seq;
      const bool live = seq < p.Sq && pos >= 0 && pos < t.len;
      uint8_t* dq_row = p.dq + (t.b * p.dq_stride[0] + t.h * p.dq_stride[1] + (long long)seq * p.dq_stride[2] + grp * 64) * 2;
      uint32_t acc[64];
      if (n > 0) {
        const long long srow = ((long long)t.b * p.Hq + t.h) * ((long long)p.Nq * 128) + seq;
        const float nlse = p.lse_log2[srow], ndlt = p.delta[srow];
        const uint64_t sc2 = pack2(p.scale_log2, p.scale_log2), nl2 = pack2(nlse, nlse), nd2 = pack2(ndlt, ndlt);
        // every row of the tile sees all keys of [free_lo, free_hi)
        const int free_lo = min(t.p_hi, t.len - 1) - p.window + 1, free_hi = t.p_lo + 1;
        for (int j = 0; j < n && ok; ++j) {
          const int j0 = t.tiles.tile(j) * 128;
          const bool whole = j0 >= free_lo && j0 + 128 <= free_hi;
          ok = mbar_wait(BAR(kSFull), s_cnt & 1, wctx, 420);
          if (!ok) break;
          ++s_cnt;
          tc_fence_after();
          const uint32_t buf = dp_cnt & 1;
          const uint32_t t_s = tS + lane_base + grp * 64, t_g = tdP + buf * 128u + lane_base + grp * 64;
          // one body for whole tiles, one for masked ones (the dK/dV kernel's has the times)
          auto tile = [&](auto masked) -> bool {
            constexpr bool kMasked = decltype(masked)::value;
            float pr[64];
            {
              uint32_t* u = reinterpret_cast<uint32_t*>(pr);
              tmem_ld32(t_s, u);
              tmem_ld32(t_s + 32, u + 32);
              tmem_wait_ld();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(kSFree));  // S_j is in registers: the next S may be computed
            const bool tail = kMasked && (j0 + 128 > t.len || p.holds_unseen(j0));
            if (tail) {  // K rows that no query sees may hold anything, and dQ contracts over them (S_j has read the tile)
              if (j0 + row >= t.len || p.unseen(j0 + row)) {
                uint4* k0 = reinterpret_cast<uint4*>(sRing + ((r_cnt + 2u * j) % NS) * kTile + grp * kSlab + row * 128);
#pragma unroll
                for (int c = 0; c < 8; ++c) k0[c] = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
            }
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              float x0, x1;
              unpack2(ffma2(pack2(pr[c], pr[c + 1]), sc2, nl2), x0, x1);
              pr[c] = ex2_approx(x0);
              pr[c + 1] = ex2_approx(x1);
            }
            uint32_t mw[2];
            if (kMasked) {
              const int c0 = j0 + grp * 64;
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mw[h] = live ? range_word(pos - p.window + 1 - c0, pos + 1 - c0, h) | low_bits(min(p.sinks, pos + 1) - c0 - 32 * h) : 0u;
#pragma unroll
              for (int c = 0; c < 64; ++c) pr[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? pr[c] : 0.f;
            }
            if (!mbar_wait(BAR(kDpFull + buf), (dp_cnt >> 1) & 1, wctx, 421)) return false;
            tc_fence_after();
            uint32_t dp[64];
            tmem_ld32(t_g, dp);
            tmem_ld32(t_g + 32, dp + 32);
            tmem_wait_ld();
            if (tail) {  // (such V rows: 0 * NaN is NaN)
#pragma unroll
              for (int c = 0; c < 64; ++c) dp[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? dp[c] : 0u;
            }
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float d0, d1;
              unpack2(fmul2(pack2(pr[2 * e], pr[2 * e + 1]),
                            fadd2(pack2(__uint_as_float(dp[2 * e]), __uint_as_float(dp[2 * e + 1])), nd2)), d0, d1);
              pk[e] = pack16<F16>(d0, d1);
            }
            tmem_st32(t_g, pk);
            return true;
          };
          ok = whole ? tile(std::false_type{}) : tile(std::true_type{});
          if (!ok) break;
          ++dp_cnt;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(kDsFull + buf));
        }
        if (!ok) break;
        r_cnt += 2 * n;
        ok = mbar_wait(BAR(kDqFinal), fin_cnt & 1, wctx, 422);
        if (!ok) break;
        ++fin_cnt;
        tc_fence_after();
        tmem_ld32(tdQ + lane_base + grp * 64, acc);
        tmem_ld32(tdQ + lane_base + grp * 64 + 32, acc + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kDqFree));
      }
      if (n == 0 || !live) {  // takes no part
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[c] = 0u;
      }
      store_half<F16>(dq_row, seq < p.Sq, acc, p.softmax_scale, cols);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------
// 3. dK/dV kernel
// ------------------------------------------------------------------------------------------------
// smem: K | V | ring of 5 tiles (Q_i, dO_i alternating) | row statistics [2][2][128] f32 | barriers.  Tensor memory:
// S @0 takes S^T_i; G @128 takes dP^T_i and then P^T_i (16 bits, first 32 of a thread's 64 columns) and dS^T_i (last
// 32), the operands of dV @256 += P^T dO and dK @384 += dS^T Q.
constexpr int kDkvStages = 5;
constexpr int kStatSlots = 2;
constexpr int kDkvSmem = 2 * kTile + kDkvStages * kTile + kStatSlots * 1024 + kBarBytes;

struct DkvItem {
  int b, hkv, nb;
  int slot;    // workspace slot of the sink rows' sums (PARTS: of every row's); -1: every row is stored directly
  bool extra;  // an item of the sinks only
  int f0, m0, nm, T;  // pair i: f = f0 + i, query head f / nm of the group, query tile m0 + f % nm
  int len, base;
};
template <bool PARTS>
__device__ __forceinline__ DkvItem dkv_item(const Params& p, int w) {
  DkvItem t;
  if (PARTS) {
    t.slot = w % p.parts;
    w /= p.parts;
    t.nb = w % p.Nkv;
    t.hkv = (w / p.Nkv) % p.Hkv;
    t.b = w / (p.Nkv * p.Hkv);
    t.extra = false;
    t.len = seq_len(p, t.b);
    t.base = p.Sk - p.Sq;
    t.f0 = t.m0 = t.T = 0;
    t.nm = 1;
    const int last = min(p.Sq, t.len - t.base) - 1;  // last query token that takes part
    const int first = max(0, t.nb * 128 - t.base);
    const int reach = (t.nb == 0 && p.sinks > 0) ? last : min(last, t.nb * 128 + 127 + p.window - 1 - t.base);
    if (t.nb * 128 < t.len && first <= reach) {
      t.m0 = first >> 7;
      t.nm = (reach >> 7) - t.m0 + 1;
      const int all = p.G * t.nm;
      t.f0 = (int)((long long)all * t.slot / p.parts);
      t.T = (int)((long long)all * (t.slot + 1) / p.parts) - t.f0;
    }
    return t;
  }
  const int extras = p.B * p.Hkv * p.sink_items;
  int bh, chunk = 0;
  t.extra = w < extras;
  if (t.extra) {
    chunk = w % p.sink_items;
    bh = w / p.sink_items;
    t.nb = 0;
    t.slot = 1 + chunk;
  } else {
    const Dealt d = deal_item(w - extras, p.B * p.Hkv, p.Nkv, p.dkv_group);
    t.nb = d.rank;  // (the first ones have the longest lists)
    bh = d.column;
    t.slot = (t.nb == 0 && p.sink_items > 0) ? 0 : -1;
  }
  t.hkv = bh % p.Hkv;
  t.b = bh / p.Hkv;
  t.len = seq_len(p, t.b);
  t.base = p.Sk - p.Sq;
  t.f0 = t.m0 = t.T = 0;
  t.nm = 1;
  const int last = min(p.Sq, t.len - t.base) - 1;  // last query token that takes part
  if (t.extra) {
    const int nm = last < 0 ? 0 : (last >> 7) + 1 - p.sink_m0;
    if (nm > 0) {
      t.nm = nm;
      t.m0 = p.sink_m0;
      const int all = p.G * nm;
      t.f0 = (int)((long long)all * chunk / p.sink_items);
      t.T = (int)((long long)all * (chunk + 1) / p.sink_items) - t.f0;
    }
  } else {
    const int first = max(0, t.nb * 128 - t.base);
    const int reach = min(last, t.nb * 128 + 127 + p.window - 1 - t.base);
    if (t.nb * 128 < t.len && first <= reach) {
      t.m0 = first >> 7;
      t.nm = (reach >> 7) - t.m0 + 1;
      t.T = p.G * t.nm;
    }
  }
  return t;
}

template <bool F16, bool PARTS>
__global__ void __launch_bounds__(kDkvThreads, 1)
window_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                  const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  constexpr int NS = kDkvStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sK = smem_raw;
  uint8_t* sV = sK + kTile;
  uint8_t* sRing = sV + kTile;
  float* sStats = reinterpret_cast<float*>(sRing + NS * kTile);  // [slot][0: lse_log2, 1: delta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStats) + kStatSlots * 1024);
  uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(bars + 32);
  volatile int& s_abort = *reinterpret_cast<volatile int*>(bars + 33);
  if ((smem_u32(smem_raw) & 1023u) != 0) {
    if (threadIdx.x == 0 && atomicCAS(p.status, 0, (int)kStatusBadIndex) == 0) p.status[2] = 994;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const uint32_t bar_base = smem_u32(bars);
  auto BAR = [&](int i) { return bar_base + (uint32_t)i * 8u; };
  constexpr int kKFull = 0, kKEmpty = 1, kVFull = 2, kVEmpty = 3, kRFull = 4, kREmpty = 4 + NS, kSFull = 4 + 2 * NS, kSFree = kSFull + 1,
                kDpFull = kSFree + 1, kPFull = kDpFull + 1, kDsFull = kPFull + 1, kGFree = kDsFull + 1,
                kFinal = kGFree + 1, kFree = kFinal + 1, kNumBars = kFree + 1;
  static_assert(kNumBars <= 32, "barrier slots");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WaitCtx wctx{&s_abort, p.status};
  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(BAR(kKFull), 1);
    mbar_init(BAR(kKEmpty), 1);
    mbar_init(BAR(kVFull), 1);
    mbar_init(BAR(kVEmpty), 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(BAR(kRFull + i), 1);
      mbar_init(BAR(kREmpty + i), 2);
    }
    mbar_init(BAR(kSFull), 1);
    mbar_init(BAR(kDpFull), 1);
    mbar_init(BAR(kSFree), 8);
    mbar_init(BAR(kPFull), 8);
    mbar_init(BAR(kDsFull), 8);
    mbar_init(BAR(kGFree), 1);
    mbar_init(BAR(kFinal), 2);
    mbar_init(BAR(kFree), 8);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  const uint32_t tS = tmem, tG = tmem + 128u, tdV = tmem + 256u, tdK = tmem + 384u;
  const int num_work = PARTS ? p.B * p.Hkv * p.Nkv * p.parts : p.B * p.Hkv * (p.Nkv + p.sink_items);

  if (warp == kDkvLoadWarp) {
    uint32_t r_cnt = 0, kv_cnt = 0, tile_cnt = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const DkvItem t = dkv_item<PARTS>(p, w);
      if (t.T == 0) continue;
      // K is read by S^T only and V by dP^T only: each is replaced as soon as the item before has issued its last one
      for (int which = 0; which < 2 && ok; ++which) {
        const int full = which ? kVFull : kKFull, empty = which ? kVEmpty : kKEmpty;
        ok = mbar_wait(BAR(empty), (kv_cnt & 1) ^ 1, wctx, 500);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(BAR(full), kTile);
          for (int sl = 0; sl < 2; ++sl)
            tma_load_4d(smem_u32((which ? sV : sK) + sl * kSlab), which ? &tm_v : &tm_k, BAR(full), sl * 64, t.nb * 128,
                        t.hkv, t.b);
        }
      }
      if (!ok) break;
      ++kv_cnt;
      for (int i = 0; i < t.T && ok; ++i) {
        const int f = t.f0 + i;
        const int hq = t.hkv * p.G + f / t.nm, m = t.m0 + f % t.nm;
        for (int which = 0; which < 2; ++which) {
          const uint32_t stage = r_cnt % NS, ph = (r_cnt / NS) & 1;
          ok = mbar_wait(BAR(kREmpty + stage), ph ^ 1, wctx, 501);
          if (!ok) break;
          if (lane == 0) {
            const CUtensorMap* tm = which ? &tm_do : &tm_q;
            mbar_arrive_expect_tx(BAR(kRFull + stage), kTile + (which ? 1024 : 0));
            for (int sl = 0; sl < 2; ++sl)
              tma_load_4d(smem_u32(sRing + stage * kTile + sl * kSlab), tm, BAR(kRFull + stage), sl * 64, m * 128, hq, t.b);
            if (which) {
              // the rows' statistics travel with their dO tile: its stage is re-used only after dK of the tile two
              // back, when the statistics slot of that tile is long free (two slots)
              float* st = sStats + (tile_cnt % kStatSlots) * 256;
              const long long at = ((long long)t.b * p.Hq + hq) * ((long long)p.Nq * 128) + (long long)m * 128;
              bulk_load_1d(smem_u32(st), p.lse_log2 + at, 512, BAR(kRFull + stage));
              bulk_load_1d(smem_u32(st + 128), p.delta + at, 512, BAR(kRFull + stage));
            }
          }
          ++r_cnt;
        }
        ++tile_cnt;
      }
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // issuer 0: S^T_i = K Q_i^T one tile ahead of the compute threads, and dV += P^T_i dO_i;
    // issuer 1: the chain through region G: dP^T_i = V dO_i^T, dK += dS^T_i Q_i, then (once dV_i has read G) dP^T_{i+1}
    const int who = warp - kMmaWarp;
    const uint32_t led = lane == 0;
    uint32_t r_cnt = 0, kv_cnt = 0, in_cnt = 0, ds_cnt = 0, free_cnt = 0;
    bool ok = true, first_item = true;
    const uint64_t k_desc = desc_k_major(smem_u32(sK)), v_desc = desc_k_major(smem_u32(sV));
    const uint64_t ring_k = desc_k_major(smem_u32(sRing)), ring_mn = desc_mn_major(smem_u32(sRing));
    const int ksteps = p.D / 16;
    const uint32_t idesc_n = Idesc<F16>::kmn(p.D);
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const int T = dkv_item<PARTS>(p, w).T;
      if (T == 0) continue;
      ok = mbar_wait(BAR(who == 0 ? kKFull : kVFull), kv_cnt & 1, wctx, 510);
      if (!ok) break;
      ++kv_cnt;
      const uint32_t base = r_cnt;  // Q_i at base + 2i, dO_i at base + 2i + 1
      auto stage_of = [&](uint32_t pos) { return pos % NS; };
      auto wait_full = [&](uint32_t pos) { return mbar_wait(BAR(kRFull + stage_of(pos)), (pos / NS) & 1, wctx, 511); };
      auto wait_free = [&]() -> bool {  // the previous item's epilogue has drained the accumulators
        if (first_item) return true;
        const bool r = mbar_wait(BAR(kFree), free_cnt & 1, wctx, 515);
        ++free_cnt;
        return r;
      };
      if (who == 0) {
        auto issue_st = [&](int i) -> bool {
          if (!wait_full(base + 2 * i)) return false;
          if (in_cnt > 0 && !mbar_wait(BAR(kSFree), (in_cnt - 1) & 1, wctx, 512)) return false;
          ++in_cnt;
          tc_fence_after();
          const uint32_t sq = stage_of(base + 2 * i);
          mma_ss_kk<F16>(tS, k_desc, ring_k + sq * kTileStep, led, ksteps);
          umma_commit_led(BAR(kSFull), led);
          umma_commit_led(BAR(kREmpty + sq), led);
          if (i == T - 1) umma_commit_led(BAR(kKEmpty), led);
          __syncwarp();
          return true;
        };
        ok = issue_st(0);
        for (int i = 0; i < T && ok; ++i) {
          if (i + 1 < T) ok = issue_st(i + 1);
          if (ok) ok = wait_full(base + 2 * i + 1);
          if (!ok) break;
          ok = mbar_wait(BAR(kPFull), ds_cnt & 1, wctx, 513);
          ++ds_cnt;
          if (ok && i == 0) ok = wait_free();
          if (!ok) break;
          tc_fence_after();
          const uint32_t sd = stage_of(base + 2 * i + 1);
          mma_ts_kmn(tdV, tG, tG + 64u, ring_mn + sd * kTileStep, i > 0, led, idesc_n);
          umma_commit_led(BAR(kREmpty + sd), led);
          umma_commit_led(BAR(kGFree), led);
          __syncwarp();
        }
      } else {
        auto issue_dp = [&](int i) -> bool {
          if (!wait_full(base + 2 * i)) return false;
          if (!wait_full(base + 2 * i + 1)) return false;
          const uint32_t sd = stage_of(base + 2 * i + 1);
          mma_ss_kk<F16>(tG, v_desc, ring_k + sd * kTileStep, led, ksteps);
          umma_commit_led(BAR(kDpFull), led);
          umma_commit_led(BAR(kREmpty + sd), led);
          if (i == T - 1) umma_commit_led(BAR(kVEmpty), led);
          __syncwarp();
          return true;
        };
        ok = issue_dp(0);
        for (int i = 0; i < T && ok; ++i) {
          ok = mbar_wait(BAR(kDsFull), ds_cnt & 1, wctx, 514);
          ++ds_cnt;
          if (ok && i == 0) ok = wait_free();
          if (!ok) break;
          tc_fence_after();
          const uint32_t sq = stage_of(base + 2 * i);
          mma_ts_kmn(tdK, tG + 32u, tG + 96u, ring_mn + sq * kTileStep, i > 0, led, idesc_n);
          umma_commit_led(BAR(kREmpty + sq), led);
          __syncwarp();
          ok = mbar_wait(BAR(kGFree), in_cnt & 1, wctx, 516);  // dV_i has read region G as well
          ++in_cnt;
          if (ok && i + 1 < T) ok = issue_dp(i + 1);
        }
      }
      if (!ok) break;
      umma_commit_led(BAR(kFinal), led);
      __syncwarp();
      r_cnt += 2 * T;
      first_item = false;
    }
  } else if (warp < 8) {
    const int grp = warp >> 2;
    const int row = threadIdx.x & 127;  // key inside the tile = tensor-memory lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s_cnt = 0, dp_cnt = 0, fin_cnt = 0, tile_cnt = 0, r_cnt = 0;
    const uint64_t sc2 = pack2(p.scale_log2, p.scale_log2);
    const int cols = p.D - grp * 64;
    bool ok = true;
    for (int w = blockIdx.x; w < num_work && ok; w += gridDim.x) {
      const DkvItem t = dkv_item<PARTS>(p, w);
      const uint32_t base = r_cnt;
      r_cnt += 2 * t.T;
      const int kv = t.nb * 128 + row;
      // query positions [kv, see_hi) see this key
      const int see_hi = kv < p.sinks ? t.len : min(t.len, kv + p.window);
      int m = t.m0 + t.f0 % t.nm;
      for (int i = 0; i < t.T && ok; ++i) {
        const float4* st_l = reinterpret_cast<const float4*>(sStats + (tile_cnt % kStatSlots) * 256 + grp * 64);
        const float4* st_d = reinterpret_cast<const float4*>(sStats + (tile_cnt % kStatSlots) * 256 + 128 + grp * 64);
        ++tile_cnt;
        const int p0 = t.base + m * 128;  // position of the query tile's first row
        if (++m == t.m0 + t.nm) m = t.m0;
        const bool whole = p0 >= t.nb * 128 + 127 && p0 + 127 < t.len && p0 + 127 < t.nb * 128 + p.window;
        ok = mbar_wait(BAR(kSFull), s_cnt & 1, wctx, 520);
        if (!ok) break;
        ++s_cnt;
        const uint32_t pos = base + 2 * (uint32_t)i + 1;  // dO_i, whose barrier also brings the statistics
        ok = mbar_wait(BAR(kRFull + pos % NS), (pos / NS) & 1, wctx, 523);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = tS + lane_base + grp * 64, t_g = tG + lane_base + grp * 64;
        // One body for whole tiles and one for masked ones: with the masked body for every tile, here and in the dQ kernel, 16
        // heads of 16384 tokens, window 1024, take 740 us for the backward instead of 685.
        auto tile = [&](auto masked) -> bool {
          constexpr bool kMasked = decltype(masked)::value;
          float pr[64];
          {
            uint32_t* u = reinterpret_cast<uint32_t*>(pr);
            tmem_ld32(t_s, u);
            tmem_ld32(t_s + 32, u + 32);
            tmem_wait_ld();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(kSFree));
#pragma unroll
          for (int c4 = 0; c4 < 16; ++c4) {
            const float4 l = st_l[c4];  // negated
            float x0, x1, x2, x3;
            unpack2(ffma2(pack2(pr[c4 * 4 + 0], pr[c4 * 4 + 1]), sc2, pack2(l.x, l.y)), x0, x1);
            unpack2(ffma2(pack2(pr[c4 * 4 + 2], pr[c4 * 4 + 3]), sc2, pack2(l.z, l.w)), x2, x3);
            pr[c4 * 4 + 0] = ex2_approx(x0);
            pr[c4 * 4 + 1] = ex2_approx(x1);
            pr[c4 * 4 + 2] = ex2_approx(x2);
            pr[c4 * 4 + 3] = ex2_approx(x3);
          }
          uint32_t mw[2];
          if (kMasked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) mw[h] = range_word(kv - p0 - grp * 64, see_hi - p0 - grp * 64, h);
#pragma unroll
            for (int c = 0; c < 64; ++c) pr[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? pr[c] : 0.f;
          }
          if (!mbar_wait(BAR(kDpFull), dp_cnt & 1, wctx, 521)) return false;
          tc_fence_after();
          // rows that take no part may hold anything: the query tile or the key tile reaches behind the end, or holds keys that
          // no query sees
          const bool tail = kMasked && (p0 < 0 || p0 + 127 >= t.len || t.nb * 128 + 127 >= t.len || p.holds_unseen(t.nb * 128));
          if (kMasked) {
            if (tail) {
              // query rows that take no part: dV contracts over the dO rows and dK over the Q rows (both tiles have been
              // read by S^T_i and dP^T_i; their stages are held until dV_i and dK_i)
              const int at = p0 + row;
              if (at < 0 || at >= t.len) {
                uint4* z0 = reinterpret_cast<uint4*>(sRing + (pos % NS) * kTile + grp * kSlab + row * 128);
                uint4* z1 = reinterpret_cast<uint4*>(sRing + ((pos - 1) % NS) * kTile + grp * kSlab + row * 128);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                  z0[c] = make_uint4(0, 0, 0, 0);
                  z1[c] = make_uint4(0, 0, 0, 0);
                }
              }
              fence_proxy_async_smem();
            }
          }
          uint32_t dp[64];
          tmem_ld32(t_g, dp);
          tmem_ld32(t_g + 32, dp + 32);
          tmem_wait_ld();
          if (tail) {  // (what dO and V hold there reaches dP^T: 0 * NaN is NaN)
#pragma unroll
            for (int c = 0; c < 64; ++c) dp[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? dp[c] : 0u;
          }
          // dP^T_i is in registers: this thread's 64 columns of region G take P^T_i (first 32) and dS^T_i (last 32)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] = pack16<F16>(pr[16 * h + 2 * e], pr[16 * h + 2 * e + 1]);
            tmem_st8(t_g + h * 8, pk);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(kPFull));
          uint32_t pk[32];
#pragma unroll
          for (int c4 = 0; c4 < 16; ++c4) {
            const float4 d = st_d[c4];  // negated
            float d0, d1, d2, d3;
            unpack2(fmul2(pack2(pr[c4 * 4 + 0], pr[c4 * 4 + 1]),
                          fadd2(pack2(__uint_as_float(dp[c4 * 4 + 0]), __uint_as_float(dp[c4 * 4 + 1])), pack2(d.x, d.y))),
                    d0, d1);
            unpack2(fmul2(pack2(pr[c4 * 4 + 2], pr[c4 * 4 + 3]),
                          fadd2(pack2(__uint_as_float(dp[c4 * 4 + 2]), __uint_as_float(dp[c4 * 4 + 3])), pack2(d.z, d.w))),
                    d2, d3);
            pk[c4 * 2] = pack16<F16>(d0, d1);
            pk[c4 * 2 + 1] = pack16<F16>(d2, d3);
          }
          tmem_st32(t_g + 32, pk);
          tmem_wait_st();
          return true;
        };
        ok = whole ? tile(std::false_type{}) : tile(std::true_type{});
        if (!ok) break;
        ++dp_cnt;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kDsFull));
      }
      if (!ok) break;
      // ---- epilogue
      const bool to_slot = PARTS || (t.slot >= 0 && row < p.sinks);
      const bool to_row = !t.extra && !to_slot && kv < p.Sk && cols > 0;
      const int slot_rows = PARTS ? 128 : p.sinks;
      float* part = p.partial;
      if (to_slot) {
        const long long bh = (long long)t.b * p.Hkv + t.hkv;
        const long long slot = PARTS ? (bh * p.Nkv + t.nb) * p.parts + t.slot : bh * (p.sink_items + 1) + t.slot;
        part += (slot * 2 * slot_rows + row) * p.D + grp * 64;
      }
      uint8_t* dk_row = p.dk + (t.b * p.dk_stride[0] + t.hkv * p.dk_stride[1] + (long long)kv * p.dk_stride[2] + grp * 64) * 2;
      uint8_t* dv_row = p.dv + (t.b * p.dv_stride[0] + t.hkv * p.dv_stride[1] + (long long)kv * p.dv_stride[2] + grp * 64) * 2;
      uint32_t acc[64];
      if (t.T > 0) {
        ok = mbar_wait(BAR(kFinal), fin_cnt & 1, wctx, 522);
        if (!ok) break;
        ++fin_cnt;
        tc_fence_after();
        tmem_ld32(tdV + lane_base + grp * 64, acc);
        tmem_ld32(tdV + lane_base + grp * 64 + 32, acc + 32);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[c] = 0u;
      }
      store_half<F16>(dv_row, to_row, acc, 1.0f, cols);
      if (to_slot) store_half_f32(part + (long long)slot_rows * p.D, acc, cols);
      if (t.T > 0) {
        __syncwarp();
        tmem_ld32(tdK + lane_base + grp * 64, acc);
        tmem_ld32(tdK + lane_base + grp * 64 + 32, acc + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kFree));
      }
      store_half<F16>(dk_row, to_row, acc, p.softmax_scale, cols);
      if (to_slot) store_half_f32(part, acc, cols);
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // (launched as the dQ kernel's dependent: what follows in the stream may rely on both having ended)
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// 4. dK and dV of the sinks: the slots' sums in order.  One thread per element.
template <bool F16>
__global__ void __launch_bounds__(256)
window_bwd_reduce_kernel(const Params p) {
  const int per = 2 * p.sinks * p.D;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)p.B * p.Hkv * per) return;
  const int e = (int)(i % per), bh = (int)(i / per);
  const int d = e % p.D, row = (e / p.D) % p.sinks, which = e / (p.D * p.sinks);
  if (row >= p.Sk) return;
  const int slots = p.sink_items + 1;
  const float* src = p.partial + (long long)bh * slots * per + e;
  float sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < slots; ++s) sum += src[(long long)s * per];
  const int hkv = bh % p.Hkv, b = bh / p.Hkv;
  const long long* st = which ? p.dv_stride : p.dk_stride;
  uint16_t* dst = reinterpret_cast<uint16_t*>(which ? p.dv : p.dk) + b * st[0] + hkv * st[1] + row * st[2] + d;
  if (!which) sum *= p.softmax_scale;
  *dst = (uint16_t)(pack16<F16>(sum, 0.f) & 0xffffu);
}

// 4. dK and dV of key tiles whose lists were cut: the parts' sums in order.  One warp per row, four channels per lane.
template <bool F16>
__global__ void __launch_bounds__(256)
window_bwd_parts_kernel(const Params p) {
  const int nb = blockIdx.x % p.Nkv, bh = blockIdx.x / p.Nkv;
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5), kv = nb * 128 + row, d = (threadIdx.x & 31) * 4;
  if (kv >= p.Sk || d >= p.D) return;
  const float* src = p.partial + (long long)blockIdx.x * p.parts * 2 * 128 * p.D + (long long)row * p.D + d;
  float4 sum[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
  for (int s = 0; s < p.parts; ++s) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float4 v = *reinterpret_cast<const float4*>(src + (long long)(2 * s + which) * 128 * p.D);
      sum[which].x += v.x;
      sum[which].y += v.y;
      sum[which].z += v.z;
      sum[which].w += v.w;
    }
  }
  const int hkv = bh % p.Hkv, b = bh / p.Hkv;
  auto store = [&](uint8_t* base, const long long* st, float4 v, float scale) {
    uint2 u;
    u.x = pack16<F16>(v.x * scale, v.y * scale);
    u.y = pack16<F16>(v.z * scale, v.w * scale);
    *reinterpret_cast<uint2*>(base + (b * st[0] + hkv * st[1] + kv * st[2] + d) * 2) = u;
  };
  store(p.dk, p.dk_stride, sum[0], p.softmax_scale);
  store(p.dv, p.dv_stride, sum[1], 1.f);
}

// How the dK/dV kernel's work is dealt.
struct Deal {
  int parts;                // few key tiles: parts of each one's list, else 0
  int sink_m0, sink_items;  // otherwise: first query tile beyond the reach of tile 0's windows, further items of tile 0
};
static Deal deal(int B, int Hq, int Hkv, int Sq, int Sk, int window, int sinks) {
  Deal r{};
  const long long Nq = (Sq + 127) / 128, Nkv = (Sk + 127) / 128, G = Hq / Hkv;
  const long long reach = 127LL + window - 1 - ((long long)Sk - Sq);
  r.sink_m0 = (int)(reach < 0 ? 0 : ((reach >> 7) + 1 < Nq ? (reach >> 7) + 1 : Nq));
  // Key tiles that leave half of the SMs or more without one are cut into as many parts as there are SMs for, where
  // that takes at least two (query head, query tile) pairs off the longest list (one takes about 3 us, the pass over the
  // parts 4).  Tile 0's list is as long as the sequence then if it holds sinks.
  const long long span = ((long long)window + 127) / 128 + 1, pairs = G * (span < Nq ? span : Nq);
  const long long longest = sinks > 0 ? G * Nq : pairs;
  long long parts = kSmsForParts / (B * Hkv * Nkv);
  if (parts > longest) parts = longest;
  if (parts >= 2 && pairs - (longest + parts - 1) / parts >= 2) {
    r.parts = (int)parts;
    return r;
  }
  if (sinks <= 0 || r.sink_m0 >= Nq) return r;
  const long long beyond = G * (Nq - r.sink_m0);
  long long per = G * ((long long)window / 128 + 2);  // pairs of an ordinary item
  if (per < 16) per = 16;                             // (below that the prologue and the slot's stores show)
  const long long n = (beyond + per - 1) / per;
  r.sink_items = (int)(n > 128 ? 128 : n);
  return r;
}
static int64_t partial_floats(const Deal& d, int B, int Hkv, int Sk, int D, int sinks) {
  if (d.parts > 0) return (int64_t)B * Hkv * ((Sk + 127) / 128) * d.parts * 2 * 128 * D;
  return d.sink_items > 0 ? (int64_t)B * Hkv * (d.sink_items + 1) * 2 * sinks * D : 0;
}

template <bool F16>
static int launch(const bsa_window_bwd_args& a, Params& p, const CUtensorMap& tq, const CUtensorMap& tdo,
                  const CUtensorMap& tk, const CUtensorMap& tv, float* lse_log2, float* delta, int num_sms, cudaStream_t st) {
  static SmemAttribute dq_attribute, dkv_attribute[2];
  auto* dkv = p.parts > 0 ? window_dkv_kernel<F16, true> : window_dkv_kernel<F16, false>;
  cudaError_t e = dq_attribute.set(reinterpret_cast<const void*>(window_dq_kernel<F16>), kDqSmem);
  if (e == cudaSuccess) e = dkv_attribute[p.parts > 0].set(reinterpret_cast<const void*>(dkv), kDkvSmem);
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "bsa_window_bwd: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const long long rows_pad = (long long)p.B * p.Hq * p.Nq * 128;
  PreParams pre{};
  pre.o = static_cast<const uint8_t*>(a.out);
  pre.d_o = static_cast<const uint8_t*>(a.dout);
  pre.q = static_cast<const uint8_t*>(a.q);
  pre.k = static_cast<const uint8_t*>(a.k);
  pre.v = static_cast<const uint8_t*>(a.v);
  pre.lse = a.lse;
  pre.lse_log2 = lse_log2;
  pre.delta = delta;
  pre.kv_lens = p.kv_lens;
  for (int i = 0; i < 3; ++i) {
    pre.o_stride[i] = a.o_stride[i];
    pre.do_stride[i] = a.do_stride[i];
    pre.q_stride[i] = a.q_stride[i];
    pre.k_stride[i] = a.k_stride[i];
    pre.v_stride[i] = a.v_stride[i];
  }
  pre.rows_pad = rows_pad;
  pre.H = p.Hq;
  pre.G = p.G;
  pre.Sq = p.Sq;
  pre.SqPad = p.Nq * 128;
  pre.D = p.D;
  pre.base = p.Sk - p.Sq;
  pre.window = p.window;
  pre.sinks = p.sinks;
  pre.scale_log2 = p.scale_log2;
  const unsigned blocks = (unsigned)((rows_pad + 63) / 64);
  if (p.window <= kFewKeys - p.sinks) {
    window_bwd_pre_few_kernel<F16><<<blocks, 256, 0, st>>>(pre);
  } else {
    pre.first_blocks = pre.base < kFewKeys ? p.B * p.Hq : 0;
    window_bwd_pre_kernel<F16><<<blocks + pre.first_blocks, 256, 0, st>>>(pre);
  }
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window backward preprocess launch: %s", cudaGetErrorString(e));
  const int work_q = p.B * p.Hq * p.Nq, work_kv = p.B * p.Hkv * (p.parts > 0 ? p.Nkv * p.parts : p.Nkv + p.sink_items);
  window_dq_kernel<F16><<<work_q < num_sms ? work_q : num_sms, kDqThreads, kDqSmem, st>>>(tq, tdo, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window dQ launch: %s", cudaGetErrorString(e));
  // The dK/dV kernel does not need the dQ kernel's results: as its dependent it starts on SMs that the dQ kernel has left
  // or never used (backward of 2 heads, 4096 tokens, window 1024: 65 -> 47 us; 2 x 12 heads, 4999 tokens: 258 -> 240).
  // Not with many items: neighbouring CTAs, which share their loads in L2, would start apart (16 heads, 16384 tokens:
  // 645 -> 667 us).
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(work_kv < num_sms ? work_kv : num_sms));
  config.blockDim = dim3(kDkvThreads);
  config.dynamicSmemBytes = kDkvSmem;
  config.stream = st;
  cudaLaunchAttribute dependent = {};
  dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  dependent.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &dependent;
  config.numAttrs = work_q < 10 * num_sms ? 1 : 0;
  e = cudaLaunchKernelEx(&config, dkv, tq, tdo, tk, tv, (const Params)p);
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window dK/dV launch: %s", cudaGetErrorString(e));
  if (p.parts > 0) {
    window_bwd_parts_kernel<F16><<<dim3((unsigned)(p.B * p.Hkv * p.Nkv), 16), 256, 0, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window backward parts launch: %s", cudaGetErrorString(e));
  }
  if (p.sink_items > 0) {
    const long long n = (long long)p.B * p.Hkv * 2 * p.sinks * p.D;
    window_bwd_reduce_kernel<F16><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window backward reduce launch: %s", cudaGetErrorString(e));
  }
  return BSA_OK;
}

}  // namespace winbwd
}  // namespace bsa

using namespace bsa;

extern "C" int64_t bsa_window_bwd_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t Sq, int32_t Sk, int32_t D,
                                                  int32_t window, int32_t sinks) {
  if (B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || Sq < 1 || Sk < 1 || D < 1 || window < 1 || sinks < 0) return 0;
  const winbwd::Deal d = winbwd::deal(B, Hq, Hkv, Sq, Sk, window < kWindowAll ? window : kWindowAll, sinks);
  const int64_t rows = (int64_t)B * Hq * ((Sq + 127) / 128) * 128;
  return (2 * rows + winbwd::partial_floats(d, B, Hkv, Sk, D, sinks)) * (int64_t)sizeof(float);
}

extern "C" int bsa_window_bwd(const bsa_window_bwd_args* a, void* cuda_stream) {
  if (!a) return set_error(BSA_ERR_INVALID, "bsa_window_bwd: null args");
  if (a->dtype != BSA_DTYPE_BF16 && a->dtype != BSA_DTYPE_F16)
    return set_error(BSA_ERR_INVALID, "bsa_window_bwd: dtype must be bf16 or f16");
  if (a->D != 64 && a->D != 96 && a->D != 128)
    return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_bwd: head dimension %d not built (64, 96 or 128)", a->D);
  if (a->B < 1 || a->Hq < 1 || a->Hkv < 1 || a->Sq < 1 || a->Sk < 1) return set_error(BSA_ERR_INVALID, "bsa_window_bwd: non-positive extent");
  if (a->Hq % a->Hkv != 0) return set_error(BSA_ERR_INVALID, "bsa_window_bwd: Hq %% Hkv != 0");
  if (a->Sq > (1 << 29) || a->Sk > (1 << 29)) return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_bwd: length out of [1, 2^29]");
  if (!a->dout || !a->q || !a->k || !a->v || !a->out || !a->lse || !a->dq || !a->dk || !a->dv || !a->workspace || !a->status)
    return set_error(BSA_ERR_INVALID, "bsa_window_bwd: null pointer");
  if (a->window < 1 || a->sinks < 0 || a->sinks > kMaxSinks)
    return set_error(BSA_ERR_INVALID, "bsa_window_bwd: window must be >= 1 and sinks in [0, %d]", kMaxSinks);
  if (!(a->softmax_scale > 0.f) || a->softmax_scale > 2.0e38f)
    return set_error(BSA_ERR_INVALID, "bsa_window_bwd: softmax_scale must be positive and finite");
  const int64_t need = bsa_window_bwd_workspace_bytes(a->B, a->Hq, a->Hkv, a->Sq, a->Sk, a->D, a->window, a->sinks);
  if (a->workspace_bytes < need) return set_error(BSA_ERR_WORKSPACE, "bsa_window_bwd: workspace of %lld bytes needed", (long long)need);
  for (int i = 0; i < 3; ++i)
    if ((a->dq_stride[i] | a->dk_stride[i] | a->dv_stride[i] | a->o_stride[i] | a->do_stride[i]) % 8 != 0)
      return set_error(BSA_ERR_INVALID, "bsa_window_bwd: strides must be multiples of 8 elements");
  {
    const void* vec16[6] = {a->out, a->dout, a->dq, a->dk, a->dv, a->workspace};
    const char* names[6] = {"out", "dout", "dq", "dk", "dv", "workspace"};
    for (int i = 0; i < 6; ++i)
      if ((reinterpret_cast<uintptr_t>(vec16[i]) & 15u) != 0)
        return set_error(BSA_ERR_INVALID, "%s: base address must be 16-byte aligned", names[i]);
  }
  int dev = 0;
  cudaGetDevice(&dev);
  const int num_sms = bsa_num_sms(dev);
  if (num_sms <= 0) return set_error(BSA_ERR_CUDA, "bsa_window_bwd: cannot query the SM count");

  winbwd::Params p{};
  p.kv_lens = a->kv_lens;
  p.dq = static_cast<uint8_t*>(a->dq);
  p.dk = static_cast<uint8_t*>(a->dk);
  p.dv = static_cast<uint8_t*>(a->dv);
  p.status = a->status;
  for (int i = 0; i < 3; ++i) {
    p.dq_stride[i] = a->dq_stride[i];
    p.dk_stride[i] = a->dk_stride[i];
    p.dv_stride[i] = a->dv_stride[i];
  }
  p.B = a->B;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.G = a->Hq / a->Hkv;
  p.Sq = a->Sq;
  p.Sk = a->Sk;
  p.Nq = (a->Sq + 127) / 128;
  p.Nkv = (a->Sk + 127) / 128;
  p.D = a->D;
  p.window = a->window < kWindowAll ? a->window : kWindowAll;
  p.dq_group = head_group((long long)a->B * a->Hq, a->Sk < p.window ? a->Sk : p.window, a->D, a->Hq / a->Hkv);
  p.dkv_group = head_group((long long)a->B * a->Hkv, (long long)(a->Hq / a->Hkv) * (a->Sq < p.window ? a->Sq : p.window), a->D, 1);
  p.sinks = a->sinks;
  p.unseen_hi = (a->Sk > a->Sq ? a->Sk - a->Sq : 0) - p.window + 1;
  const winbwd::Deal d = winbwd::deal(a->B, a->Hq, a->Hkv, a->Sq, a->Sk, p.window, a->sinks);
  p.parts = d.parts;
  p.sink_m0 = d.sink_m0;
  p.sink_items = d.sink_items;
  p.softmax_scale = a->softmax_scale;
  p.scale_log2 = a->softmax_scale * kLog2e;
  const long long rows_pad = (long long)p.B * p.Hq * p.Nq * 128;
  if (rows_pad / 64 >= 0x7fffffffLL || (long long)p.B * p.Hkv * (p.Nkv + p.sink_items) > 0x7fffffffLL ||
      (long long)p.G * p.Nq > 0x3fffffffLL)
    return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_bwd: too many tiles");
  float* lse_log2 = static_cast<float*>(a->workspace);
  float* delta = lse_log2 + rows_pad;
  p.lse_log2 = lse_log2;
  p.delta = delta;
  p.partial = delta + rows_pad;

  const CUtensorMapDataType dt = a->dtype == BSA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tdo, tk, tv;
  {
    uint64_t qd[4] = {(uint64_t)a->D, (uint64_t)a->Sq, (uint64_t)a->Hq, (uint64_t)a->B};
    uint64_t kd[4] = {(uint64_t)a->D, (uint64_t)a->Sk, (uint64_t)a->Hkv, (uint64_t)a->B};
    uint32_t box[4] = {64, 128, 1, 1};
    auto map = [&](CUtensorMap* m, const void* base, const int64_t* s, const uint64_t* dims, const char* name) {
      uint64_t sb[3] = {(uint64_t)s[2] * 2, (uint64_t)s[1] * 2, (uint64_t)s[0] * 2};
      return make_tensor_map(m, dt, 4, base, dims, sb, box, name);
    };
    int rc;
    if ((rc = map(&tq, a->q, a->q_stride, qd, "q"))) return rc;
    if ((rc = map(&tdo, a->dout, a->do_stride, qd, "dout"))) return rc;
    if ((rc = map(&tk, a->k, a->k_stride, kd, "k"))) return rc;
    if ((rc = map(&tv, a->v, a->v_stride, kd, "v"))) return rc;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  if (a->dtype == BSA_DTYPE_F16) return winbwd::launch<true>(*a, p, tq, tdo, tk, tv, lse_log2, delta, num_sms, st);
  return winbwd::launch<false>(*a, p, tq, tdo, tk, tv, lse_log2, delta, num_sms, st);
}
