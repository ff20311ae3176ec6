// Causal sliding-window attention with sink tokens, forward, for sm_100a: contiguous keys (training, prefill) or a
// paged cache (decoding of single tokens, chunks of a prompt, trees of drafted tokens).
//
//   out_i = sum_j softmax_j(scale q_i k_j | visible(i, j)) v_j,   lse_i = log sum_j exp(scale q_i k_j)
//
// One pass over the visible keys with the running maximum and sum of the softmax; see bsa_window.cuh for visible().
// The structure is the one that measured best for the block-sparse forward: two persistent CTAs per SM, each walking
// (query tile, split) items; warps 0-3 softmax (thread = query row = tensor-memory lane, all 128 scores of a tile),
// warp 4 MMA issue (QK(0), then PV(i), QK(i+1)), warp 5 TMA producer (Q tile and a ring K(0), V(0), K(1), ...),
// warps 6-7 idle (setmaxnreg works on whole warpgroups).  Tensor memory: S @0, O @128; P overwrites the head of S and
// is the A operand of PV.
//
// Rows of a query tile: 128 positions of one head, or, packed, seq_per_tile = floor(128 / G) positions x the G heads
// that share a KV head, so that a key tile is read once for the group.  Packing pays when one head cannot fill a
// tile; the host packs below 128 query tokens.  With few items the key tiles of an item are dealt to several splits,
// whose fp32 partial rows window_combine_kernel joins.
//
// Keys behind the sequence's end may hold anything (padding, the unused end of a page): their scores are replaced,
// not added to, and their V rows are set to zero in shared memory before PV reads them (0 * NaN is NaN).
#include "bsa_b200.h"
#include "bsa_common.cuh"
#include "bsa_host.h"
#include "bsa_window.cuh"

#include <type_traits>

namespace bsa {

struct WinFwdParams {
  const int32_t* __restrict__ kv_lens;     // [B] or null
  const int32_t* __restrict__ page_table;  // [B, max_pages] or null (contiguous keys)
  const unsigned long long* __restrict__ tree_mask;  // [B, Sq] or null
  uint8_t* out;
  long long o_stride_b, o_stride_h, o_stride_s;  // bytes
  float* lse;
  float* partial_o;
  float* partial_lse;
  int* status;
  int B, Hq, Hkv, G, Hidx, packed;
  int Sq, Sk, NqT, seq_per_tile;
  int D;
  int window, sinks;
  int max_pages, page_size, num_pages, seg, seg_log2;  // seg = rows of one key box: min(page_size, 128), 128 when contiguous
  int splits, num_work;
  float scale_log2;
};

namespace winfwd {
constexpr int kThreads = 256;
constexpr int kSoftmaxThreads = 128;
constexpr int kMmaWarp = 4;
constexpr int kLoadWarp = 5;
constexpr int kCtasPerSm = 2;
constexpr int kTileBytes = 128 * 128 * 2;
constexpr int kSlabBytes = 128 * 128;
constexpr int kStages = 2;
constexpr int kSmemBytes = kTileBytes + kStages * kTileBytes + 256 + 16;
static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 196 * 1024, "two CTAs per SM");

struct Item {
  int b, m, split;
  int hkv, g, hidx;
  int len, base;  // tokens of the sequence, position of query row 0
  int seq0, nseq; // query tokens of the tile
  int p_lo, p_hi; // range of the positions of its rows
  TileList tiles;
  int it_begin, it_end;
};

__device__ __forceinline__ Item decode_item(const WinFwdParams& p, int w) {
  Item t;
  t.split = w % p.splits;
  int r = w / p.splits;
  t.m = r % p.NqT;
  r /= p.NqT;
  t.hidx = r % p.Hidx;
  t.b = r / p.Hidx;
  t.hkv = p.packed ? t.hidx : t.hidx / p.G;
  t.g = p.packed ? 0 : t.hidx % p.G;
  t.len = p.kv_lens ? max(0, min(p.kv_lens[t.b], p.Sk)) : p.Sk;
  t.base = (p.page_table ? t.len : p.Sk) - p.Sq;
  t.seq0 = t.m * p.seq_per_tile;
  t.nseq = min(p.seq_per_tile, p.Sq - t.seq0);
  if (p.tree_mask) {  // positions go by depth: anywhere between the first draft's and the last's
    t.p_lo = t.base;
    t.p_hi = t.base + p.Sq - 1;
  } else {
    t.p_lo = t.base + t.seq0;
    t.p_hi = t.p_lo + t.nseq - 1;
  }
  t.tiles = window_tiles(t.p_lo, t.p_hi, t.len, p.window, p.sinks);
  t.it_begin = (int)(((long long)t.tiles.n * t.split) / p.splits);
  t.it_end = (int)(((long long)t.tiles.n * (t.split + 1)) / p.splits);
  return t;
}

// What a query row sees: keys [lo, hi) and [0, sinks) below hi, and the drafts of `tree` (bit u = key base + u).
struct Row {
  int lo, hi;
  unsigned long long tree;
  bool live;  // sees anything at all
};

__device__ __forceinline__ Row make_row(const WinFwdParams& p, const Item& t, int seq, bool valid) {
  Row r;
  r.tree = 0;
  r.lo = 0;
  r.hi = 0;
  r.live = false;
  if (!valid) return r;
  if (p.tree_mask) {
    const unsigned long long* masks = p.tree_mask + (long long)t.b * p.Sq;
    // drafts that exist: u < Sq, at a position that exists
    unsigned long long all = p.Sq >= 64 ? ~0ull : ((1ull << p.Sq) - 1ull);
    if (t.base < 0) all = (-t.base >= 64) ? 0ull : (all & (~0ull << (-t.base)));
    const unsigned long long mine = masks[seq];
    const int depth = __popcll(mine & all) - 1;
    r.tree = mine & all;
    if (depth >= p.window) {  // (only a window shorter than the branch leaves ancestors behind)
      for (int u = 0; u < p.Sq; ++u) {
        const int du = __popcll(masks[u] & all) - 1;
        if (((r.tree >> u) & 1ull) && depth - du >= p.window && t.base + du >= p.sinks) r.tree &= ~(1ull << u);
      }
    }
    if (mine & all) {
      r.lo = t.base + depth - p.window + 1;
      r.hi = max(t.base, 0);
      r.live = true;
    }
  } else {
    const int pos = t.base + seq;
    if (pos >= 0 && pos < t.len) {
      r.lo = pos - p.window + 1;
      r.hi = pos + 1;
      r.live = true;
    }
  }
  return r;
}

// Visibility bits of the row among the 32 keys from c0 on.
__device__ __forceinline__ uint32_t row_word(const Row& r, int base, int sinks, int c0) {
  uint32_t w = range_word(r.lo - c0, r.hi - c0, 0) | low_bits(min(sinks, r.hi) - c0);
  const int d = base - c0;  // draft 0 is column d
  if (r.tree != 0 && d < 32 && d > -64) w |= d >= 0 ? (uint32_t)r.tree << d : (uint32_t)(r.tree >> (-d));
  return w;
}

template <bool F16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const WinFwdParams p) {
  constexpr int NS = kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sQ = smem_raw;
  uint8_t* sKV = sQ + kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + NS * kTileBytes);
  const uint32_t bar_base = smem_u32(bars);
  auto BAR = [&](int i) { return bar_base + (uint32_t)i * 8u; };
  constexpr int kQFull = 0, kQEmpty = 1, kKvFull = 2, kKvEmpty = 2 + NS, kSFull = 2 + 2 * NS, kPHalf = kSFull + 1,
                kPFull = kPHalf + 1, kOFinal = kPFull + 1, kNumBars = kOFinal + 1;
  static_assert(kNumBars <= 32, "barrier slots");
  uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(bars + 32);
  volatile int& s_abort = *reinterpret_cast<volatile int*>(bars + 33);
  if ((smem_u32(smem_raw) & 1023u) != 0) {  // uniform over the CTA: nothing has been set up yet
    if (threadIdx.x == 0 && atomicCAS(p.status, 0, (int)kStatusBadIndex) == 0) p.status[2] = 996;
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  WaitCtx wctx{&s_abort, p.status};

  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(BAR(kQFull), 1);
    mbar_init(BAR(kQEmpty), 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(BAR(kKvFull + i), 1);
      mbar_init(BAR(kKvEmpty + i), 1);
    }
    mbar_init(BAR(kSFull), 1);
    mbar_init(BAR(kPHalf), kSoftmaxThreads);
    mbar_init(BAR(kPFull), kSoftmaxThreads);
    mbar_init(BAR(kOFinal), 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    // half of the SM's tensor memory: the other half belongs to the CTA that shares the SM
    tmem_alloc(smem_u32(&s_tmem_base), 256);
    tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  const uint32_t tS = tmem, tO = tmem + 128u;

  if (warp == kLoadWarp) {
    // ======================================= TMA producer =======================================
    setmaxnreg_dec<40>();
    uint32_t ring_cnt = 0, q_cnt = 0;
    bool ok = true;
    const uint32_t q_bytes = 2u * 128u * (uint32_t)(p.packed ? p.G * p.seq_per_tile : 128);
    const int segs = 128 / p.seg;  // key boxes of a tile
    for (int w = blockIdx.x; w < p.num_work && ok; w += gridDim.x) {
      const Item t = decode_item(p, w);
      const int n_it = t.it_end - t.it_begin;
      if (n_it <= 0) continue;
      ok = mbar_wait(BAR(kQEmpty), (q_cnt & 1) ^ 1, wctx, 100);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(BAR(kQFull), q_bytes);
#pragma unroll
        for (int sl = 0; sl < 2; ++sl)
          tma_load_5d(smem_u32(sQ + sl * kSlabBytes), &tm_q, BAR(kQFull), sl * 64, t.g, t.seq0, t.hkv, t.b);
      }
      ++q_cnt;
      for (int i = 0; i < n_it && ok; ++i) {
        const int it = t.it_begin + i;
        const int j0 = t.tiles.tile(it) * 128;
        // lane s holds where box s of this tile comes from.  Boxes that no row can see (behind the end, before the
        // windows, behind the sinks of the sink tile) and pages outside the pool are loaded from beyond the tensor's
        // last page: zeros, no memory traffic.
        int page = 0, row = j0;
        if (p.page_table) {
          page = p.num_pages;
          row = 0;
          if (lane < segs) {
            const int tok = j0 + lane * p.seg;
            const bool needed = tok < t.len && (tok < p.sinks || (it < t.tiles.n_win && tok + p.seg > t.tiles.k_lo));
            const int slot = tok / p.page_size;
            if (needed && slot < p.max_pages) {
              const int id = p.page_table[(long long)t.b * p.max_pages + slot];
              if (id >= 0 && id < p.num_pages) {
                page = id;
                row = tok - slot * p.page_size;
              }
            }
          }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {  // K(i), then V(i)
          const CUtensorMap* tm = which ? &tm_v : &tm_k;
          const uint32_t stage = ring_cnt % NS;
          ok = mbar_wait(BAR(kKvEmpty + stage), ((ring_cnt / NS) & 1) ^ 1, wctx, 101);
          if (!ok) break;
          uint8_t* dst = sKV + stage * kTileBytes;
          if (lane == 0) mbar_arrive_expect_tx(BAR(kKvFull + stage), kTileBytes);
          __syncwarp();
          if (lane < segs) {
#pragma unroll
            for (int sl = 0; sl < 2; ++sl) {
              const uint32_t at = smem_u32(dst + sl * kSlabBytes + lane * p.seg * 128);
              if (p.page_table) tma_load_4d(at, tm, BAR(kKvFull + stage), sl * 64, row, t.hkv, page);
              else tma_load_4d(at, tm, BAR(kKvFull + stage), sl * 64, row, t.hkv, t.b);
            }
          }
          __syncwarp();
          ++ring_cnt;
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ========================================= MMA issue ========================================
    setmaxnreg_dec<40>();
    constexpr uint32_t kFmt = F16 ? 0u : 1u;
    const uint32_t idesc_qk = umma_idesc(kFmt, kFmt, 0, 0, 128, 128);
    const uint32_t idesc_pv = umma_idesc(kFmt, kFmt, 0, 1, 128, (uint32_t)p.D);
    const int qk_steps = p.D / 16;
    const uint32_t led = lane == 0;
    uint32_t ring_pos = 0, q_cnt = 0, p_cnt = 0;
    const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ), 0, 1024);
    const uint64_t k_desc0 = umma_desc_sw128(smem_u32(sKV), 0, 1024);                     // K-major view
    const uint64_t v_desc0 = umma_desc_sw128(smem_u32(sKV), (uint32_t)kSlabBytes, 1024);  // MN-major view
    bool ok = true;
    for (int w = blockIdx.x; w < p.num_work && ok; w += gridDim.x) {
      const Item t = decode_item(p, w);
      const int n_it = t.it_end - t.it_begin;
      if (n_it <= 0) continue;
      ok = mbar_wait(BAR(kQFull), q_cnt & 1, wctx, 200);
      if (!ok) break;
      ++q_cnt;
      auto issue_qk = [&](bool last) -> bool {
        const uint32_t stage = ring_pos % NS;
        if (!mbar_wait(BAR(kKvFull + stage), (ring_pos / NS) & 1, wctx, 201)) return false;
        ++ring_pos;
        tc_fence_after();
        const uint64_t kd = k_desc0 + (uint64_t)stage * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)((k >> 2) * (kSlabBytes >> 4) + (k & 3) * 2);
          umma_f16_ss_led(tS, q_desc + off, kd + off, idesc_qk, k > 0, (k < qk_steps) ? led : 0u);
        }
        umma_commit_led(BAR(kSFull), led);
        umma_commit_led(BAR(kKvEmpty + stage), led);
        if (last) umma_commit_led(BAR(kQEmpty), led);
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](int i, bool last) -> bool {
        const uint32_t stage = ring_pos % NS;
        if (!mbar_wait(BAR(kKvFull + stage), (ring_pos / NS) & 1, wctx, 202)) return false;
        ++ring_pos;
        if (!mbar_wait(BAR(kPHalf), p_cnt & 1, wctx, 203)) return false;
        tc_fence_after();
        const uint64_t vd = v_desc0 + (uint64_t)stage * (kTileBytes >> 4);
        auto pv_steps = [&](int k0, int k1) {
#pragma unroll
          for (int k = k0; k < k1; ++k)
            umma_f16_ts_led(tO, tS + (uint32_t)k * 8u, vd + (uint64_t)(k * 128), idesc_pv, (i > 0) || (k > 0), led);
        };
        pv_steps(0, 4);
        if (!mbar_wait(BAR(kPFull), p_cnt & 1, wctx, 204)) return false;
        ++p_cnt;
        tc_fence_after();
        pv_steps(4, 8);
        umma_commit_led(BAR(kKvEmpty + stage), led);
        if (last) umma_commit_led(BAR(kOFinal), led);
        __syncwarp();
        return true;
      };
      ok = issue_qk(n_it == 1);
      for (int i = 0; i < n_it && ok; ++i) {
        ok = issue_pv(i, i == n_it - 1);
        if (ok && i + 1 < n_it) ok = issue_qk(i + 2 == n_it);
      }
    }
  } else if (warp < 4) {
    // ===================================== softmax + epilogue ===================================
    setmaxnreg_inc<216>();
    const int row = threadIdx.x;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    uint32_t s_cnt = 0, of_cnt = 0, ring_cnt = 0;
    bool ok = true;
    constexpr float kRescaleThreshold = 8.0f;
    const int heads = p.packed ? p.G : 1;  // heads of a tile's rows
    const int segs = 128 / p.seg;

    for (int w = blockIdx.x; w < p.num_work && ok; w += gridDim.x) {
      const Item t = decode_item(p, w);
      const int n_it = t.it_end - t.it_begin;
      float m_cur = -INFINITY;  // running max, log2 domain (scale applied)
      float l_sum = 0.f;        // running sum relative to m_cur
      const int seq = t.seq0 + row / heads;
      const int hq = t.hkv * p.G + (p.packed ? row % heads : t.g);
      const bool row_valid = row < heads * t.nseq;
      const bool warp_active = (warp * 32) < heads * t.nseq;  // some row of this warp exists
      const Row r = make_row(p, t, seq, row_valid && n_it > 0);
      // every row of the tile sees all keys of [free_lo, free_hi) that exist
      const int free_lo = min(t.p_hi, t.len - 1) - p.window + 1;
      const int free_hi = p.tree_mask ? t.base : t.p_lo + 1;

      for (int i = 0; i < n_it && ok; ++i) {
        const int it = t.it_begin + i;
        const int j0 = t.tiles.tile(it) * 128;
        uint32_t pages_ok = 0xffffffffu;
        if (p.page_table) {
          bool good = true;
          if (lane < segs) {
            const int tok = j0 + lane * p.seg;
            const int slot = tok / p.page_size;
            if (tok < t.len) {
              const int id = slot < p.max_pages ? p.page_table[(long long)t.b * p.max_pages + slot] : -1;
              good = id >= 0 && id < p.num_pages;
            }
          }
          pages_ok = __ballot_sync(0xffffffffu, good);
        }
        const bool whole = j0 >= free_lo && j0 + 128 <= free_hi && pages_ok == 0xffffffffu;  // uniform over the warp
        ok = mbar_wait(BAR(kSFull), s_cnt & 1, wctx, 300);
        if (!ok) break;
        ++s_cnt;
        tc_fence_after();
        if (j0 + 128 > t.len) {
          // V rows behind the end may hold anything: zero them.  PV(i) of this tile waits for our P, so the stage
          // cannot have been refilled when its arrival is observed here.
          const uint32_t pos = ring_cnt + 2u * (uint32_t)i + 1u;
          const uint32_t stage = pos % NS;
          ok = mbar_wait(BAR(kKvFull + stage), (pos / NS) & 1, wctx, 301);
          if (!ok) break;
          if (j0 + row >= t.len) {
            uint4* v0 = reinterpret_cast<uint4*>(sKV + stage * kTileBytes + row * 128);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              v0[c] = make_uint4(0, 0, 0, 0);
              v0[c + kSlabBytes / 16] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
        }
        if (!warp_active) {  // no row of this warp exists: only the barrier protocol
          tc_fence_before();
          mbar_arrive(BAR(kPHalf));
          mbar_arrive(BAR(kPFull));
          continue;
        }
        const uint32_t t_row = tS + lane_base;
        uint64_t s0 = pack2(0.f, 0.f), s1 = s0;
        // One body for whole tiles and one for masked tiles, both straight-line: tests inside one body slowed every
        // tile, and loops over the 32-column groups that a warp sees doubled the time of a tile on the diagonal (4000
        // clocks against 2000 for the warp that sees all groups; the others wait for it).
        auto tile = [&](auto masked) {
          constexpr bool kMasked = decltype(masked)::value;
          float sv[128];
          uint32_t* su = reinterpret_cast<uint32_t*>(sv);
          float m0, m1;
          tmem_ld32(t_row + 0, su + 0);
          tmem_ld32(t_row + 32, su + 32);
          uint32_t mw[4];
          if (kMasked) {
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) {
              mw[c4] = row_word(r, t.base, p.sinks, j0 + c4 * 32);
              if (pages_ok != 0xffffffffu) {  // keys of pages that are not in the pool
                if (!((pages_ok >> ((c4 * 32) >> p.seg_log2)) & 1u)) mw[c4] &= 0xffff0000u;
                if (!((pages_ok >> ((c4 * 32 + 16) >> p.seg_log2)) & 1u)) mw[c4] &= 0x0000ffffu;
              }
            }
          }
          tmem_wait_ld();
          // two 64-column halves; the second arrives while the maximum of the first is taken
          tmem_ld32(t_row + 64, su + 64);
          tmem_ld32(t_row + 96, su + 96);
          if (kMasked) {
#pragma unroll
            for (int c = 0; c < 64; ++c) sv[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? sv[c] : -INFINITY;
          }
          m0 = fmax3(sv[0], sv[1], sv[2]);
          m1 = fmax3(sv[3], sv[4], sv[5]);
#pragma unroll
          for (int c = 6; c < 62; c += 4) {
            m0 = fmax3(m0, sv[c], sv[c + 1]);
            m1 = fmax3(m1, sv[c + 2], sv[c + 3]);
          }
          m0 = fmax3(m0, sv[62], sv[63]);
          tmem_wait_ld();
          if (kMasked) {
#pragma unroll
            for (int c = 64; c < 128; ++c) sv[c] = ((mw[c >> 5] >> (c & 31)) & 1u) ? sv[c] : -INFINITY;
          }
#pragma unroll
          for (int c = 64; c < 128; c += 4) {
            m0 = fmax3(m0, sv[c], sv[c + 1]);
            m1 = fmax3(m1, sv[c + 2], sv[c + 3]);
          }
          // the running maximum; O and the sum are rescaled only when it grew by more than the threshold in some row
          const float m_new = fmaxf(m_cur, fmaxf(m0, m1) * p.scale_log2);
          if (i == 0) {
            m_cur = m_new;
          } else if (__any_sync(0xffffffffu, (m_new - m_cur) > kRescaleThreshold)) {
            const float sc = (m_new == -INFINITY) ? 1.f : ex2_approx(m_cur - m_new);
            m_cur = m_new;
            l_sum *= sc;
            // (the previous PV has completed: the commit that signalled this S was issued after it)
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + lane_base + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * sc);
              tmem_st32(tO + lane_base + c * 32, o);
            }
            tmem_wait_st();
          }
          const float neg_m = (m_cur == -INFINITY) ? 0.f : -m_cur;
          // exponentials, row sum (fp32, before P is rounded to 16 bits for the tensor cores), P to tensor memory
          const uint64_t sc2 = pack2(p.scale_log2, p.scale_log2);
          const uint64_t nm2 = pack2(neg_m, neg_m);
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int c = c4 * 32 + e * 2;
              float x0, x1;
              unpack2(ffma2(pack2(sv[c], sv[c + 1]), sc2, nm2), x0, x1);
              x0 = ex2_approx(x0);
              x1 = ex2_approx(x1);
              if (e & 1) s1 = fadd2(s1, pack2(x0, x1));
              else s0 = fadd2(s0, pack2(x0, x1));
              pk[e] = F16 ? pack_f16x2(x0, x1) : pack_bf16x2(x0, x1);
            }
            if (c4 == 2) {  // the first half of P is released on its own barrier, its stores long landed
              tmem_wait_st();
              tc_fence_before();
              mbar_arrive(BAR(kPHalf));
            }
            tmem_st16(t_row + c4 * 16, pk);
          }
          tmem_wait_st();
        };
        if (whole) tile(std::false_type{});
        else tile(std::true_type{});
        float y0, y1, y2, y3;
        unpack2(s0, y0, y1);
        unpack2(s1, y2, y3);
        l_sum += (y0 + y1) + (y2 + y3);
        tc_fence_before();
        mbar_arrive(BAR(kPFull));
      }
      if (!ok) break;
      ring_cnt += 2u * (uint32_t)max(n_it, 0);

      // ------------------------------------ tile epilogue ------------------------------------
      const bool seen = r.live && l_sum > 0.f;
      const float inv = seen ? (1.f / l_sum) : 0.f;
      const float lse = seen ? (m_cur + lg2_approx(l_sum)) * kLn2 : -INFINITY;
      if (n_it > 0) {
        ok = mbar_wait(BAR(kOFinal), of_cnt & 1, wctx, 310);
        if (!ok) break;
        ++of_cnt;
        tc_fence_after();
      }
      long long prow = 0;
      float4* dst_f = nullptr;
      uint4* dst_h = nullptr;
      if (SPLIT) {
        prow = (((long long)t.split * p.B + t.b) * p.Hq + hq) * p.Sq + seq;
        dst_f = reinterpret_cast<float4*>(p.partial_o + prow * p.D);
      } else {
        dst_h = reinterpret_cast<uint4*>(p.out + (long long)t.b * p.o_stride_b + (long long)hq * p.o_stride_h +
                                         (long long)seq * p.o_stride_s);
      }
      // an empty split writes its -inf LSE only: the combine does not read its rows
      if (warp_active && !(SPLIT && n_it <= 0)) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          if (c * 32 < p.D) {
            float acc[32];
            if (n_it > 0) {
              uint32_t o[32];
              tmem_ld32(tO + lane_base + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) acc[e] = seen ? __uint_as_float(o[e]) * inv : 0.f;
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) acc[e] = 0.f;
            }
            if (row_valid) {
              if (SPLIT) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  dst_f[c * 8 + e] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
              } else {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                  uint32_t u[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float a = acc[ch * 8 + 2 * e], b = acc[ch * 8 + 2 * e + 1];
                    u[e] = F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
                  }
                  dst_h[c * 4 + ch] = make_uint4(u[0], u[1], u[2], u[3]);
                }
              }
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      if (row_valid) {
        if (SPLIT) p.partial_lse[prow] = lse;
        else if (p.lse != nullptr) p.lse[((long long)t.b * p.Hq + hq) * p.Sq + seq] = lse;
      }
    }
  } else {
    setmaxnreg_dec<40>();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// Joins the splits of a row: lse = log sum_s exp(lse_s), out = sum_s exp(lse_s - lse) O_s.  One warp per row, four
// channels per lane; splits without a visible key carry -inf and are not read.
template <bool F16>
__global__ void __launch_bounds__(256)
window_combine_kernel(const float* __restrict__ po, const float* __restrict__ plse, uint8_t* __restrict__ out,
                      float* __restrict__ lse, int splits, long long rows, int H, int Sq, int D, long long os_b,
                      long long os_h, long long os_s) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, plse[(long long)s * rows + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float sum = 0.f;
  if (m != -INFINITY)
    for (int s = lane; s < splits; s += 32) sum += __expf(plse[(long long)s * rows + row] - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  if (lane == 0 && lse != nullptr) lse[row] = sum > 0.f ? m + __logf(sum) : -INFINITY;
  if (lane * 4 >= D) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < splits; s0 += 8) {  // eight partial rows in flight
    float w[8];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u;
      const float l = s < splits ? plse[(long long)s * rows + row] : -INFINITY;
      w[u] = l == -INFINITY ? 0.f : __expf(l - m) * inv;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (l != -INFINITY) v[u] = *reinterpret_cast<const float4*>(po + ((long long)s * rows + row) * D + lane * 4);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      acc.x = fmaf(w[u], v[u].x, acc.x);
      acc.y = fmaf(w[u], v[u].y, acc.y);
      acc.z = fmaf(w[u], v[u].z, acc.z);
      acc.w = fmaf(w[u], v[u].w, acc.w);
    }
  }
  const int sq = (int)(row % Sq);
  const long long bh = row / Sq;
  uint2 packed;
  packed.x = F16 ? pack_f16x2(acc.x, acc.y) : pack_bf16x2(acc.x, acc.y);
  packed.y = F16 ? pack_f16x2(acc.z, acc.w) : pack_bf16x2(acc.z, acc.w);
  *reinterpret_cast<uint2*>(out + (bh / H) * os_b + (bh % H) * os_h + (long long)sq * os_s + lane * 8) = packed;
}

template <bool F16, bool SPLIT>
static int launch(const WinFwdParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  int num_sms, cudaStream_t stream) {
  auto kern = window_fwd_kernel<F16, SPLIT>;
  static SmemAttribute attribute;
  cudaError_t e = attribute.set(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "cudaFuncSetAttribute(smem): %s", cudaGetErrorString(e));
  const int grid = p.num_work < kCtasPerSm * num_sms ? p.num_work : kCtasPerSm * num_sms;
  kern<<<grid, kThreads, kSmemBytes, stream>>>(tq, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window forward launch: %s", cudaGetErrorString(e));
  if (SPLIT) {
    const long long rows = (long long)p.B * p.Hq * p.Sq;
    window_combine_kernel<F16><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(
        p.partial_o, p.partial_lse, p.out, p.lse, p.splits, rows, p.Hq, p.Sq, p.D, p.o_stride_b, p.o_stride_h,
        p.o_stride_s);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window combine launch: %s", cudaGetErrorString(e));
  }
  return BSA_OK;
}

}  // namespace winfwd
}  // namespace bsa

using namespace bsa;

extern "C" int bsa_window_fwd(const bsa_window_fwd_args* a, void* cuda_stream) {
  if (!a) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: null args");
  if (a->dtype != BSA_DTYPE_BF16 && a->dtype != BSA_DTYPE_F16)
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: dtype must be bf16 or f16");
  if (a->D != 64 && a->D != 96 && a->D != 128)
    return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: head dimension %d not built (64, 96 or 128)", a->D);
  if (a->B < 1 || a->Hq < 1 || a->Hkv < 1 || a->Sq < 1) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: non-positive extent");
  if (a->Hq % a->Hkv != 0) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: Hq %% Hkv != 0");
  if (!a->q || !a->k || !a->v || !a->out || !a->status) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: null tensor pointer");
  if (a->window < 1 || a->sinks < 0 || a->sinks > kMaxSinks)
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: window must be >= 1 and sinks in [0, %d]", kMaxSinks);
  const bool paged = a->page_table != nullptr;
  long long Sk = a->Sk;
  if (paged) {
    const int ps = a->page_size;
    if (ps < 16 || (ps < 128 ? (ps & (ps - 1)) != 0 : ps % 128 != 0))
      return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: page size %d not built (16, 32, 64 or a multiple of 128)", ps);
    if (a->max_pages < 1 || a->num_pages < 1) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: empty page table or pool");
    if (!a->kv_lens) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: a paged cache needs its lengths");
    Sk = (long long)a->max_pages * ps;
  }
  // positions, windows and their sums stay inside 32 bits
  if (Sk < 1 || Sk > (1 << 29) || a->Sq > (1 << 29)) return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: length out of [1, 2^29]");
  if (a->tree_mask && (a->Sq > kMaxTreeNodes || !paged))
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: a tree has at most %d drafts, over a paged cache", kMaxTreeNodes);
  if (!(a->softmax_scale > 0.f) || a->softmax_scale > 3.0e38f)  // the running maximum is taken before scaling
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: softmax_scale must be positive and finite");
  if (a->splits < 1 || a->splits > 256) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: splits out of [1, 256]");
  if (a->splits > 1 && (!a->partial_o || !a->partial_lse))
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: a split run needs partial buffers");
  if ((reinterpret_cast<uintptr_t>(a->out) & 15u) != 0 || (reinterpret_cast<uintptr_t>(a->partial_o) & 15u) != 0)
    return set_error(BSA_ERR_INVALID, "out: base address must be 16-byte aligned");
  if ((a->o_stride[0] | a->o_stride[1] | a->o_stride[2]) % 8 != 0)
    return set_error(BSA_ERR_INVALID, "out: strides must be multiples of 8 elements");
  const int G = a->Hq / a->Hkv;
  const int packed = a->pack_gqa != 0 && G > 1;
  if (packed && G > 128) return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: more than 128 heads per KV head cannot be packed");

  int dev = 0;
  cudaGetDevice(&dev);
  const int num_sms = bsa_num_sms(dev);
  if (num_sms <= 0) return set_error(BSA_ERR_CUDA, "bsa_window_fwd: cannot query the SM count");

  WinFwdParams p{};
  p.kv_lens = a->kv_lens;
  p.page_table = a->page_table;
  p.tree_mask = reinterpret_cast<const unsigned long long*>(a->tree_mask);
  p.out = static_cast<uint8_t*>(a->out);
  p.o_stride_b = (long long)a->o_stride[0] * 2;
  p.o_stride_h = (long long)a->o_stride[1] * 2;
  p.o_stride_s = (long long)a->o_stride[2] * 2;
  p.lse = a->lse;
  p.partial_o = a->partial_o;
  p.partial_lse = a->partial_lse;
  p.status = a->status;
  p.B = a->B;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.G = G;
  p.packed = packed;
  p.Hidx = packed ? a->Hkv : a->Hq;
  p.Sq = a->Sq;
  p.Sk = (int)Sk;
  p.seq_per_tile = packed ? 128 / G : 128;
  p.NqT = (a->Sq + p.seq_per_tile - 1) / p.seq_per_tile;
  p.D = a->D;
  p.window = a->window < kWindowAll ? a->window : kWindowAll;
  p.sinks = a->sinks;
  p.max_pages = a->max_pages;
  p.page_size = paged ? a->page_size : 1;
  p.num_pages = a->num_pages;
  p.seg = paged ? (a->page_size < 128 ? a->page_size : 128) : 128;
  for (p.seg_log2 = 4; (1 << p.seg_log2) < p.seg;) ++p.seg_log2;
  p.splits = a->splits;
  const long long work = (long long)p.B * p.Hidx * p.NqT * p.splits;
  if (work > 0x7fffffffLL) return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: more than 2^31 work items");
  if ((long long)p.B * p.Hq * p.Sq / 8 >= 0x7fffffffLL) return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: too many rows");
  p.num_work = (int)work;
  p.scale_log2 = a->softmax_scale * kLog2e;

  const CUtensorMapDataType dt = a->dtype == BSA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tk, tv;
  {
    uint64_t dims[5] = {(uint64_t)a->D, (uint64_t)G, (uint64_t)a->Sq, (uint64_t)a->Hkv, (uint64_t)a->B};
    uint64_t str[4] = {(uint64_t)a->q_stride[1] * 2, (uint64_t)a->q_stride[2] * 2, (uint64_t)a->q_stride[1] * G * 2,
                       (uint64_t)a->q_stride[0] * 2};
    uint32_t box[5] = {64, packed ? (uint32_t)G : 1u, (uint32_t)p.seq_per_tile, 1, 1};
    int rc = make_tensor_map(&tq, dt, 5, a->q, dims, str, box, "q");
    if (rc) return rc;
  }
  {
    // contiguous: (D, Sk, Hkv, B); paged: (D, page_size, Hkv, num_pages)
    uint64_t dims[4] = {(uint64_t)a->D, paged ? (uint64_t)a->page_size : (uint64_t)Sk, (uint64_t)a->Hkv,
                        paged ? (uint64_t)a->num_pages : (uint64_t)a->B};
    uint64_t kstr[3] = {(uint64_t)a->k_stride[2] * 2, (uint64_t)a->k_stride[1] * 2, (uint64_t)a->k_stride[0] * 2};
    uint64_t vstr[3] = {(uint64_t)a->v_stride[2] * 2, (uint64_t)a->v_stride[1] * 2, (uint64_t)a->v_stride[0] * 2};
    uint32_t box[4] = {64, (uint32_t)p.seg, 1, 1};
    int rc = make_tensor_map(&tk, dt, 4, a->k, dims, kstr, box, "k");
    if (rc) return rc;
    rc = make_tensor_map(&tv, dt, 4, a->v, dims, vstr, box, "v");
    if (rc) return rc;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  if (a->dtype == BSA_DTYPE_F16)
    return p.splits > 1 ? winfwd::launch<true, true>(p, tq, tk, tv, num_sms, st)
                        : winfwd::launch<true, false>(p, tq, tk, tv, num_sms, st);
  return p.splits > 1 ? winfwd::launch<false, true>(p, tq, tk, tv, num_sms, st)
                      : winfwd::launch<false, false>(p, tq, tk, tv, num_sms, st);
}
