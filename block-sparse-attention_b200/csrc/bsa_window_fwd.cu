// Causal sliding-window attention with sink tokens, forward, for sm_100a: contiguous keys (training, prefill) or a
// paged cache (decoding of single tokens, chunks of a prompt, trees of drafted tokens).
//
//   out_i = sum_j softmax_j(scale q_i k_j | visible(i, j)) v_j,   lse_i = log sum_j exp(scale q_i k_j)
//
// One pass over the visible keys with the running maximum and sum of the softmax; see bsa_window.cuh for visible().
// The structure is the one that measured best for the block-sparse forward: two persistent CTAs per SM, each with its own
// share of the query tiles; warps 0-3 softmax (thread = query row = tensor-memory lane, all 128 scores of a tile),
// warp 4 MMA issue (QK(0), then PV(i), QK(i+1)), warp 5 TMA producer (Q tile and a ring K(0), V(0), K(1), ...),
// warps 6-7 idle (setmaxnreg works on whole warpgroups).  Tensor memory: S @0, O @128; P overwrites the head of S and
// is the A operand of PV.
//
// Rows of a query tile: 128 positions of one head, or, packed, seq_per_tile = floor(128 / G) positions x the G heads
// that share a KV head, so that a key tile is read once for the group.  Packing pays when one head cannot fill a
// tile; the host packs below 128 query tokens.
//
// Three ways of dealing the work: whole query tiles in turn; for few query tiles with short lists of key tiles (decoding
// within a window), a cluster of up to eight CTAs for each ("team"), which join their results through one another's
// shared memory; for few or unequal ones with longer lists, equal runs of the list of all key tiles of all query tiles
// ("stream").  A run may begin and end inside a query tile: such pieces leave fp32 rows and their LSE in one of the CTA's
// two slots of the workspace, and window_join_kernel joins them.  The lengths are on the device only, so every warp finds
// its CTA's run itself from the lengths' prefix sums.  (The host's rule has the times of the three.)
//
// Bound, where many rows share a key, by the chain QK - softmax - PV of a tile, two of which overlap on an SM; where few
// do, by the reads of the keys.  Measured: 32 heads (8 of keys) of 32768 tokens, window 2048, 1219 us, 875 TFLOP/s of the
// visible pairs; one token of each of 64 sequences, 4096 visible keys, 196 us, 5.5 TB/s; one token of one sequence, 1024
// visible keys, 13 us; trees of 48 drafts over 8 sequences of up to 16384 tokens, 137 us; 2048 new tokens over 65536 cached,
// window 4096, 32 (8) heads, 159 us in pages of 64, 153 contiguous.
//
// Roundings: scores, maximum, sums and O are fp32.  P is rounded to the inputs' type for the tensor cores; the sum is that of
// the unrounded P, so a rounding does not shift the others.
//
// Keys that no query of the call sees may hold anything (padding, the unused end of a page, an unused draft, what every window
// has left behind): their scores are replaced, not added to, and their V rows are set to zero in shared memory before PV
// reads them (0 * NaN is NaN).
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
  float* partial_o;    // stream: [2 * CTAs, D / 4, slot_rows, 4]
  float* partial_lse;  // [2 * CTAs, slot_rows]
  int4* joins;         // [CTAs]: the query tile whose first piece ends the CTA's run (b, hidx, m, pieces), pieces 0: none
  int* status;
  int B, Hq, Hkv, G, Hidx, packed;
  int Sq, Sk, NqT, seq_per_tile, slot_rows;
  int D;
  int window, sinks;
  int max_pages, page_size, num_pages, seg, seg_log2;  // seg = rows of one key box: min(page_size, 128), 128 when contiguous
  int ctas, lists;  // stream
  int team;         // CTAs of a cluster
  int group;        // of deal_item
  int num_work;     // query tiles
  float scale_log2;
};

namespace winfwd {
enum Deal { kWhole, kStream, kTeam };
constexpr int kMaxTeam = 8;  // (the portable cluster size)
constexpr int kThreads = 256;
constexpr int kSoftmaxThreads = 128;
constexpr int kMmaWarp = 4;
constexpr int kLoadWarp = 5;
constexpr int kCtasPerSm = 2;
constexpr int kSoftmaxRegs = 208, kOtherRegs = 48;  // 128 threads each: together the 256 x 128 the CTA is launched with
static_assert(kSoftmaxRegs + kOtherRegs == 2 * 128, "register split");
constexpr int kTileBytes = 128 * 128 * 2;
constexpr int kSlabBytes = 128 * 128;
constexpr int kStages = 2;
constexpr int kSmemBytes = kTileBytes + kStages * kTileBytes + 256 + 16 + 8 * 32;  // tiles, barriers, misc, places
static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 196 * 1024, "two CTAs per SM");

struct Item {
  int b, m, hkv, g, hidx;
  int len, base;   // tokens of the sequence, position of query row 0
  int seq0, nseq;  // query tokens of the tile
  int p_lo, p_hi;  // range of the positions of its rows
  TileList tiles;
  int it_begin, it_end;  // this piece of the list of key tiles
  int slot;              // workspace slot of the piece, -1: the piece is the whole list
};

// Length, positions and key tiles of query tile (b, m): the same for all heads.
__device__ __forceinline__ void describe(const WinFwdParams& p, Item& t) {
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
}
__device__ __forceinline__ void describe_heads(const WinFwdParams& p, Item& t) {
  t.hkv = p.packed ? t.hidx : t.hidx / p.G;
  t.g = p.packed ? 0 : t.hidx % p.G;
}

// A query tile without key tiles still has its zeros to write: it counts as one.
__device__ __forceinline__ int item_cost(const WinFwdParams& p, int b, int m) {
  Item t;
  t.b = b;
  t.m = m;
  describe(p, t);
  return max(t.tiles.n, 1);
}

// The list that a stream run is cut from: (head, sequence, query tile) in this order, all query tiles or only the CTA's
// one (p.lists = NqT lists side by side, whose CTAs walk the same keys at the same time: one read from HBM serves them).
__device__ __forceinline__ int list_first(const WinFwdParams& p) { return p.lists > 1 ? (int)blockIdx.x % p.lists : 0; }
__device__ __forceinline__ int list_size(const WinFwdParams& p) { return p.lists > 1 ? 1 : p.NqT; }

// Where the next piece of a CTA begins.  Kept in shared memory, one copy for each warp: in registers it cost the
// softmax warps spills.
struct Place {
  int b, hidx, m, it;
  int left;  // key tiles left of the CTA's run
  int q, r;  // of Runs
};

// Called by whole warps.  (All sums fit 32 bits: the host deals whole query tiles otherwise.)
__device__ __forceinline__ void first_place(const WinFwdParams& p, Place* at) {
  const int lane = threadIdx.x & 31;
  const int m0 = list_first(p), nm = list_size(p), pairs = p.B * nm;  // (sequence, query tile) pairs of a head
  auto cost = [&](int i) { return item_cost(p, i / nm, m0 + i % nm); };
  Place s;
  s.b = s.hidx = s.m = s.it = s.left = 0;
  const int per_head = total_cost(pairs, cost), all = per_head * p.Hidx;
  const int cta = (int)blockIdx.x / p.lists, n = min(all, p.ctas / p.lists);
  const Runs runs{all / n, all % n};
  s.q = runs.q;
  s.r = runs.r;
  if (cta < n) {
    int lo = runs.begin(cta);
    s.left = runs.begin(cta + 1) - lo;
    s.hidx = lo / per_head;
    lo -= s.hidx * per_head;
    const int pair = find_item(pairs, lo, cost);
    s.b = pair / nm;
    s.m = m0 + pair % nm;
    s.it = lo;
  }
  if (lane == 0) *at = s;
  __syncwarp();
}

// The CTA's next piece.  `whole` counts the query tiles when whole ones are dealt.
template <int DEAL>
__device__ __forceinline__ bool next_piece(const WinFwdParams& p, Place* at, int& whole, Item& t) {
  if (DEAL == kStream) {
    Place s = *at;
    __syncwarp();
    if (s.left <= 0) return false;
    t.b = s.b;
    t.hidx = s.hidx;
    t.m = s.m;
    describe(p, t);
    describe_heads(p, t);
    const int cost = max(t.tiles.n, 1);
    const int end = min(cost, s.it + s.left);
    t.it_begin = s.it;
    t.it_end = min(end, t.tiles.n);
    t.slot = (s.it == 0 && end == cost) ? -1 : 2 * (int)blockIdx.x + (s.it > 0 ? 0 : 1);
    s.left -= end - s.it;
    s.it = 0;
    if (++s.m == list_first(p) + list_size(p)) {
      s.m = list_first(p);
      if (++s.b == p.B) {
        s.b = 0;
        ++s.hidx;
      }
    }
    if ((threadIdx.x & 31) == 0) *at = s;
    __syncwarp();
    return true;
  }
  if (whole >= p.num_work) return false;
  const Dealt d = deal_item(whole, p.B * p.Hidx, p.NqT, p.group);
  t.m = p.NqT - 1 - d.rank;  // (the last ones have the longest lists)
  t.hidx = d.column % p.Hidx;
  t.b = d.column / p.Hidx;
  describe(p, t);
  describe_heads(p, t);
  t.it_begin = 0;
  t.it_end = t.tiles.n;
  t.slot = -1;
  if (DEAL == kTeam) {
    t.slot = (int)blockIdx.x % p.team;
    t.it_begin = (int)((long long)t.tiles.n * t.slot / p.team);
    t.it_end = (int)((long long)t.tiles.n * (t.slot + 1) / p.team);
  }
  whole += gridDim.x;  // (past the end, for a team)
  return true;
}

// Cluster-wide barrier (all threads of all CTAs) and reads of another CTA's shared memory.
__device__ __forceinline__ void team_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t team_address(uint32_t local, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  return a;
}
__device__ __forceinline__ float team_load(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ float4 team_load4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}
// A team's piece in shared memory, over the tiles, which are done with by then: fp32 rows, four channels c of row r at
// place (c + r) mod D / 4 (a thread writes a whole row: without the shift the writes of a warp would share a bank), and
// behind them the rows' LSE.
__device__ __forceinline__ uint32_t team_place(int row, int c, int D) {
  return (uint32_t)(row * (D / 4) + (c + row) % (D / 4)) * 16u;
}
constexpr uint32_t kTeamLse = 128 * 128 * 4;
static_assert(kTeamLse + 512 <= (1 + kStages) * kTileBytes, "a team's piece fits the tiles");

// The sinks' tile takes MMAs of 32 or 64 columns where that holds them all (32768 tokens, window 2048: 1169 -> 1131 us).
__device__ __forceinline__ bool narrow_end(const WinFwdParams& p, const Item& t) {
  return p.sinks <= 64 && t.tiles.n > t.tiles.n_win && t.it_end == t.tiles.n && t.it_begin < t.it_end;
}

// What a query row sees: keys [lo, hi) and [0, sinks) below hi, and the drafts of `tree` (bit u = key base + u).
struct Row {
  int lo, hi;
  unsigned long long tree;
  bool live;  // sees anything at all
};

__device__ __forceinline__ unsigned long long all_drafts(const WinFwdParams& p) {
  return p.Sq >= 64 ? ~0ull : ((1ull << p.Sq) - 1ull);
}
// The drafts whose keys a row with the (non-empty) mask `mine` sees.  Positions go by all bits of a mask; keys exist from the
// sequence's start on (a short sequence holds the last drafts).
__device__ __forceinline__ unsigned long long seen_drafts(const WinFwdParams& p, int base, const unsigned long long* masks,
                                                          unsigned long long mine) {
  unsigned long long seen = mine;
  if (base < 0) seen = -base >= 64 ? 0ull : (mine & (~0ull << (-base)));
  const int depth = __popcll(mine) - 1;
  if (depth >= p.window) {  // (only a window shorter than the branch leaves ancestors behind)
    for (int u = 0; u < p.Sq; ++u) {
      const int du = __popcll(masks[u] & all_drafts(p)) - 1;
      if (((seen >> u) & 1ull) && depth - du >= p.window && base + du >= p.sinks) seen &= ~(1ull << u);
    }
  }
  return seen;
}
// The drafts that no draft of the sequence sees: unused slots.  Called by whole warps.
__device__ __forceinline__ unsigned long long unseen_drafts(const WinFwdParams& p, const Item& t) {
  const unsigned long long* masks = p.tree_mask + (long long)t.b * p.Sq;
  unsigned long long seen = 0;
  for (int u = threadIdx.x & 31; u < p.Sq; u += 32) {
    const unsigned long long mine = masks[u] & all_drafts(p);
    if (mine != 0 && t.base + __popcll(mine) - 1 >= 0) seen |= seen_drafts(p, t.base, masks, mine);
  }
  const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)seen), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(seen >> 32));
  return all_drafts(p) & ~((unsigned long long)hi << 32 | lo);
}

__device__ __forceinline__ Row make_row(const WinFwdParams& p, const Item& t, int seq, bool valid) {
  Row r;
  r.tree = 0;
  r.lo = 0;
  r.hi = 0;
  r.live = false;
  if (!valid) return r;
  if (p.tree_mask) {
    const unsigned long long* masks = p.tree_mask + (long long)t.b * p.Sq;
    const unsigned long long mine = masks[seq] & all_drafts(p);
    const int depth = __popcll(mine) - 1;
    if (mine != 0 && t.base + depth >= 0) {
      r.tree = seen_drafts(p, t.base, masks, mine);
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

// Joins a team's pieces (window_join_kernel has the formula): the rows are dealt to the CTAs, a warp takes a row, a lane
// four channels.  Called by the softmax warps - they have the registers - behind their last piece, while the other warps
// only wait with them; also when a wait expired (the result is marked invalid then).
template <bool F16>
__device__ __forceinline__ void join_team(const WinFwdParams& p, uint32_t base) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  team_sync();
  Item t;
  const Dealt d = deal_item((int)blockIdx.x / p.team, p.B * p.Hidx, p.NqT, p.group);
  t.m = p.NqT - 1 - d.rank;
  t.hidx = d.column % p.Hidx;
  t.b = d.column / p.Hidx;
  describe(p, t);
  describe_heads(p, t);
  const int heads = p.packed ? p.G : 1, rows = heads * t.nseq, step = 4 * p.team;
  constexpr int kRows = 2;  // of a warp at a time, all their loads in flight
  for (int row0 = ((int)blockIdx.x % p.team) * 4 + warp; row0 < rows; row0 += kRows * step) {
    float l[kRows][kMaxTeam];
    float4 v[kRows][kMaxTeam];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int row = row0 + u * step;
#pragma unroll
      for (int s = 0; s < kMaxTeam; ++s) {
        l[u][s] = -INFINITY;
        v[u][s] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < p.team && row < rows) {
          l[u][s] = team_load(team_address(base + kTeamLse + row * 4, s));
          if (lane * 4 < p.D) v[u][s] = team_load4(team_address(base + team_place(row, lane, p.D), s));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int row = row0 + u * step;
      if (row >= rows) break;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxTeam; ++s) top = fmaxf(top, l[u][s]);
      if (top == -INFINITY) top = 0.f;  // (a row that sees nothing, or NaN, which the maximum passes over)
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kMaxTeam; ++s) {  // (rows of a piece that sees nothing are zeros)
        const float w = __expf(l[u][s] - top);
        sum += w;
        acc.x = fmaf(w, v[u][s].x, acc.x);
        acc.y = fmaf(w, v[u][s].y, acc.y);
        acc.z = fmaf(w, v[u][s].z, acc.z);
        acc.w = fmaf(w, v[u][s].w, acc.w);
      }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      const int seq = t.seq0 + row / heads, hq = t.hkv * p.G + (p.packed ? row % heads : t.g);
      if (lane == 0 && p.lse != nullptr)
        p.lse[((long long)t.b * p.Hq + hq) * p.Sq + seq] = sum != 0.f ? top + __logf(sum) : -INFINITY;
      if (lane * 4 < p.D) {
        uint2 packed;
        packed.x = F16 ? pack_f16x2(acc.x * inv, acc.y * inv) : pack_bf16x2(acc.x * inv, acc.y * inv);
        packed.y = F16 ? pack_f16x2(acc.z * inv, acc.w * inv) : pack_bf16x2(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(p.out + (long long)t.b * p.o_stride_b + (long long)hq * p.o_stride_h +
                                  (long long)seq * p.o_stride_s + lane * 8) = packed;
      }
    }
  }
}

template <bool F16, int DEAL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const WinFwdParams p) {
  constexpr int NS = kStages;
  constexpr bool STREAM = DEAL == kStream;
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
    if (DEAL == kTeam) {  // (the others of the team wait twice)
      team_sync();
      team_sync();
    }
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  WaitCtx wctx{&s_abort, p.status};
  Place* place = reinterpret_cast<Place*>(reinterpret_cast<uint8_t*>(bars) + 272 + warp * 32);
  static_assert(sizeof(Place) <= 32, "place");

  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(BAR(kQFull), 1);
    mbar_init(BAR(kQEmpty), 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(BAR(kKvFull + i), 1);
      mbar_init(BAR(kKvEmpty + i), 1);
    }
    mbar_init(BAR(kSFull), 1);
    mbar_init(BAR(kPHalf), kSoftmaxThreads / 32);  // (one arrival a warp: those of its lanes are taken in turn)
    mbar_init(BAR(kPFull), kSoftmaxThreads / 32);
    mbar_init(BAR(kOFinal), 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    // half of the SM's tensor memory: the other half belongs to the CTA that shares the SM
    tmem_alloc(smem_u32(&s_tmem_base), 256);
    tmem_relinquish();
  }
  if (STREAM && warp <= kLoadWarp) first_place(p, place);  // every warp for itself
  int whole_next = DEAL == kTeam ? (int)blockIdx.x / p.team : (int)blockIdx.x;
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
    setmaxnreg_dec<kOtherRegs>();
    uint32_t ring_cnt = 0, q_cnt = 0;
    bool ok = true;
    const uint32_t q_bytes = 2u * 128u * (uint32_t)(p.packed ? p.G * p.seq_per_tile : 128);
    const int segs = 128 / p.seg;  // key boxes of a tile
    int4 join = make_int4(0, 0, 0, 0);
    Item t;
    while (ok && next_piece<DEAL>(p, place, whole_next, t)) {
      const int n_it = t.it_end - t.it_begin;
      if (n_it <= 0) continue;
      if (STREAM && t.slot >= 0 && (t.slot & 1)) {  // the rest of this query tile begins the runs of the CTAs behind
        const Runs runs{place->q, place->r};
        const int cta = (int)blockIdx.x / p.lists;
        const int last = runs.holder(runs.begin(cta + 1) + t.tiles.n - t.it_end - 1);
        join = make_int4(t.b, t.hidx, t.m, last - cta + 1);
      }
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
    if (STREAM && lane == 0) p.joins[blockIdx.x] = join;
    if (DEAL == kTeam) team_sync();
  } else if (warp == kMmaWarp) {
    // ========================================= MMA issue ========================================
    setmaxnreg_dec<kOtherRegs>();
    constexpr uint32_t kFmt = F16 ? 0u : 1u;
    const uint32_t idesc_qk = umma_idesc(kFmt, kFmt, 0, 0, 128, 128);
    const uint32_t idesc_pv = umma_idesc(kFmt, kFmt, 0, 1, 128, (uint32_t)p.D);
    const uint32_t led = lane == 0;
    uint32_t ring_pos = 0, q_cnt = 0, p_cnt = 0;
    const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ), 0, 1024);
    const uint64_t k_desc0 = umma_desc_sw128(smem_u32(sKV), 0, 1024);                     // K-major view
    const uint64_t v_desc0 = umma_desc_sw128(smem_u32(sKV), (uint32_t)kSlabBytes, 1024);  // MN-major view
    bool ok = true;
    Item t;
    while (ok && next_piece<DEAL>(p, place, whole_next, t)) {
      const int n_it = t.it_end - t.it_begin;
      if (n_it <= 0) continue;
      ok = mbar_wait(BAR(kQFull), q_cnt & 1, wctx, 200);
      if (!ok) break;
      ++q_cnt;
      const bool narrow = narrow_end(p, t);
      const int n_main = n_it - (narrow ? 1 : 0);
      const int groups = (p.sinks + 31) / 32;  // of the narrow tile
      auto issue_qk = [&](auto is_narrow, bool last) -> bool {
        const uint32_t stage = ring_pos % NS;
        if (!mbar_wait(BAR(kKvFull + stage), (ring_pos / NS) & 1, wctx, 201)) return false;
        ++ring_pos;
        tc_fence_after();
        const uint64_t kd = k_desc0 + (uint64_t)stage * (kTileBytes >> 4);
        // (the columns of whole tiles are a constant: with a computed number every tile's MMAs were issued more slowly)
        const uint32_t idesc = decltype(is_narrow)::value ? umma_idesc(kFmt, kFmt, 0, 0, 128, 32u * groups) : idesc_qk;
        auto steps = [&](int k0, int k1) {
#pragma unroll
          for (int k = k0; k < k1; ++k) {
            const uint64_t off = (uint64_t)((k >> 2) * (kSlabBytes >> 4) + (k & 3) * 2);
            umma_f16_ss_led(tS, q_desc + off, kd + off, idesc, k > 0, led);
          }
        };
        steps(0, 4);
        if (p.D > 64) steps(4, 6);  // (an MMA that is predicated off takes as long to issue as one that runs)
        if (p.D > 96) steps(6, 8);
        umma_commit_led(BAR(kSFull), led);
        umma_commit_led(BAR(kKvEmpty + stage), led);
        if (last) umma_commit_led(BAR(kQEmpty), led);
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](auto is_narrow, int i, bool last) -> bool {
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
        if (decltype(is_narrow)::value) {
          pv_steps(0, 2);
          if (groups > 1) pv_steps(2, 4);
        } else {
          pv_steps(0, 4);
        }
        if (!mbar_wait(BAR(kPFull), p_cnt & 1, wctx, 204)) return false;
        ++p_cnt;
        tc_fence_after();
        if (!decltype(is_narrow)::value) pv_steps(4, 8);
        umma_commit_led(BAR(kKvEmpty + stage), led);
        if (last) umma_commit_led(BAR(kOFinal), led);
        __syncwarp();
        return true;
      };
      ok = n_main > 0 ? issue_qk(std::false_type{}, n_it == 1) : true;
      for (int i = 0; i < n_main && ok; ++i) {
        ok = issue_pv(std::false_type{}, i, i == n_it - 1);
        if (ok && i + 1 < n_main) ok = issue_qk(std::false_type{}, i + 2 == n_it);
      }
      if (narrow && ok) {
        ok = issue_qk(std::true_type{}, true);
        if (ok) ok = issue_pv(std::true_type{}, n_main, true);
      }
    }
    if (DEAL == kTeam) team_sync();
  } else if (warp < 4) {
    // ===================================== softmax + epilogue ===================================
    setmaxnreg_inc<kSoftmaxRegs>();
    const int row = threadIdx.x;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    uint32_t s_cnt = 0, of_cnt = 0, ring_cnt = 0;
    bool ok = true;
    const int heads = p.packed ? p.G : 1;  // heads of a tile's rows
    const int row_seq = p.packed ? row / heads : row, row_head = p.packed ? row % heads : 0;
    const int segs = 128 / p.seg;

    Item t;
    bool more = next_piece<DEAL>(p, place, whole_next, t);
    while (ok && more) {
      const int n_it = t.it_end - t.it_begin;
      float m_cur = -INFINITY;  // running max, log2 domain (scale applied)
      float l_sum = 0.f;        // running sum relative to m_cur
      const int seq = t.seq0 + row_seq;
      const int hq = t.hkv * p.G + t.g + row_head;
      const bool row_valid = row < heads * t.nseq;
      const bool warp_active = (warp * 32) < heads * t.nseq;  // some row of this warp exists
      const Row r = make_row(p, t, seq, row_valid && n_it > 0);
      // every row of the tile sees all keys of [free_lo, free_hi) that exist
      const int free_lo = min(t.p_hi, t.len - 1) - p.window + 1;
      const int free_hi = p.tree_mask ? t.base : t.p_lo + 1;
      const bool narrow = narrow_end(p, t);
      // no query of the call sees keys [sinks, unseen_hi): they lie before every window
      const int unseen_hi = max(t.base, 0) - p.window + 1;

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
        const unsigned long long unused = p.tree_mask && j0 + 128 > t.base ? unseen_drafts(p, t) : 0ull;
        ok = mbar_wait(BAR(kSFull), s_cnt & 1, wctx, 300);
        if (!ok) break;
        ++s_cnt;
        tc_fence_after();
        if (j0 + 128 > t.len || (j0 < unseen_hi && j0 + 128 > p.sinks) || unused != 0) {
          // V rows behind the end, and others that no query of the call sees, may hold anything: zero them.  PV(i) of this
          // tile waits for our P, so the stage cannot have been refilled when its arrival is observed here.
          const uint32_t pos = ring_cnt + 2u * (uint32_t)i + 1u;
          const uint32_t stage = pos % NS;
          ok = mbar_wait(BAR(kKvFull + stage), (pos / NS) & 1, wctx, 301);
          if (!ok) break;
          const int j = j0 + row, u = j - t.base;
          if (j >= t.len || (j >= p.sinks && j < unseen_hi) || (u >= 0 && u < 64 && ((unused >> u) & 1ull))) {
            uint4* v0 = reinterpret_cast<uint4*>(sKV + stage * kTileBytes + row * 128);
#pragma unroll
            for (int c = 0; c < 8; ++c) {  // (each row begins at another chunk: other banks than its neighbours')
              v0[(c + row) & 7] = make_uint4(0, 0, 0, 0);
              v0[((c + row) & 7) + kSlabBytes / 16] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
        }
        if (!warp_active) {  // no row of this warp exists: only the barrier protocol
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(BAR(kPHalf));
            mbar_arrive(BAR(kPFull));
          }
          continue;
        }
        const uint32_t t_row = tS + lane_base;
        uint64_t s0 = pack2(0.f, 0.f), s1 = s0;
        // The running maximum takes in a tile's largest score; O and the sum are rescaled only when it grew by more than
        // 2^8 in some row of the warp.  Rows that see nothing have no say: they may hold anything, and the others' roundings
        // must not depend on it.  Returns the addend of the exponents.
        auto grow = [&](float top) -> float {
          const float m_new = fmaxf(m_cur, top * p.scale_log2);
          if (i == 0) {
            m_cur = m_new;
          } else if (__any_sync(0xffffffffu, r.live && (m_new - m_cur) > 8.f)) {
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
          return (m_cur == -INFINITY) ? 0.f : -m_cur;
        };
        // P of 32 columns, rounded to 16 bits for the tensor cores, and their sum, in fp32 before the rounding
        auto exponentials = [&](const float* sv, uint64_t sc2, uint64_t nm2, uint32_t* pk) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            unpack2(ffma2(pack2(sv[2 * e], sv[2 * e + 1]), sc2, nm2), x0, x1);
            x0 = ex2_approx(x0);
            x1 = ex2_approx(x1);
            if (e & 1) s1 = fadd2(s1, pack2(x0, x1));
            else s0 = fadd2(s0, pack2(x0, x1));
            pk[e] = F16 ? pack_f16x2(x0, x1) : pack_bf16x2(x0, x1);
          }
        };
        // One body for whole tiles and one for masked tiles, both straight-line: with the masked body for every tile 16 heads
        // of 16384 tokens, window 1024, take 220 us instead of 200, and loops over the 32-column groups that a warp sees
        // doubled the time of a tile on the diagonal (4000 clocks against 2000 for the warp that sees all groups; the
        // others wait for it).
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
          const float neg_m = grow(fmaxf(m0, m1));
          const uint64_t sc2 = pack2(p.scale_log2, p.scale_log2), nm2 = pack2(neg_m, neg_m);
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            uint32_t pk[16];
            exponentials(sv + c4 * 32, sc2, nm2, pk);
            if (c4 == 2) {  // the first half of P is released on its own barrier, its stores long landed
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(BAR(kPHalf));
            }
            tmem_st16(t_row + c4 * 16, pk);
          }
          tmem_wait_st();
        };
        // the sinks' tile, 32 columns at a time
        auto narrow_tile = [&]() {
          float bm = -INFINITY;
          const int groups = (p.sinks + 31) / 32;
          auto load_group = [&](int g, float* sv) {
            uint32_t w = low_bits(p.sinks - 32 * g);
            if (!((pages_ok >> ((g * 32) >> p.seg_log2)) & 1u)) w &= 0xffff0000u;
            if (!((pages_ok >> ((g * 32 + 16) >> p.seg_log2)) & 1u)) w &= 0x0000ffffu;
            tmem_ld32(t_row + g * 32, reinterpret_cast<uint32_t*>(sv));
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[e] = ((w >> e) & 1u) ? sv[e] : -INFINITY;
          };
#pragma unroll 1
          for (int g = 0; g < groups; ++g) {
            float sv[32];
            load_group(g, sv);
#pragma unroll
            for (int e = 0; e < 32; e += 2) bm = fmax3(bm, sv[e], sv[e + 1]);
          }
          const float neg_m = grow(bm);
          const uint64_t sc2 = pack2(p.scale_log2, p.scale_log2), nm2 = pack2(neg_m, neg_m);
#pragma unroll 1
          for (int g = 0; g < groups; ++g) {  // (P of group 1 overwrites scores of group 0)
            float sv[32];
            uint32_t pk[16];
            load_group(g, sv);
            exponentials(sv, sc2, nm2, pk);
            tmem_st16(t_row + g * 16, pk);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(kPHalf));
        };
        if (whole) tile(std::false_type{});
        else if (narrow && i == n_it - 1) narrow_tile();
        else tile(std::true_type{});
        float y0, y1, y2, y3;
        unpack2(s0, y0, y1);
        unpack2(s1, y2, y3);
        l_sum += (y0 + y1) + (y2 + y3);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kPFull));
      }
      if (!ok) break;
      ring_cnt += 2u * (uint32_t)max(n_it, 0);

      Item next;
      more = next_piece<DEAL>(p, place, whole_next, next);  // (while the last PV runs)

      // ------------------------------------ tile epilogue ------------------------------------
      const bool seen = r.live && l_sum != 0.f;  // (NaN, where the inputs hold one, is passed on)
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
      const bool piece = STREAM && t.slot >= 0;  // uniform
      if (piece) {
        prow = (long long)t.slot * p.slot_rows + row;
        // (four channels of all rows side by side: a thread has a row, so the writes of a warp are one run of memory)
        dst_f = reinterpret_cast<float4*>(p.partial_o + (long long)t.slot * p.slot_rows * p.D) + row;
      } else {
        dst_h = reinterpret_cast<uint4*>(p.out + (long long)t.b * p.o_stride_b + (long long)hq * p.o_stride_h +
                                         (long long)seq * p.o_stride_s);
      }
      if (warp_active) {
        const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_valid) >> (lane & ~3);
        uint4* dst[4];
        exchange_rows(dst_h, dst);
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
            if (DEAL == kTeam) {
              if (row_valid) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  *reinterpret_cast<float4*>(smem_raw + team_place(row, c * 8 + e, p.D)) =
                      make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
              }
            } else if (piece) {
              if (row_valid) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  dst_f[(long long)(c * 8 + e) * p.slot_rows] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
              }
            } else {
              uint32_t u[4][4];
#pragma unroll
              for (int e = 0; e < 16; ++e)
                u[e >> 2][e & 3] = F16 ? pack_f16x2(acc[2 * e], acc[2 * e + 1]) : pack_bf16x2(acc[2 * e], acc[2 * e + 1]);
              store_exchanged(dst, c * 4, u, rows_ok);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      if (row_valid) {
        if (DEAL == kTeam) *reinterpret_cast<float*>(smem_raw + kTeamLse + row * 4) = lse;
        else if (piece) p.partial_lse[prow] = lse;
        else if (p.lse != nullptr) p.lse[((long long)t.b * p.Hq + hq) * p.Sq + seq] = lse;
      }
      t = next;
    }
    if (DEAL == kTeam) join_team<F16>(p, smem_u32(smem_raw));
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (DEAL == kTeam) team_sync();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
  if (DEAL == kTeam) team_sync();  // nobody leaves while another may read its memory
}

// Joins the pieces of cut query tiles: lse = log sum_s exp(lse_s), out = sum_s exp(lse_s - lse) O_s.  Block (c, y) takes
// kJoinRows * R rows of the query tile whose first piece ended CTA c's run, if there is one: first each row's statistics,
// then a thread for four channels of R rows, eight rows side by side as the pieces hold them.  Pieces in which the row
// sees nothing carry -inf and are not read.
// Bound by the latency of its chain of loads, so eight are in flight: of eight pieces of one row where tiles have few rows
// or many pieces, of two pieces of four rows otherwise (128 query tiles of 128 rows, two or three pieces each: 12 us, with
// one row a thread 24).
constexpr int kJoinRows = 8;
template <bool F16, int R>
__global__ void __launch_bounds__(256)
window_join_kernel(const WinFwdParams p) {
  constexpr int kFly = 8 / R;  // pieces of a row in flight
  __shared__ float s_top[kJoinRows * R], s_inv[kJoinRows * R];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (a dependent launch: the forward kernel has ended behind this)
  const int4 j = p.joins[blockIdx.x];
  const int pieces = j.w;
  // (the list is written by the forward kernel, also when one of its waits expired; never trust it with an address)
  if (pieces < 2 || pieces > p.ctas || (int)blockIdx.x + (pieces - 1) * p.lists >= p.ctas || j.x < 0 || j.x >= p.B ||
      j.y < 0 || j.y >= p.Hidx || j.z < 0 || j.z >= p.NqT)
    return;
  const int heads = p.packed ? p.G : 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = min(p.slot_rows, heads * (p.Sq - j.z * p.seq_per_tile)), row0 = (int)blockIdx.y * kJoinRows * R;
  // the first piece is the last of its CTA's run, each of the others the first of its CTA's
  auto slot = [&](int s) { return (long long)(2 * ((int)blockIdx.x + s * p.lists) + (s == 0 ? 1 : 0)); };
  auto piece_lse = [&](int s, int row) { return p.partial_lse[slot(s) * p.slot_rows + row]; };
  auto seq_of = [&](int row) { return j.z * p.seq_per_tile + row / heads; };
  auto head_of = [&](int row) { return p.packed ? j.y * p.G + row % heads : j.y; };
  auto statistics = [&](int at, float top, float sum) {
    const int row = row0 + at;
    s_top[at] = top;
    s_inv[at] = sum != 0.f ? 1.f / sum : 0.f;
    if (p.lse != nullptr)
      p.lse[((long long)j.x * p.Hq + head_of(row)) * p.Sq + seq_of(row)] = sum != 0.f ? top + __logf(sum) : -INFINITY;
  };
  if (R == 1) {  // a warp for a row
    const int row = row0 + warp;
    if (row < rows) {
      float m = -INFINITY, sum = 0.f;
      for (int s = lane; s < pieces; s += 32) m = fmaxf(m, piece_lse(s, row));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float top = m == -INFINITY ? 0.f : m;  // (the maximum passes over NaN, the sum does not)
      for (int s = lane; s < pieces; s += 32) sum += __expf(piece_lse(s, row) - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) statistics(warp, top, sum);
    }
  } else if (warp == 0) {  // a lane for a row
    const int row = row0 + lane;
    if (row < rows) {
      float m = -INFINITY, sum = 0.f;
#pragma unroll 4
      for (int s = 0; s < pieces; ++s) m = fmaxf(m, piece_lse(s, row));
      const float top = m == -INFINITY ? 0.f : m;
#pragma unroll 4
      for (int s = 0; s < pieces; ++s) sum += __expf(piece_lse(s, row) - top);
      statistics(lane, top, sum);
    }
  }
  static_assert(R == 1 || kJoinRows * R == 32, "a lane for a row");
  const int u = threadIdx.x & 7, c = threadIdx.x >> 3;
  float w[R][kFly];
  float4 v[R][kFly], acc[R];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = row0 + u + i * kJoinRows;
#pragma unroll
      for (int e = 0; e < kFly; ++e) {
        w[i][e] = -INFINITY;
        v[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s0 + e < pieces && row < rows && c * 4 < p.D) {
          w[i][e] = piece_lse(s0 + e, row);
          v[i][e] = reinterpret_cast<const float4*>(p.partial_o)[(slot(s0 + e) * (p.D / 4) + c) * p.slot_rows + row];
        }
      }
    }
  };
  load(0);  // (under the statistics)
  __syncthreads();
  if (c * 4 >= p.D) return;
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0;;) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float top = s_top[u + i * kJoinRows], inv = s_inv[u + i * kJoinRows];
#pragma unroll
      for (int e = 0; e < kFly; ++e) {
        if (w[i][e] != -INFINITY) {
          const float f = __expf(w[i][e] - top) * inv;
          acc[i].x = fmaf(f, v[i][e].x, acc[i].x);
          acc[i].y = fmaf(f, v[i][e].y, acc[i].y);
          acc[i].z = fmaf(f, v[i][e].z, acc[i].z);
          acc[i].w = fmaf(f, v[i][e].w, acc[i].w);
        }
      }
    }
    s0 += kFly;
    if (s0 >= pieces) break;
    load(s0);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + u + i * kJoinRows;
    if (row >= rows) break;
    uint2 packed;
    packed.x = F16 ? pack_f16x2(acc[i].x, acc[i].y) : pack_bf16x2(acc[i].x, acc[i].y);
    packed.y = F16 ? pack_f16x2(acc[i].z, acc[i].w) : pack_bf16x2(acc[i].z, acc[i].w);
    *reinterpret_cast<uint2*>(p.out + (long long)j.x * p.o_stride_b + (long long)head_of(row) * p.o_stride_h +
                              (long long)seq_of(row) * p.o_stride_s + c * 8) = packed;
  }
}

template <bool F16, int DEAL>
static int launch(const WinFwdParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  int num_sms, cudaStream_t stream) {
  auto kern = window_fwd_kernel<F16, DEAL>;
  static SmemAttribute attribute;
  cudaError_t e = attribute.set(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "cudaFuncSetAttribute(smem): %s", cudaGetErrorString(e));
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr = {};
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSmemBytes;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 0;
  if (DEAL == kTeam) {
    config.gridDim = dim3((unsigned)(p.num_work * p.team));
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.team;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.numAttrs = 1;
  } else if (DEAL == kStream) {
    config.gridDim = dim3((unsigned)p.ctas);
  } else {
    config.gridDim = dim3((unsigned)(p.num_work < kCtasPerSm * num_sms ? p.num_work : kCtasPerSm * num_sms));
  }
  e = cudaLaunchKernelEx(&config, kern, tq, tk, tv, p);
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window forward launch: %s", cudaGetErrorString(e));
  if (DEAL == kStream) {
    // a dependent launch, set up while the forward kernel runs (1.3 us less a call for small ones)
    // (32 query tiles of 128 rows, nine pieces each: equal; 16 with 18 pieces: 28.8 us for the call against 35.1)
    const bool one_row = p.slot_rows <= kJoinRows || p.ctas > 12LL * p.num_work;
    const int block_rows = one_row ? kJoinRows : 4 * kJoinRows;
    config.gridDim = dim3((unsigned)p.ctas, (unsigned)((p.slot_rows + block_rows - 1) / block_rows));
    config.blockDim = dim3(256);
    config.dynamicSmemBytes = 0;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.numAttrs = 1;
    e = one_row ? cudaLaunchKernelEx(&config, window_join_kernel<F16, 1>, p)
                : cudaLaunchKernelEx(&config, window_join_kernel<F16, 4>, p);
    if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "window join launch: %s", cudaGetErrorString(e));
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
  if (!(a->softmax_scale > 0.f) || a->softmax_scale > 2.0e38f)  // the running maximum is taken before scaling
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: softmax_scale must be positive and finite");
  if (a->stream_ctas < 0 || a->stream_ctas > 65535) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: stream_ctas out of [0, 65535]");
  if (a->team < 0 || a->team > winfwd::kMaxTeam || (a->team > 1 && a->stream_ctas > 0))
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: team out of [0, %d], or together with stream_ctas", winfwd::kMaxTeam);
  if (a->stream_lists > 1 && a->stream_ctas % a->stream_lists != 0)
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: stream_ctas must be a multiple of stream_lists");
  if (a->stream_ctas > 0 && (!a->partial_o || !a->partial_lse || !a->joins))
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: a stream run needs its workspace");
  if ((reinterpret_cast<uintptr_t>(a->out) & 15u) != 0 || ((reinterpret_cast<uintptr_t>(a->partial_o) | reinterpret_cast<uintptr_t>(a->joins)) & 15u) != 0)
    return set_error(BSA_ERR_INVALID, "out, partial_o, joins: base address must be 16-byte aligned");
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
  p.joins = reinterpret_cast<int4*>(a->joins);
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
  p.ctas = a->stream_ctas;
  p.lists = a->stream_lists > 1 ? a->stream_lists : 1;
  p.team = a->team > 1 ? a->team : 1;
  p.slot_rows = (packed ? G : 1) * (a->Sq < p.seq_per_tile ? a->Sq : p.seq_per_tile);
  const long long work = (long long)p.B * p.Hidx * p.NqT;
  if (work > 0x7f000000LL)  // (a grid's width is added to an item's index)
    return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: more than 2^31 work items");
  p.num_work = (int)work;
  p.group = head_group((long long)p.B * p.Hidx, Sk < p.window ? Sk : p.window, p.D, packed ? 1 : G);
  if (p.team > 1 && work * p.team > 65535) return set_error(BSA_ERR_INVALID, "bsa_window_fwd: more than 65535 CTAs in teams");
  if (p.ctas > 0 && p.lists > 1 && p.lists != p.NqT)
    return set_error(BSA_ERR_INVALID, "bsa_window_fwd: stream_lists must be 1 or the number of query tiles per head (%d)", p.NqT);
  // key tiles of a query tile: those that its rows' windows touch, and the sinks'
  const long long rows = a->Sq < p.seq_per_tile ? a->Sq : p.seq_per_tile, touched = (rows + p.window + 127) / 128 + 1;
  const long long most = (Sk + 127) / 128 < touched ? (Sk + 127) / 128 : touched;
  if (p.ctas > 0 && work * (most + 1) > 0x7fffffffLL)
    return set_error(BSA_ERR_UNSUPPORTED, "bsa_window_fwd: more than 2^31 key tiles in a stream run");
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
  auto run = [&](auto f16) {
    constexpr bool kF16 = decltype(f16)::value;
    if (p.team > 1) return winfwd::launch<kF16, winfwd::kTeam>(p, tq, tk, tv, num_sms, st);
    if (p.ctas > 0) return winfwd::launch<kF16, winfwd::kStream>(p, tq, tk, tv, num_sms, st);
    return winfwd::launch<kF16, winfwd::kWhole>(p, tq, tk, tv, num_sms, st);
  };
  return a->dtype == BSA_DTYPE_F16 ? run(std::true_type{}) : run(std::false_type{});
}
