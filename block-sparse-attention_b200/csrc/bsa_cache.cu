// Writes of the paged key/value cache that bsa_window_fwd reads, and the ancestor masks of trees of drafts.
//
// The token at position j of sequence b lies in page page_table[b][j / page_size] at row j % page_size.  All of it is
// bound by HBM (append) or by latency (keep, masks): 16 bytes per thread and access, K and V together.  Measured at 8 heads
// of 128 channels (changing inputs, in a captured graph): append of 2048 tokens to each of 8 sequences 23.7 us, 5.7 TB/s; append of 32
// drafts to 64 sequences and keep of 8 of them 9.2 us together (in keep one load waits for the path's entry, which waits for the
// length).
#include "bsa_b200.h"
#include "bsa_common.cuh"
#include "bsa_host.h"

namespace bsa {
namespace cache {

struct Pages {
  uint8_t* k;
  uint8_t* v;
  long long k_page, k_head, k_row, v_page, v_head, v_row;  // bytes
  const int32_t* __restrict__ table;
  int max_pages, page_size, num_pages;

  // A length beyond the table counts as the tokens that the table holds, as in the attention over the cache.
  __device__ __forceinline__ int cut(int len) const { return max(0, min(len, max_pages * page_size)); }
  // Byte offsets of (sequence, head, position) in K and V; false when the position has no page in the pool.
  __device__ __forceinline__ bool at(int b, int h, int pos, long long& ko, long long& vo) const {
    if (pos < 0) return false;
    const int slot = pos / page_size;
    if (slot >= max_pages) return false;
    const int id = table[(long long)b * max_pages + slot];
    if (id < 0 || id >= num_pages) return false;
    const int row = pos - slot * page_size;
    ko = id * k_page + h * k_head + row * k_row;
    vo = id * v_page + h * v_head + row * v_row;
    return true;
  }
};

struct Source {
  const uint8_t* k;
  const uint8_t* v;
  long long k_b, k_h, k_t, v_b, v_h, v_t;  // bytes
};

// One thread: one 16-byte chunk of K and of V of kRows consecutive tokens (all loads in flight before the stores).
constexpr int kRows = 4;
__global__ void __launch_bounds__(256)
cache_append_kernel(const Source s, const Pages pg, const int32_t* __restrict__ lens, int B, int H, int T, int chunks,
                    long long units) {
  const long long unit = (long long)blockIdx.x * 256 + threadIdx.x;
  if (unit >= units) return;
  const int c = (int)(unit % chunks);
  long long r = unit / chunks;
  const int groups = (T + kRows - 1) / kRows;
  const int t0 = (int)(r % groups) * kRows;
  r /= groups;
  const int h = (int)(r % H), b = (int)(r / H);
  const int base = pg.cut(lens[b]) - T;
  uint4 kv[kRows], vv[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int t = min(t0 + i, T - 1);
    kv[i] = *(reinterpret_cast<const uint4*>(s.k + b * s.k_b + h * s.k_h + t * s.k_t) + c);
    vv[i] = *(reinterpret_cast<const uint4*>(s.v + b * s.v_b + h * s.v_h + t * s.v_t) + c);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    long long ko, vo;
    if (t0 + i < T && pg.at(b, h, base + t0 + i, ko, vo)) {
      *(reinterpret_cast<uint4*>(pg.k + ko) + c) = kv[i];
      *(reinterpret_cast<uint4*>(pg.v + vo) + c) = vv[i];
    }
  }
}

// Accepted draft path[i] moves to place i.  A path is ascending, so path[i] >= i: with the moves of a sequence done in
// order, none overwrites a source that a later one reads.  One thread carries one chunk of K and V through the whole
// path, eight moves at a time (their loads before their stores, the order kept between the eights).
__global__ void __launch_bounds__(128)
cache_keep_kernel(const Pages pg, const int32_t* __restrict__ lens, const int32_t* __restrict__ path,
                  const int32_t* __restrict__ path_lens, int32_t* __restrict__ new_lens, int B, int H, int T,
                  int path_cap, int chunks, long long units) {
  constexpr int kMoves = 8;
  const long long unit = (long long)blockIdx.x * 128 + threadIdx.x;
  if (unit >= units) return;
  const int c = (int)(unit % chunks);
  const long long r = unit / chunks;
  const int h = (int)(r % H), b = (int)(r / H);
  const int len = lens[b], base = pg.cut(len) - T;
  const int32_t* mine = path + (long long)b * path_cap;
  int n = base < 0 ? 0 : max(0, min(path_lens[b], path_cap));
  int last = -1, kept = 0;
  for (int i0 = 0; i0 < n; i0 += kMoves) {
    uint4 kv[kMoves], vv[kMoves];
    bool have[kMoves];
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      have[i] = false;
      if (i0 + i < n) {
        const int u = mine[i0 + i];
        if (u <= last || u >= T) {
          n = i0 + i;  // the path ends here
        } else {
          last = u;
          kept = i0 + i + 1;
          long long ko, vo;
          if (u != i0 + i && pg.at(b, h, base + u, ko, vo)) {
            have[i] = true;
            kv[i] = *(reinterpret_cast<const uint4*>(pg.k + ko) + c);
            vv[i] = *(reinterpret_cast<const uint4*>(pg.v + vo) + c);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      long long ko, vo;
      if (have[i] && pg.at(b, h, base + i0 + i, ko, vo)) {
        *(reinterpret_cast<uint4*>(pg.k + ko) + c) = kv[i];
        *(reinterpret_cast<uint4*>(pg.v + vo) + c) = vv[i];
      }
    }
  }
  if (h == 0 && c == 0) new_lens[b] = base < 0 ? len : base + kept;
}

// One thread per draft walks up its parents: at most T steps, as every parent is an earlier draft.
__global__ void __launch_bounds__(64)
tree_mask_kernel(const int32_t* __restrict__ parents, long long* __restrict__ mask, int T) {
  __shared__ int up[64];
  const int t = threadIdx.x;
  const long long row = (long long)blockIdx.x * T;
  if (t < T) up[t] = parents[row + t];
  __syncthreads();
  if (t >= T) return;
  unsigned long long m = 0;
  for (int u = t; u >= 0;) {
    const int above = up[u];
    if (above >= u || above < -1) {  // not a tree: an unused slot
      m = 0;
      break;
    }
    m |= 1ull << u;
    u = above;
  }
  mask[row + t] = (long long)m;
}

static int check_pages(const char* what, const bsa_cache_args* a) {
  if (!a) return set_error(BSA_ERR_INVALID, "%s: null args", what);
  if (!a->k_cache || !a->v_cache || !a->page_table || !a->lens) return set_error(BSA_ERR_INVALID, "%s: null pointer", what);
  if (a->B < 1 || a->H < 1 || a->T < 1 || a->max_pages < 1 || a->page_size < 1 || a->num_pages < 1)
    return set_error(BSA_ERR_INVALID, "%s: non-positive extent", what);
  if (a->D < 8 || a->D % 8 != 0) return set_error(BSA_ERR_INVALID, "%s: D must be a multiple of 8", what);
  if ((long long)a->max_pages * a->page_size > (1 << 29))
    return set_error(BSA_ERR_UNSUPPORTED, "%s: more than 2^29 tokens per sequence", what);
  if (a->k_cache == a->v_cache) return set_error(BSA_ERR_INVALID, "%s: keys and values share a pool", what);
  if (((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15u) != 0)
    return set_error(BSA_ERR_INVALID, "%s: the caches must be 16-byte aligned", what);
  for (int i = 0; i < 3; ++i)
    if ((a->kc_stride[i] | a->vc_stride[i]) % 8 != 0)
      return set_error(BSA_ERR_INVALID, "%s: cache strides must be multiples of 8 elements", what);
  return BSA_OK;
}

static Pages make_pages(const bsa_cache_args* a) {
  Pages pg{};
  pg.k = static_cast<uint8_t*>(a->k_cache);
  pg.v = static_cast<uint8_t*>(a->v_cache);
  pg.k_page = a->kc_stride[0] * 2; pg.k_head = a->kc_stride[1] * 2; pg.k_row = a->kc_stride[2] * 2;
  pg.v_page = a->vc_stride[0] * 2; pg.v_head = a->vc_stride[1] * 2; pg.v_row = a->vc_stride[2] * 2;
  pg.table = a->page_table;
  pg.max_pages = a->max_pages;
  pg.page_size = a->page_size;
  pg.num_pages = a->num_pages;
  return pg;
}

}  // namespace cache
}  // namespace bsa

using namespace bsa;

extern "C" int bsa_tree_mask(const int32_t* parents, int32_t B, int32_t T, int64_t* mask, void* cuda_stream) {
  if (!parents || !mask) return set_error(BSA_ERR_INVALID, "bsa_tree_mask: null pointer");
  if (B < 1 || T < 1 || T > 64) return set_error(BSA_ERR_INVALID, "bsa_tree_mask: 1 to 64 drafts");
  cache::tree_mask_kernel<<<(unsigned)B, 64, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      parents, reinterpret_cast<long long*>(mask), T);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "tree mask launch: %s", cudaGetErrorString(e));
  return BSA_OK;
}

extern "C" int bsa_cache_append(const bsa_cache_args* a, void* cuda_stream) {
  int rc = cache::check_pages("bsa_cache_append", a);
  if (rc) return rc;
  if (!a->k || !a->v) return set_error(BSA_ERR_INVALID, "bsa_cache_append: null pointer");
  if (((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15u) != 0)
    return set_error(BSA_ERR_INVALID, "bsa_cache_append: k and v must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if ((a->k_stride[i] | a->v_stride[i]) % 8 != 0)
      return set_error(BSA_ERR_INVALID, "bsa_cache_append: strides must be multiples of 8 elements");
  cache::Source s{};
  s.k = static_cast<const uint8_t*>(a->k);
  s.v = static_cast<const uint8_t*>(a->v);
  s.k_b = a->k_stride[0] * 2; s.k_h = a->k_stride[1] * 2; s.k_t = a->k_stride[2] * 2;
  s.v_b = a->v_stride[0] * 2; s.v_h = a->v_stride[1] * 2; s.v_t = a->v_stride[2] * 2;
  const int chunks = a->D / 8;
  const long long units = (long long)a->B * a->H * ((a->T + cache::kRows - 1) / cache::kRows) * chunks;
  const long long blocks = (units + 255) / 256;
  if (blocks > 0x7fffffffLL) return set_error(BSA_ERR_UNSUPPORTED, "bsa_cache_append: too many tokens");
  cache::cache_append_kernel<<<(unsigned)blocks, 256, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      s, cache::make_pages(a), a->lens, a->B, a->H, a->T, chunks, units);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "cache append launch: %s", cudaGetErrorString(e));
  return BSA_OK;
}

extern "C" int bsa_cache_keep(const bsa_cache_args* a, void* cuda_stream) {
  int rc = cache::check_pages("bsa_cache_keep", a);
  if (rc) return rc;
  if (!a->path || !a->path_lens || !a->new_lens) return set_error(BSA_ERR_INVALID, "bsa_cache_keep: null pointer");
  if (a->path_cap < 1) return set_error(BSA_ERR_INVALID, "bsa_cache_keep: non-positive extent");
  const int chunks = a->D / 8;
  const long long units = (long long)a->B * a->H * chunks;
  const long long blocks = (units + 127) / 128;
  if (blocks > 0x7fffffffLL) return set_error(BSA_ERR_UNSUPPORTED, "bsa_cache_keep: too many heads");
  cache::cache_keep_kernel<<<(unsigned)blocks, 128, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      cache::make_pages(a), a->lens, a->path, a->path_lens, a->new_lens, a->B, a->H, a->T, a->path_cap, chunks, units);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "cache keep launch: %s", cudaGetErrorString(e));
  return BSA_OK;
}
