// Rotary positions with several axes (text, images, video): pair p of a head turns by
//   angle(b, s, p) = positions[b, s, axis(p)] * inv_freq[p].
//
// Bound by HBM: q and k are read and written once, three multiply-adds per element.  A block holds a few whole tokens:
// its threads first compute the sines and cosines of the tokens' pairs, about one each, into shared memory; then a
// thread owns one 16-byte chunk of a token (half-split pairing: the two chunks its pairs connect), takes its pairs'
// values into registers and walks over every head_lanes-th head of q and k, four heads in flight at a time.
//
// The angle of position 10^5 at frequency 1 is 10^5 radians; in 32 bits its fraction of a turn would be off by 10^-3.
// So position * (inv_freq / 2 pi) is formed and reduced to [-1/2, 1/2] turns in 64 bits, and only the reduced turn is
// rounded to 32 bits (sincospi of twice that: an error below 2^-24 turns).
#include "bsa_b200.h"
#include "bsa_common.cuh"
#include "bsa_host.h"

#include <cuda_fp16.h>

namespace bsa {
namespace rotary {

constexpr int kThreads = 256;

struct Params {
  const uint8_t* q;
  const uint8_t* k;
  uint8_t* qo;
  uint8_t* ko;
  const int32_t* __restrict__ positions;
  const float* __restrict__ inv_freq;
  long long q_b, q_h, q_s, k_b, k_h, k_s;      // bytes
  long long qo_b, qo_h, qo_s, ko_b, ko_h, ko_s;
  long long pos_b, pos_s;  // elements
  long long units;         // element form: B * S * units per token
  int end0, end1, end2;    // first pair of axes 1, 2, 3
  int Hq, heads, S, D, P;
  int per_token;           // units per token
  int heads_per_cta;
  long long tokens;        // B * S
  int tokens_per_block;    // vector form: whole tokens of a block, at most kThreads units
  int head_lanes;          // ... and the heads its threads work on side by side
  float sign;
};

template <typename T>
struct Io;
template <>
struct Io<float> {
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(uint4 u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(uint4 u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(uint4 u, float* f) {
    unpack_f16x2(u.x, f[0], f[1]);
    unpack_f16x2(u.y, f[2], f[3]);
    unpack_f16x2(u.z, f[4], f[5]);
    unpack_f16x2(u.w, f[6], f[7]);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
  }
};

__device__ __forceinline__ void pair_sincos(const Params& p, const int32_t* pos, int pair, float& c, float& s) {
  const int axis = (pair >= p.end0) + (pair >= p.end1) + (pair >= p.end2);
  constexpr double kInvTwoPi = 0.15915494309189533576888;
  const double turns = (double)pos[axis] * ((double)p.inv_freq[pair] * kInvTwoPi);
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  s *= p.sign;
}

// Address of the row of (head slot h, batch, token): q heads first, then k heads.
__device__ __forceinline__ void row_of(const Params& p, int h, long long b, int tok, const uint8_t*& src, uint8_t*& dst) {
  if (h < p.Hq) {
    src = p.q + b * p.q_b + h * p.q_h + tok * p.q_s;
    dst = p.qo + b * p.qo_b + h * p.qo_h + tok * p.qo_s;
  } else {
    src = p.k + b * p.k_b + (h - p.Hq) * p.k_h + tok * p.k_s;
    dst = p.ko + b * p.ko_b + (h - p.Hq) * p.ko_h + tok * p.ko_s;
  }
}

// Vector form: 16-byte chunks.  Interleaved: unit c = chunk c (its pairs lie inside it; pairs from P on are copied).
// Half-split: units 0 .. P/V-1 are pairs of chunks (c, P/V + c), the rest single chunks that are copied.
constexpr int kTable = 2048;  // P <= V * units per token, V <= 8, and a block's tokens have at most kThreads units
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
rotary_vec_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int kPairs = INTERLEAVED ? V / 2 : V;
  constexpr int kFly = 4;  // heads in flight
  __shared__ float2 table[kTable];
  const long long token0 = (long long)blockIdx.x * p.tokens_per_block;
  const int here = (int)min((long long)p.tokens_per_block, p.tokens - token0);
  for (int i = threadIdx.x; i < here * p.P; i += kThreads) {
    const int t = i / p.P, pair = i - t * p.P;
    const long long token = token0 + t, b = token / p.S;
    float c, s;
    pair_sincos(p, p.positions + b * p.pos_b + (token - b * p.S) * p.pos_s, pair, c, s);
    table[i] = make_float2(c, s);
  }
  __syncthreads();
  const int units = p.tokens_per_block * p.per_token;
  const int lane = threadIdx.x / units, unit = threadIdx.x - lane * units;  // head lane, unit inside the block
  const int t = unit / p.per_token, c = unit - t * p.per_token;
  if (lane >= p.head_lanes || t >= here) return;
  const long long b = (token0 + t) / p.S;
  const int tok = (int)(token0 + t - b * p.S);
  const int half_chunks = p.P / V;
  const bool turned = INTERLEAVED || c < half_chunks;  // half-split: the tail units only copy
  float cs[kPairs], sn[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int pair = c * kPairs + i;
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (turned && pair < p.P) {
      const float2 v = table[t * p.P + pair];
      cs[i] = v.x;
      sn[i] = v.y;
    }
  }
  const int chunk_a = turned ? c : half_chunks + c;
  const int chunk_b = half_chunks + c;  // half-split only
  const int h1 = min(p.heads, ((int)blockIdx.y + 1) * p.heads_per_cta), step = p.head_lanes;
  for (int h = blockIdx.y * p.heads_per_cta + lane; h < h1; h += kFly * step) {
    uint4 a[kFly], z[kFly];
    uint8_t* out[kFly];
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      const uint8_t* src;
      row_of(p, min(h + i * step, h1 - 1), b, tok, src, out[i]);
      if (h + i * step < h1) {
        a[i] = __ldcs(reinterpret_cast<const uint4*>(src) + chunk_a);
        if (!INTERLEAVED && turned) z[i] = __ldcs(reinterpret_cast<const uint4*>(src) + chunk_b);
      }
    }
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      if (h + i * step >= h1) break;
      uint4* dst = reinterpret_cast<uint4*>(out[i]);
      if (INTERLEAVED) {
        float x[V];
        Io<T>::unpack(a[i], x);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          const float x0 = x[2 * e], x1 = x[2 * e + 1];
          x[2 * e] = x0 * cs[e] - x1 * sn[e];
          x[2 * e + 1] = x0 * sn[e] + x1 * cs[e];
        }
        uint4 r = Io<T>::pack(x);
        if ((c + 1) * kPairs > p.P) {
          // the chunk reaches behind the turned channels: those leave with their bits unchanged
          const int turned_words = max(0, p.P - c * kPairs) * (int)(2 * sizeof(T)) / 4;
          if (turned_words <= 0) r.x = a[i].x;
          if (turned_words <= 1) r.y = a[i].y;
          if (turned_words <= 2) r.z = a[i].z;
          if (turned_words <= 3) r.w = a[i].w;
        }
        dst[chunk_a] = r;
      } else if (turned) {
        float x[V], y[V];
        Io<T>::unpack(a[i], x);
        Io<T>::unpack(z[i], y);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x0 = x[e], x1 = y[e];
          x[e] = x0 * cs[e] - x1 * sn[e];
          y[e] = x0 * sn[e] + x1 * cs[e];
        }
        dst[chunk_a] = Io<T>::pack(x);
        dst[chunk_b] = Io<T>::pack(y);
      } else {
        dst[chunk_a] = a[i];
      }
    }
  }
}

// Element form, for rows, strides or halves that 16-byte chunks do not fit: unit < P = one pair, else one copied channel.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
rotary_elt_kernel(const Params p) {
  const long long unit = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (unit >= p.units) return;
  const long long token = unit / p.per_token;
  const int c = (int)(unit - token * p.per_token);
  const long long b = token / p.S;
  const int tok = (int)(token - b * p.S);
  const bool turned = c < p.P;
  float cs = 1.f, sn = 0.f;
  if (turned) pair_sincos(p, p.positions + b * p.pos_b + tok * p.pos_s, c, cs, sn);
  const int ia = turned ? (INTERLEAVED ? 2 * c : c) : p.P + c;
  const int ib = INTERLEAVED ? 2 * c + 1 : p.P + c;
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(p.heads, h0 + p.heads_per_cta);
  for (int h = h0; h < h1; ++h) {
    const uint8_t* src;
    uint8_t* out;
    row_of(p, h, b, tok, src, out);
    const T* x = reinterpret_cast<const T*>(src);
    T* y = reinterpret_cast<T*>(out);
    if (turned) {
      const float x0 = Io<T>::load(x + ia), x1 = Io<T>::load(x + ib);
      Io<T>::store(y + ia, x0 * cs - x1 * sn);
      Io<T>::store(y + ib, x0 * sn + x1 * cs);
    } else {
      y[ia] = x[ia];
    }
  }
}

template <typename T>
static int launch(Params& p, const bsa_rotary_args& a, bool vec, int num_sms, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  p.tokens = (long long)a.B * a.S;
  long long blocks, groups;
  if (vec) {
    p.per_token = a.interleaved ? a.D / V : p.P / V + (a.D - 2 * p.P) / V;
    // Many tokens to a block (head-major rows of neighbouring tokens are neighbours in memory), one head at a time; while
    // that leaves SMs with less than four blocks, fewer tokens and more heads side by side.
    p.head_lanes = 1;
    p.tokens_per_block = kThreads / p.per_token;
    while (p.tokens_per_block > 1 && 2 * p.head_lanes <= p.heads && p.tokens < 4LL * num_sms * p.tokens_per_block) {
      p.head_lanes *= 2;
      p.tokens_per_block = kThreads / (p.per_token * p.head_lanes);
      if (p.tokens_per_block < 1) p.tokens_per_block = 1;
    }
    p.head_lanes = kThreads / (p.tokens_per_block * p.per_token);
    if (p.head_lanes > p.heads) p.head_lanes = p.heads;
    blocks = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    groups = (2LL * num_sms + blocks - 1) / blocks;  // blocks that share tokens, on different heads
    const long long rounds = (p.heads + p.head_lanes - 1) / p.head_lanes;
    if (groups > rounds) groups = rounds;
  } else {
    p.per_token = p.P + (a.D - 2 * p.P);
    p.units = p.tokens * p.per_token;
    blocks = (p.units + kThreads - 1) / kThreads;
    // one thread serves every head of its pair; heads are dealt to more threads while SMs are short of warps
    groups = (8LL * num_sms + blocks - 1) / blocks;
    if (groups > p.heads) groups = p.heads;
  }
  if (blocks > 0x7fffffffLL) return set_error(BSA_ERR_UNSUPPORTED, "bsa_rotary_nd: too many tokens");
  if (groups > 65535) groups = 65535;
  p.heads_per_cta = (int)((p.heads + groups - 1) / groups);
  const dim3 grid((unsigned)blocks, (unsigned)((p.heads + p.heads_per_cta - 1) / p.heads_per_cta));
  if (vec) {
    if (a.interleaved) rotary_vec_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
    else rotary_vec_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
  } else {
    if (a.interleaved) rotary_elt_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
    else rotary_elt_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(BSA_ERR_CUDA, "rotary launch: %s", cudaGetErrorString(e));
  return BSA_OK;
}

}  // namespace rotary
}  // namespace bsa

using namespace bsa;

extern "C" int bsa_rotary_nd(const bsa_rotary_args* a, void* cuda_stream) {
  if (!a) return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: null args");
  if (a->dtype != BSA_ROTARY_BF16 && a->dtype != BSA_ROTARY_F16 && a->dtype != BSA_ROTARY_F32)
    return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: unknown dtype %d", a->dtype);
  if (a->B < 1 || a->Hq < 1 || a->Hk < 0 || a->S < 1 || a->D < 2 || a->D > 512 || a->D % 2 != 0)
    return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: bad extent (even D in [2, 512])");
  if (a->num_axes < 1 || a->num_axes > 4) return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: 1 to 4 axes");
  int P = 0, ends[4] = {0, 0, 0, 0};
  for (int i = 0; i < a->num_axes; ++i) {
    if (a->axis_pairs[i] < 0 || a->axis_pairs[i] > 256) return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: bad axis_pairs");
    P += a->axis_pairs[i];
    ends[i] = P;
  }
  for (int i = a->num_axes; i < 4; ++i) ends[i] = 1 << 30;
  for (int i = 0; i < 4; ++i)
    if (i >= a->num_axes - 1) ends[i] = 1 << 30;  // the last axis runs to the end
  if (P < 1 || 2 * P > a->D) return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: %d pairs do not fit %d channels", P, a->D);
  if (!a->q || !a->q_out || !a->positions || !a->inv_freq || (a->Hk > 0 && (!a->k || !a->k_out)))
    return set_error(BSA_ERR_INVALID, "bsa_rotary_nd: null pointer");
  int dev = 0;
  cudaGetDevice(&dev);
  const int num_sms = bsa_num_sms(dev);
  if (num_sms <= 0) return set_error(BSA_ERR_CUDA, "bsa_rotary_nd: cannot query the SM count");

  const int size = a->dtype == BSA_ROTARY_F32 ? 4 : 2;
  const int V = 16 / size;
  rotary::Params p{};
  p.q = static_cast<const uint8_t*>(a->q);
  p.k = static_cast<const uint8_t*>(a->k);
  p.qo = static_cast<uint8_t*>(a->q_out);
  p.ko = static_cast<uint8_t*>(a->k_out);
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  p.q_b = a->q_stride[0] * size; p.q_h = a->q_stride[1] * size; p.q_s = a->q_stride[2] * size;
  p.k_b = a->k_stride[0] * size; p.k_h = a->k_stride[1] * size; p.k_s = a->k_stride[2] * size;
  p.qo_b = a->qo_stride[0] * size; p.qo_h = a->qo_stride[1] * size; p.qo_s = a->qo_stride[2] * size;
  p.ko_b = a->ko_stride[0] * size; p.ko_h = a->ko_stride[1] * size; p.ko_s = a->ko_stride[2] * size;
  p.pos_b = a->pos_stride[0];
  p.pos_s = a->pos_stride[1];
  p.end0 = ends[0];
  p.end1 = ends[1];
  p.end2 = ends[2];
  p.Hq = a->Hq;
  p.heads = a->Hq + a->Hk;
  p.S = a->S;
  p.D = a->D;
  p.P = P;
  p.sign = a->inverse ? -1.f : 1.f;
  // 16-byte chunks where every row starts on one and (half-split) both halves are whole chunks
  bool vec = a->D % V == 0 && (a->interleaved || P % V == 0);
  const void* base[4] = {a->q, a->q_out, a->Hk ? a->k : nullptr, a->Hk ? a->k_out : nullptr};
  for (const void* q : base) vec = vec && (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
  for (int i = 0; i < 3; ++i) {
    vec = vec && (a->q_stride[i] | a->qo_stride[i]) % V == 0;
    if (a->Hk) vec = vec && (a->k_stride[i] | a->ko_stride[i]) % V == 0;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  if (a->dtype == BSA_ROTARY_F32) return rotary::launch<float>(p, *a, vec, num_sms, st);
  if (a->dtype == BSA_ROTARY_F16) return rotary::launch<__half>(p, *a, vec, num_sms, st);
  return rotary::launch<__nv_bfloat16>(p, *a, vec, num_sms, st);
}
