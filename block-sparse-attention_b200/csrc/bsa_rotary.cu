// Rotary positions with several axes (text, images, video): pair p of a head turns by
//   angle(b, s, p) = positions[b, s, axis(p)] * inv_freq[p].
//
// Bound by HBM: q and k are read and written once, three multiply-adds per element.  A block holds a few whole tokens:
// its threads first compute the sines and cosines of the tokens' pairs, about one each, into shared memory; a thread
// owns one 16-byte chunk of a token (half-split pairing: the two chunks its pairs connect), takes its pairs' values
// into registers and walks over every head_lanes-th head of q and k.  Four loads are in flight while the four before are
// worked on, the first four under the sines.  Measured (changing
// inputs, in a captured graph): 76800 tokens of 24 + 24 heads of 128 channels, bf16, 309 us, 6.1 TB/s (93 % of a plain copy's
// rate); 16384 tokens of 16 + 16 heads, fp32, 91 us, 5.9 TB/s; 3 x 4097 tokens of 16 + 4 heads of 96, fp16, 18.1 us; 64 tokens of
// 32 + 8 heads, 2.9 us.
//
// The angle of position 10^5 at frequency 1 is 10^5 radians; in 32 bits its fraction of a turn would be off by 10^-3.
// So a frequency becomes a 64-bit fraction of a turn per position, whose product with the position wraps around whole
// turns by itself (integer arithmetic modulo 2^64; frequencies up to 1 are off by 2^-55 turns, their products with any
// 32-bit position by 2^-24), and only the wrapped turn is rounded to 32 bits.
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
  int tokens;              // B * S
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

// inv_freq in turns per position, modulo 1, as a 64-bit fraction.
__device__ __forceinline__ unsigned long long turn_fraction(float inv_freq) {
  constexpr double kInvTwoPi = 0.15915494309189533576888, kTwo64 = 18446744073709551616.0;
  const double turns = (double)inv_freq * kInvTwoPi;
  return (unsigned long long)((turns - floor(turns)) * kTwo64);  // (a tiny negative one rounds to a whole turn: the conversion saturates)
}
// 0, or NaN for a frequency that is infinite or NaN (the integers above would hide it).
__device__ __forceinline__ float poison_of(float inv_freq) { return inv_freq - inv_freq; }
__device__ __forceinline__ int axis_of(const Params& p, int pair) {
  return (pair >= p.end0) + (pair >= p.end1) + (pair >= p.end2);
}
__device__ __forceinline__ float2 position_sincos(const Params& p, int position, unsigned long long turns, float poison) {
  const int wrapped = (int)((turns * (unsigned long long)(long long)position) >> 32);  // [-1/2, 1/2) turns, times 2^32
  float s, c;
  sincospif((float)wrapped * 0x1p-31f, &s, &c);
  return make_float2(c + poison, s * p.sign + poison);
}

// The rows of one token: q heads first, then k heads.
struct Rows {
  const uint8_t* q;
  const uint8_t* k;
  uint8_t* qo;
  uint8_t* ko;
  __device__ __forceinline__ Rows(const Params& p, int b, int tok)
      : q(p.q + b * p.q_b + tok * p.q_s), k(p.k + b * p.k_b + tok * p.k_s - p.Hq * p.k_h),
        qo(p.qo + b * p.qo_b + tok * p.qo_s), ko(p.ko + b * p.ko_b + tok * p.ko_s - p.Hq * p.ko_h) {}
  __device__ __forceinline__ const uint8_t* from(const Params& p, int h) const { return h < p.Hq ? q + h * p.q_h : k + h * p.k_h; }
  __device__ __forceinline__ uint8_t* to(const Params& p, int h) const { return h < p.Hq ? qo + h * p.qo_h : ko + h * p.ko_h; }
};

// Vector form: 16-byte chunks.  Interleaved: unit c = chunk c (its pairs lie inside it; pairs from P on are copied).
// Half-split: units 0 .. P/V-1 are pairs of chunks (c, P/V + c), the rest single chunks that are copied.
constexpr int kTable = 2048;  // P <= V * units per token, V <= 8, and a block's tokens have at most kThreads units
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 3)
rotary_vec_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int kPairs = INTERLEAVED ? V / 2 : V;
  constexpr int kFly = INTERLEAVED ? 4 : 2;  // heads in flight: four 16-byte loads, twice
  __shared__ float2 table[kTable];
  __shared__ unsigned long long turns[kTable / 8];  // P <= D / 2 <= 256
  __shared__ float poison[kTable / 8];
  const int token0 = blockIdx.x * p.tokens_per_block;
  const int here = min(p.tokens_per_block, p.tokens - token0);
  const int units = p.tokens_per_block * p.per_token;
  const int lane = threadIdx.x / units, unit = threadIdx.x - lane * units;  // head lane, unit inside the block
  const int t = unit / p.per_token, c = unit - t * p.per_token;
  const bool works = lane < p.head_lanes && t < here;
  const int b = (token0 + t) / p.S, tok = token0 + t - b * p.S;
  const Rows rows(p, b, tok);
  const int half_chunks = p.P / V;
  const bool turned = INTERLEAVED || c < half_chunks;  // half-split: the tail units only copy
  const int chunk_a = turned ? c : half_chunks + c;
  const int chunk_b = half_chunks + c;  // half-split only
  const int h1 = min(p.heads, ((int)blockIdx.y + 1) * p.heads_per_cta), step = p.head_lanes;
  struct Batch {
    uint4 a[kFly], z[kFly];
  };
  auto load = [&](int h, Batch& x) {
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      if (h + i * step < h1) {
        const uint8_t* src = rows.from(p, h + i * step);
        x.a[i] = __ldcs(reinterpret_cast<const uint4*>(src) + chunk_a);
        if (!INTERLEAVED && turned) x.z[i] = __ldcs(reinterpret_cast<const uint4*>(src) + chunk_b);
      }
    }
  };
  int h = blockIdx.y * p.heads_per_cta + lane;
  Batch now, then;
  if (works) load(h, now);  // on their way while the sines are computed

  for (int i = threadIdx.x; i < p.P; i += kThreads) {
    const float f = p.inv_freq[i];
    turns[i] = turn_fraction(f);
    poison[i] = poison_of(f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < here * p.P; i += kThreads) {
    const int at = i / p.P, pair = i - at * p.P;
    const int bt = (token0 + at) / p.S;
    const int position = p.positions[bt * p.pos_b + (token0 + at - bt * p.S) * p.pos_s + axis_of(p, pair)];
    table[i] = position_sincos(p, position, turns[pair], poison[pair]);
  }
  __syncthreads();
  if (!works) return;
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
  for (; h < h1; h += kFly * step) {
    load(h + kFly * step, then);
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      if (h + i * step >= h1) break;
      uint4* dst = reinterpret_cast<uint4*>(rows.to(p, h + i * step));
      if (INTERLEAVED) {
        float x[V];
        Io<T>::unpack(now.a[i], x);
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
          if (turned_words <= 0) r.x = now.a[i].x;
          if (turned_words <= 1) r.y = now.a[i].y;
          if (turned_words <= 2) r.z = now.a[i].z;
          if (turned_words <= 3) r.w = now.a[i].w;
        }
        dst[chunk_a] = r;
      } else if (turned) {
        float x[V], y[V];
        Io<T>::unpack(now.a[i], x);
        Io<T>::unpack(now.z[i], y);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x0 = x[e], x1 = y[e];
          x[e] = x0 * cs[e] - x1 * sn[e];
          y[e] = x0 * sn[e] + x1 * cs[e];
        }
        dst[chunk_a] = Io<T>::pack(x);
        dst[chunk_b] = Io<T>::pack(y);
      } else {
        dst[chunk_a] = now.a[i];
      }
    }
    now = then;
  }
}

// Element form, for rows, strides or halves that 16-byte chunks do not fit: unit < P = one pair, else one copied channel.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
rotary_elt_kernel(const Params p) {
  const long long unit = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (unit >= p.units) return;
  const int token = (int)(unit / p.per_token), c = (int)(unit - (long long)token * p.per_token);
  const int b = token / p.S, tok = token - b * p.S;
  const Rows rows(p, b, tok);
  const bool turned = c < p.P;
  float2 cs = make_float2(1.f, 0.f);
  if (turned) {
    const float f = p.inv_freq[c];
    cs = position_sincos(p, p.positions[b * p.pos_b + tok * p.pos_s + axis_of(p, c)], turn_fraction(f), poison_of(f));
  }
  const int ia = turned ? (INTERLEAVED ? 2 * c : c) : p.P + c;
  const int ib = INTERLEAVED ? 2 * c + 1 : p.P + c;
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(p.heads, h0 + p.heads_per_cta);
  for (int h = h0; h < h1; ++h) {
    const T* x = reinterpret_cast<const T*>(rows.from(p, h));
    T* y = reinterpret_cast<T*>(rows.to(p, h));
    if (turned) {
      const float x0 = Io<T>::load(x + ia), x1 = Io<T>::load(x + ib);
      Io<T>::store(y + ia, x0 * cs.x - x1 * cs.y);
      Io<T>::store(y + ib, x0 * cs.y + x1 * cs.x);
    } else {
      y[ia] = x[ia];
    }
  }
}

template <typename T>
static int launch(Params& p, const bsa_rotary_args& a, bool vec, int num_sms, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if ((long long)a.B * a.S > 0x7fffffffLL - kThreads) return set_error(BSA_ERR_UNSUPPORTED, "bsa_rotary_nd: more than 2^31 tokens");
  p.tokens = a.B * a.S;
  long long blocks, groups;
  if (vec) {
    p.per_token = a.interleaved ? a.D / V : p.P / V + (a.D - 2 * p.P) / V;
    // Many tokens to a block (head-major rows of neighbouring tokens are neighbours in memory), one head at a time; while
    // that leaves SMs with less than two blocks, fewer tokens and more heads side by side.
    p.head_lanes = 1;
    p.tokens_per_block = kThreads / p.per_token;
    while (p.tokens_per_block > 1 && 2 * p.head_lanes <= p.heads && p.tokens < 2LL * num_sms * p.tokens_per_block) {
      p.head_lanes *= 2;
      p.tokens_per_block = kThreads / (p.per_token * p.head_lanes);
      if (p.tokens_per_block < 1) p.tokens_per_block = 1;
    }
    p.head_lanes = kThreads / (p.tokens_per_block * p.per_token);
    if (p.head_lanes > p.heads) p.head_lanes = p.heads;
    blocks = ((long long)p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    groups = (2LL * num_sms + blocks - 1) / blocks;  // blocks that share tokens, on different heads
    const long long rounds = (p.heads + p.head_lanes - 1) / p.head_lanes;
    if (groups > rounds) groups = rounds;
  } else {
    p.per_token = p.P + (a.D - 2 * p.P);
    p.units = (long long)p.tokens * p.per_token;
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
