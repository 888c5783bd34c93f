// Rotary positions, and the append of new tokens to the paged caches with the rotation applied on the way.
//
// Pair j of the rotated features, as one complex number, is turned by the angle p f_j (gradient: by minus that angle,
// the transpose of a rotation); with several axes (time, height, width) the pairs are dealt out to the axes in
// order and p is the position on the pair's axis.  A pair is two neighbours (interleaved) or feature j of either half.
//
// The angle is taken in turns, p * (f / 2 pi), in 64 bits and reduced there to [-1/2, 1/2]: at position 10^5 its
// fraction is right to 10^-11, where a 32-bit product has lost 10^-2.  Sine and cosine of the fraction are 32 bits, the
// rotation is 32 bits, and the only rounding to fewer is the store.
#pragma once

#include <algorithm>

#include "dsa_common.cuh"

namespace dsa {

constexpr int kRopeThreads = 256;
constexpr int kRopeAngles = 2048;   // (token, pair) angles that a block keeps: 16 KB
constexpr int kRopeTokens = 64;     // tokens per block at most

// cos and sin of p f, p an integer position
__device__ __forceinline__ float2 rope_angle(int64_t p, float f, float sign) {
  const double turns = (double)p * ((double)f * 0.15915494309189533577);
  float s, c;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c, sign * s);
}
__device__ __forceinline__ int64_t rope_position(const void* positions, int32_t is64, int64_t i) {
  return is64 ? ((const int64_t*)positions)[i] : (int64_t)((const int32_t*)positions)[i];
}
// Axis of a pair: ends[] are the running sums of the pairs per axis (entries past the last axis hold all pairs).
__device__ __forceinline__ int rope_axis(const int32_t* ends, int32_t pair) {
  return (pair >= ends[0]) + (pair >= ends[1]) + (pair >= ends[2]);
}

struct RopeDev {
  const void* x;
  void* out;               // contiguous [tokens, n, d]
  const void* positions;   // [axes, tokens]
  const float* inv_freq;
  int64_t stride_b, stride_s, stride_n, tokens;
  int32_t s1, n, d, pairs, offset, interleaved, pos64;
  int32_t ends[3];
  int32_t tokens_per_block;
  float sign;
};

template <typename T, int V>
struct alignas(V * sizeof(T)) RopeVec { T v[V]; };

// Quotient of numbers below 2^31 by a divisor that the host knows: x * mul >> shift with mul = ceil(2^(31 + l) / d),
// 2^l >= d.
struct RopeDiv {
  uint32_t mul, shift, d;
  explicit RopeDiv(int64_t div = 1) {
    uint32_t l = 0;
    while ((1ll << l) < div) ++l;
    shift = 31 + l;
    mul = (uint32_t)(((1ull << shift) + div - 1) / (uint64_t)div);
    d = (uint32_t)div;
  }
  __device__ __forceinline__ int32_t operator()(int32_t x) const { return (int32_t)(((uint64_t)(uint32_t)x * mul) >> shift); }
};

// A block takes a few tokens: one angle per (token, pair), shared by all heads, then units of 2 V features (V pairs, or two
// vectors of features that pass through).  V features are 16 bytes, or one feature where sizes, strides or pointers
// are not multiples of that.  Bound by memory once the 64-bit angles of a block (a microsecond of latency) hide behind
// the loads of the others, and its divisions are multiplications: 15360 tokens x 128 heads x 64 features from rows of 192 in
// bf16, 503 MB: 88 us = 5.7 TB/s (with divisions and four units a thread in flight 200 us; multiplied, two in flight
// 105, four 148: what they take in registers costs blocks); the same bytes in fp32 80 us = 6.3 TB/s; one feature a unit (66 wide,
// bf16, 69 MB) 32 us = 2.2 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(kRopeThreads, 6) rope_kernel(const RopeDev a, const RopeDiv per_token, const RopeDiv units,
                                                            const RopeDiv pairs) {
  __shared__ float2 angle[kRopeAngles];
  __shared__ int64_t base[kRopeTokens];
  grid_dep_launch();
  grid_dep_wait();
  const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_block;
  const int nt = (int)min((int64_t)a.tokens_per_block, a.tokens - tok0);
  const int rot = a.pairs / V;                                // units of pairs per head
  const int pass = (a.d - 2 * a.pairs) / V;                   // vectors that pass through
  const int items = nt * (int)per_token.d;
  using Vec = RopeVec<T, V>;
  for (int t = threadIdx.x; t < nt; t += kRopeThreads) {
    const int64_t tok = tok0 + t, b = tok / a.s1;
    base[t] = b * a.stride_b + (tok - b * a.s1) * a.stride_s;
  }
  for (int i = threadIdx.x; i < nt * a.pairs; i += kRopeThreads) {
    const int t = pairs(i), j = i - t * a.pairs;
    const int64_t p = rope_position(a.positions, a.pos64, rope_axis(a.ends, j) * a.tokens + tok0 + t);
    angle[i] = rope_angle(p, a.inv_freq[j], a.sign);
  }
  __syncthreads();
  // first features of a unit's two vectors (the second of the last passing unit may not exist: -1)
  auto place = [&](int u, int& lo, int& hi) {
    if (u < rot) {
      lo = a.offset + (a.interleaved ? 2 * V * u : V * u);
      hi = a.interleaved ? lo + V : lo + a.pairs;
    } else {
      const int k = 2 * (u - rot);
      lo = k * V;
      hi = (k + 1) * V;
      if (lo >= a.offset) lo += 2 * a.pairs;
      if (hi >= a.offset) hi += 2 * a.pairs;
      if (k + 1 >= pass) hi = -1;
    }
  };
  for (int i = threadIdx.x; i < items; i += kRopeThreads) {
    const int t = per_token(i), r = i - t * (int)per_token.d, h = units(r), u = r - h * (int)units.d;
    int fl, fh;
    place(u, fl, fh);
    const T* x = (const T*)a.x + base[t] + h * a.stride_n;
    Vec lo = *reinterpret_cast<const Vec*>(x + fl), hi;
    if (fh >= 0) hi = *reinterpret_cast<const Vec*>(x + fh);
    if (u < rot) {
      const float2* cs = angle + t * a.pairs + V * u;
      auto turn = [&](T& re, T& im, float2 w) {
        const float x = to_f32<T>(re), y = to_f32<T>(im);
        re = from_f32<T>(x * w.x - y * w.y);
        im = from_f32<T>(x * w.y + y * w.x);
      };
      if (V > 1 && a.interleaved) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          turn(lo.v[2 * e], lo.v[2 * e + 1], cs[e]);
          turn(hi.v[2 * e], hi.v[2 * e + 1], cs[V / 2 + e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) turn(lo.v[e], hi.v[e], cs[e]);
      }
    }
    T* y = (T*)a.out + ((tok0 + t) * a.n + h) * a.d;
    *reinterpret_cast<Vec*>(y + fl) = lo;
    if (fh >= 0) *reinterpret_cast<Vec*>(y + fh) = hi;
  }
}

template <typename T, int V>
inline int rope_launch(RopeDev a, cudaStream_t st) {
  const int64_t units = a.pairs / V + ((a.d - 2 * a.pairs) / V + 1) / 2;
  // about 1024 units per block (512: 96 us for the 503 MB above, 1024: 88, 2048: 90), but blocks enough for two on every SM, and tokens and angles that fit the block's arrays
  int64_t t = std::max<int64_t>(1, 4 * kRopeThreads / (a.n * units));
  t = std::min({t, std::max<int64_t>(1, a.tokens / (2 * 148)), (int64_t)std::max(1, kRopeAngles / a.pairs), (int64_t)kRopeTokens});
  a.tokens_per_block = (int32_t)t;
  const int64_t blocks = (a.tokens + t - 1) / t;
  if (blocks > 0x7FFFFFFF) return DSA_ERR_TOO_LARGE;
  if (launch_after(rope_kernel<T, V>, dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a, RopeDiv(a.n * units), RopeDiv(units),
                   RopeDiv(a.pairs)) != cudaSuccess)
    return DSA_ERR_CUDA;
  count_launch();
  return DSA_OK;
}

// ---- append to the paged caches -----------------------------------------------------------------------
struct AppendDev {
  SeqDesc seq;             // seq_k: lengths with the new tokens; token pos of a sequence goes to act_k - act_q + pos
  const void* latent;
  const void* key_rope;
  const void* index_key;   // NULL: no index keys
  const void* norm_weight; // NULL: latents are stored as they are
  const void* positions;   // NULL: a token's position in its sequence; else [axes, tokens]
  const float* inv_freq;   // [32]
  void* latent_cache;
  void* rope_cache;
  void* index_cache;
  int64_t latent_b, latent_s, rope_b, rope_s, index_b, index_s;   // strides in elements (TND: the first is unused)
  int64_t tokens;
  int32_t d, d_index, index_offset;
  int32_t interleaved, index_interleaved, pos64, weight_fp32;
  int32_t ends[3];
  float eps;
};

constexpr int kAppendWarps = 4;   // tokens per block

// Pair j (of lane j) of a 64-wide rotated part: features (2 j, 2 j + 1) or (j, j + 32).
template <typename T>
__device__ __forceinline__ RopeVec<T, 2> rope_pair_load(const T* src, int lane, bool interleaved) {
  if (interleaved) return *reinterpret_cast<const RopeVec<T, 2>*>(src + 2 * lane);
  RopeVec<T, 2> v;
  v.v[0] = src[lane];
  v.v[1] = src[lane + 32];
  return v;
}
template <typename T>
__device__ __forceinline__ void rope_pair_store(RopeVec<T, 2> v, T* dst, int lane, bool interleaved, float2 w) {
  const float x = to_f32<T>(v.v[0]), y = to_f32<T>(v.v[1]);
  v.v[0] = from_f32<T>(x * w.x - y * w.y);
  v.v[1] = from_f32<T>(x * w.y + y * w.x);
  if (interleaved) *reinterpret_cast<RopeVec<T, 2>*>(dst + 2 * lane) = v;
  else { dst[lane] = v.v[0]; dst[lane + 32] = v.v[1]; }
}

// One warp per token: lane j has pair j of the 32 (rope key and index key share the angle), 8 latent features at a time
// for the mean square and the store.  A token without a slot (past its sequence's query length, before position 0, past
// the table, on an absent page or one beyond the cache) writes nothing; every slot that no token goes to keeps what it holds.
template <typename T>
__global__ void __launch_bounds__(kAppendWarps * 32) latent_append_kernel(const AppendDev a) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  if (tok >= a.tokens) return;
  // the token's own data first: the look-ups of where it goes (lengths, block table) take as long
  const bool tnd = a.seq.layout_q == DSA_LAYOUT_TND;
  const int64_t b = tnd ? 0 : tok / a.seq.s1, s = tok - b * a.seq.s1;
  const T* src = (const T*)a.latent + b * a.latent_b + s * a.latent_s;
  RopeVec<T, 8> v[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if ((k * 32 + lane) * 8 < a.d) v[k] = *reinterpret_cast<const RopeVec<T, 8>*>(src + (k * 32 + lane) * 8);
  const T* xr = (const T*)a.key_rope + b * a.rope_b + s * a.rope_s;
  const RopeVec<T, 2> pr = rope_pair_load<T>(xr, lane, a.interleaved != 0);
  RopeVec<T, 2> pi = {};
  const T* xi = (const T*)a.index_key + b * a.index_b + s * a.index_s;
  if (a.index_key != nullptr) pi = rope_pair_load<T>(xi + a.index_offset, lane, a.index_interleaved != 0);
  const float freq = a.inv_freq[lane];
  const RowInfo ri = row_info(a.seq, (int32_t)tok);
  if (ri.pos >= ri.act_q) return;
  const int64_t p = (int64_t)ri.act_k - ri.act_q + ri.pos;
  if (p < 0 || p >= a.seq.s2) return;
  const int64_t row = key_row(a.seq, ri, (int32_t)p);
  if (row < 0) return;
  T* dst = (T*)a.latent_cache + row * a.d;
  {
    const int64_t at = a.positions ? rope_position(a.positions, a.pos64, rope_axis(a.ends, lane) * a.tokens + tok) : p;
    const float2 turn = rope_angle(at, freq, 1.f);
    rope_pair_store<T>(pr, (T*)a.rope_cache + row * 64, lane, a.interleaved != 0, turn);
    if (a.index_key != nullptr) {
      T* yi = (T*)a.index_cache + row * a.d_index;
      rope_pair_store<T>(pi, yi + a.index_offset, lane, a.index_interleaved != 0, turn);
      for (int k = lane * 2; k < a.d_index - 64; k += 64) {
        const int f = k < a.index_offset ? k : k + 64;
        *reinterpret_cast<RopeVec<T, 2>*>(yi + f) = *reinterpret_cast<const RopeVec<T, 2>*>(xi + f);
      }
    }
  }
  if (a.norm_weight != nullptr) {
    float w[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = (k * 32 + lane) * 8;
      if (c >= a.d) continue;
      if (a.weight_fp32) {
        *reinterpret_cast<float4*>(&w[k][0]) = reinterpret_cast<const float4*>((const float*)a.norm_weight + c)[0];
        *reinterpret_cast<float4*>(&w[k][4]) = reinterpret_cast<const float4*>((const float*)a.norm_weight + c)[1];
      } else {
        const RopeVec<T, 8> g = *reinterpret_cast<const RopeVec<T, 8>*>((const T*)a.norm_weight + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[k][e] = to_f32<T>(g.v[e]);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if ((k * 32 + lane) * 8 >= a.d) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float x = to_f32<T>(v[k].v[e]); ss += x * x; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss / (float)a.d + a.eps);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if ((k * 32 + lane) * 8 >= a.d) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k].v[e] = from_f32<T>(to_f32<T>(v[k].v[e]) * r * w[k][e]);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = (k * 32 + lane) * 8;
    if (c < a.d) *reinterpret_cast<RopeVec<T, 8>*>(dst + c) = v[k];
  }
}

}  // namespace dsa
