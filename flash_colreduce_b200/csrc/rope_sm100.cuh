// Norm of queries and keys for each head and position rotation, in one pass.
//
//   y = x * rsqrt(mean_d x_d^2 + eps) * w_d          (without weights: y = x)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t)  t = position * inv_freq[i]
//
// with the pairs (i, i + R/2) of the first R dimensions, or (2i, 2i + 1).  Everything is fp32 and rounded once; the
// angle is the exception: positions reach millions, where a 32-bit product is off by hundredths of a radian, so
// position * inv_freq / 2 pi is formed in 64 bits, reduced to a fraction of a turn there, and only that fraction goes
// to sincospif.
//
// Bound by HBM: each row is read and written once and the arithmetic is about ten operations per element.  Two kernels: rows
// that can be read 16 bytes at a time, and all others.  2 x 16384 tokens of 32 + 8 heads of 128 in bf16: 137 us (4.9 TB/s) with
// the first, 638 us with the second; in fp32 211 us (6.4 TB/s); heads of 80 with 80 or 64 rotated dimensions 130 us, with 40 or 20
// (half of them is no multiple of 8: the second kernel) 550 us; one token of one sequence 2.6 us.
//
// Included by colreduce_sm100.cu.
#pragma once

namespace fcr {

struct RopeParams {
  const void* x[2];        // queries, keys
  void* y[2];              // contiguous (B, heads, M, D)
  const void* weight[2];   // [D] or null
  long long sb[2], sh[2], sm[2];  // strides of x in elements
  int heads[2];
  int B, M, D, half;       // half = number of rotated pairs
  int weight_f32;          // weights are fp32 (else of x's type)
  int interleaved;
  int heads_per_warp;      // vector kernel: heads of a token that one warp takes
  const void* positions;
  int pos_bits;
  long long pos_sb, pos_sm;  // strides of positions in elements
  const float* inv_freq;   // [half]
  float eps;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ long long load_index(const void* p, int bits, long long i) {
  return bits == 64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

// cos and sin of position * inv_freq.  The product in turns is good to 2^-53 of its size; sincospif takes half turns.
__device__ __forceinline__ void rope_turn(long long position, float inv_freq, float& c, float& s) {
  const double turns = (double)position * ((double)inv_freq * 0.15915494309189533577);
  sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
}

// 16 consecutive bytes' worth of values, twice eight values of a lane.
template <typename T>
struct Vec8 {
  uint4 raw[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void rope_load8(const T* x, Vec8<T>& v) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.raw[i] = reinterpret_cast<const uint4*>(x)[i];
}
__device__ __forceinline__ void rope_unpack(const Vec8<float>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = reinterpret_cast<const float*>(v.raw)[i];
}
__device__ __forceinline__ void rope_unpack(const Vec8<__half>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(reinterpret_cast<const __half2*>(v.raw)[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void rope_unpack(const Vec8<__nv_bfloat16>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(v.raw)[i];
    f[2 * i] = __uint_as_float(w << 16);
    f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ void rope_store8(T* y, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(y)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(y)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(f[i]);
    *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(o);
  }
}

// The rows that can be read 16 bytes at a time: D and R multiples of 16, D <= 16 * LPR.  LPR lanes share a row, each with
// two pieces of eight values: the two halves of eight pairs (or 16 neighbours, interleaved or beyond R).  A warp takes
// one token and 32 / LPR of its heads at a time: the token's angles are worked out once, R / 64 per lane, and handed round.
// Blocks are eight neighbouring tokens, so that they write whole stretches of every head.
template <typename T, int LPR, bool INTERLEAVED>
__global__ void __launch_bounds__(256)
rope_vector_kernel(const RopeParams p) {
  constexpr int kHeads = 32 / LPR;            // heads at a time
  constexpr int K = LPR / 4;                  // angles per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.heads[0] + p.heads[1];
  const int chunks = (heads + p.heads_per_warp - 1) / p.heads_per_warp;
  const long long token = (long long)(blockIdx.x / chunks) * 8 + warp;
  if (token >= (long long)p.B * p.M) return;
  const int chunk = blockIdx.x % chunks;
  const long long b = token / p.M, m = token - b * p.M;
  const int l = lane % LPR;
  const bool on = 16 * l < p.D;
  const bool rotated = l < p.half / 8;        // 16 of the R rotated dimensions
  const int d0 = INTERLEAVED || !rotated ? 16 * l : 8 * l, d1 = INTERLEAVED || !rotated ? 16 * l + 8 : p.half + 8 * l;
  const int h_lo = chunk * p.heads_per_warp, h_hi = min(heads, h_lo + p.heads_per_warp);
  // rows of this warp, two at a time: their loads go out before the angles are worked out
  Vec8<T> va[2], vb[2];
  auto load = [&](int h, int u) {
    if (h < h_hi && on) {
      const int which = h >= p.heads[0], hh = which ? h - p.heads[0] : h;
      const T* x = reinterpret_cast<const T*>(p.x[which]) + b * p.sb[which] + hh * p.sh[which] + m * p.sm[which];
      rope_load8(x + d0, va[u]);
      rope_load8(x + d1, vb[u]);
    }
  };
  int h = h_lo + lane / LPR;
  load(h, 0);
  load(h + kHeads, 1);
  const long long pos = load_index(p.positions, p.pos_bits, b * p.pos_sb + m * p.pos_sm);
  float ck[K], sk[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int f = lane * K + k;
    ck[k] = 1.f;
    sk[k] = 0.f;
    if (f < p.half) rope_turn(pos, p.inv_freq[f], ck[k], sk[k]);
  }
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {  // pair 8 l + j
    const int from = (8 * l + j) / K;
    c[j] = __shfl_sync(0xffffffffu, ck[j % K], from & 31);
    s[j] = __shfl_sync(0xffffffffu, sk[j % K], from & 31);
  }
  const float inv_d = 1.f / (float)p.D;
  for (int h0 = h_lo; h0 < h_hi; h0 += 2 * kHeads) {
#pragma unroll
    for (int u = 0; u < 2; ++u, h += kHeads) {
      float a[8], e[8];
      rope_unpack(va[u], a);
      rope_unpack(vb[u], e);
      load(h + 2 * kHeads, u);
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(a[j], a[j], fmaf(e[j], e[j], sq));
      if (!on) sq = 0.f;
#pragma unroll
      for (int o = LPR / 2; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      if (h >= h_hi || !on) continue;
      const int which = h >= p.heads[0], hh = which ? h - p.heads[0] : h;
      const void* w = p.weight[which];
      if (w) {
        const float inv = rsqrtf(fmaf(sq, inv_d, p.eps));
        float wa[8], we[8];
        if (p.weight_f32) {
          Vec8<float> r0, r1;
          rope_load8(reinterpret_cast<const float*>(w) + d0, r0);
          rope_load8(reinterpret_cast<const float*>(w) + d1, r1);
          rope_unpack(r0, wa);
          rope_unpack(r1, we);
        } else {
          Vec8<T> r0, r1;
          rope_load8(reinterpret_cast<const T*>(w) + d0, r0);
          rope_load8(reinterpret_cast<const T*>(w) + d1, r1);
          rope_unpack(r0, wa);
          rope_unpack(r1, we);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] = a[j] * inv * wa[j];
          e[j] = e[j] * inv * we[j];
        }
      }
      if (rotated) {
        if (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a0 = a[2 * j], a1 = a[2 * j + 1], e0 = e[2 * j], e1 = e[2 * j + 1];
            a[2 * j] = a0 * c[j] - a1 * s[j];
            a[2 * j + 1] = a0 * s[j] + a1 * c[j];
            e[2 * j] = e0 * c[4 + j] - e1 * s[4 + j];
            e[2 * j + 1] = e0 * s[4 + j] + e1 * c[4 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = a[j], y = e[j];
            a[j] = x * c[j] - y * s[j];
            e[j] = x * s[j] + y * c[j];
          }
        }
      }
      T* y = reinterpret_cast<T*>(p.y[which]) + ((b * p.heads[which] + hh) * p.M + m) * p.D;
      rope_store8(y + d0, a);
      rope_store8(y + d1, e);
    }
  }
}

// One warp per row of any layout: D <= 256, any strides, R <= D.
template <typename T>
__global__ void __launch_bounds__(256)
rope_rows_kernel(const RopeParams p) {
  __shared__ float row_s[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.heads[0] + p.heads[1];
  const long long rows = (long long)p.B * p.M * heads;
  float* row = row_s[warp];
  for (long long r = (long long)blockIdx.x * 8 + warp; r < rows; r += (long long)gridDim.x * 8) {
    const long long token = r / heads;
    int h = (int)(r - token * heads);
    const long long b = token / p.M, m = token - b * p.M;
    const int which = h >= p.heads[0];
    if (which) h -= p.heads[0];
    const T* x = reinterpret_cast<const T*>(p.x[which]) + b * p.sb[which] + h * p.sh[which] + m * p.sm[which];
    float v[8], sq = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      v[j] = d < p.D ? to_f32(x[d]) : 0.f;
      sq = fmaf(v[j], v[j], sq);
    }
    const void* w = p.weight[which];
    if (w) {
#pragma unroll
      for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const float inv = rsqrtf(sq / (float)p.D + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = lane + 32 * j;
        if (d < p.D) v[j] = v[j] * inv * (p.weight_f32 ? reinterpret_cast<const float*>(w)[d] : to_f32(reinterpret_cast<const T*>(w)[d]));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) row[lane + 32 * j] = v[j];
    __syncwarp();
    T* y = reinterpret_cast<T*>(p.y[which]) + ((b * p.heads[which] + h) * p.M + m) * p.D;
    const long long pos = load_index(p.positions, p.pos_bits, b * p.pos_sb + m * p.pos_sm);
    for (int i = lane; i < p.half; i += 32) {
      float c, s;
      rope_turn(pos, p.inv_freq[i], c, s);
      const int d0 = p.interleaved ? 2 * i : i, d1 = p.interleaved ? 2 * i + 1 : i + p.half;
      const float a = row[d0], e = row[d1];
      y[d0] = from_f32<T>(a * c - e * s);
      y[d1] = from_f32<T>(a * s + e * c);
    }
    for (int d = 2 * p.half + lane; d < p.D; d += 32) y[d] = from_f32<T>(row[d]);
    __syncwarp();
  }
}

}  // namespace fcr
