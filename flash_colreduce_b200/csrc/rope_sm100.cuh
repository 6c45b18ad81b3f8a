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
// Bound by HBM: each row is read and written once and the arithmetic is about ten operations per element.
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
  int heads_per_warp;      // fast kernel: heads of a token that one warp takes
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
