// Attention of M drafted tokens per sequence over a KV cache: the tokens attend the sequence's first lengths[b]
// cached positions, and of the drafted tokens themselves, which lie in the cache at lengths[b] .. lengths[b] + M - 1,
// those that a mask names.
//
//   S_ij = q_i . k_j * scale,   out_i = sum_j softmax_j(S_ij) v_j,   lse_i = log sum_j exp(S_ij)
//
// A row that attends nothing has out = 0 and lse = -inf.
//
// Included by colreduce_sm100.cu after kvcache_sm100.cuh.
#pragma once

namespace fcr {

struct TreeParams {
  const void* q;
  const void* cache[2];    // K, V
  const unsigned char* scales[2];
  const void* lengths;
  const unsigned char* mask;
  void* out;
  float* lse;
  long long qb, qh, qm;
  long long cb[2], ch[2], cn[2];
  long long sb[2], sh[2], sn[2];
  long long mask_b, mask_m;
  int B, Hq, Hk, M, N, D, G;
  int index_bits;
  float scale2;            // scale * log2(e)
};

template <typename T, int FORMAT>
__device__ __forceinline__ float tree_load(const TreeParams& p, int which, int b, int h, long long n, int d) {
  const long long at = b * p.cb[which] + h * p.ch[which] + n * p.cn[which] + d;
  if (FORMAT == FCR_KV_16BIT) return to_f32(reinterpret_cast<const T*>(p.cache[which])[at]);
  const uint32_t byte = reinterpret_cast<const unsigned char*>(p.cache[which])[at];
  float v[4];
  unpack_codes4<FORMAT>(byte, v);
  return v[0] * kv_scale(p.scales[which][b * p.sb[which] + h * p.sh[which] + n * p.sn[which]]);
}

// One warp per query row.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(128)
tree_rows_kernel(const TreeParams p) {
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)p.B * p.Hq * p.M;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int m = (int)(r % p.M);
  const int h = (int)(r / p.M % p.Hq), b = (int)(r / p.M / p.Hq);
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.qb + h * p.qh + m * p.qm;
  float qv[4], o[4], mx = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 32 * j;
    qv[j] = d < p.D ? to_f32(q[d]) * p.scale2 : 0.f;
    o[j] = 0.f;
  }
  const long long have = max(0LL, min(load_index(p.lengths, p.index_bits, b), (long long)p.N));
  const long long end = min(have + p.M, (long long)p.N);
  for (long long n = 0; n < end; ++n) {
    if (n >= have) {
      const int j = (int)(n - have);
      if (p.mask ? !p.mask[b * p.mask_b + m * p.mask_m + j] : j > m) continue;
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 32 * j;
      if (d < p.D) s = fmaf(qv[j], tree_load<T, FORMAT>(p, 0, b, h / p.G, n, d), s);
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    const float m_new = fmaxf(mx, s);
    const float at = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(mx - at), w = exp2f(s - at);
    l = l * alpha + w;
    mx = m_new;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 32 * j;
      if (d < p.D) o[j] = o[j] * alpha + w * tree_load<T, FORMAT>(p, 1, b, h / p.G, n, d);
    }
  }
  T* out = reinterpret_cast<T*>(p.out) + r * p.D;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 32 * j;
    if (d < p.D) out[d] = from_f32<T>(l == 0.f ? 0.f : o[j] / l);
  }
  if (p.lse && lane == 0) p.lse[r] = l == 0.f ? -INFINITY : (mx + log2f(l)) * 0.69314718055994531f;
}

}  // namespace fcr
