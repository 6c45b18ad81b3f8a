// A KV cache (B, H, N, D) in 16 bits, e4m3 or int8: rows are quantised as they are written and read back whole or at
// selected positions.
//
// A row x of D values (one token, one head, K or V) is held as codes c_d and one scale 2^e:
//
//   a = max_d |x_d|,   e = max(-127, ceil(log2(a / top))),   c_d = rne(x_d * 2^-e),   top = 448 (e4m3) or 127 (int8)
//
// The scale is a power of two, held as one E8M0 byte (e + 127).  It costs e4m3 nothing (the codes float) and int8 half a
// bit on average, and in return the division is exact, the code is the nearest one in every precision, and code * 2^e
// has at most 8 significant bits: reading a row back in the type it was written from is exact, and so is writing it
// again.  Values whose code * 2^e would pass the type's largest finite value are clamped to the largest that does not.
// A row that holds a NaN or an infinity has scale byte 255, E8M0's NaN, and reads back as NaN.
//
// Bound by HBM: 2 D bytes in and D + 1 out to write a row, the reverse to read one.
//
// Included by colreduce_sm100.cu after rope_sm100.cuh.
#pragma once
#include <cuda_fp8.h>

namespace fcr {

struct KvTensor {
  void* data;
  unsigned char* scales;  // null for 16-bit formats
  long long sb, sh, sn;   // strides of data in elements
  long long ssb, ssh, ssn;
};

struct KvAppendParams {
  KvTensor t[2];           // K, V
  const void* x[2];
  long long xb[2], xh[2], xm[2];
  int B, H, N, D, M;
  int group;               // lanes per row: the power of two that covers D in steps of 8
  const void* lengths;
  const void* counts;      // null: all M tokens
  int index_bits;
};

struct KvReadParams {
  KvTensor t[2];
  void* y[2];              // contiguous (B, H, n, D)
  int B, H, N, D, n;
  int group;
  const void* positions;   // (B, H, n) contiguous or null: 0 .. n-1
  int index_bits;
};

// Smallest e with a <= top * 2^e, at least -127; top = 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8).  a is finite.
template <int FORMAT>
__device__ __forceinline__ int kv_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int t = (int)(u >> 23) - 127;
  const uint32_t mant = u & 0x7fffffu;
  const int e = FORMAT == FCR_KV_FP8 ? t - 8 + (mant > 0x600000u) : t - 6 + (mant > 0x7e0000u);
  return max(e, -127);
}
// 2^e for e in [-127, 127]; -127 is a subnormal.
__device__ __forceinline__ float kv_pow2(int e) {
  return __uint_as_float(e == -127 ? 0x00400000u : (uint32_t)(e + 127) << 23);
}
// The scale a byte stands for.
__device__ __forceinline__ float kv_scale(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : kv_pow2((int)byte - 127);
}

// Eight 16-bit values as fp32.
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8], __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(h[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8], __nv_bfloat16) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four codes of a word as fp32.
template <int FORMAT>
__device__ __forceinline__ void unpack_codes4(uint32_t w, float* v) {
  if (FORMAT == FCR_KV_FP8) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * j)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  } else {
    // byte + 128 under the exponent of 2^23 is the float 2^23 + 128 + code
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + j)) - 8388736.f;
  }
}

// Largest magnitude whose code * 2^e stays finite in the type: 1.875 * 2^top (e4m3, 4 bits) or 1.96875 * 2^top (6 bits).
template <typename T, int FORMAT>
__device__ __forceinline__ float kv_largest() {
  const float m = FORMAT == FCR_KV_FP8 ? 1.875f : 1.96875f;
  return sizeof(T) == 2 && std::is_same<T, __half>::value ? m * 32768.f : m * 1.7014118346046923e38f;
}

// Both kernels: a block takes kKvRows rows per lane group of one (K or V, sequence, head); `group` lanes per row, eight
// consecutive values each.  A thread's rows are read together, so that four loads are under way.  2 x 8 heads of 32768 tokens,
// D = 128, e4m3: 111 us to write (3.6 TB/s, short of the memory's rate by the quantiser's instructions, about 100 per eight
// values) and 71 us to read (5.7 TB/s); int8 118 and 81; 16 bits 83 each (6.5 TB/s).  For both in e4m3, 181 us: two rows per
// thread take 234, eight 186, one with its place found by 64-bit divisions 295.
constexpr int kKvRows = 4;
struct KvPlace {
  int kv, b, h, row0, step;  // first row of this thread, distance to its next
};
__device__ __forceinline__ KvPlace kv_place(int B, int H, int group) {
  // neighbouring blocks take the same rows of all heads, which lie side by side in a projection's output
  const int combos = 2 * B * H, block = blockIdx.x / combos, combo = blockIdx.x - block * combos;
  KvPlace r;
  r.kv = combo / (B * H);
  const int bh = combo - r.kv * (B * H);
  r.b = bh / H;
  r.h = bh - r.b * H;
  r.step = (int)blockDim.x / group;
  r.row0 = block * r.step * kKvRows + (int)threadIdx.x / group;
  return r;
}

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256)
kv_append_kernel(const __grid_constant__ KvAppendParams p) {
  const int group = p.group;
  const int gl = threadIdx.x & (group - 1), d0 = gl * 8;
  const bool on = d0 < p.D;
  const KvPlace at = kv_place(p.B, p.H, group);
  const KvTensor& t = p.t[at.kv];
  const T* x = reinterpret_cast<const T*>(p.x[at.kv]) + at.b * p.xb[at.kv] + at.h * p.xh[at.kv] + d0;
  // (the rows are read whether they will be written or not: the loads need not wait for the lengths)
  uint4 raw[kKvRows];
#pragma unroll
  for (int u = 0; u < kKvRows; ++u) {
    const int m = at.row0 + u * at.step;
    raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (m < p.M && on) {
      if (VEC) {
        raw[u] = *reinterpret_cast<const uint4*>(x + m * p.xm[at.kv]);
      } else {
        unsigned short e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = d0 + j < p.D ? reinterpret_cast<const unsigned short*>(x + m * p.xm[at.kv])[j] : (unsigned short)0;
        raw[u] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
      }
    }
  }
  const long long first = load_index(p.lengths, p.index_bits, at.b);
  // tokens that are written: m < count, and their positions exist
  long long count = p.counts ? min(load_index(p.counts, p.index_bits, at.b), (long long)p.M) : p.M;
  count = first < 0 ? 0 : min(count, (long long)p.N - first);
#pragma unroll
  for (int u = 0; u < kKvRows; ++u) {
    const int m = at.row0 + u * at.step;
    const bool live = m < count;
    const long long n = first + m;
    if (FORMAT == FCR_KV_16BIT) {
      if (live && on) {
        unsigned short* y = reinterpret_cast<unsigned short*>(t.data) + at.b * t.sb + at.h * t.sh + n * t.sn + d0;
        if (VEC) {
          *reinterpret_cast<uint4*>(y) = raw[u];
        } else {
          const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (d0 + j < p.D) y[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
        }
      }
      continue;
    }
    float v[8];
    unpack8(raw[u], v, T());
    // the largest magnitude by its bits: a NaN or infinity is then larger than every finite value
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    for (int o = group >> 1; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    const bool fine = top < 0x7f800000u;
    const int e = fine ? kv_exponent<FORMAT>(__uint_as_float(top)) : 128;
    // exact: 2^-e is a float (e >= -127), and a product too small for the format's grid rounds to zero either way
    const float inv = fine ? kv_pow2(-e) : 0.f;
    const float lim = kv_largest<T, FORMAT>();
    uint32_t code[2] = {0u, 0u};
    if (fine) {
      if (__uint_as_float(top) > lim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -lim), lim);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv;
      if (FORMAT == FCR_KV_FP8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * j], v[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
          code[j >> 1] |= two << (16 * (j & 1));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) code[j >> 2] |= ((uint32_t)__float2int_rn(v[j]) & 255u) << (8 * (j & 3));
      }
    }
    if (on) {
      unsigned char* y = reinterpret_cast<unsigned char*>(t.data) + at.b * t.sb + at.h * t.sh + n * t.sn + d0;
      if (VEC) {
        *reinterpret_cast<uint2*>(y) = make_uint2(code[0], code[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d0 + j < p.D) y[j] = (unsigned char)(code[j >> 2] >> (8 * (j & 3)));
      }
    }
    if (gl == 0) t.scales[at.b * t.ssb + at.h * t.ssh + n * t.ssn] = (unsigned char)(e + 127);
  }
}

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256)
kv_read_kernel(const __grid_constant__ KvReadParams p) {
  const int group = p.group;
  const int gl = threadIdx.x & (group - 1), d0 = gl * 8;
  if (d0 >= p.D) return;
  const KvPlace at = kv_place(p.B, p.H, group);
  const KvTensor& t = p.t[at.kv];
  const long long row_base = ((long long)at.b * p.H + at.h) * p.n;
  const long long data_base = at.b * t.sb + at.h * t.sh + d0, scale_base = at.b * t.ssb + at.h * t.ssh;
  constexpr int kWords = FORMAT == FCR_KV_16BIT ? 4 : 2;
  long long pos[kKvRows];
  uint32_t raw[kKvRows][kWords];
  uint32_t byte[kKvRows];
#pragma unroll
  for (int u = 0; u < kKvRows; ++u) {
    const int i = at.row0 + u * at.step;
    pos[u] = -1;
    if (i < p.n) pos[u] = p.positions ? load_index(p.positions, p.index_bits, row_base + i) : i;
  }
#pragma unroll
  for (int u = 0; u < kKvRows; ++u) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) raw[u][j] = 0u;
    byte[u] = 127u;
    if (pos[u] >= 0 && pos[u] < p.N) {
      const long long from = data_base + pos[u] * t.sn;
      if (FORMAT == FCR_KV_16BIT) {
        const unsigned short* x = reinterpret_cast<const unsigned short*>(t.data) + from;
        if (VEC) {
          const uint4 q = *reinterpret_cast<const uint4*>(x);
          raw[u][0] = q.x, raw[u][1] = q.y, raw[u][kWords - 2] = q.z, raw[u][kWords - 1] = q.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (d0 + j < p.D) raw[u][(j >> 1) % kWords] |= (uint32_t)x[j] << (16 * (j & 1));
        }
      } else {
        const unsigned char* x = reinterpret_cast<const unsigned char*>(t.data) + from;
        if (VEC) {
          const uint2 q = *reinterpret_cast<const uint2*>(x);
          raw[u][0] = q.x, raw[u][1] = q.y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (d0 + j < p.D) raw[u][(j >> 2) % kWords] |= (uint32_t)x[j] << (8 * (j & 3));
        }
        byte[u] = t.scales[scale_base + pos[u] * t.ssn];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kKvRows; ++u) {
    const int i = at.row0 + u * at.step;
    if (i >= p.n) continue;
    uint32_t o[4];
    if constexpr (FORMAT == FCR_KV_16BIT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = raw[u][j];
    } else {
      const float s = kv_scale(byte[u]);
      float v[8];
      unpack_codes4<FORMAT>(raw[u][0], v);
      unpack_codes4<FORMAT>(raw[u][1], v + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = pack2(v[2 * j] * s, v[2 * j + 1] * s, T());
    }
    unsigned short* y = reinterpret_cast<unsigned short*>(p.y[at.kv]) + (row_base + i) * p.D + d0;
    if (VEC) {
      *reinterpret_cast<uint4*>(y) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (d0 + j < p.D) y[j] = (unsigned short)(o[j >> 1] >> (16 * (j & 1)));
    }
  }
}

}  // namespace fcr
