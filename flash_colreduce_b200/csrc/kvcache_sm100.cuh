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

// `group` lanes per row, 8 consecutive values each.  A row's K and V, tokens, heads and sequences are all one index.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256)
kv_append_kernel(const KvAppendParams p) {
  const int group = p.group;
  const int gl = threadIdx.x & (group - 1);
  const long long rows = 2LL * p.B * p.H * p.M;
  const int d0 = gl * 8;
  const bool on = d0 < p.D;
  const long long per_block = blockDim.x / group;
  const long long stride = (long long)gridDim.x * per_block;
  // every lane of a warp makes the same number of trips: the shuffles below need them all
  for (long long base = (long long)blockIdx.x * per_block; base < rows; base += stride) {
    const long long r = base + threadIdx.x / group;
    bool live = r < rows;
    long long rest = live ? r : 0;
    const long long m = rest % p.M;
    rest /= p.M;
    const int h = (int)(rest % p.H);
    rest /= p.H;
    const int b = (int)(rest % p.B), kv = (int)(rest / p.B);
    long long n = -1;
    if (live) {
      n = load_index(p.lengths, p.index_bits, b);
      if (n < 0 || (p.counts && m >= load_index(p.counts, p.index_bits, b))) live = false;
      n += m;
      if (n >= p.N) live = false;
    }
    const T* x = reinterpret_cast<const T*>(p.x[kv]) + b * p.xb[kv] + h * p.xh[kv] + m * p.xm[kv] + d0;
    const KvTensor& t = p.t[kv];
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (live && on) {
      if (VEC) {
        raw = *reinterpret_cast<const uint4*>(x);
      } else {
        unsigned short* e = reinterpret_cast<unsigned short*>(&raw);
        for (int j = 0; j < 8; ++j) e[j] = d0 + j < p.D ? reinterpret_cast<const unsigned short*>(x)[j] : (unsigned short)0;
      }
    }
    if (FORMAT == FCR_KV_16BIT) {
      if (live && on) {
        T* y = reinterpret_cast<T*>(t.data) + b * t.sb + h * t.sh + n * t.sn + d0;
        if (VEC)
          *reinterpret_cast<uint4*>(y) = raw;
        else
          for (int j = 0; j < 8 && d0 + j < p.D; ++j) y[j] = reinterpret_cast<const T*>(&raw)[j];
      }
      continue;
    }
    float v[8];
    unpack8(raw, v, T());
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
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -lim), lim) * inv;
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
      unsigned char* y = reinterpret_cast<unsigned char*>(t.data) + b * t.sb + h * t.sh + n * t.sn + d0;
      if (VEC)
        *reinterpret_cast<uint2*>(y) = make_uint2(code[0], code[1]);
      else
        for (int j = 0; j < 8 && d0 + j < p.D; ++j) y[j] = (unsigned char)(code[j >> 2] >> (8 * (j & 3)));
    }
    if (gl == 0) t.scales[b * t.ssb + h * t.ssh + n * t.ssn] = (unsigned char)(e + 127);
  }
}

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(256)
kv_read_kernel(const KvReadParams p) {
  const int group = p.group;
  const int gl = threadIdx.x & (group - 1);
  const long long rows = 2LL * p.B * p.H * p.n;
  const int d0 = gl * 8;
  if (d0 >= p.D) return;
  const long long per_block = blockDim.x / group;
  for (long long r = (long long)blockIdx.x * per_block + threadIdx.x / group; r < rows; r += (long long)gridDim.x * per_block) {
    long long rest = r;
    const long long i = rest % p.n;
    rest /= p.n;
    const int h = (int)(rest % p.H);
    rest /= p.H;
    const int b = (int)(rest % p.B), kv = (int)(rest / p.B);
    const KvTensor& t = p.t[kv];
    const long long row = ((long long)b * p.H + h) * p.n + i;
    const long long pos = p.positions ? load_index(p.positions, p.index_bits, row) : i;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (pos >= 0 && pos < p.N) {
      const long long at = b * t.sb + h * t.sh + pos * t.sn + d0;
      if (FORMAT == FCR_KV_16BIT) {
        const unsigned short* x = reinterpret_cast<const unsigned short*>(t.data) + at;
        if (VEC)
          raw = *reinterpret_cast<const uint4*>(x);
        else
          for (int j = 0; j < 8 && d0 + j < p.D; ++j) reinterpret_cast<unsigned short*>(&raw)[j] = x[j];
      } else {
        const unsigned char* x = reinterpret_cast<const unsigned char*>(t.data) + at;
        uint2 c = make_uint2(0u, 0u);
        if (VEC)
          c = *reinterpret_cast<const uint2*>(x);
        else
          for (int j = 0; j < 8 && d0 + j < p.D; ++j) reinterpret_cast<unsigned char*>(&c)[j] = x[j];
        const float s = kv_scale(t.scales[b * t.ssb + h * t.ssh + pos * t.ssn]);
        float v[8];
        unpack_codes4<FORMAT>(c.x, v);
        unpack_codes4<FORMAT>(c.y, v + 4);
        uint32_t* o = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = pack2(v[2 * j] * s, v[2 * j + 1] * s, T());
      }
    }
    T* y = reinterpret_cast<T*>(p.y[kv]) + row * p.D + d0;
    if (VEC)
      *reinterpret_cast<uint4*>(y) = raw;
    else
      for (int j = 0; j < 8 && d0 + j < p.D; ++j) reinterpret_cast<unsigned short*>(y)[j] = reinterpret_cast<const unsigned short*>(&raw)[j];
  }
}

}  // namespace fcr
