// Attention of M drafted tokens per sequence over a KV cache: the tokens attend the sequence's first lengths[b]
// cached positions, and of the drafted tokens themselves, which lie in the cache at lengths[b] .. lengths[b] + M - 1,
// those that a mask names.
//
//   S_ij = q_i . k_j * scale,   out_i = sum_j softmax_j(S_ij) v_j,   lse_i = log sum_j exp(S_ij)
//
// A row that attends nothing has out = 0 and lse = -inf.
//
// The G query heads of a key head and their M tokens are G * M rows that read the same keys.  One CTA runs a row tile
// of them against a run of 128-key tiles:
//
//   S = Q K^T    tcgen05, 128 rows x 128 keys, fp32 in tensor memory
//   P = 2^(S * scale * log2 e - m)   one thread per row, 16 bits, back to tensor memory over S
//   O += P V     tcgen05, A = P from tensor memory, B = V as it lies in the cache (rows are the K dimension)
//
// with m a reference that follows the running maximum only when that has grown by more than 2^8: O is then rescaled in
// tensor memory, otherwise the loop carries no correction.  For fp16 the reference is kept 7 below the maximum it follows, so that
// a row's largest weight lies in 2^7 .. 2^15: fp16 keeps 11 bits down to 2^-14 only and nothing below 2^-25, and many small
// weights add up.  What is lost of a row is at most 2^-32 of its sum per key.  Two warpgroups take turns, so that the exponentials of one
// tile run under the products of the other.  With more than 128 rows (PAIR) they are two row tiles over the same keys;
// with 65 to 128, two runs of keys (every other tile) whose results are merged.  Up to 64 rows treedecode_sm100.cuh takes.
//
// The key tiles of all rows of all sequences are one line that the CTAs share equally (plan.h), so ragged lengths cost
// nothing and a single long sequence uses every SM.  A piece that covers a group's keys only in part leaves its
// (m, l, O) in the workspace and tree_combine_kernel joins them, in the order of the keys.
//
// A cache in 8 bits: TMA brings the codes, one warp the scales, and eight warps turn code * 2^e into 16 bits (exactly) and write
// the swizzled tile that TMA writes for a 16-bit cache.  Multiplying codes as they are (kind::f8f6f4) would need the queries and
// the weights in 8 bits.
//
// What bounds it: 64 tokens of 8 sequences over 8 heads of up to 16384 bf16 keys (256 rows per head) take 145 us against 54 of
// the tensor cores: a warpgroup's exponentials (3400 cycles per tile, in two passes over tensor memory) and its two products
// follow one another, and the other warpgroup's products hide only part of that.
//
// Masked scores are selected away, so NaN in masked keys is harmless; a masked value is not, being multiplied by zero,
// so values behind the last drafted token are zeroed and non-finite ones among the drafted tokens too; a row that does attend such
// a token gets it back in the epilogue.
//
// Included by colreduce_sm100.cu after kvcache_sm100.cuh.
#pragma once

namespace fcr {

constexpr int kTreeMaxM = 256;        // drafted tokens per sequence
constexpr int kTreeSoftmaxWarps = 8;  // two warpgroups
constexpr int kTreeMmaWarp = 8;       // two warps, one per warpgroup
constexpr int kTreeQWarp = 10;        // first of those that bring the queries
template <bool QUANT>
__host__ __device__ constexpr int tree_q_warps() { return QUANT ? 1 : 4; }  // with an 8-bit cache one, which brings its scales too
// then TMA, and for an 8-bit cache the warps that convert codes
constexpr int kTreeConvertWarps = 8;
constexpr int kTreeConvertWarpsOf = kTreeConvertWarps / 2;  // for the keys, and for the values
template <bool QUANT>
constexpr int tree_threads() { return 32 * (kTreeQWarp + tree_q_warps<QUANT>() + 1 + (QUANT ? kTreeConvertWarps : 0)); }

enum {
  ST_TR_WAIT_Q_EMPTY = 87,
  ST_TR_WAIT_K_EMPTY = 88,
  ST_TR_WAIT_V_EMPTY = 89,
  ST_TR_WAIT_Q_FULL = 90,
  ST_TR_WAIT_K_FULL = 75,
  ST_TR_WAIT_V_FULL = 76,
  ST_TR_WAIT_P = 77,
  ST_TR_WAIT_S = 78,
  ST_TR_WAIT_O = 79,
  ST_TR_WAIT_MERGE = 80,
  ST_TR_WAIT_V_FULL_SM = 81,
  ST_TR_WAIT_DRAIN = 82,
  ST_TR_WAIT_C_EMPTY = 83,
  ST_TR_WAIT_C_FULL = 84,
  ST_TR_WAIT_SC_EMPTY = 85,
  ST_TR_WAIT_SC_FULL = 86,
};

// A bounded wait as elsewhere, but with its loop out of line.  These kernels have up to seven kinds of warps, and the code
// that is running must fit the instruction cache: with the loops inline and the converters unrolled 44 % of its
// requests missed, warps waited for instructions nearly as much as for data (4.8 against 5.4 of them at each issue), and a
// change of a few instructions anywhere moved the time of 16 x 8 heads of 4096 int8 keys between 82 and 129 us; it is 58 now, with 9 % misses.
__device__ __noinline__ bool tree_wait_loop(uint32_t bar, uint32_t parity, volatile int* abort_flag, const WaitParams* p, int code, int bounds) {
  const long long t0 = clock64();
  while (true) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
    const bool late = clock64() - t0 > bounds * p->wait_limit;
    if (__any_sync(0xffffffffu, late || *abort_flag != 0)) {
      if (late && *abort_flag == 0) {
        *abort_flag = 1;
        report_status(*p, code, (int)parity);
      }
      __syncwarp();
      return false;
    }
  }
}
__device__ __forceinline__ bool tree_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const WaitParams& p, int code, int bounds) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  return tree_wait_loop(bar, parity, abort_flag, &p, code, bounds);
}
#define TREE_WAIT(bar, par, code) tree_wait(bar, par, abort_flag, p, code, 1)
#define TREE_WAIT_BEHIND(bar, par, code) tree_wait(bar, par, abort_flag, p, code, 2)

struct TreeParams : WaitParams {
  const void* q;
  const void* cache[2];             // K, V
  const unsigned char* scales[2];
  const void* lengths;
  const uint32_t* mask;             // packed (mask_rows, M, words); null: a chain
  void* out;
  float* lse;
  float* part_o;                    // [ctas][2][part_rows][DPAD]
  float2* part_ml;                  // [ctas][2][part_rows]
  long long qb, qh, qm;
  long long cb[2], ch[2], cn[2];    // 8-bit cache: byte strides
  long long sb[2], sh[2], sn[2];
  int B, Hq, Hk, M, N, D, G, rows;  // rows = G * M
  int row_tiles, groups;            // groups = Hk * row_tiles
  int part_rows;
  int words, mask_shared;
  int index_bits;
  float scale2;                     // |scale| * log2(e)
  uint32_t idesc_s, idesc_o;
  int k_steps;                      // 32-byte steps of a key row that hold data
  int skip_ring_load;
};

struct TreeLengths {
  const void* p;
  int bits;
  FCR_HD long long operator()(int b) const {
    return bits == 64 ? reinterpret_cast<const long long*>(p)[b] : (long long)reinterpret_cast<const int*>(p)[b];
  }
};

template <int DPAD, bool PAIR, bool QUANT>
struct TreeSmem {
  static constexpr int kTileBytes = 128 * DPAD * 2;
  static constexpr int kSlabBytes = 128 * 128;
  static constexpr int kQBuffers = PAIR ? 1 : 2;
  // a query buffer doubles as the space in which the two warpgroups merge: 256 lanes x 32 columns of fp32
  static constexpr int kQBytes = PAIR ? 2 * kTileBytes : 32768;
  // Key and value tiles in flight.  Where the warpgroups take turns the numbers are even: a slot then always belongs to the
  // same warpgroup, which sees every phase of its barriers.
  static constexpr int KS = DPAD == 64 ? (QUANT ? 2 : 4) : (QUANT || !PAIR ? 2 : 3);
  static constexpr int VS = DPAD == 64 ? (QUANT ? 2 : 4) : 2;
  static constexpr int SS = QUANT ? (DPAD == 64 ? 8 : 2) : 0;               // tiles of codes in flight
  static_assert(PAIR || (KS % 2 == 0 && VS % 2 == 0), "see above");
  static constexpr int off_q = 0;
  static constexpr int off_k = off_q + kQBuffers * kQBytes;
  static constexpr int off_v = off_k + KS * kTileBytes;
  static constexpr int off_codes = off_v + VS * kTileBytes;
  static constexpr int off_stat = off_codes + SS * 128 * DPAD;  // float2 [256]; PAIR keeps none, scale bytes then lie there
  static constexpr int off_scales = PAIR ? off_stat : off_stat + 2048;
  static constexpr int off_bars = off_stat + 2048 + (PAIR || !QUANT ? 0 : 520);
  static constexpr int kNumBars = 4 + 2 * KS + 2 * VS + 2 + 2 + 2 + 1 + (QUANT ? 2 * SS + 4 : 0);
  static constexpr int off_misc = off_bars + 8 * kNumBars;
  static constexpr int kDynamicBytes = off_misc + 48;
  static_assert(kDynamicBytes <= 232448, "exceeds the 227 KB shared memory of an sm_100 CTA");
};

// Bits of the keys n0 .. n0 + 31 that row m attends.
__device__ __noinline__ uint32_t tree_bits(const TreeParams& p, const uint32_t* words, int m, int n0, int have, int end) {
  if (n0 + 32 <= have) return 0xffffffffu;
  if (n0 >= end) return 0u;
  const int j0 = n0 - have;  // place of the first key among the drafted tokens, negative: cached positions come first
  uint32_t bits;
  if (words == nullptr) {
    const int last = m - j0;  // attended: bit <= last
    bits = last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u;
  } else {
    const int first = max(j0, 0), w = first >> 5;
    const uint32_t lo = words[w], hi = w + 1 < p.words ? words[w + 1] : 0u;
    bits = __funnelshift_r(lo, hi, first & 31);
    if (j0 < 0) bits = bits << -j0 | ((1u << -j0) - 1u);
  }
  if (n0 + 32 > end) bits &= (1u << (end - n0)) - 1u;
  return bits;
}

// log2 of the weight that a row's largest score gets when the reference moves.
template <typename T>
__host__ __device__ constexpr float tree_aim() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

template <typename T>
__device__ __forceinline__ bool non_finite16(uint32_t h) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (h & kExp) == kExp;
}

// Sixteen codes times 2^(byte - 127), exactly, as eight words of two 16-bit values.  The short form holds for the scales of
// ordinary keys and values, 2^-24 .. 2^5; the caller says whether all of a warp's are such.  Instructions per four codes:
// fp16 4 (e4m3) or 5 (int8), bf16 10 or 9.
__device__ __forceinline__ bool tree_short_scale(uint32_t byte) { return byte >= 103u && byte <= 132u; }
template <typename T, int FORMAT>
__device__ __forceinline__ void tree_convert16(const uint4& codes, uint32_t byte, uint32_t (&o)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&codes);
  const float s = __uint_as_float(byte << 23);
  if (std::is_same<T, __half>::value) {
    const __half2 s2 = __float2half2_rn(s);  // 2^-24 is fp16's least subnormal
    if (FORMAT == FCR_KV_FP8) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const __half2 v = __hmul2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[q >> 1] >> (16 * (q & 1))), __NV_E4M3)), s2);
        o[q] = *reinterpret_cast<const uint32_t*>(&v);
      }
    } else {
      // byte + 128 under the exponent of 1024 is the fp16 value 1152 + code; one multiplication-addition takes 1152 * s away
      const __half2 off = __hmul2(s2, __float2half2_rn(-1152.f));
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t u = __byte_perm(w[q >> 1] ^ 0x80808080u, 0x64646464u, (q & 1) ? 0x4342 : 0x4140);
        const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&u), s2, off);
        o[q] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    return;
  }
  const float2 s2 = make_float2(s, s);
  const float2 off = make_float2(-8388736.f * s, -8388736.f * s);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float2 a, b;
    if (FORMAT == FCR_KV_FP8) {
      a = __fmul2_rn(__half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w[q], __NV_E4M3))), s2);
      b = __fmul2_rn(__half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[q] >> 16), __NV_E4M3))), s2);
    } else {  // the same with 2^23 + 128 in fp32
      const uint32_t u = w[q] ^ 0x80808080u;
      a = __ffma2_rn(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441))), s2, off);
      b = __ffma2_rn(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))), s2, off);
    }
    o[2 * q] = pack2(a.x, a.y, T());
    o[2 * q + 1] = pack2(b.x, b.y, T());
  }
}
// Any scale, NaN included.  Out of line, for the instruction cache's sake.
template <typename T, int FORMAT>
__device__ __noinline__ uint4 tree_convert8_any(uint2 codes, uint32_t byte) {
  const float s = kv_scale(byte);
  float v[8];
  unpack_codes4<FORMAT>(codes.x, v);
  unpack_codes4<FORMAT>(codes.y, v + 4);
  return make_uint4(pack2(v[0] * s, v[1] * s, T()), pack2(v[2] * s, v[3] * s, T()), pack2(v[4] * s, v[5] * s, T()), pack2(v[6] * s, v[7] * s, T()));
}
// Zeros in place of what is not finite; whether there was any.
template <typename T>
__device__ __forceinline__ bool clean_words(uint32_t* e, int n) {
  bool bad = false;
  for (int i = 0; i < n; ++i) {
    const bool lo = non_finite16<T>(e[i] & 0xffffu), hi = non_finite16<T>(e[i] >> 16);
    if (lo) e[i] &= 0xffff0000u;
    if (hi) e[i] &= 0xffffu;
    bad = bad || lo || hi;
  }
  return bad;
}

// The values of a drafted token that the product left out because they are not finite; 0 for a finite one.
template <typename T, int FORMAT>
__device__ __forceinline__ float tree_non_finite(const TreeParams& p, int b, int h, int n, int d) {
  const long long at = b * p.cb[1] + h * p.ch[1] + n * p.cn[1] + d;
  float v;
  if (FORMAT != FCR_KV_16BIT) {
    float c[4];
    const uint32_t byte = reinterpret_cast<const unsigned char*>(p.cache[1])[at];
    unpack_codes4<FORMAT>(byte, c);
    v = c[0] * kv_scale(p.scales[1][b * p.sb[1] + h * p.sh[1] + n * p.sn[1]]);
  } else {
    v = to_f32(reinterpret_cast<const T*>(p.cache[1])[at]);
  }
  v = to_f32(from_f32<T>(v));  // as the product would have had it
  return fabsf(v) < INFINITY ? 0.f : v;
}
template <typename T, int FORMAT>
__device__ __noinline__ void tree_add_non_finite(const TreeParams& p, const TreeSegment& s, const uint32_t* words, int m, int d0, int nd,
                                                 float* o) {
  const int h = s.group / p.row_tiles;
  const int hi = min(s.end, s.hi * kTreeTile);
  for (int n = max(s.have, s.lo * kTreeTile); n < hi; ++n) {
    const int j = n - s.have;
    if (words ? !(words[j >> 5] >> (j & 31) & 1u) : j > m) continue;
    for (int d = 0; d < nd && d0 + d < p.D; ++d) o[d] += tree_non_finite<T, FORMAT>(p, s.b, h, n, d0 + d);
  }
}

// Packs a bool mask (mask_b, M, M) into words of 32 tokens; a warp per word.
__global__ void __launch_bounds__(256)
tree_pack_mask_kernel(const unsigned char* __restrict__ mask, long long stride_b, long long stride_m, int M, int words, int n_words,
                      uint32_t* __restrict__ out) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= n_words) return;
  const int w = i % words, m = i / words % M, b = i / words / M;
  const int j = 32 * w + lane;
  const bool on = j < M && mask[b * stride_b + m * stride_m + j] != 0;
  const uint32_t bits = __ballot_sync(0xffffffffu, on);
  if (lane == 0) out[i] = bits;
}

// ------------------------------------------------------------------ what both kernels share
// Pieces c0 .. c1 - 1 of row `row` (key n) of a value tile: zeros behind the last drafted token, and in place of what is not
// finite in a drafted token's values.
template <typename T, int DPAD>
__device__ __noinline__ void tree_clean_values(uint32_t tile, int row, int n, const TreeSegment& s, int c0, int c1, volatile int* bad_flag) {
  if (n < s.have) return;
  for (int c = c0; c < c1; ++c) {
    const uint32_t a = tile + (uint32_t)(c >> 3) * (128u * 128u) + (uint32_t)row * 128u + (((uint32_t)c & 7u) ^ ((uint32_t)row & 7u)) * 16u;
    if (n >= s.end) {
      ptx::sts128(a, make_uint4(0u, 0u, 0u, 0u));
      continue;
    }
    uint32_t e[4];
    *reinterpret_cast<uint4*>(e) = ptx::lds128(a);
    if (clean_words<T>(e, 4)) {
      ptx::sts128(a, make_uint4(e[0], e[1], e[2], e[3]));
      *bad_flag = 1;
    }
  }
}

// The rings of key and value tiles in shared memory (swizzled 16-bit tiles of 128 keys) and their barriers; for an 8-bit cache
// also the rings of codes (key and value tiles in turn, slabs of 64 bytes by 128 rows) and of scale bytes (two batches of SB tiles: 128
// keys, then 128 values, per tile; then a byte per tile and kind: are all scales ordinary?) that the tiles are made from.
struct TreeRing {
  uint32_t k, v;
  uint32_t bar_k_full, bar_k_empty, bar_v_full, bar_v_empty;
  uint32_t codes, scales;
  uint32_t bar_c_full, bar_c_empty, bar_sc_full, bar_sc_empty;
};

// No arrival may be outstanding when the CTA retires: wait until the products have given back every slot.
template <int KS, int VS>
__device__ __forceinline__ void tree_drain(const TreeParams& p, const TreeRing& r, uint32_t seq, bool ok, volatile int* abort_flag) {
  for (uint32_t i = 0; ok && i < (KS > VS ? KS : VS) && i < seq; ++i) {
    const uint32_t last = seq - 1 - i;
    if (i < KS) ok = TREE_WAIT_BEHIND(r.bar_k_empty + 8u * (last % KS), (last / KS) & 1u, ST_TR_WAIT_DRAIN);
    if (ok && i < VS) ok = TREE_WAIT_BEHIND(r.bar_v_empty + 8u * (last % VS), (last / VS) & 1u, ST_TR_WAIT_DRAIN);
  }
}

// One warp: the tiles of a 16-bit cache by TMA.
template <int DPAD, int KS, int VS>
__device__ __forceinline__ void tree_tma_tiles(const TreeParams& p, const TreeRing& r, const CUtensorMap* tmap_k, const CUtensorMap* tmap_v,
                                               TreeWalk<TreeLengths> walk, int lane, volatile int* abort_flag) {
  constexpr uint32_t kTileBytes = 128 * DPAD * 2, kSlabBytes = 128 * 128;
  uint32_t seq = 0;
  bool ok = true;
  TreeSegment seg{};
  auto load = [&](auto is_v, int t, int h) {
    constexpr bool kv = decltype(is_v)::value;
    constexpr uint32_t kSlots = kv ? VS : KS;
    const uint32_t slot = seq % kSlots, ph = (seq / kSlots) & 1u;
    const uint32_t full = (kv ? r.bar_v_full : r.bar_k_full) + 8u * slot;
    ok = TREE_WAIT_BEHIND((kv ? r.bar_v_empty : r.bar_k_empty) + 8u * slot, ph ^ 1u, kv ? ST_TR_WAIT_V_EMPTY : ST_TR_WAIT_K_EMPTY);
    if (!ok) return;
    const bool left_out = blockIdx.x == 0 && !kv && (int)seq == p.skip_ring_load;  // self-test of the bounded waits
    if (lane == 0 && !left_out) {
      const uint32_t dst = (kv ? r.v : r.k) + slot * kTileBytes;
      ptx::mbar_arrive_expect_tx(full, kTileBytes);
#pragma unroll
      for (int sl = 0; sl < DPAD / 64; ++sl)
        ptx::tma_load_4d(dst + sl * kSlabBytes, kv ? tmap_v : tmap_k, full, sl * 64, t * kTreeTile, h, seg.b);
    }
    __syncwarp();
  };
  while (ok && walk.next(seg)) {
    const int h = seg.group / p.row_tiles;
    for (int t = seg.lo; ok && t < seg.hi; ++t) {
      load(std::false_type{}, t, h);
      if (!ok) break;
      load(std::true_type{}, t, h);
      ++seq;
    }
  }
  tree_drain<KS, VS>(p, r, seq, ok, abort_flag);
}

// An 8-bit cache takes three roles.  One warp: the codes by TMA, SS tiles of them under way.
template <int DPAD, int SS>
__device__ __forceinline__ void tree_tma_codes(const TreeParams& p, const TreeRing& r, const CUtensorMap* tmap_k, const CUtensorMap* tmap_v,
                                               TreeWalk<TreeLengths> walk, int lane, volatile int* abort_flag) {
  uint32_t seq = 0;
  bool ok = true;
  TreeSegment seg{};
  while (ok && walk.next(seg)) {
    const int h = seg.group / p.row_tiles;
    for (int t2 = 2 * seg.lo; t2 < 2 * seg.hi; ++t2, ++seq) {
      const uint32_t slot = seq % SS, full = r.bar_c_full + 8u * slot;
      ok = TREE_WAIT_BEHIND(r.bar_c_empty + 8u * slot, ((seq / SS) & 1u) ^ 1u, ST_TR_WAIT_C_EMPTY);
      if (!ok) break;
      const bool left_out = blockIdx.x == 0 && (int)seq == p.skip_ring_load;  // self-test of the bounded waits
      if (lane == 0 && !left_out) {
        ptx::mbar_arrive_expect_tx(full, 128 * DPAD);
#pragma unroll
        for (int sl = 0; sl < DPAD / 64; ++sl)  // slabs of 64 codes, like those of the tiles they become
          ptx::tma_load_4d(r.codes + slot * (128 * DPAD) + sl * 8192, (t2 & 1) ? tmap_v : tmap_k, full, sl * 64, (t2 >> 1) * kTreeTile, h, seg.b);
      }
      __syncwarp();
    }
  }
}

// One warp: the scale bytes, SB tiles at a time so that their loads' latencies overlap.  They may lie anywhere, at any
// stride, so plain loads bring them.  After each batch `also(tiles so far)` may do other work; it returns whether to go on.
template <int SB, typename Also>
__device__ __forceinline__ void tree_load_scales(const TreeParams& p, const TreeRing& r, TreeWalk<TreeLengths> walk, int lane,
                                                 volatile int* abort_flag, Also also) {
  TreeSegment seg{};
  int t = 0;
  bool more = walk.next(seg);
  if (more) t = seg.lo;
  for (uint32_t batch = 0; more; ++batch) {
    uint32_t word[SB][2];  // a lane has four neighbouring keys
    bool all[SB][2];
#pragma unroll
    for (int i = 0; i < SB; ++i) {
      const int h = more ? seg.group / p.row_tiles : 0, n0 = t * kTreeTile + 4 * lane;
      const int upto = more ? seg.end - n0 : 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const long long step = p.sn[kv];
        const unsigned char* src = p.scales[kv] + seg.b * p.sb[kv] + h * p.sh[kv] + n0 * step;
        uint32_t byte[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          byte[k] = 127u;
          if (k < upto) byte[k] = *src;
          src += step;
        }
        word[i][kv] = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
        all[i][kv] = tree_short_scale(byte[0]) && tree_short_scale(byte[1]) && tree_short_scale(byte[2]) && tree_short_scale(byte[3]);
      }
      if (more && ++t == seg.hi) {
        more = walk.next(seg);
        if (more) t = seg.lo;
      }
    }
    const uint32_t buf = batch & 1u;
    if (!TREE_WAIT_BEHIND(r.bar_sc_empty + 8u * buf, ((batch >> 1) & 1u) ^ 1u, ST_TR_WAIT_SC_EMPTY)) return;
#pragma unroll
    for (int i = 0; i < SB; ++i) {
      const uint32_t at = SB * buf + i;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        ptx::sts32(r.scales + at * 256u + kv * 128u + 4u * lane, word[i][kv]);
        const uint32_t ordinary = __all_sync(0xffffffffu, all[i][kv]) ? 1u : 0u;
        if (lane == 0) ptx::sts8(r.scales + 512u * SB + at * 2u + kv, ordinary);
      }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(r.bar_sc_full + 8u * buf);
    if (!also((long long)SB * (batch + 1))) return;
  }
}

// Zeros in place of what is not finite in a converter's rows of drafted tokens.  Out of line: the last tiles only.
template <typename T, int kSlabs, int kRows>
__device__ __noinline__ void tree_clean_rows(uint32_t dst, uint32_t at0, uint32_t at1, int row0, int drafted, volatile int* bad_flag) {
  for (int k = 0; k < kRows; k += 8) {
    if (row0 + k < drafted) continue;
    for (int sl = 0; sl < 2 * kSlabs; ++sl) {
      const uint32_t a = dst + (sl >> 1) * (128u * 128u) + k * 128u + ((sl & 1) ? at1 : at0);
      uint32_t e[4];
      *reinterpret_cast<uint4*>(e) = ptx::lds128(a);
      if (clean_words<T>(e, 4)) {
        ptx::sts128(a, make_uint4(e[0], e[1], e[2], e[3]));
        *bad_flag = 1;
      }
    }
  }
}

// kTreeConvertWarps warps: codes times scale in 16 bits.  `tid` counts these warps' threads.  (Loading the codes straight
// into registers was built first: a warp's wait for a load includes the younger loads behind it, so that there was
// never more than one tile under way; 365 us for 32 x 8 heads of 8191 int8 keys, against 292 with this ring.)
template <typename T, int FORMAT, int DPAD, int KS, int VS, int SS, int SB>
__device__ __forceinline__ void tree_convert_tiles(const TreeParams& p, const TreeRing& r, TreeWalk<TreeLengths> walk, int tid,
                                                   volatile int* abort_flag, volatile int* bad_flag) {
  constexpr uint32_t kTileBytes = 128 * DPAD * 2;
  constexpr int kSlabs = DPAD / 64;
  constexpr int kRows = 128 / kTreeConvertWarpsOf;  // a warp takes this many rows of each tile, eight of one slab at a time
  const int lane = tid & 31, role = tid / 32, kv = role / kTreeConvertWarpsOf;  // half the warps take the keys, half the values
  const int row0 = (role % kTreeConvertWarpsOf) * kRows + (lane >> 2), piece = lane & 3;
  // Eight lanes read two rows of 64 codes and write 16-byte pieces 2 * piece (then 2 * piece + 1) of two rows of opposite
  // parity: the swizzle puts them in eight different places, so neither access meets a bank twice.
  const uint32_t from = r.codes + row0 * 64 + piece * 16;
  const uint32_t to = (kv ? r.v : r.k) + row0 * 128u, at0 = ((2u * piece) ^ (lane >> 2)) << 4, at1 = at0 ^ 16u;
  const uint32_t bar_full = kv ? r.bar_v_full : r.bar_k_full, bar_empty = kv ? r.bar_v_empty : r.bar_k_empty;
  const uint32_t scales = r.scales + kv * 128u + row0;
  uint32_t seq = 0;  // tiles so far
  bool ok = true;
  TreeSegment seg{};
  while (ok && walk.next(seg)) {
    for (int t = seg.lo; t < seg.hi; ++t, ++seq) {
      // rows from `drafted` on are drafted tokens', rows from `end` on nobody's
      const int drafted = seg.have - t * kTreeTile, end = seg.end - t * kTreeTile;
      const uint32_t c_seq = 2u * seq + kv, c_slot = c_seq % SS;
      const uint32_t slot = kv ? seq % VS : seq % KS, use = kv ? seq / VS : seq / KS;
      // the codes are there, the slot is free, the scales are there: asked for together, waited for in turn
      const uint32_t bar_c = r.bar_c_full + 8u * c_slot, par_c = (c_seq / SS) & 1u;
      const uint32_t bar_e = bar_empty + 8u * slot, par_e = (use & 1u) ^ 1u;
      const uint32_t bar_sc = r.bar_sc_full + 8u * ((seq / SB) & 1u), par_sc = (seq / (2 * SB)) & 1u, sc_at = seq % (2 * SB);
      const uint32_t now = ptx::mbar_try_wait(bar_c, par_c) & ptx::mbar_try_wait(bar_e, par_e) & ptx::mbar_try_wait(bar_sc, par_sc);
      if (!__all_sync(0xffffffffu, now)) {
        ok = TREE_WAIT(bar_c, par_c, ST_TR_WAIT_C_FULL) && TREE_WAIT(bar_sc, par_sc, ST_TR_WAIT_SC_FULL) &&
             TREE_WAIT_BEHIND(bar_e, par_e, kv ? ST_TR_WAIT_V_EMPTY : ST_TR_WAIT_K_EMPTY);
        if (!ok) break;
      }
      const uint32_t sc = scales + sc_at * 256u, src = from + c_slot * (128 * DPAD), dst = to + slot * kTileBytes;
      // (a byte per tile and kind says whether all of its scales allow the short conversion)
      const bool plain = ptx::lds8(r.scales + 512u * SB + sc_at * 2u + kv) != 0u;
      const bool check = kv == 1 && drafted < kTreeTile;  // values of drafted tokens must be finite
#pragma unroll 1
      for (int k = 0; k < kRows; k += 8) {
        const uint32_t scale = ptx::lds8(sc + k);
        uint4 codes[kSlabs];
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl) codes[sl] = ptx::lds128(src + sl * 8192 + k * 64);
        if (row0 + k >= end) {
#pragma unroll
          for (int sl = 0; sl < kSlabs; ++sl) codes[sl] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl) {
          uint32_t o[8];
          if (plain) {
            tree_convert16<T, FORMAT>(codes[sl], scale, o);
          } else {
            *reinterpret_cast<uint4*>(o) = tree_convert8_any<T, FORMAT>(make_uint2(codes[sl].x, codes[sl].y), scale);
            *reinterpret_cast<uint4*>(o + 4) = tree_convert8_any<T, FORMAT>(make_uint2(codes[sl].z, codes[sl].w), scale);
          }
          const uint32_t a = dst + sl * (128u * 128u) + k * 128u;
          ptx::sts128(a + at0, make_uint4(o[0], o[1], o[2], o[3]));
          ptx::sts128(a + at1, make_uint4(o[4], o[5], o[6], o[7]));
        }
      }
      if (check) tree_clean_rows<T, kSlabs, kRows>(dst, at0, at1, row0, drafted, bad_flag);
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(r.bar_c_empty + 8u * c_slot);
        ptx::mbar_arrive(bar_full + 8u * slot);
        if (seq % SB == SB - 1) ptx::mbar_arrive(r.bar_sc_empty + 8u * ((seq / SB) & 1u));
      }
    }
  }
  tree_drain<KS, VS>(p, r, seq, ok, abort_flag);
}

// The query warp: load(segment, its number) brings a segment's queries.  With an 8-bit cache it also brings the scales; a segment's queries
// follow the scales of its first tiles, which never wait for queries, while those may wait for the products of the segment before.
template <int SB, bool QUANT, typename Load>
__device__ __forceinline__ void tree_query_role(const TreeParams& p, const TreeRing& ring, TreeWalk<TreeLengths> walk, int lane,
                                                volatile int* abort_flag, Load load) {
  uint32_t number = 0;
  if constexpr (QUANT) {
    TreeWalk<TreeLengths> scale_walk = walk;
    long long next_at = 0;  // first tile of the next segment whose queries are to come
    tree_load_scales<SB>(p, ring, scale_walk, lane, abort_flag, [&](long long tiles) {
      while (next_at < tiles) {
        TreeSegment s;
        if (!walk.next(s)) return true;
        next_at += s.hi - s.lo;
        if (!load(s, number++)) return false;
      }
      return true;
    });
  } else {
    TreeSegment s;
    while (walk.next(s) && load(s, number)) ++number;
  }
}

template <int SS>
__device__ __forceinline__ void tree_init_code_bars(const TreeRing& r) {
  for (int i = 0; i < SS; ++i) {
    ptx::mbar_init(r.bar_c_full + 8u * i, 1);
    ptx::mbar_init(r.bar_c_empty + 8u * i, kTreeConvertWarpsOf);
  }
  for (int i = 0; i < 2; ++i) {
    ptx::mbar_init(r.bar_sc_full + 8u * i, 1);
    ptx::mbar_init(r.bar_sc_empty + 8u * i, kTreeConvertWarps);
  }
}

// What the load warps do; `role` counts them.
template <typename T, int DPAD, int KS, int VS, int SS, int SB, int FORMAT>
__device__ __forceinline__ void tree_load_roles(const TreeParams& p, const TreeRing& ring, const CUtensorMap* tmap_k, const CUtensorMap* tmap_v,
                                                const TreeWalk<TreeLengths>& walk, int role, int lane, volatile int* abort_flag,
                                                volatile int* bad_flag) {
  if constexpr (FORMAT == FCR_KV_16BIT) {
    tree_tma_tiles<DPAD, KS, VS>(p, ring, tmap_k, tmap_v, walk, lane, abort_flag);
  } else {
    if (role == 0)
      tree_tma_codes<DPAD, SS>(p, ring, tmap_k, tmap_v, walk, lane, abort_flag);
    else
      tree_convert_tiles<T, FORMAT, DPAD, KS, VS, SS, SB>(p, ring, walk, 32 * (role - 1) + lane, abort_flag, bad_flag);
  }
}

// One warp: this CTA's piece of the line of tiles, as the sequence it begins in, the tile there and its length.
__device__ __forceinline__ void tree_find_piece(const TreeParams& p, const TreeLengths& lengths, int lane, volatile int* start_b,
                                                volatile long long* start_off, volatile long long* start_n) {
  auto tiles_of = [&](int b) { return b < p.B ? tree_tiles(tree_have(lengths(b), p.M, p.N), p.M, p.N) : 0; };
  const int mine0 = tiles_of(lane);
  long long total = mine0;
  for (int b = lane + 32; b < p.B; b += 32) total += tiles_of(b);
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= p.groups;
  const int ctas = tree_ctas(total, gridDim.x), c = min((int)blockIdx.x, ctas);
  const long long lo = tree_piece(total, ctas, c), hi = c < ctas ? tree_piece(total, ctas, c + 1) : lo;
  long long before = 0;
  for (int b0 = 0; b0 < p.B && before <= lo; b0 += 32) {
    const long long mine = (long long)(b0 == 0 ? mine0 : tiles_of(b0 + lane)) * p.groups;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (mine > 0 && before + incl - mine <= lo && lo < before + incl) {
      *start_b = b0 + lane;
      *start_off = lo - (before + incl - mine);
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) *start_n = hi - lo;
}

template <typename T, int DPAD, bool PAIR, int FORMAT>
__global__ void __launch_bounds__(tree_threads<FORMAT != FCR_KV_16BIT>(), 1)
tree_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ TreeParams p) {
  constexpr bool QUANT = FORMAT != FCR_KV_16BIT;
  using L = TreeSmem<DPAD, PAIR, QUANT>;
  constexpr int KS = L::KS, VS = L::VS, kLoadWarp = kTreeQWarp + tree_q_warps<QUANT>();
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(p, ST_SMEM_MISALIGNED, (int)base);
    return;
  }
  const uint32_t bar0 = base + L::off_bars;
  auto bar_q_full = [&](uint32_t i) { return bar0 + 8u * i; };
  auto bar_q_empty = [&](uint32_t i) { return bar0 + 8u * (2 + i); };
  auto bar_k_full = [&](uint32_t i) { return bar0 + 8u * (4 + i); };
  auto bar_k_empty = [&](uint32_t i) { return bar0 + 8u * (4 + KS + i); };
  auto bar_v_full = [&](uint32_t i) { return bar0 + 8u * (4 + 2 * KS + i); };
  auto bar_v_empty = [&](uint32_t i) { return bar0 + 8u * (4 + 2 * KS + VS + i); };
  auto bar_s = [&](uint32_t w) { return bar0 + 8u * (4 + 2 * KS + 2 * VS + w); };
  auto bar_p = [&](uint32_t w) { return bar0 + 8u * (6 + 2 * KS + 2 * VS + w); };
  auto bar_o = [&](uint32_t w) { return bar0 + 8u * (8 + 2 * KS + 2 * VS + w); };
  const uint32_t bar_merge = bar0 + 8u * (10 + 2 * KS + 2 * VS);
  const uint32_t bar_c = bar_merge + 8u;
  const TreeRing ring{base + L::off_k, base + L::off_v, bar_k_full(0), bar_k_empty(0), bar_v_full(0), bar_v_empty(0), base + L::off_codes,
                      base + L::off_scales, bar_c, bar_c + 8u * L::SS, bar_c + 16u * L::SS, bar_c + 16u * L::SS + 16u};
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::off_misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 8);  // a drafted value was not finite
  volatile int* start_b = reinterpret_cast<volatile int*>(smem + L::off_misc + 12);
  volatile long long* start_off = reinterpret_cast<volatile long long*>(smem + L::off_misc + 16);
  volatile long long* start_n = reinterpret_cast<volatile long long*>(smem + L::off_misc + 24);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // warp-uniform for the compiler
  const int lane = (int)(threadIdx.x & 31);

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kQBuffers; ++i) {
      ptx::mbar_init(bar_q_full(i), tree_q_warps<QUANT>());
      ptx::mbar_init(bar_q_empty(i), PAIR ? 2 : kTreeSoftmaxWarps + 2);
    }
    for (int i = 0; i < KS; ++i) {
      ptx::mbar_init(bar_k_full(i), QUANT ? kTreeConvertWarpsOf : 1);
      ptx::mbar_init(bar_k_empty(i), PAIR ? 2 : 1);
    }
    for (int i = 0; i < VS; ++i) {
      ptx::mbar_init(bar_v_full(i), QUANT ? kTreeConvertWarpsOf : 1);
      ptx::mbar_init(bar_v_empty(i), PAIR ? 2 : 1);
    }
    for (int w = 0; w < 2; ++w) {
      ptx::mbar_init(bar_s(w), 1);
      ptx::mbar_init(bar_p(w), 4);
      ptx::mbar_init(bar_o(w), 1);
    }
    ptx::mbar_init(bar_merge, kTreeSoftmaxWarps);
    if (QUANT) tree_init_code_bars<L::SS>(ring);
    *abort_flag = 0;
    *bad_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kTreeMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
    ptx::tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    ptx::prefetch_tensormap(&tmap_k);
    ptx::prefetch_tensormap(&tmap_v);
  }
  if (threadIdx.x == 0) ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();  // the kernel before this one may have written lengths, cache or queries
  if (blockIdx.x == 0 && threadIdx.x < 4) p.status[threadIdx.x] = 0;
  const TreeLengths lengths{p.lengths, p.index_bits};
  if (warp >= kTreeQWarp && warp < kLoadWarp) {
    tree_find_piece(p, lengths, lane, start_b, start_off, start_n);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  TreeWalk<TreeLengths> walk{lengths, p.B, p.groups, p.M, p.N};
  const long long n_tiles = *start_n;
  walk.start(n_tiles > 0 ? *start_b : 0, *start_off, n_tiles);
  TreeSegment seg{};

  if (warp >= kTreeQWarp && warp < kLoadWarp) {
    // ----------------------------------------------------- queries of the next segment
    // (all copies of a segment under way at once: behind the flood of key and value tiles each wait costs microseconds)
    auto load_queries = [&](const TreeSegment s, uint32_t number) {
      const uint32_t buf = number % L::kQBuffers;
      if (!TREE_WAIT_BEHIND(bar_q_empty(buf), ((number / L::kQBuffers) & 1u) ^ 1u, ST_TR_WAIT_Q_EMPTY)) return false;
      const int kh = s.group / p.row_tiles, r0 = (s.group - kh * p.row_tiles) * 256;
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p.q) + s.b * p.qb + (long long)kh * p.G * p.qh;
      const uint32_t dst0 = base + L::off_q + buf * L::kQBytes;
      const long long qh = p.qh, qm = p.qm;
      const int M = p.M, rows = p.rows - r0;
      constexpr int kChunks = DPAD / 8;  // 16-byte pieces of a row
      constexpr int kStep = 32 * tree_q_warps<QUANT>() / kChunks;
      const int first = 32 * (warp - kTreeQWarp) + lane, c = first % kChunks, d0 = c * 8;
      const bool on_d = d0 < p.D;
      int row = first / kChunks, g = (r0 + row) / M, m = r0 + row - g * M;
#pragma unroll 4
      for (int i = 0; i < (PAIR ? 256 : 128) / kStep; ++i) {
        const bool on = row < rows && on_d;
        const uint32_t tile = dst0 + (uint32_t)(row >> 7) * L::kTileBytes, in = (uint32_t)(row & 127);
        ptx::cp_async16(tile + (uint32_t)(c >> 3) * L::kSlabBytes + in * 128u + (((uint32_t)c & 7u) ^ (in & 7u)) * 16u,
                        on ? q + g * qh + m * qm + d0 : q, on);
        row += kStep;
        for (m += kStep; m >= M; m -= M) ++g;
      }
      ptx::cp_async_wait_all();
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_q_full(buf));
      return true;
    };
    tree_query_role<1, QUANT>(p, ring, walk, lane, abort_flag, load_queries);
  } else if (warp == kTreeMmaWarp || warp == kTreeMmaWarp + 1) {
    // ------------------------------------------------------------------- products
    // A warp per warpgroup: S of its next tile follows P V of the last one, which orders the buffer they share (S
    // overwrites the P that the product has read), and while one warpgroup takes exponentials the other's products run.
    // (One warp that issued for both in turn: 62 instead of 55 us for 64 tokens over 4 x 8 heads of 4096 keys, 145 either
    // way over 8 x 8 heads of up to 16384.)
    const uint32_t w = (uint32_t)(warp - kTreeMmaWarp);
    struct Cursor {
      TreeWalk<TreeLengths> walk;
      TreeSegment s;
      int t;
      uint32_t tile, seg;
      bool on;
      __device__ __forceinline__ void step() {
        ++tile;
        if (++t < s.hi) return;
        on = walk.next(s);
        t = s.lo;
        ++seg;
      }
    };
    constexpr int kStride = PAIR ? 1 : 2;  // own tiles: all, or every other one
    auto first_own = [&]() {
      Cursor c{walk, TreeSegment{}, 0, 0, 0, false};
      c.on = c.walk.next(c.s);
      c.t = c.s.lo;
      if (!PAIR && w == 1 && c.on) c.step();
      return c;
    };
    auto next_own = [&](Cursor& c) {
      c.step();
      if (!PAIR && c.on) c.step();
    };
    Cursor sc = first_own(), oc = sc;
    uint32_t q_waited = 0, p_use = 0;
    bool ok = true;
    auto issue_s = [&]() {
      // every segment's queries in turn, also those of a segment without a tile for this warpgroup: no phase is skipped,
      // and none can pass unseen, as the buffer is given back by this warp too
      for (; ok && q_waited <= sc.seg; ++q_waited) {
        if (!PAIR && q_waited > 0 && lane == 0) ptx::mbar_arrive(bar_q_empty((q_waited - 1u) % L::kQBuffers));
        ok = TREE_WAIT(bar_q_full(q_waited % L::kQBuffers), (q_waited / L::kQBuffers) & 1u, ST_TR_WAIT_Q_FULL);
      }
      if (ok) ok = TREE_WAIT(bar_k_full(sc.tile % KS), (sc.tile / KS) & 1u, ST_TR_WAIT_K_FULL);
      if (!ok) return;
      ptx::tc_fence_after_sync();
      if (ptx::elect_one()) {
        const uint32_t a_lo = ptx::smem_desc_lo(base + L::off_q + (sc.seg % L::kQBuffers) * L::kQBytes + (PAIR ? w * L::kTileBytes : 0));
        const uint32_t b_lo = ptx::smem_desc_lo(base + L::off_k + (sc.tile % KS) * L::kTileBytes);
        const uint32_t d = tmem_base + 2 * DPAD + w * 128;
#pragma unroll
        for (int kk = 0; kk < DPAD / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk >> 2) * (L::kSlabBytes >> 4) + (uint32_t)(kk & 3) * 2u;
          if (kk < p.k_steps) ptx::umma_step<false>(d, a_lo + off, b_lo + off, p.idesc_s, kk == 0);
        }
        ptx::umma_commit(bar_s(w));
        ptx::umma_commit(bar_k_empty(sc.tile % KS));
        if (PAIR && sc.t + 1 == sc.s.hi) ptx::umma_commit(bar_q_empty(sc.seg % L::kQBuffers));
      }
      __syncwarp();
      next_own(sc);
    };
    if (sc.on) issue_s();
    while (ok && oc.on) {
      ok = TREE_WAIT(bar_v_full(oc.tile % VS), (oc.tile / VS) & 1u, ST_TR_WAIT_V_FULL);
      if (!ok) break;
      ok = TREE_WAIT_BEHIND(bar_p(w), p_use & 1u, ST_TR_WAIT_P);
      if (!ok) break;
      ++p_use;
      ptx::tc_fence_after_sync();
      if (ptx::elect_one()) {
        const uint32_t b_lo = ptx::smem_desc_lo_mn(base + L::off_v + (oc.tile % VS) * L::kTileBytes, L::kSlabBytes);
        const uint32_t a = tmem_base + 2 * DPAD + w * 128, d = tmem_base + w * DPAD;
        const bool first = oc.t - oc.s.lo < kStride;  // this warpgroup's first tile of the segment
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) ptx::umma_f16_ts(d, a + 8 * kk, b_lo + kk * (2048u >> 4), p.idesc_o, !(first && kk == 0));
        ptx::umma_commit(bar_v_empty(oc.tile % VS));
        if (oc.s.hi - oc.t <= kStride) ptx::umma_commit(bar_o(w));  // ... and its last one
      }
      __syncwarp();
      next_own(oc);
      if (sc.on) issue_s();
    }
  } else if (warp >= kLoadWarp) {
    // -------------------------------------------------------- key and value tiles
    tree_load_roles<T, DPAD, KS, VS, L::SS, 1, FORMAT>(p, ring, &tmap_k, &tmap_v, walk, warp - kLoadWarp, lane, abort_flag, bad_flag);
  } else {
    // -------------------------------------------------------------- softmax warps
    const int w = warp >> 2;
    const int lane_row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lanes + 2 * DPAD + w * 128, o_addr = tmem_base + lanes + w * DPAD;
    uint32_t tile_seq = 0;   // tiles of this CTA so far
    uint32_t s_use = 0, o_use = 0, merge_use = 0, q_seq = 0;
    bool ok = true;
    auto sync_all = [&]() {  // a bounded barrier over the eight warps
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_merge);
      ok = TREE_WAIT_BEHIND(bar_merge, merge_use & 1u, ST_TR_WAIT_MERGE);
      ++merge_use;
      return ok;
    };
    while (ok && walk.next(seg)) {
      const int kh = seg.group / p.row_tiles;
      const int row = (seg.group - kh * p.row_tiles) * 256 + (PAIR ? w * 128 : 0) + lane_row;  // of the G * M
      const bool real = row < p.rows;
      const int m = real ? row % p.M : 0;
      const uint32_t* words = p.mask ? p.mask + ((size_t)(p.mask_shared ? 0 : seg.b) * p.M + m) * p.words : nullptr;
      float m_ref = -INFINITY, l = 0.f;
      int mine = 0;  // tiles this warpgroup has taken
      for (int t = seg.lo; t < seg.hi; ++t, ++tile_seq) {
        if (!PAIR && (int)(tile_seq & 1u) != w) continue;
        ok = TREE_WAIT(bar_s(w), s_use & 1u, ST_TR_WAIT_S);
        if (!ok) break;
        ++s_use;
        ptx::tc_fence_after_sync();
        const bool edge = (t + 1) * kTreeTile > seg.have;
        uint32_t bits[4];  // the tile's keys that this row attends
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; ++c) bits[c] = tree_bits(p, words, m, t * kTreeTile + 32 * c, seg.have, seg.end);
          __syncwarp();  // the lanes took different ways; tensor memory is read by a converged warp
        }
        auto load_scores = [&](int c, uint32_t (&x)[32]) {
          ptx::tmem_ld<32>(s_addr + 32 * c, x);
          ptx::tmem_ld_wait<32>(x);
          if (edge) {
            const uint32_t now = c == 0 ? bits[0] : c == 1 ? bits[1] : c == 2 ? bits[2] : bits[3];
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = (now >> e) & 1u ? x[e] : 0xff800000u;
          }
        };
        auto largest = [&](const uint32_t (&x)[32], float top) {
          float t0 = top, t1 = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            t0 = ptx::max3(t0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
            t1 = ptx::max3(t1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          }
          return fmaxf(t0, t1);
        };
        float2 s01, s23;
        auto weigh = [&](const uint32_t (&x)[32], uint32_t (&pk)[16]) {
          const float nm = m_ref == -INFINITY ? 0.f : -m_ref;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float2 a = __ffma2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), make_float2(p.scale2, p.scale2),
                                  make_float2(nm, nm));
            float2 b = __ffma2_rn(make_float2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), make_float2(p.scale2, p.scale2),
                                  make_float2(nm, nm));
            a.x = ptx::ex2(a.x);
            a.y = ptx::ex2(a.y);
            b.x = ptx::ex2(b.x);
            b.y = ptx::ex2(b.y);
            s01 = __fadd2_rn(s01, a);
            s23 = __fadd2_rn(s23, b);
            pk[e / 2] = pack2(a.x, a.y, T());
            pk[e / 2 + 1] = pack2(b.x, b.y, T());
          }
        };
        // The reference moves when the maximum has grown by more than 2^8: P stays within 2^15.
        constexpr float kAim = tree_aim<T>();
        auto follow = [&](float top) {
          const bool grow = real && top > m_ref + (8.f + kAim);
          if (!__any_sync(0xffffffffu, grow)) return;
          const float m_new = grow ? top - kAim : m_ref;
          const float alpha = m_new == m_ref ? 1.f : ptx::ex2(m_ref - m_new);
          m_ref = m_new;
          l *= alpha;
          if (mine > 0) {
            __syncwarp();
            uint32_t o[32];
            for (int c = 0; c < DPAD / 32; ++c) {
              ptx::tmem_ld<32>(o_addr + 32 * c, o);
              ptx::tmem_ld_wait<32>(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              ptx::tmem_st32(o_addr + 32 * c, o);
            }
          }
        };
        // Two passes over the scores, for the maximum and for the weights.  (One pass that keeps the tile's weights in registers
        // until the maximum beside them is known spilled 700 bytes a thread, with 168 registers: 151 -> 212 us for 64
        // tokens over 8 x 8 heads of 16384 keys.)
        uint32_t x[32];
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          load_scores(c, x);
          top = largest(x, top);
        }
        follow(top * p.scale2);
        s01 = s23 = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
          load_scores(c, x);
          weigh(x, pk);
          // P chunk c covers columns 16 c .. 16 c + 15: scores that this thread has read
          ptx::tmem_st16(s_addr + 16 * c, pk);
        }
        l += (s01.x + s01.y) + (s23.x + s23.y);
        ptx::tmem_st_wait();
        ++mine;
        if (!QUANT && edge) {
          // values behind the last drafted token become zeros, and non-finite ones of the drafted tokens
          const uint32_t slot = tile_seq % VS;
          ok = TREE_WAIT(bar_v_full(slot), (tile_seq / VS) & 1u, ST_TR_WAIT_V_FULL_SM);
          if (!ok) break;
          // (PAIR: each warpgroup takes half of the 16-byte pieces)
          constexpr int kPieces = PAIR ? DPAD / 16 : DPAD / 8;
          tree_clean_values<T, DPAD>(base + L::off_v + slot * L::kTileBytes, lane_row, t * kTreeTile + lane_row, seg, PAIR ? w * kPieces : 0,
                                     PAIR ? (w + 1) * kPieces : kPieces, bad_flag);
          ptx::fence_proxy_async_smem();
          if (PAIR && !sync_all()) break;  // both warpgroups' halves are done before either's product
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_p(w));
      }
      if (!ok) break;
      // ------------------------------------------------ the segment's results
      if (mine > 0) {
        ok = TREE_WAIT(bar_o(w), o_use & 1u, ST_TR_WAIT_O);
        if (!ok) break;
        ++o_use;
        ptx::tc_fence_after_sync();
      }
      const bool whole = seg.whole();
      const size_t part = ((size_t)blockIdx.x * 2 + seg.slot()) * p.part_rows;
      const size_t out_row0 = (size_t)(seg.b * p.Hk + kh) * p.rows;
      if constexpr (PAIR) {
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
        const int in_part = w * 128 + lane_row;
        for (int c = 0; c < DPAD / 32; ++c) {
          __syncwarp();  // rows beyond the last one leave the previous step early
          uint32_t ra[32];
          ptx::tmem_ld<32>(o_addr + 32 * c, ra);
          ptx::tmem_ld_wait<32>(ra);
          if (!real || 32 * c >= p.D) continue;
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = l == 0.f ? 0.f : __uint_as_float(ra[e]) * inv;
          if (*bad_flag) {
            float fix[32];
            for (int e = 0; e < 32; ++e) fix[e] = o[e];
            tree_add_non_finite<T, FORMAT>(p, seg, words, m, 32 * c, 32, fix);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fix[e];
          }
          if (whole) {
            T* dst = reinterpret_cast<T*>(p.out) + (out_row0 + row) * p.D + 32 * c;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              if (32 * c + e < p.D)
                *reinterpret_cast<uint4*>(dst + e) = make_uint4(pack2(o[e], o[e + 1], T()), pack2(o[e + 2], o[e + 3], T()),
                                                                pack2(o[e + 4], o[e + 5], T()), pack2(o[e + 6], o[e + 7], T()));
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(p.part_o + (part + in_part) * DPAD + 32 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (real) {
          if (!whole)
            p.part_ml[part + in_part] = make_float2(m_ref, l);
          else if (p.lse)
            p.lse[out_row0 + row] = l == 0.f ? -INFINITY : (m_ref + log2f(l)) * 0.69314718055994531f;
        }
      } else {
        // merge the two warpgroups: lane_row is the same row in both
        float2* stat = reinterpret_cast<float2*>(smem + L::off_stat);
        float* buf = reinterpret_cast<float*>(smem + L::off_q + (q_seq % L::kQBuffers) * L::kQBytes);
        const int tid = (int)threadIdx.x;
        stat[tid] = make_float2(m_ref, l);
        if (!sync_all()) break;
        const float2 other = stat[tid ^ 128];
        const float m_all = fmaxf(m_ref, other.x), m_use = m_all == -INFINITY ? 0.f : m_all;
        float f = ptx::ex2(m_ref - m_use);
        // (in warpgroup order, so that both find the same sum)
        const float a0 = l * f, a1 = other.y * ptx::ex2(other.x - m_use), l_all = w == 0 ? a0 + a1 : a1 + a0;
        if (whole) f *= l_all == 0.f ? 0.f : 1.f / l_all;
        const bool none = mine == 0 || l == 0.f;  // nothing summed here: the accumulator may hold anything
        if (w == 0 && real) {
          if (!whole)
            p.part_ml[part + lane_row] = make_float2(m_all, l_all);
          else if (p.lse)
            p.lse[out_row0 + row] = l_all == 0.f ? -INFINITY : (m_all + log2f(l_all)) * 0.69314718055994531f;
        }
        for (int c = 0; ok && 32 * c < p.D; ++c) {
          __syncwarp();  // only some lanes had statistics to write
          uint32_t ra[32];
          if (mine > 0) {
            ptx::tmem_ld<32>(o_addr + 32 * c, ra);
            ptx::tmem_ld_wait<32>(ra);
          }
          float4* dst = reinterpret_cast<float4*>(buf) + tid * 8;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float4 v = make_float4(__uint_as_float(ra[4 * e]) * f, __uint_as_float(ra[4 * e + 1]) * f, __uint_as_float(ra[4 * e + 2]) * f,
                                   __uint_as_float(ra[4 * e + 3]) * f);
            if (none) v = make_float4(0.f, 0.f, 0.f, 0.f);
            dst[e ^ (tid & 7)] = v;  // 16-byte pieces in another order per row: no bank is asked for twice
          }
          if (!sync_all()) break;
          for (int i = tid; i < 128 * 8; i += 256) {
            const int r = i >> 3, piece = i & 7;
            const float4* src = reinterpret_cast<const float4*>(buf) + r * 8 + (piece ^ (r & 7));
            const float4 v0 = src[0], v1 = src[128 * 8];
            float4 sum = make_float4(v0.x + v1.x, v0.y + v1.y, v0.z + v1.z, v0.w + v1.w);
            const int d = 32 * c + 4 * piece;
            if (r < p.rows && d < p.D) {
              if (*bad_flag) {
                float o[4] = {sum.x, sum.y, sum.z, sum.w};
                const int rm = r % p.M;
                tree_add_non_finite<T, FORMAT>(p, seg, p.mask ? p.mask + ((size_t)(p.mask_shared ? 0 : seg.b) * p.M + rm) * p.words : nullptr,
                                              rm, d, 4, o);
                sum = make_float4(o[0], o[1], o[2], o[3]);
              }
              if (whole)
                *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + (out_row0 + r) * p.D + d) =
                    make_uint2(pack2(sum.x, sum.y, T()), pack2(sum.z, sum.w, T()));
              else
                *reinterpret_cast<float4*>(p.part_o + (part + r) * DPAD + d) = sum;
            }
          }
          if (!sync_all()) break;
        }
        if (!ok) break;
        if (lane == 0) ptx::mbar_arrive(bar_q_empty(q_seq % L::kQBuffers));
        ++q_seq;
      }
    }
  }

  // ------------------------------------------------------------- teardown
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    // A wait expired somewhere: give loads that may still be in flight time to
    // land in this CTA's shared memory before it is released.
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kTreeMmaWarp) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// Joins the partial results of groups whose keys more than one CTA took, in the order of the keys.  A block per group and
// eight rows of it; a warp per row.
template <typename T, int DPAD>
__global__ void __launch_bounds__(256)
tree_combine_kernel(const __grid_constant__ TreeParams p, int ctas, int rows_per_tile, int blocks_per_group) {
  __shared__ long long warp_sum[2][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int item = blockIdx.x / blocks_per_group;  // sequence * groups + group
  const int b = item / p.groups, group = item - b * p.groups;
  const TreeLengths lengths{p.lengths, p.index_bits};
  long long before = 0, total = 0;
  for (int i = threadIdx.x; i < p.B; i += 256) {
    const int t = tree_tiles(tree_have(lengths(i), p.M, p.N), p.M, p.N);
    total += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    warp_sum[0][warp] = total;
    warp_sum[1][warp] = before;
  }
  __syncthreads();
  total = before = 0;
  for (int i = 0; i < 8; ++i) {
    total += warp_sum[0][i];
    before += warp_sum[1][i];
  }
  total *= p.groups;
  ctas = tree_ctas(total, ctas);
  const int tiles = tree_tiles(tree_have(lengths(b), p.M, p.N), p.M, p.N);
  const long long first = before * p.groups + (long long)group * tiles;
  const int c0 = tree_owner(total, ctas, first), c1 = tree_owner(total, ctas, first + tiles - 1);
  if (c0 == c1) return;  // one CTA took all of it and has written the result
  const int kh = group / p.row_tiles, r0 = (group - kh * p.row_tiles) * 256;
  const int local = (blockIdx.x - item * blocks_per_group) * 8 + warp;
  const int row = r0 + local;
  if (local >= rows_per_tile || row >= p.rows) return;
  // the first CTA's part starts the group (its second slot), the others' continue it (their first slot)
  auto slot_row = [&](int c) { return ((size_t)c * 2 + (c == c0 ? 1 : 0)) * p.part_rows + local; };
  float m_all = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m_all = fmaxf(m_all, p.part_ml[slot_row(c)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
  const float m_use = m_all == -INFINITY ? 0.f : m_all;
  float l_all = 0.f;
  constexpr int kVec = DPAD / 32;  // columns per lane
  float acc[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) acc[e] = 0.f;
  for (int cb = c0; cb <= c1; cb += 32) {
    // a lane per part for the statistics, then all lanes over the parts' values, several loads under way at a time
    float f_mine = 0.f, l_mine = 0.f;
    if (cb + lane <= c1) {
      const float2 ml = p.part_ml[slot_row(cb + lane)];
      f_mine = ptx::ex2(ml.x - m_use);
      l_mine = ml.y;
    }
    const int n = min(32, c1 - cb + 1);
    constexpr int kAhead = 4;
    for (int i0 = 0; i0 < n; i0 += kAhead) {
      float v[kAhead][kVec];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = min(i0 + u, n - 1);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[u][e] = 0.f;
        if (lane * kVec < p.D) {
          const float* o = p.part_o + slot_row(cb + i) * DPAD + lane * kVec;
          if constexpr (kVec == 4) {
            const float4 q = *reinterpret_cast<const float4*>(o);
            v[u][0] = q.x, v[u][1] = q.y, v[u][2] = q.z, v[u][3] = q.w;
          } else {
            const float2 q = *reinterpret_cast<const float2*>(o);
            v[u][0] = q.x, v[u][1] = q.y;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = (i0 + u) & 31;
        const float f = __shfl_sync(0xffffffffu, f_mine, i), l = __shfl_sync(0xffffffffu, l_mine, i);
        if (i0 + u < n && l != 0.f) {  // a part that saw nothing may hold anything
          l_all += l * f;
#pragma unroll
          for (int e = 0; e < kVec; ++e) acc[e] += v[u][e] * f;
        }
      }
    }
  }
  const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
  const size_t out_row = (size_t)(b * p.Hk + kh) * p.rows + row;
  if (lane * kVec < p.D) {
    T* dst = reinterpret_cast<T*>(p.out) + out_row * p.D + lane * kVec;
#pragma unroll
    for (int e = 0; e < kVec; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2(acc[e] * inv, acc[e + 1] * inv, T());
  }
  if (p.lse && lane == 0) p.lse[out_row] = l_all == 0.f ? -INFINITY : (m_all + log2f(l_all)) * 0.69314718055994531f;
}

}  // namespace fcr
