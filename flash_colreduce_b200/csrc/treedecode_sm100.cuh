// Attention of drafted tokens with at most 64 query rows per key head (plain decoding, short trees): the operands of
// treeattn_sm100.cuh's products swap roles, so that the keys lie on the 128 lanes and the NR = 16, 32 or 64 rows are columns.
//
//   S^T = K Q^T     tcgen05, 128 keys x NR rows
//   P^T = 2^(S^T * scale * log2 e - m)   a thread owns a key, its NR weights go to shared memory in 16 bits
//   O^T += V^T P^T  A = V as it lies in the cache (MN-major), 128 values of D x NR rows in tensor memory
//
// A product then costs NR / 128 of what the rows-on-lanes form pays whatever the rows are, each thread has NR scores per tile
// to take the exponential of instead of 128, and four softmax warps keep up with the memory.  A maximum would need the
// threads to exchange values for every tile; instead they share a reference m per row and only agree (one barrier of
// four warps) whether any score has passed it by more than 2^8.  That happens in a segment's first tile and rarely after; then the
// rows' maxima are formed, O^T and the sums are rescaled and the reference moves.  Sums stay in registers, a
// thread's keys apart from the others', and are added up when a segment ends.
//
// What bounds it: reading the cache.  The chain of a tile (scores, exponentials, barrier, weights, products) runs under the loads of the
// next ones.
//
// Included by colreduce_sm100.cu after treeattn_sm100.cuh (TreeParams, the rings, the walk over the tiles).
#pragma once

namespace fcr {

constexpr int kDecodeMmaWarp = 4;   // warps 0 - 3: softmax
constexpr int kDecodeQWarp = 5;
constexpr int kDecodeLoadWarp = 6;  // one TMA warp, or the warps that convert codes
template <bool QUANT>
constexpr int decode_threads() { return 32 * (kDecodeLoadWarp + (QUANT ? kTreeConvertWarps : 1)); }

enum {
  ST_TD_WAIT_VOTE = 91,
  ST_TD_WAIT_PV = 92,
};

template <int DPAD, int NR>
struct DecodeSmem {
  static constexpr int kTileBytes = 128 * DPAD * 2;
  static constexpr int kSlabBytes = 128 * 128;
  static constexpr int kQSlabBytes = NR * 128;               // 64 values of each row
  static constexpr int kQBytes = NR * DPAD * 2;
  static constexpr int kPBytes = NR * 256;                   // a weight per row and key
  static constexpr int KS = DPAD == 64 ? 5 : 3, VS = DPAD == 64 ? 5 : NR == 64 ? 2 : 3;
  static constexpr int off_k = 0;
  static constexpr int off_v = off_k + KS * kTileBytes;
  static constexpr int off_q = off_v + VS * kTileBytes;      // two buffers
  static constexpr int off_p = off_q + 2 * kQBytes;          // two buffers
  static constexpr int off_ref = off_p + 2 * kPBytes;        // float [4 warps][NR]: minus the reference of a row
  static constexpr int off_top = off_ref + 4 * NR * 4;       // float [4 warps][NR]: maxima
  static constexpr int off_bars = off_top + 4 * NR * 4;
  static constexpr int kNumBars = 4 + 2 * KS + 2 * VS + 2 + 2 + 2 + 1;
  static constexpr int off_misc = off_bars + 8 * kNumBars;
  // with 64 values per row the V^T operand's upper 64 lanes are whatever follows the tile: that must be this block's memory
  static constexpr int kEnd = off_misc + 48;
  static constexpr int kDynamicBytes = kEnd > off_q + kSlabBytes ? kEnd : off_q + kSlabBytes;
  static_assert(kDynamicBytes <= 232448, "exceeds the 227 KB shared memory of an sm_100 CTA");
};

// W columns of this thread's lane.
template <int W>
__device__ __forceinline__ void tmem_row_ld(uint32_t taddr, uint32_t (&r)[W]) {
  static_assert(W == 16 || W == 32, "");
  if constexpr (W == 32) {
    ptx::tmem_ld32(taddr, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    ptx::pin32(r);
  } else {
    ptx::tmem_ld16(taddr, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    ptx::pin16(r);
  }
}
template <int W>
__device__ __forceinline__ void tmem_row_st(uint32_t taddr, const uint32_t (&r)[W]) {
  if constexpr (W == 32) ptx::tmem_st32(taddr, r); else ptx::tmem_st16(taddr, r);
}

// Bits of the rows r0 .. r0 + width - 1 that attend key n; what it says of rows beyond the last one does not matter.
__device__ __forceinline__ uint32_t decode_row_bits(const TreeParams& p, const TreeSegment& s, int n, int r0, int width) {
  if (n < s.have) return 0xffffffffu;
  if (n >= s.end) return 0u;
  const int j = n - s.have;
  const uint32_t* words = p.mask ? p.mask + (size_t)(p.mask_shared ? 0 : s.b) * p.M * p.words + (j >> 5) : nullptr;
  uint32_t bits = 0;
  int m = r0 % p.M;
#pragma unroll 4
  for (int e = 0; e < width; ++e) {
    const bool on = words ? (words[m * p.words] >> (j & 31)) & 1u : j <= m;
    bits |= (uint32_t)on << e;
    m = m + 1 == p.M ? 0 : m + 1;
  }
  return bits;
}

template <typename T, int DPAD, int NR, bool QUANT>
__global__ void __launch_bounds__(decode_threads<QUANT>(), 1)
tree_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ TreeParams p) {
  using L = DecodeSmem<DPAD, NR>;
  constexpr int KS = L::KS, VS = L::VS;
  constexpr int W = NR < 32 ? NR : 32;  // rows a thread has in registers at a time
  constexpr uint32_t kTmem = NR == 64 ? 256 : 128;  // two score buffers and O^T: 3 * NR columns
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(p, ST_SMEM_MISALIGNED, (int)base);
    return;
  }
  const uint32_t bar0 = base + L::off_bars;
  auto bar_q_full = [&](uint32_t i) { return bar0 + 8u * i; };
  auto bar_q_empty = [&](uint32_t i) { return bar0 + 8u * (2 + i); };
  const uint32_t bar_k_full = bar0 + 8u * 4, bar_k_empty = bar_k_full + 8u * KS;
  const uint32_t bar_v_full = bar_k_empty + 8u * KS, bar_v_empty = bar_v_full + 8u * VS;
  const uint32_t bar_s = bar_v_empty + 8u * VS, bar_p = bar_s + 16u, bar_pv = bar_p + 16u, bar_vote = bar_pv + 16u;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::off_misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 8);  // a drafted value was not finite
  volatile int* start_b = reinterpret_cast<volatile int*>(smem + L::off_misc + 12);
  volatile long long* start_off = reinterpret_cast<volatile long long*>(smem + L::off_misc + 16);
  volatile long long* start_n = reinterpret_cast<volatile long long*>(smem + L::off_misc + 24);
  volatile int* vote = reinterpret_cast<volatile int*>(smem + L::off_misc + 32);     // [2]

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // warp-uniform for the compiler
  const int lane = (int)(threadIdx.x & 31);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_q_full(i), 1);
      ptx::mbar_init(bar_q_empty(i), 1);
      ptx::mbar_init(bar_s + 8u * i, 1);
      ptx::mbar_init(bar_p + 8u * i, 4);
      ptx::mbar_init(bar_pv + 8u * i, 1);
    }
    for (int i = 0; i < KS; ++i) {
      ptx::mbar_init(bar_k_full + 8u * i, QUANT ? kTreeConvertWarps : 1);
      ptx::mbar_init(bar_k_empty + 8u * i, 1);
    }
    for (int i = 0; i < VS; ++i) {
      ptx::mbar_init(bar_v_full + 8u * i, QUANT ? kTreeConvertWarps : 1);
      ptx::mbar_init(bar_v_empty + 8u * i, 1);
    }
    ptx::mbar_init(bar_vote, 4);
    *abort_flag = 0;
    *bad_flag = 0;
    vote[0] = vote[1] = -1;
    ptx::fence_mbar_init();
  }
  if (warp == kDecodeMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmem);
    ptx::tmem_relinquish();
  }
  if (!QUANT && warp == kDecodeLoadWarp && lane == 0) {
    ptx::prefetch_tensormap(&tmap_k);
    ptx::prefetch_tensormap(&tmap_v);
  }
  if (threadIdx.x == 0) ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();  // the kernel before this one may have written lengths, cache or queries
  if (blockIdx.x == 0 && threadIdx.x < 4) p.status[threadIdx.x] = 0;
  const TreeLengths lengths{p.lengths, p.index_bits};
  if (warp == kDecodeQWarp) tree_find_piece(p, lengths, lane, start_b, start_off, start_n);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  TreeWalk<TreeLengths> walk{lengths, p.B, p.groups, p.M, p.N};
  const long long n_tiles = *start_n;
  walk.start(n_tiles > 0 ? *start_b : 0, *start_off, n_tiles);
  TreeSegment seg{};

  if (warp == kDecodeQWarp) {
    // ----------------------------------------------------- queries of the next segment
    uint32_t seq = 0;
    while (walk.next(seg)) {
      const uint32_t buf = seq & 1u;
      if (!WAIT_BEHIND(bar_q_empty(buf), ((seq >> 1) & 1u) ^ 1u, ST_TR_WAIT_Q_EMPTY)) break;
      ++seq;
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p.q) + seg.b * p.qb + (long long)seg.group * p.G * p.qh;
      const uint32_t dst = base + L::off_q + buf * L::kQBytes;
      constexpr int kChunks = DPAD / 8;  // 16-byte pieces of a row
      constexpr int kRowsAtATime = 32 / kChunks;
      const int c = lane % kChunks, d0 = c * 8;
      int row = lane / kChunks, g = row / p.M, m = row - g * p.M;
#pragma unroll 4
      for (int i = 0; i < NR / kRowsAtATime; ++i) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < p.rows && d0 < p.D) {
          const unsigned short* src = q + g * p.qh + m * p.qm + d0;
          if (p.q_vec) {
            v = *reinterpret_cast<const uint4*>(src);
          } else {
            unsigned short* e = reinterpret_cast<unsigned short*>(&v);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = src[j];
          }
        }
        ptx::sts128(dst + (uint32_t)(c >> 3) * L::kQSlabBytes + (uint32_t)row * 128u + (((uint32_t)c & 7u) ^ ((uint32_t)row & 7u)) * 16u, v);
        row += kRowsAtATime;
        for (m += kRowsAtATime; m >= p.M; m -= p.M) ++g;
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_q_full(buf));
    }
  } else if (warp == kDecodeMmaWarp) {
    // ------------------------------------------------------------------- products
    // S^T of tile j + 2 follows the product of tile j: it overwrites the scores that the weights of tile j came from.
    TreeWalk<TreeLengths> ahead = walk;
    TreeSegment sa{};
    int s_left = 0, o_left = 0;
    uint32_t s_tile = 0, o_tile = 0, q_seq = 0;
    bool ok = true, fresh = true;
    auto issue_s = [&]() {
      if (s_left == 0) {
        ahead.next(sa);
        s_left = sa.hi - sa.lo;
        ok = WAIT(bar_q_full(q_seq & 1u), (q_seq >> 1) & 1u, ST_TR_WAIT_Q_FULL);
        if (!ok) return;
      }
      ok = WAIT(bar_k_full + 8u * (s_tile % KS), (s_tile / KS) & 1u, ST_TR_WAIT_K_FULL);
      if (!ok) return;
      ptx::tc_fence_after_sync();
      if (ptx::elect_one()) {
        const uint32_t a_lo = ptx::smem_desc_lo(base + L::off_k + (s_tile % KS) * L::kTileBytes);
        const uint32_t b_lo = ptx::smem_desc_lo(base + L::off_q + (q_seq & 1u) * L::kQBytes);
        const uint32_t d = tmem_base + (s_tile & 1u) * NR;
#pragma unroll
        for (int kk = 0; kk < DPAD / 16; ++kk) {
          const uint32_t in = (uint32_t)(kk & 3) * 2u;
          if (kk < p.k_steps)
            ptx::umma_step<false>(d, a_lo + (uint32_t)(kk >> 2) * (L::kSlabBytes >> 4) + in, b_lo + (uint32_t)(kk >> 2) * (L::kQSlabBytes >> 4) + in,
                                  p.idesc_s, kk == 0);
        }
        ptx::umma_commit(bar_s + 8u * (s_tile & 1u));
        ptx::umma_commit(bar_k_empty + 8u * (s_tile % KS));
        if (s_left == 1) ptx::umma_commit(bar_q_empty(q_seq & 1u));
      }
      __syncwarp();
      ++s_tile;
      if (--s_left == 0) ++q_seq;
    };
    if (n_tiles > 0) issue_s();
    if (ok && n_tiles > 1) issue_s();
    for (long long j = 0; ok && j < n_tiles; ++j) {
      if (o_left == 0) {
        walk.next(seg);
        o_left = seg.hi - seg.lo;
        fresh = true;
      }
      ok = WAIT(bar_v_full + 8u * (o_tile % VS), (o_tile / VS) & 1u, ST_TR_WAIT_V_FULL);
      if (!ok) break;
      ok = WAIT_BEHIND(bar_p + 8u * (o_tile & 1u), (o_tile >> 1) & 1u, ST_TR_WAIT_P);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      if (ptx::elect_one()) {
        const uint32_t a_lo = ptx::smem_desc_lo_mn(base + L::off_v + (o_tile % VS) * L::kTileBytes, L::kSlabBytes);
        const uint32_t b_lo = ptx::smem_desc_lo(base + L::off_p + (o_tile & 1u) * L::kPBytes);
        const uint32_t d = tmem_base + 2 * NR;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          ptx::umma_step<false>(d, a_lo + kk * (2048u >> 4), b_lo + (uint32_t)(kk >> 2) * (L::kQSlabBytes >> 4) + (uint32_t)(kk & 3) * 2u, p.idesc_o,
                                fresh && kk == 0);
        ptx::umma_commit(bar_v_empty + 8u * (o_tile % VS));
        ptx::umma_commit(bar_pv + 8u * (o_tile & 1u));
      }
      __syncwarp();
      fresh = false;
      ++o_tile;
      --o_left;
      if (j + 2 < n_tiles) issue_s();
    }
  } else if (warp >= kDecodeLoadWarp) {
    // -------------------------------------------------------- key and value tiles
    const TreeRing ring{base + L::off_k, base + L::off_v, bar_k_full, bar_k_empty, bar_v_full, bar_v_empty};
    if constexpr (QUANT)
      tree_convert_tiles<T, DPAD, KS, VS>(p, ring, walk, n_tiles, threadIdx.x - 32 * kDecodeLoadWarp, abort_flag, bad_flag);
    else
      tree_tma_tiles<DPAD, KS, VS>(p, ring, &tmap_k, &tmap_v, walk, lane, abort_flag);
  } else {
    // -------------------------------------------------------------- softmax warps
    const int key = warp * 32 + lane;  // of the tile; of D in O^T
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t o_addr = tmem_base + lanes + 2 * NR;
    float* const ref_s = reinterpret_cast<float*>(smem + L::off_ref) + warp * NR;  // this warp's copy, minus the reference
    float* const top_s = reinterpret_cast<float*>(smem + L::off_top);
    const uint32_t p_at = base + L::off_p + (uint32_t)(key >> 6) * L::kQSlabBytes + (uint32_t)(key & 7) * 2u;
    const uint32_t p_chunk = (uint32_t)(key & 63) >> 3;
    uint32_t tile_seq = 0, votes = 0;
    bool ok = true;
    // The product of the tile before this one.  A barrier per buffer: the product two tiles earlier on the same one is known to
    // be done (the scores of tile j come after the product of tile j - 2), so that no parity can be mistaken for an older phase's.
    auto wait_pv = [&](int code) {
      ok = WAIT(bar_pv + 8u * ((tile_seq - 1u) & 1u), ((tile_seq - 1u) >> 1) & 1u, code);
      if (ok) ptx::tc_fence_after_sync();
      return ok;
    };
    auto sync_all = [&]() {  // a bounded barrier over the four warps
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_vote);
      ok = WAIT_BEHIND(bar_vote, votes & 1u, ST_TD_WAIT_VOTE);
      ++votes;
      return ok;
    };
    while (ok && walk.next(seg)) {
      float l[NR];
#pragma unroll
      for (int e = 0; e < NR; ++e) l[e] = 0.f;
      __syncwarp();
      for (int e = lane; e < NR; e += 32) ref_s[e] = INFINITY;  // the reference is -inf: nothing seen
      __syncwarp();
      for (int t = seg.lo; t < seg.hi; ++t, ++tile_seq) {
        const uint32_t buf = tile_seq & 1u;
        const uint32_t s_addr = tmem_base + lanes + buf * NR;
        ok = WAIT(bar_s + 8u * buf, (tile_seq >> 1) & 1u, ST_TR_WAIT_S);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const bool edge = (t + 1) * kTreeTile > seg.have;
        const int n = t * kTreeTile + key;
        uint32_t x[W];
        // has a score passed its row's reference by more than 2^8?
        bool grow = false;
#pragma unroll
        for (int c = 0; c < NR / W; ++c) {
          tmem_row_ld<W>(s_addr + c * W, x);
          if (edge) {
            const uint32_t bits = decode_row_bits(p, seg, n, c * W, W);
#pragma unroll
            for (int e = 0; e < W; ++e) x[e] = (bits >> e) & 1u ? x[e] : 0xff800000u;
          }
          float most = -INFINITY;
#pragma unroll
          for (int e = 0; e < W; e += 4) {
            const float4 nm = *reinterpret_cast<const float4*>(ref_s + c * W + e);
            most = ptx::max3(most, fmaf(__uint_as_float(x[e]), p.scale2, nm.x), fmaf(__uint_as_float(x[e + 1]), p.scale2, nm.y));
            most = ptx::max3(most, fmaf(__uint_as_float(x[e + 2]), p.scale2, nm.z), fmaf(__uint_as_float(x[e + 3]), p.scale2, nm.w));
          }
          grow = grow || most > 8.f;
        }
        if (__any_sync(0xffffffffu, grow) && lane == 0) vote[buf] = (int)tile_seq;
        if (!sync_all()) break;
        if (vote[buf] == (int)tile_seq) {
          // the rows' maxima over the tile's 128 keys; O^T, the sums and the reference follow where a row has grown
#pragma unroll
          for (int c = 0; c < NR / W; ++c) {
            if (NR > W) {
              tmem_row_ld<W>(s_addr + c * W, x);
              if (edge) {
                const uint32_t bits = decode_row_bits(p, seg, n, c * W, W);
#pragma unroll
                for (int e = 0; e < W; ++e) x[e] = (bits >> e) & 1u ? x[e] : 0xff800000u;
              }
            }
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const float most = ptx::redux_max(__uint_as_float(x[e]));
              if (lane == e) top = most;
            }
            if (lane < W) top_s[warp * NR + c * W + lane] = top;
          }
          if (!sync_all()) break;
          const bool rescale = t > seg.lo;
          if (rescale) {
            // the product before this one may still be adding to O^T
            if (!wait_pv(ST_TD_WAIT_PV)) break;
          }
#pragma unroll
          for (int c = 0; c < NR / W; ++c) {
            float alpha = 1.f;
            if (lane < W) {
              const int e = c * W + lane;
              const float top = fmaxf(fmaxf(top_s[e], top_s[NR + e]), fmaxf(top_s[2 * NR + e], top_s[3 * NR + e])) * p.scale2;
              const float nm = ref_s[e];
              if (top + nm > 8.f) {
                alpha = nm == INFINITY ? 0.f : ptx::ex2(-nm - top);
                ref_s[e] = -top;
              }
            }
            if (__any_sync(0xffffffffu, alpha != 1.f) && rescale) {
              uint32_t o[W];
              tmem_row_ld<W>(o_addr + c * W, o);
#pragma unroll
              for (int e = 0; e < W; ++e) {
                const float f = __shfl_sync(0xffffffffu, alpha, e);
                o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                l[c * W + e] *= f;
              }
              tmem_row_st<W>(o_addr + c * W, o);
              ptx::tmem_st_wait();
            }
          }
          __syncwarp();
        }
        const uint32_t p_buf = p_at + buf * L::kPBytes;
#pragma unroll
        for (int c = 0; c < NR / W; ++c) {
          if (NR > W) tmem_row_ld<W>(s_addr + c * W, x);
          uint32_t bits = 0xffffffffu;
          if (edge) bits = decode_row_bits(p, seg, n, c * W, W);
#pragma unroll
          for (int e = 0; e < W; e += 4) {
            const float4 nm = *reinterpret_cast<const float4*>(ref_s + c * W + e);
            float w[4] = {ptx::ex2(fmaf(__uint_as_float(x[e]), p.scale2, nm.x)), ptx::ex2(fmaf(__uint_as_float(x[e + 1]), p.scale2, nm.y)),
                          ptx::ex2(fmaf(__uint_as_float(x[e + 2]), p.scale2, nm.z)), ptx::ex2(fmaf(__uint_as_float(x[e + 3]), p.scale2, nm.w))};
            if (edge) {
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = (bits >> (e + i)) & 1u ? w[i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              l[c * W + e + i] += w[i];
              l[c * W + e + i + 1] += w[i + 1];
              const uint32_t two = pack2(w[i], w[i + 1], T());
              const uint32_t row = (uint32_t)(c * W + e + i);
              ptx::sts16(p_buf + row * 128u + ((p_chunk ^ (row & 7u)) << 4), two);
              ptx::sts16(p_buf + (row + 1u) * 128u + ((p_chunk ^ ((row + 1u) & 7u)) << 4), two >> 16);
            }
          }
        }
        if (!QUANT && edge) {
          const uint32_t slot = tile_seq % VS;
          ok = WAIT(bar_v_full + 8u * slot, (tile_seq / VS) & 1u, ST_TR_WAIT_V_FULL_SM);
          if (!ok) break;
          tree_clean_values<T, DPAD>(base + L::off_v + slot * L::kTileBytes, key, n, seg, 0, DPAD / 8, bad_flag);
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_p + 8u * buf);
      }
      if (!ok) break;
      // ------------------------------------------------ the segment's results
      if (!wait_pv(ST_TR_WAIT_O)) break;
      float* const sum_s = reinterpret_cast<float*>(smem + L::off_p);  // [4 warps][NR]: the products have read the weights
      // the sums over the keys: a warp's by exchanging halves until lane e has row e's, then over the warps
#pragma unroll
      for (int c = 0; c < NR / W; ++c) {
        float v[W];
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = l[c * W + e];
#pragma unroll
        for (int o = W / 2; o; o >>= 1) {
          const bool up = (lane & o) != 0;
#pragma unroll
          for (int e = 0; e < o; ++e) {
            const float keep = up ? v[e + o] : v[e], give = up ? v[e] : v[e + o];
            v[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        }
        if (W == 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
        if (lane < W) sum_s[warp * NR + c * W + lane] = v[0];
      }
      if (!sync_all()) break;
      const bool whole = seg.whole();
      const size_t part = ((size_t)blockIdx.x * 2 + seg.slot()) * p.part_rows;
      const size_t out_row0 = (size_t)(seg.b * p.Hk + seg.group) * p.rows;
#pragma unroll
      for (int c = 0; c < NR / W; ++c) {
        if (c * W >= p.rows) break;
        const int mine = c * W + (lane & (W - 1));
        const float sum = (sum_s[mine] + sum_s[NR + mine]) + (sum_s[2 * NR + mine] + sum_s[3 * NR + mine]);
        const float factor = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
        if (warp == 0 && lane < W && mine < p.rows) {
          const float m_ref = -ref_s[mine];
          if (!whole)
            p.part_ml[part + mine] = make_float2(m_ref, sum);
          else if (p.lse)
            p.lse[out_row0 + mine] = sum == 0.f ? -INFINITY : (m_ref + log2f(sum)) * 0.69314718055994531f;
        }
        uint32_t o[W];
        tmem_row_ld<W>(o_addr + c * W, o);
        if (*bad_flag && key < p.D) {
          for (int r = c * W; r < min(c * W + W, p.rows); ++r) {
            const int m = r % p.M;
            float fix = 0.f;
            tree_add_non_finite<T, QUANT>(p, seg, p.mask ? p.mask + ((size_t)(p.mask_shared ? 0 : seg.b) * p.M + m) * p.words : nullptr, m, key, 1, &fix);
#pragma unroll
            for (int e = 0; e < W; ++e)
              if (e == r - c * W) o[e] = __float_as_uint(__uint_as_float(o[e]) + fix);
          }
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float v = __uint_as_float(o[e]) * __shfl_sync(0xffffffffu, factor, e);
          const int row = c * W + e;
          if (row < p.rows && key < p.D) {
            if (whole)
              reinterpret_cast<T*>(p.out)[(out_row0 + row) * p.D + key] = from_f32<T>(v);
            else
              p.part_o[(part + row) * DPAD + key] = v;
          }
        }
      }
      // the next segment's sums and first product may overwrite what has been read here
      ptx::tc_fence_before_sync();
      if (!sync_all()) break;
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
  if (warp == kDecodeMmaWarp) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmem);
  }
}

}  // namespace fcr
