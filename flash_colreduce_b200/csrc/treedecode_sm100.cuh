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
// four warps) whether any score has passed it by more than 2^8 (for fp16, whose reference lies 7 below the maximum, 2^15).  That happens in a segment's first tile and rarely after; then the
// rows' maxima are formed, O^T and the sums are rescaled and the reference moves.  Sums stay in registers, a
// thread's keys apart from the others', and are added up when a segment ends.
//
// What bounds it: with a 16-bit cache reading it (32 x 8 heads of 8191 bf16 keys, 4 rows: 171 us, 1.03 of the measured copy
// rate's floor; 8 heads of 131072 fp16 keys: 93 us, 1.12 of it).  With an 8-bit cache the latency of the converters: 32 x 8
// heads of 8191 int8 keys take 162 us, the floor is 84.  That is 2900 cycles per pair of tiles, of which the converters' seven
// integer instructions per four codes fill about 900; the rest are load, conversion and store of one step after the other, and
// waits.  So an 8-bit cache saves memory, and time only for single tokens: 16 x 8 heads of 4096 keys take 52 us in bf16 and 54 in 8
// bits with 4 rows, 64 and 70 with 32, 70 and 86 with 64.
//
// Up to 16 and 32 rows the rows-on-lanes form, with the rows held in 4 or 2 copies, was slower (188 and 501 us for 32 x 8 heads
// of 8191 keys in bf16 and int8, where this form's first version took 171 and 365).  For 33 to 64 rows the two present forms,
// keys on the lanes / rows on the lanes:
//   D = 128   16 x 8 heads of 4096 keys: bf16 68..71 / 70..74 us, 8 bits 82..86 / 99..103;
//             8 heads of 32768: bf16 55..57 / 52..54, 8 bits 59..62 / 65..67
//   D = 64    16 x 8 heads of 4096 keys: bf16 59..62 / 58..60, 8 bits 71..74 / 68..70;
//             8 heads of 32768: bf16 44..47 / 41..42, 8 bits 50..53 / 46..47
// This form gains up to 17 % with long rows and an 8-bit cache and loses up to 12 % with short rows; one border, 64 rows, is
// kept for all.
//
// Included by colreduce_sm100.cu after treeattn_sm100.cuh (TreeParams, the rings, the walk over the tiles).
#pragma once

namespace fcr {

// Warps: 4 per 32 rows for the softmax, one that issues S^T, one that issues O^T, one for the queries (and an 8-bit cache's
// scales), one for TMA, and those that convert codes.
template <int NR>
__host__ __device__ constexpr int decode_softmax_warps() { return NR == 64 ? 8 : 4; }
template <int NR, bool QUANT>
__host__ __device__ constexpr int decode_threads() { return 32 * (decode_softmax_warps<NR>() + 4 + (QUANT ? kTreeConvertWarps : 0)); }

// Minus the reference of a row that has seen no key: any finite score passes it, and a masked one (-inf) stays at weight 0.
constexpr float kNothingSeen = 3e38f;

enum {
  ST_TD_WAIT_VOTE = 91,
  ST_TD_WAIT_PV = 92,
};

template <int DPAD, int NR, bool QUANT>
struct DecodeSmem {
  static constexpr int kTileBytes = 128 * DPAD * 2;
  static constexpr int kSlabBytes = 128 * 128;
  static constexpr int kQSlabBytes = NR * 128;               // 64 values of each row
  static constexpr int kQBytes = NR * DPAD * 2;
  static constexpr int kQBuffers = NR == 64 && QUANT ? 1 : 2;
  // Weights: a key's are one row of 128 bytes, swizzled like the tiles (MN-major operand).  Up to 32 rows fill half of
  // that, and the two buffers lie side by side.
  static constexpr int kPBytes = NR == 64 ? 2 * kSlabBytes : kSlabBytes;
  static constexpr int kPStep = NR == 64 ? kSlabBytes : 64;  // from one buffer to the other
  static constexpr int kValueSlots = NR == 64 ? 1 : 2, kCodeSlots = 4;
  static constexpr int KS = DPAD == 64 ? (QUANT ? 4 : 5) : (QUANT ? 2 : 3);
  static constexpr int VS = DPAD == 64 ? (QUANT ? 4 : 5) : (QUANT ? kValueSlots : NR == 64 ? 2 : 3);
  static constexpr int SS = QUANT ? (DPAD == 64 ? 6 : kCodeSlots) : 0;  // tiles of codes in flight
  static constexpr int off_k = 0;
  static constexpr int off_v = off_k + KS * kTileBytes;
  static constexpr int off_p = off_v + VS * kTileBytes;
  static constexpr int off_q = off_p + kPBytes;
  static constexpr int off_codes = off_q + kQBuffers * kQBytes;
  static constexpr int off_scales = off_codes + SS * 128 * DPAD;
  static constexpr int off_ref = off_scales + (QUANT ? 1040 : 0);  // float [4 warps][NR]: minus the reference of a row
  static constexpr int off_top = off_ref + 4 * NR * 4;       // float [4 warps][NR]: maxima
  static constexpr int off_bars = off_top + 4 * NR * 4;
  static constexpr int kNumBars = 4 + 2 * KS + 2 * VS + 2 + 2 + 2 + 2 + (QUANT ? 2 * SS + 4 : 0);
  static constexpr int off_misc = off_bars + 8 * kNumBars;
  // with 64 values per row the V^T operand's upper 64 lanes are whatever follows the tile: that must be this block's memory
  static constexpr int kDynamicBytes = off_misc + 64;
  static_assert(kPBytes >= kSlabBytes, "the weights' space follows the value tiles");
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
__device__ __noinline__ uint32_t decode_row_bits(const TreeParams& p, const TreeSegment& s, int n, int r0, int width) {
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

template <typename T, int DPAD, int NR, int FORMAT>
__global__ void __launch_bounds__((decode_threads<NR, FORMAT != FCR_KV_16BIT>()), 1)
tree_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ TreeParams p) {
  constexpr bool QUANT = FORMAT != FCR_KV_16BIT;
  using L = DecodeSmem<DPAD, NR, QUANT>;
  constexpr int KS = L::KS, VS = L::VS;
  constexpr int W = NR < 32 ? NR : 32;                 // rows that a warpgroup owns
  constexpr int kGroups = NR / W;                      // warpgroups
  constexpr int kSWarp = decode_softmax_warps<NR>(), kOWarp = kSWarp + 1, kQWarp = kSWarp + 2, kLoadWarp = kSWarp + 3;
  constexpr uint32_t kTmem = NR == 64 ? 256 : 128;     // two score buffers and O^T: 3 * NR columns
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(p, ST_SMEM_MISALIGNED, (int)base);
    return;
  }
  const uint32_t bar_q_full = base + L::off_bars, bar_q_empty = bar_q_full + 16u;
  const uint32_t bar_k_full = bar_q_empty + 16u, bar_k_empty = bar_k_full + 8u * KS;
  const uint32_t bar_v_full = bar_k_empty + 8u * KS, bar_v_empty = bar_v_full + 8u * VS;
  const uint32_t bar_s = bar_v_empty + 8u * VS, bar_p = bar_s + 16u, bar_pv = bar_p + 16u, bar_vote = bar_pv + 16u;
  const uint32_t bar_c = bar_vote + 16u;
  const TreeRing ring{base + L::off_k, base + L::off_v, bar_k_full, bar_k_empty, bar_v_full, bar_v_empty, base + L::off_codes,
                      base + L::off_scales, bar_c, bar_c + 8u * L::SS, bar_c + 16u * L::SS, bar_c + 16u * L::SS + 16u};
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::off_misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 8);  // a drafted value was not finite
  volatile int* start_b = reinterpret_cast<volatile int*>(smem + L::off_misc + 12);
  volatile long long* start_off = reinterpret_cast<volatile long long*>(smem + L::off_misc + 16);
  volatile long long* start_n = reinterpret_cast<volatile long long*>(smem + L::off_misc + 24);
  volatile int* votes_s = reinterpret_cast<volatile int*>(smem + L::off_misc + 32);  // [warpgroup][2]

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // warp-uniform for the compiler
  const int lane = (int)(threadIdx.x & 31);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_q_full + 8u * i, 1);
      ptx::mbar_init(bar_q_empty + 8u * i, 1);
      ptx::mbar_init(bar_s + 8u * i, 1);
      ptx::mbar_init(bar_p + 8u * i, decode_softmax_warps<NR>());
      ptx::mbar_init(bar_pv + 8u * i, 1);
      ptx::mbar_init(bar_vote + 8u * i, 4);
    }
    for (int i = 0; i < KS; ++i) {
      ptx::mbar_init(bar_k_full + 8u * i, QUANT ? kTreeConvertWarpsOf : 1);
      ptx::mbar_init(bar_k_empty + 8u * i, 1);
    }
    for (int i = 0; i < VS; ++i) {
      ptx::mbar_init(bar_v_full + 8u * i, QUANT ? kTreeConvertWarpsOf : 1);
      ptx::mbar_init(bar_v_empty + 8u * i, 1);
    }
    if (QUANT) tree_init_code_bars<L::SS>(ring);
    *abort_flag = 0;
    *bad_flag = 0;
    for (int i = 0; i < 4; ++i) votes_s[i] = -1;
    ptx::fence_mbar_init();
  }
  if (warp == kSWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmem);
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
  if (warp == kQWarp) tree_find_piece(p, lengths, lane, start_b, start_off, start_n);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  TreeWalk<TreeLengths> walk{lengths, p.B, p.groups, p.M, p.N};
  const long long n_tiles = *start_n;
  walk.start(n_tiles > 0 ? *start_b : 0, *start_off, n_tiles);
  TreeSegment seg{};

  if (warp == kQWarp) {
    // ----------------------------------------------------- queries of the next segment
    // (all copies of a segment under way at once: behind the flood of key and value tiles each wait costs microseconds)
    auto load_queries = [&](const TreeSegment s, uint32_t number) {
      const uint32_t buf = number % L::kQBuffers;
      if (!TREE_WAIT_BEHIND(bar_q_empty + 8u * buf, ((number / L::kQBuffers) & 1u) ^ 1u, ST_TR_WAIT_Q_EMPTY)) return false;
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p.q) + s.b * p.qb + (long long)s.group * p.G * p.qh;
      const long long qh = p.qh, qm = p.qm;
      const int M = p.M, rows = p.rows;
      const uint32_t dst = base + L::off_q + buf * L::kQBytes;
      constexpr int kChunks = DPAD / 8;  // 16-byte pieces of a row
      constexpr int kRowsAtATime = 32 / kChunks;
      const int c = lane % kChunks, d0 = c * 8;
      int row = lane / kChunks, g = row / M, m = row - g * M;
#pragma unroll 4
      for (int i = 0; i < NR / kRowsAtATime; ++i) {
        const bool on = row < rows && d0 < p.D;
        ptx::cp_async16(dst + (uint32_t)(c >> 3) * L::kQSlabBytes + (uint32_t)row * 128u + (((uint32_t)c & 7u) ^ ((uint32_t)row & 7u)) * 16u,
                        on ? q + g * qh + m * qm + d0 : q, on);
        row += kRowsAtATime;
        for (m += kRowsAtATime; m >= M; m -= M) ++g;
      }
      ptx::cp_async_wait_all();
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_q_full + 8u * buf);
      return true;
    };
    tree_query_role<2, QUANT>(p, ring, walk, lane, abort_flag, load_queries);
  } else if (warp == kSWarp) {
    // ------------------------------------------------------------------- S^T = K Q^T
    // Two score buffers: tile j may be written once the weights of tile j - 2 have been made.  (One warp that issued
    // both products was busy for 1230 cycles per tile, more than reading an 8-bit tile takes.)
    uint32_t tile = 0, q_seq = 0;
    bool ok = true;
    while (ok && walk.next(seg)) {
      ok = TREE_WAIT(bar_q_full + 8u * (q_seq % L::kQBuffers), (q_seq / L::kQBuffers) & 1u, ST_TR_WAIT_Q_FULL);
      const uint32_t b_lo = ptx::smem_desc_lo(base + L::off_q + (q_seq % L::kQBuffers) * L::kQBytes);
      for (int t = seg.lo; ok && t < seg.hi; ++t, ++tile) {
        const uint32_t buf = tile & 1u, slot = tile % KS;
        ok = TREE_WAIT(bar_k_full + 8u * slot, (tile / KS) & 1u, ST_TR_WAIT_K_FULL);
        if (!ok) break;
        if (tile >= 2) ok = TREE_WAIT_BEHIND(bar_p + 8u * buf, ((tile - 2u) >> 1) & 1u, ST_TR_WAIT_P);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        if (ptx::elect_one()) {
          const uint32_t a_lo = ptx::smem_desc_lo(base + L::off_k + slot * L::kTileBytes);
          const uint32_t d = tmem_base + buf * NR;
#pragma unroll
          for (int kk = 0; kk < DPAD / 16; ++kk) {
            const uint32_t in = (uint32_t)(kk & 3) * 2u;
            if (kk < p.k_steps)
              ptx::umma_step<false>(d, a_lo + (uint32_t)(kk >> 2) * (L::kSlabBytes >> 4) + in,
                                    b_lo + (uint32_t)(kk >> 2) * (L::kQSlabBytes >> 4) + in, p.idesc_s, kk == 0);
          }
          ptx::umma_commit(bar_s + 8u * buf);
          ptx::umma_commit(bar_k_empty + 8u * slot);
          if (t + 1 == seg.hi) ptx::umma_commit(bar_q_empty + 8u * (q_seq % L::kQBuffers));
        }
        __syncwarp();
      }
      ++q_seq;
    }
  } else if (warp == kOWarp) {
    // ------------------------------------------------------------------- O^T += V^T P^T
    uint32_t tile = 0;
    bool ok = true;
    while (ok && walk.next(seg)) {
      for (int t = seg.lo; ok && t < seg.hi; ++t, ++tile) {
        const uint32_t buf = tile & 1u, slot = tile % VS;
        ok = TREE_WAIT(bar_v_full + 8u * slot, (tile / VS) & 1u, ST_TR_WAIT_V_FULL);
        if (!ok) break;
        ok = TREE_WAIT_BEHIND(bar_p + 8u * buf, (tile >> 1) & 1u, ST_TR_WAIT_P);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        if (ptx::elect_one()) {
          const uint32_t a_lo = ptx::smem_desc_lo_mn(base + L::off_v + slot * L::kTileBytes, L::kSlabBytes);
          const uint32_t b_lo = ptx::smem_desc_lo_mn(base + L::off_p + buf * L::kPStep, L::kSlabBytes);
          const uint32_t d = tmem_base + 2 * NR;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys: 2048 bytes of either operand
            ptx::umma_f16(d, a_lo + kk * (2048u >> 4), b_lo + kk * (2048u >> 4), p.idesc_o, t > seg.lo || kk > 0);
          ptx::umma_commit(bar_pv + 8u * buf);
          ptx::umma_commit(bar_v_empty + 8u * slot);
        }
        __syncwarp();
      }
    }
  } else if (warp >= kLoadWarp) {
    // -------------------------------------------------------- key and value tiles
    tree_load_roles<T, DPAD, KS, VS, L::SS, 2, FORMAT>(p, ring, &tmap_k, &tmap_v, walk, warp - kLoadWarp, lane, abort_flag, bad_flag);
  } else {
    // -------------------------------------------------------------- softmax warps
    const int wg = warp >> 2, wq = warp & 3;
    const int r0 = wg * W;             // this warpgroup's first row
    const int key = wq * 32 + lane;    // of the tile; of D in O^T
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const uint32_t o_addr = tmem_base + lanes + 2 * NR + r0;
    const uint32_t vote_bar = bar_vote + 8u * wg;
    volatile int* const vote = votes_s + 2 * wg;
    float* const ref_s = reinterpret_cast<float*>(smem + L::off_ref) + wq * NR + r0;  // this warp's copy, minus the reference
    float* const top_s = reinterpret_cast<float*>(smem + L::off_top) + r0;            // [4 warps], NR apart
    const uint32_t p_row = base + L::off_p + (uint32_t)key * 128u, x7 = (uint32_t)key & 7u;
    uint32_t tile_seq = 0, votes = 0;
    bool ok = true;
    auto sync_group = [&]() {  // a bounded barrier over the warpgroup
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(vote_bar);
      ok = TREE_WAIT_BEHIND(vote_bar, votes & 1u, ST_TD_WAIT_VOTE);
      ++votes;
      return ok;
    };
    // The product of tile `i`, at most the one before the last whose weights have been made: every product is waited for in
    // turn (tile j's weights overwrite tile j - 2's), so that no parity can be mistaken for an older phase's.
    auto wait_pv = [&](uint32_t i, int code) {
      ok = TREE_WAIT(bar_pv + 8u * (i & 1u), (i >> 1) & 1u, code);
      if (ok) ptx::tc_fence_after_sync();
      return ok;
    };
    while (ok && walk.next(seg)) {
      float l[W];
#pragma unroll
      for (int e = 0; e < W; ++e) l[e] = 0.f;
      __syncwarp();
      if (lane < W) ref_s[lane] = kNothingSeen;
      __syncwarp();
      for (int t = seg.lo; t < seg.hi; ++t, ++tile_seq) {
        const uint32_t buf = tile_seq & 1u;
        const uint32_t s_addr = tmem_base + lanes + buf * NR + r0;
        ok = TREE_WAIT(bar_s + 8u * buf, (tile_seq >> 1) & 1u, ST_TR_WAIT_S);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const bool edge = (t + 1) * kTreeTile > seg.have;
        const uint32_t bits = edge ? decode_row_bits(p, seg, t * kTreeTile + key, r0, W) : 0xffffffffu;
        if (edge) __syncwarp();  // the lanes took different ways; tensor memory is read by a converged warp
        auto load_scores = [&](uint32_t (&x)[W]) {
          tmem_row_ld<W>(s_addr, x);
          int masked = edge;
          asm volatile("" : "+r"(masked));  // (or the compiler makes a second copy of the whole tile for edge tiles)
          if (masked) {
#pragma unroll
            for (int e = 0; e < W; ++e) x[e] = (bits >> e) & 1u ? x[e] : 0xff800000u;
          }
        };
        uint32_t x[W];
        load_scores(x);
        // exponents against the reference as it is: has one passed 8 above the aim?
        constexpr float kAim = tree_aim<T>();
        float w[W];
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < W; e += 4) {
          const float4 nm = *reinterpret_cast<const float4*>(ref_s + e);
          const float2 a = __ffma2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), make_float2(p.scale2, p.scale2), make_float2(nm.x, nm.y));
          const float2 b = __ffma2_rn(make_float2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), make_float2(p.scale2, p.scale2), make_float2(nm.z, nm.w));
          most = ptx::max3(ptx::max3(most, a.x, a.y), b.x, b.y);
          w[e] = a.x, w[e + 1] = a.y, w[e + 2] = b.x, w[e + 3] = b.y;
        }
        if (__any_sync(0xffffffffu, most > 8.f + kAim) && lane == 0) vote[buf] = (int)tile_seq;
        if (!sync_group()) break;
        if (vote[buf] == (int)tile_seq) {
          // the rows' maxima over the tile's 128 keys; O^T, the sums and the reference follow where a row has grown
          float top = -INFINITY;
          // (Scores and references are read again: kept in registers for this rare path they spilled the common one's values,
          // 64 bf16 rows over 16 x 8 heads of 4096 keys took 90 us instead of 70.)
          asm volatile("" ::: "memory");
          load_scores(x);
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float largest = ptx::redux_max(__uint_as_float(x[e]));
            if (lane == e) top = largest;
          }
          if (lane < W) top_s[wq * NR + lane] = top;
          if (!sync_group()) break;
          float alpha = 1.f;
          if (lane < W) {
            top = fmaxf(fmaxf(top_s[lane], top_s[NR + lane]), fmaxf(top_s[2 * NR + lane], top_s[3 * NR + lane])) * p.scale2;
            const float nm = ref_s[lane];
            if (top + nm > 8.f + kAim) {
              const float now = kAim - top;
              alpha = nm == kNothingSeen ? 0.f : ptx::ex2(now - nm);
              ref_s[lane] = now;
            }
          }
          __syncwarp();
          if (t > seg.lo) {
            if (!wait_pv(tile_seq - 1u, ST_TD_WAIT_PV)) break;  // it may still be adding to O^T
            uint32_t o[W];
            tmem_row_ld<W>(o_addr, o);
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const float f = __shfl_sync(0xffffffffu, alpha, e);
              o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              l[e] *= f;
            }
            tmem_row_st<W>(o_addr, o);
            ptx::tmem_st_wait();
          }
          load_scores(x);
#pragma unroll
          for (int e = 0; e < W; ++e) w[e] = fmaf(__uint_as_float(x[e]), p.scale2, ref_s[e]);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) w[e] = ptx::ex2(w[e]);
        if (tile_seq >= 2 && !wait_pv(tile_seq - 2u, ST_TD_WAIT_PV)) break;  // it read this buffer
        const uint32_t p_buf = p_row + (NR == 64 ? buf * L::kPStep : 0u);
        const uint32_t c0 = NR == 64 ? (uint32_t)wg * 4u : buf * 4u;  // first 16-byte piece of the key's row
#pragma unroll
        for (int e = 0; e < W; e += 8) {
          const uint4 v = make_uint4(pack2(w[e], w[e + 1], T()), pack2(w[e + 2], w[e + 3], T()), pack2(w[e + 4], w[e + 5], T()),
                                     pack2(w[e + 6], w[e + 7], T()));
          ptx::sts128(p_buf + (((c0 + (uint32_t)(e >> 3)) ^ x7) << 4), v);
        }
        if (!QUANT && edge) {
          const uint32_t slot = tile_seq % VS;
          ok = TREE_WAIT(bar_v_full + 8u * slot, (tile_seq / VS) & 1u, ST_TR_WAIT_V_FULL_SM);
          if (!ok) break;
          constexpr int kPieces = DPAD / 8 / kGroups;  // each warpgroup takes its share of the 16-byte pieces
          tree_clean_values<T, DPAD>(base + L::off_v + slot * L::kTileBytes, key, t * kTreeTile + key, seg, wg * kPieces, (wg + 1) * kPieces, bad_flag);
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_p + 8u * buf);
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          const float2 sum = __fadd2_rn(make_float2(l[e], l[e + 1]), make_float2(w[e], w[e + 1]));
          l[e] = sum.x, l[e + 1] = sum.y;
        }
      }
      if (!ok) break;
      // ------------------------------------------------ the segment's results
      // the sums over the keys: a warp's by exchanging halves until lane e has row e's, then over the warps
#pragma unroll
      for (int o = W / 2; o; o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int e = 0; e < o; ++e) {
          const float keep = up ? l[e + o] : l[e], give = up ? l[e] : l[e + o];
          l[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      if (W == 16) l[0] += __shfl_xor_sync(0xffffffffu, l[0], 16);
      if (!wait_pv(tile_seq - 1u, ST_TR_WAIT_O)) break;
      float* const sum_s = reinterpret_cast<float*>(smem + L::off_top) + r0;  // the maxima are not needed any more
      if (!sync_group()) break;
      if (lane < W) sum_s[wq * NR + lane] = l[0];
      if (!sync_group()) break;
      const bool whole = seg.whole();
      const size_t part = ((size_t)blockIdx.x * 2 + seg.slot()) * p.part_rows;
      const size_t out_row0 = (size_t)(seg.b * p.Hk + seg.group) * p.rows;
      const int mine = lane & (W - 1), my_row = r0 + mine;
      const float sum = (sum_s[mine] + sum_s[NR + mine]) + (sum_s[2 * NR + mine] + sum_s[3 * NR + mine]);
      const float factor = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      if (wq == 0 && lane < W && my_row < p.rows) {
        const float m_ref = -ref_s[mine];
        if (!whole)
          p.part_ml[part + my_row] = make_float2(m_ref, sum);
        else if (p.lse)
          p.lse[out_row0 + my_row] = sum == 0.f ? -INFINITY : (m_ref + log2f(sum)) * 0.69314718055994531f;
      }
      __syncwarp();  // only some lanes had statistics to write
      uint32_t o[W];
      tmem_row_ld<W>(o_addr, o);
      if (*bad_flag && key < p.D) {
        for (int r = r0; r < min(r0 + W, p.rows); ++r) {
          const int m = r % p.M;
          float fix = 0.f;
          tree_add_non_finite<T, FORMAT>(p, seg, p.mask ? p.mask + ((size_t)(p.mask_shared ? 0 : seg.b) * p.M + m) * p.words : nullptr, m, key, 1, &fix);
#pragma unroll
          for (int e = 0; e < W; ++e)
            if (e == r - r0) o[e] = __float_as_uint(__uint_as_float(o[e]) + fix);
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float v = __uint_as_float(o[e]) * __shfl_sync(0xffffffffu, factor, e);
        const int row = r0 + e;
        if (row < p.rows && key < p.D) {
          if (whole)
            reinterpret_cast<T*>(p.out)[(out_row0 + row) * p.D + key] = from_f32<T>(v);
          else
            p.part_o[(part + row) * DPAD + key] = v;
        }
      }
      // the next segment's maxima and first product may overwrite what has been read here
      ptx::tc_fence_before_sync();
      if (!sync_group()) break;
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
  if (warp == kSWarp) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmem);
  }
}

}  // namespace fcr
