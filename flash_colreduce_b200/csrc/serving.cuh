// C entries of the serving operators: norm + rotation, the KV cache, attention of drafted tokens.
//
// Included by colreduce_sm100.cu after the other entry points (needs fail, cuda_fail, launch_kernel, device_info).
#pragma once

#include <cfloat>

namespace fcr {

constexpr float kLog2E = 1.4426950408889634f;

constexpr int32_t kMaxRows = 1 << 30;  // rows, positions and heads are counted in 32 bits, in steps of up to 1024
static int too_many(const char* what) { return fail(FCR_ERR_UNSUPPORTED, std::string("more than ") + std::to_string(kMaxRows) + " " + what); }

static bool kv_aligned(const void* ptr, const int64_t* strides, const int32_t* sizes, int dims, int elem_bytes, int bytes) {
  if (reinterpret_cast<uintptr_t>(ptr) % bytes) return false;
  for (int i = 0; i < dims; ++i)
    if (sizes[i] > 1 && (strides[i] * elem_bytes) % bytes) return false;
  return true;
}

template <typename T, int LPR>
static cudaError_t launch_rope_vector(const RopeParams& p, dim3 grid, cudaStream_t stream) {
  return p.interleaved ? launch_kernel(rope_vector_kernel<T, LPR, true>, grid, dim3(256), 0, stream, false, p)
                       : launch_kernel(rope_vector_kernel<T, LPR, false>, grid, dim3(256), 0, stream, false, p);
}
template <typename T>
static cudaError_t launch_rope(RopeParams& p, int sms, cudaStream_t stream) {
  const int heads = p.heads[0] + p.heads[1];
  bool vec = p.D % 16 == 0 && p.half % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    const int64_t st[3] = {p.sb[i], p.sh[i], p.sm[i]};
    const int32_t sizes[3] = {p.B, p.heads[i], p.M};
    vec = vec && kv_aligned(p.x[i], st, sizes, 3, sizeof(T), 16) && reinterpret_cast<uintptr_t>(p.y[i]) % 16 == 0 &&
          reinterpret_cast<uintptr_t>(p.weight[i]) % 16 == 0;
  }
  const long long tokens = (long long)p.B * p.M;
  if (vec) {
    const int lpr = p.D <= 64 ? 4 : p.D <= 128 ? 8 : 16, at_a_time = 32 / lpr;
    // All heads of a token in one warp spare it angles; with few tokens the heads are spread until there are 8 warps per SM.
    const long long want = std::max<long long>(1, (8LL * sms + tokens - 1) / tokens);
    const int chunks = (int)std::min<long long>(want, (heads + at_a_time - 1) / at_a_time);
    p.heads_per_warp = ((heads + chunks - 1) / chunks + at_a_time - 1) / at_a_time * at_a_time;
    const long long blocks = (tokens + 7) / 8 * ((heads + p.heads_per_warp - 1) / p.heads_per_warp);
    if (blocks <= 0x7fffffffLL) {
      const dim3 grid((unsigned)blocks);
      return lpr == 4 ? launch_rope_vector<T, 4>(p, grid, stream) : lpr == 8 ? launch_rope_vector<T, 8>(p, grid, stream) : launch_rope_vector<T, 16>(p, grid, stream);
    }
  }
  const long long rows = tokens * heads;
  return launch_kernel(rope_rows_kernel<T>, dim3((unsigned)std::min<long long>((rows + 7) / 8, (long long)sms * 64)), dim3(256), 0, stream, false, p);
}

static int check_cache(const fcr_kv_cache& c, const void* k, const void* v, const void* ks, const void* vs) {
  if (!k || !v) return fail(FCR_ERR_BAD_ARG, "null cache");
  if (c.B <= 0 || c.H <= 0 || c.N <= 0 || c.D <= 0) return fail(FCR_ERR_BAD_ARG, "cache sizes must be positive");
  if (c.D > 256) return fail(FCR_ERR_UNSUPPORTED, "head dimension " + std::to_string(c.D) + " exceeds 256");
  if (c.N > kMaxRows) return too_many("positions");
  if ((long long)c.B * c.H > kMaxRows) return too_many("heads of sequences");
  if (c.dtype != FCR_F16 && c.dtype != FCR_BF16) return fail(FCR_ERR_UNSUPPORTED, "a cache holds fp16 or bf16 values");
  if (c.format != FCR_KV_16BIT && c.format != FCR_KV_FP8 && c.format != FCR_KV_INT8)
    return fail(FCR_ERR_BAD_ARG, "invalid cache format");
  if (c.k_strides[3] != 1 || c.v_strides[3] != 1) return fail(FCR_ERR_UNSUPPORTED, "innermost stride of the cache must be 1");
  if (c.format != FCR_KV_16BIT && (!ks || !vs)) return fail(FCR_ERR_BAD_ARG, "an 8-bit cache needs its scales");
  return FCR_OK;
}

static void fill_kv(KvTensor (&t)[2], const fcr_kv_cache& c, const void* k, const void* v, const void* ks, const void* vs) {
  const void* data[2] = {k, v};
  const void* scales[2] = {ks, vs};
  const int64_t* st[2] = {c.k_strides, c.v_strides};
  const int64_t* ss[2] = {c.k_scale_strides, c.v_scale_strides};
  for (int i = 0; i < 2; ++i) {
    t[i].data = const_cast<void*>(data[i]);
    t[i].scales = static_cast<unsigned char*>(const_cast<void*>(scales[i]));
    t[i].sb = st[i][0];
    t[i].sh = st[i][1];
    t[i].sn = st[i][2];
    t[i].ssb = ss[i][0];
    t[i].ssh = ss[i][1];
    t[i].ssn = ss[i][2];
  }
}

static bool cache_vectors(const fcr_kv_cache& c, const void* k, const void* v) {
  const int elem = c.format == FCR_KV_16BIT ? 2 : 1;
  const int32_t sizes[3] = {c.B, c.H, c.N};
  return c.D % 8 == 0 && kv_aligned(k, c.k_strides, sizes, 3, elem, 8 * elem) && kv_aligned(v, c.v_strides, sizes, 3, elem, 8 * elem);
}

static int kv_group(int D) {
  int g = 1;
  while (8 * g < D) g *= 2;
  return g;
}

// Blocks for `rows` rows of each of 2 * B * H (K or V, sequence, head); 0 when the grid would be too large.
static unsigned kv_blocks(int B, int H, int rows, int group) {
  const int per_block = 256 / group * kKvRows;
  const long long blocks = 2LL * B * H * ((rows + per_block - 1) / per_block);
  return blocks > 0x7fffffffLL ? 0u : (unsigned)blocks;
}

template <typename T, int FORMAT>
static cudaError_t launch_append(const KvAppendParams& p, bool vec, unsigned blocks, cudaStream_t stream) {
  return vec ? launch_kernel(kv_append_kernel<T, FORMAT, true>, dim3(blocks), dim3(256), 0, stream, false, p)
             : launch_kernel(kv_append_kernel<T, FORMAT, false>, dim3(blocks), dim3(256), 0, stream, false, p);
}
template <typename T>
static cudaError_t launch_append_f(int format, const KvAppendParams& p, bool vec, unsigned blocks, cudaStream_t stream) {
  if (format == FCR_KV_FP8) return launch_append<T, FCR_KV_FP8>(p, vec, blocks, stream);
  if (format == FCR_KV_INT8) return launch_append<T, FCR_KV_INT8>(p, vec, blocks, stream);
  return launch_append<T, FCR_KV_16BIT>(p, vec, blocks, stream);
}
template <typename T, int FORMAT>
static cudaError_t launch_read(const KvReadParams& p, bool vec, unsigned blocks, cudaStream_t stream) {
  return vec ? launch_kernel(kv_read_kernel<T, FORMAT, true>, dim3(blocks), dim3(256), 0, stream, false, p)
             : launch_kernel(kv_read_kernel<T, FORMAT, false>, dim3(blocks), dim3(256), 0, stream, false, p);
}
template <typename T>
static cudaError_t launch_read_f(int format, const KvReadParams& p, bool vec, unsigned blocks, cudaStream_t stream) {
  if (format == FCR_KV_FP8) return launch_read<T, FCR_KV_FP8>(p, vec, blocks, stream);
  if (format == FCR_KV_INT8) return launch_read<T, FCR_KV_INT8>(p, vec, blocks, stream);
  return launch_read<T, FCR_KV_16BIT>(p, vec, blocks, stream);
}

static int check_tree(const fcr_kv_cache& c, const fcr_tree& t) {
  if (c.B <= 0 || c.H <= 0 || c.N <= 0 || c.D <= 0 || t.Hq <= 0 || t.M <= 0)
    return fail(FCR_ERR_BAD_ARG, "attention sizes must be positive");
  if (c.N > kMaxRows) return too_many("positions");
  if ((long long)c.B * c.H > kMaxRows) return too_many("heads of sequences");
  if ((long long)(t.Hq / c.H) * t.M > kMaxRows) return too_many("query rows per cache head");
  if (t.Hq % c.H) return fail(FCR_ERR_BAD_ARG, "query heads must be a multiple of the cache's heads");
  if (t.M > kTreeMaxM) return fail(FCR_ERR_UNSUPPORTED, std::to_string(t.M) + " drafted tokens exceed " + std::to_string(kTreeMaxM));
  if (c.D > 128 || c.D % (c.format == FCR_KV_16BIT ? 8 : 16))
    return fail(FCR_ERR_UNSUPPORTED, "attention takes head dimensions up to 128, multiples of 8 for a 16-bit cache and of 16 for an 8-bit one");
  if (t.index_bits != 32 && t.index_bits != 64) return fail(FCR_ERR_BAD_ARG, "index_bits must be 32 or 64");
  if (t.q_strides[3] != 1) return fail(FCR_ERR_UNSUPPORTED, "innermost stride of the queries must be 1");
  if (!(fabsf(t.scale) * kLog2E <= FLT_MAX)) return fail(FCR_ERR_BAD_ARG, "the scale must be finite in fp32, and times log2(e)");
  const int32_t sizes[3] = {c.B, c.H, c.N};
  const int elem = c.format == FCR_KV_16BIT ? 2 : 1;
  for (const int64_t* st : {c.k_strides, c.v_strides}) {
    if (st[3] != 1) return fail(FCR_ERR_UNSUPPORTED, "innermost stride of the cache must be 1");
    for (int i = 0; i < 3; ++i)
      if (sizes[i] > 1 && (st[i] <= 0 || (st[i] * elem) % 16))
        return fail(FCR_ERR_UNSUPPORTED, "strides of the cache must be positive multiples of 16 bytes");
  }
  return FCR_OK;
}

// Tensor map over an 8-bit cache's codes: a box is 128 rows of 64 codes of one head, as they lie; codes beyond D or
// beyond the capacity read as zero.
static int make_code_map(CUtensorMap* map, const void* ptr, const fcr_kv_cache& c, const int64_t* strides) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return fail(FCR_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  auto stride = [&](int64_t s) -> cuuint64_t { return s > 0 && s % 16 == 0 ? (cuuint64_t)s : 256u; };  // of a dimension of one: never used
  cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.N, (cuuint64_t)c.H, (cuuint64_t)c.B};
  cuuint64_t gstr[3] = {stride(strides[2]), stride(strides[1]), stride(strides[0])};
  cuuint32_t box[4] = {64u, (cuuint32_t)kTreeTile, 1u, 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FCR_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult " + std::to_string((int)r));
  return FCR_OK;
}

struct HostLengths {
  const int64_t* p;
  FCR_HD long long operator()(int b) const { return (long long)p[b]; }
};

// What the host decides of an attention call: the kernel's variant and the workspace.
struct TreePlan {
  int rows, decode_rows, part_rows, row_tiles, ctas, words, mask_rows;
  bool pair;
  int d_pad;
  size_t off_mask, off_ml, off_o, bytes;
};
static TreePlan plan_tree(const fcr_kv_cache& c, const fcr_tree& t, int sms) {
  TreePlan pl;
  pl.rows = t.Hq / c.H * t.M;
  pl.pair = pl.rows > 128;
  pl.row_tiles = pl.pair ? (pl.rows + 255) / 256 : 1;
  pl.decode_rows = pl.rows > 64 ? 0 : pl.rows <= 16 ? 16 : pl.rows <= 32 ? 32 : 64;
  pl.part_rows = pl.pair ? 256 : pl.decode_rows ? pl.decode_rows : 128;
  pl.d_pad = c.D <= 64 ? 64 : 128;
  const long long most = (long long)c.B * c.H * pl.row_tiles * ((c.N + kTreeTile - 1) / kTreeTile);
  pl.ctas = (int)std::min<long long>(most, sms);
  pl.words = (t.M + 31) / 32;
  pl.mask_rows = t.mask_strides[0] == 0 ? 1 : c.B;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  pl.off_mask = kStatusWords * 4;
  pl.off_ml = up(pl.off_mask + (size_t)pl.mask_rows * t.M * pl.words * 4);
  pl.off_o = up(pl.off_ml + (size_t)pl.ctas * 2 * pl.part_rows * 8);
  pl.bytes = up(pl.off_o + (size_t)pl.ctas * 2 * pl.part_rows * pl.d_pad * 4);
  return pl;
}

template <typename T, int DPAD>
static int launch_tree_kernel(void (*kern)(const CUtensorMap, const CUtensorMap, const TreeParams), int smem, int threads,
                              std::atomic<unsigned long long>& opted_in, const CUtensorMap& map_k, const CUtensorMap& map_v,
                              const TreeParams& p, const TreePlan& pl, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const unsigned long long bit = 1ULL << (t_device & 63);
  if (!(opted_in.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    opted_in.fetch_or(bit, std::memory_order_release);
  }
  e = launch_kernel(kern, dim3(pl.ctas), dim3(threads), smem, stream, true, map_k, map_v, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree attention launch");
  if (p.N > kTreeTile && pl.ctas > 1) {  // a group of one tile is never shared
    const int rows_per_tile = std::min(p.rows, 256), blocks_per_group = (rows_per_tile + 7) / 8;
    const long long blocks = (long long)p.B * p.groups * blocks_per_group;
    if (blocks > 0x7fffffffLL) return fail(FCR_ERR_UNSUPPORTED, "too many rows");
    e = launch_kernel(tree_combine_kernel<T, DPAD>, dim3((unsigned)blocks), dim3(256), 0, stream, true, p, pl.ctas, rows_per_tile,
                      blocks_per_group);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "tree combine launch");
  }
  return FCR_OK;
}
template <typename T, int DPAD, bool PAIR, int FORMAT>
static int launch_tree_rows(const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, const TreePlan& pl, cudaStream_t stream) {
  static std::atomic<unsigned long long> opted_in{0};
  constexpr bool kQuant = FORMAT != FCR_KV_16BIT;
  return launch_tree_kernel<T, DPAD>(tree_attention_kernel<T, DPAD, PAIR, FORMAT>, TreeSmem<DPAD, PAIR, kQuant>::kDynamicBytes, tree_threads<kQuant>(),
                                     opted_in, map_k, map_v, p, pl, stream);
}
template <typename T, int DPAD, int NR, int FORMAT>
static int launch_tree_keys(const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, const TreePlan& pl, cudaStream_t stream) {
  static std::atomic<unsigned long long> opted_in{0};
  constexpr bool kQuant = FORMAT != FCR_KV_16BIT;
  return launch_tree_kernel<T, DPAD>(tree_decode_kernel<T, DPAD, NR, FORMAT>, DecodeSmem<DPAD, NR, kQuant>::kDynamicBytes, decode_threads<NR, kQuant>(),
                                     opted_in,
                                     map_k, map_v, p, pl, stream);
}
template <typename T, int DPAD, int FORMAT>
static int launch_tree(const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, const TreePlan& pl, cudaStream_t stream) {
  if (pl.pair) return launch_tree_rows<T, DPAD, true, FORMAT>(map_k, map_v, p, pl, stream);
  if (pl.decode_rows == 0) return launch_tree_rows<T, DPAD, false, FORMAT>(map_k, map_v, p, pl, stream);
  if (pl.decode_rows == 16) return launch_tree_keys<T, DPAD, 16, FORMAT>(map_k, map_v, p, pl, stream);
  if (pl.decode_rows == 32) return launch_tree_keys<T, DPAD, 32, FORMAT>(map_k, map_v, p, pl, stream);
  return launch_tree_keys<T, DPAD, 64, FORMAT>(map_k, map_v, p, pl, stream);
}
template <typename T, int DPAD>
static int launch_tree_f(int format, const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, const TreePlan& pl,
                         cudaStream_t stream) {
  if (format == FCR_KV_FP8) return launch_tree<T, DPAD, FCR_KV_FP8>(map_k, map_v, p, pl, stream);
  if (format == FCR_KV_INT8) return launch_tree<T, DPAD, FCR_KV_INT8>(map_k, map_v, p, pl, stream);
  return launch_tree<T, DPAD, FCR_KV_16BIT>(map_k, map_v, p, pl, stream);
}
template <typename T>
static int launch_tree_d(int d_pad, int format, const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, const TreePlan& pl,
                         cudaStream_t stream) {
  return d_pad == 64 ? launch_tree_f<T, 64>(format, map_k, map_v, p, pl, stream) : launch_tree_f<T, 128>(format, map_k, map_v, p, pl, stream);
}

}  // namespace fcr

extern "C" {

int fcr_qk_norm_rope(const fcr_rope* problem, const void* q, const void* k, const void* positions,
                     const float* inv_freq, const void* q_weight, const void* k_weight, void* q_out,
                     void* k_out, void* stream_v) {
  if (!problem) return fail(FCR_ERR_BAD_ARG, "null argument");
  const fcr_rope& r = *problem;
  if (r.B <= 0 || r.M <= 0 || r.D <= 0 || r.Hq < 0 || r.Hk < 0 || (r.Hq == 0 && r.Hk == 0))
    return fail(FCR_ERR_BAD_ARG, "sizes must be positive");
  if (r.M > kMaxRows) return too_many("tokens");
  if ((long long)r.Hq + r.Hk > kMaxRows) return too_many("heads");
  if (r.D > 256) return fail(FCR_ERR_UNSUPPORTED, "head dimension " + std::to_string(r.D) + " exceeds 256");
  if (r.rotary < 0 || r.rotary > r.D || r.rotary % 2) return fail(FCR_ERR_BAD_ARG, "rotary must be even and lie in [0, D]");
  if ((r.Hq > 0 && (!q || !q_out)) || (r.Hk > 0 && (!k || !k_out)) || !positions || (r.rotary > 0 && !inv_freq))
    return fail(FCR_ERR_BAD_ARG, "null argument");
  if (r.dtype != FCR_F16 && r.dtype != FCR_BF16 && r.dtype != FCR_F32) return fail(FCR_ERR_BAD_ARG, "invalid dtype");
  if ((q_weight || k_weight) && r.weight_dtype != r.dtype && r.weight_dtype != FCR_F32)
    return fail(FCR_ERR_BAD_ARG, "weights must be of the inputs' type or fp32");
  if (r.position_bits != 32 && r.position_bits != 64) return fail(FCR_ERR_BAD_ARG, "position_bits must be 32 or 64");
  if ((r.Hq > 0 && r.q_strides[3] != 1) || (r.Hk > 0 && r.k_strides[3] != 1))
    return fail(FCR_ERR_UNSUPPORTED, "innermost stride must be 1");
  RopeParams p;
  memset(&p, 0, sizeof(p));
  const int64_t* st[2] = {r.q_strides, r.k_strides};
  p.x[0] = q;
  p.x[1] = k;
  p.y[0] = q_out;
  p.y[1] = k_out;
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.heads[0] = r.Hq;
  p.heads[1] = r.Hk;
  for (int i = 0; i < 2; ++i) {
    p.sb[i] = st[i][0];
    p.sh[i] = st[i][1];
    p.sm[i] = st[i][2];
  }
  p.B = r.B;
  p.M = r.M;
  p.D = r.D;
  p.half = r.rotary / 2;
  p.weight_f32 = r.weight_dtype == FCR_F32;
  p.interleaved = r.interleaved != 0;
  p.positions = positions;
  p.pos_bits = r.position_bits;
  p.pos_sb = r.position_strides[0];
  p.pos_sm = r.position_strides[1];
  p.inv_freq = inv_freq;
  p.eps = r.eps;
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != FCR_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  if (r.dtype == FCR_F16)
    e = launch_rope<__half>(p, sms, stream);
  else if (r.dtype == FCR_BF16)
    e = launch_rope<__nv_bfloat16>(p, sms, stream);
  else
    e = launch_rope<float>(p, sms, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "qk_norm_rope launch");
  return FCR_OK;
}

int fcr_kv_append(const fcr_kv_cache* cache, void* k_cache, void* v_cache, void* k_scales, void* v_scales,
                  const void* key, const int64_t key_strides[4], const void* value,
                  const int64_t value_strides[4], int32_t M, const void* lengths, const void* counts,
                  int32_t index_bits, void* stream_v) {
  if (!cache || !key || !value || !key_strides || !value_strides || !lengths) return fail(FCR_ERR_BAD_ARG, "null argument");
  const fcr_kv_cache& c = *cache;
  int rc = check_cache(c, k_cache, v_cache, k_scales, v_scales);
  if (rc != FCR_OK) return rc;
  if (M <= 0) return fail(FCR_ERR_BAD_ARG, "sizes must be positive");
  if (M > kMaxRows) return too_many("tokens");
  if (index_bits != 32 && index_bits != 64) return fail(FCR_ERR_BAD_ARG, "index_bits must be 32 or 64");
  if (key_strides[3] != 1 || value_strides[3] != 1) return fail(FCR_ERR_UNSUPPORTED, "innermost stride must be 1");
  KvAppendParams p;
  memset(&p, 0, sizeof(p));
  fill_kv(p.t, c, k_cache, v_cache, k_scales, v_scales);
  const int64_t* st[2] = {key_strides, value_strides};
  p.x[0] = key;
  p.x[1] = value;
  for (int i = 0; i < 2; ++i) {
    p.xb[i] = st[i][0];
    p.xh[i] = st[i][1];
    p.xm[i] = st[i][2];
  }
  p.B = c.B;
  p.H = c.H;
  p.N = c.N;
  p.D = c.D;
  p.M = M;
  p.group = kv_group(c.D);
  p.lengths = lengths;
  p.counts = counts;
  p.index_bits = index_bits;
  const int32_t sizes[3] = {c.B, c.H, M};
  const bool vec = cache_vectors(c, k_cache, v_cache) && kv_aligned(key, key_strides, sizes, 3, 2, 16) &&
                   kv_aligned(value, value_strides, sizes, 3, 2, 16);
  const unsigned blocks = kv_blocks(c.B, c.H, M, p.group);
  if (blocks == 0) return fail(FCR_ERR_UNSUPPORTED, "too many rows");
  int sms = 0;
  rc = device_sm_count(&sms);  // refuses a device that this library has no code for
  if (rc != FCR_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  cudaError_t e = c.dtype == FCR_F16 ? launch_append_f<__half>(c.format, p, vec, blocks, stream)
                                     : launch_append_f<__nv_bfloat16>(c.format, p, vec, blocks, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "kv_append launch");
  return FCR_OK;
}

int fcr_kv_read(const fcr_kv_cache* cache, const void* k_cache, const void* v_cache, const void* k_scales,
                const void* v_scales, const void* positions, int32_t index_bits, int32_t n, void* k_out,
                void* v_out, void* stream_v) {
  if (!cache || !k_out || !v_out) return fail(FCR_ERR_BAD_ARG, "null argument");
  const fcr_kv_cache& c = *cache;
  int rc = check_cache(c, k_cache, v_cache, k_scales, v_scales);
  if (rc != FCR_OK) return rc;
  if (n <= 0) return fail(FCR_ERR_BAD_ARG, "sizes must be positive");
  if (n > kMaxRows) return too_many("positions");
  if (positions && index_bits != 32 && index_bits != 64) return fail(FCR_ERR_BAD_ARG, "index_bits must be 32 or 64");
  KvReadParams p;
  memset(&p, 0, sizeof(p));
  fill_kv(p.t, c, k_cache, v_cache, k_scales, v_scales);
  p.y[0] = k_out;
  p.y[1] = v_out;
  p.B = c.B;
  p.H = c.H;
  p.N = c.N;
  p.D = c.D;
  p.n = n;
  p.group = kv_group(c.D);
  p.positions = positions;
  p.index_bits = index_bits;
  const bool vec = cache_vectors(c, k_cache, v_cache) && reinterpret_cast<uintptr_t>(k_out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_out) % 16 == 0;
  const unsigned blocks = kv_blocks(c.B, c.H, n, p.group);
  if (blocks == 0) return fail(FCR_ERR_UNSUPPORTED, "too many rows");
  int sms = 0;
  rc = device_sm_count(&sms);  // refuses a device that this library has no code for
  if (rc != FCR_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  cudaError_t e = c.dtype == FCR_F16 ? launch_read_f<__half>(c.format, p, vec, blocks, stream)
                                     : launch_read_f<__nv_bfloat16>(c.format, p, vec, blocks, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "kv_read launch");
  return FCR_OK;
}

size_t fcr_tree_workspace_bytes(const fcr_kv_cache* cache, const fcr_tree* tree, int32_t num_sms) {
  if (!cache || !tree) {
    fail(FCR_ERR_BAD_ARG, "null argument");
    return 0;
  }
  if (check_tree(*cache, *tree) != FCR_OK) return 0;
  int sms = num_sms;
  if (sms <= 0 && device_sm_count(&sms) != FCR_OK) return 0;
  return plan_tree(*cache, *tree, sms).bytes;
}

int fcr_tree_segment(const fcr_kv_cache* cache, const fcr_tree* tree, int32_t num_sms, const int64_t* lengths, int32_t cta,
                     int32_t index, int32_t* out) {
  if (!cache || !tree || !lengths || !out || num_sms <= 0) return fail(FCR_ERR_BAD_ARG, "null argument");
  const int rc = check_tree(*cache, *tree);
  if (rc != FCR_OK) return rc;
  const fcr_kv_cache& c = *cache;
  const TreePlan pl = plan_tree(c, *tree, num_sms);
  if (cta < 0 || cta >= pl.ctas || index < 0) return fail(FCR_ERR_BAD_ARG, "no such CTA or segment");
  const int groups = c.H * pl.row_tiles;
  long long total = 0;
  for (int b = 0; b < c.B; ++b) total += (long long)tree_tiles(tree_have(lengths[b], tree->M, c.N), tree->M, c.N) * groups;
  const int ctas = tree_ctas(total, pl.ctas);
  if (cta >= ctas) return fail(FCR_ERR_BAD_ARG, "no such CTA or segment");
  const long long lo = tree_piece(total, ctas, cta), hi = tree_piece(total, ctas, cta + 1);
  long long before = 0;
  int first = 0;
  for (; first < c.B; ++first) {
    const long long mine = (long long)tree_tiles(tree_have(lengths[first], tree->M, c.N), tree->M, c.N) * groups;
    if (lo < before + mine) break;
    before += mine;
  }
  TreeWalk<HostLengths> walk{{lengths}, c.B, groups, tree->M, c.N};
  walk.start(first, lo - before, hi - lo);
  TreeSegment s;
  for (int i = 0; i <= index; ++i)
    if (!walk.next(s)) return fail(FCR_ERR_BAD_ARG, "no such CTA or segment");
  long long group_first = (long long)s.group * s.tiles;
  for (int b = 0; b < s.b; ++b) group_first += (long long)tree_tiles(tree_have(lengths[b], tree->M, c.N), tree->M, c.N) * groups;
  const int v[10] = {s.b, s.group / pl.row_tiles, s.group % pl.row_tiles, s.lo, s.hi, s.tiles, s.whole() ? -1 : s.slot(),
                     tree_owner(total, ctas, group_first), tree_owner(total, ctas, group_first + s.tiles - 1), ctas};
  for (int i = 0; i < 10; ++i) out[i] = v[i];
  return FCR_OK;
}

int fcr_tree_attention(const fcr_kv_cache* cache, const fcr_tree* tree, const void* q, const void* k_cache,
                       const void* v_cache, const void* k_scales, const void* v_scales, const void* lengths,
                       const void* mask, void* out, float* lse, void* workspace, size_t workspace_bytes,
                       void* stream_v) {
  if (!cache || !tree || !q || !lengths || !out) return fail(FCR_ERR_BAD_ARG, "null argument");
  const fcr_kv_cache& c = *cache;
  const fcr_tree& t = *tree;
  int rc = check_cache(c, k_cache, v_cache, k_scales, v_scales);
  if (rc != FCR_OK) return rc;
  rc = check_tree(c, t);
  if (rc != FCR_OK) return rc;
  if (reinterpret_cast<uintptr_t>(k_cache) % 16 || reinterpret_cast<uintptr_t>(v_cache) % 16)
    return fail(FCR_ERR_UNSUPPORTED, "cache base address must be 16-byte aligned");
  const int32_t q_sizes[3] = {c.B, t.Hq, t.M};
  if (!kv_aligned(q, t.q_strides, q_sizes, 3, 2, 16))
    return fail(FCR_ERR_UNSUPPORTED, "base address and strides of the queries must be multiples of 16 bytes");
  if (reinterpret_cast<uintptr_t>(out) % 16) return fail(FCR_ERR_UNSUPPORTED, "output must be 16-byte aligned");
  const DeviceInfo* dev = nullptr;
  rc = device_info(&dev, true);
  if (rc != FCR_OK) return rc;
  rc = check_mailbox(*dev, nullptr);  // a wait that expired in an earlier call is reported here
  if (rc != FCR_OK) return rc;
  t_device = dev->index;
  const TreePlan pl = plan_tree(c, t, dev->sms);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < pl.bytes)
    return fail(FCR_ERR_WORKSPACE, "workspace missing, misaligned or smaller than " + std::to_string(pl.bytes) + " bytes");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const bool quant = c.format != FCR_KV_16BIT;
  TreeParams p;
  memset(&p, 0, sizeof(p));
  p.status = reinterpret_cast<int*>(ws);
  p.host_status = dev->mailbox_dev;
  p.wait_limit = g_wait_limit_override > 0 ? g_wait_limit_override : kWaitLimitCycles;
  p.skip_ring_load = g_skip_ring_load;
  p.q = q;
  p.cache[0] = k_cache;
  p.cache[1] = v_cache;
  p.scales[0] = static_cast<const unsigned char*>(k_scales);
  p.scales[1] = static_cast<const unsigned char*>(v_scales);
  p.lengths = lengths;
  p.out = out;
  p.lse = lse;
  p.part_ml = reinterpret_cast<float2*>(ws + pl.off_ml);
  p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  p.qb = t.q_strides[0];
  p.qh = t.q_strides[1];
  p.qm = t.q_strides[2];
  const int64_t* st[2] = {c.k_strides, c.v_strides};
  const int64_t* ss[2] = {c.k_scale_strides, c.v_scale_strides};
  for (int i = 0; i < 2; ++i) {
    p.cb[i] = st[i][0];
    p.ch[i] = st[i][1];
    p.cn[i] = st[i][2];
    p.sb[i] = ss[i][0];
    p.sh[i] = ss[i][1];
    p.sn[i] = ss[i][2];
  }
  p.B = c.B;
  p.Hq = t.Hq;
  p.Hk = c.H;
  p.M = t.M;
  p.N = c.N;
  p.D = c.D;
  p.G = t.Hq / c.H;
  p.rows = pl.rows;
  p.row_tiles = pl.row_tiles;
  p.groups = c.H * pl.row_tiles;
  p.part_rows = pl.part_rows;
  p.words = pl.words;
  p.mask_shared = t.mask_strides[0] == 0;
  p.index_bits = t.index_bits;
  float s2 = fabsf(t.scale) * kLog2E;
  if (!(s2 >= 1e-30f)) s2 = 1e-30f;  // scale 0: every score becomes (numerically) zero
  p.scale2 = s2;
  p.idesc_s = instr_desc(c.dtype, t.scale < 0.f);
  p.idesc_o = instr_desc(c.dtype, false);
  const uint32_t n_field = 63u << 17;
  if (pl.decode_rows) {  // N = the rows; in V^T P^T both operands are MN-major (bits 15 and 16)
    p.idesc_s = (p.idesc_s & ~n_field) | ((uint32_t)(pl.decode_rows >> 3) << 17);
    p.idesc_o = (p.idesc_o & ~n_field) | (3u << 15) | ((uint32_t)(pl.decode_rows >> 3) << 17);
  } else {  // P V: the second operand is MN-major (bit 16), N = the padded head dimension
    p.idesc_o = (p.idesc_o & ~n_field) | (1u << 16) | ((uint32_t)(pl.d_pad >> 3) << 17);
  }
  p.k_steps = (c.D + 15) / 16;
  CUtensorMap map_k, map_v;
  memset(&map_k, 0, sizeof(map_k));
  memset(&map_v, 0, sizeof(map_v));
  if (quant) {
    rc = make_code_map(&map_k, k_cache, c, c.k_strides);
    if (rc == FCR_OK) rc = make_code_map(&map_v, v_cache, c, c.v_strides);
    if (rc != FCR_OK) return rc;
  } else {
    rc = make_tensor_map(&map_k, k_cache, c.dtype, c.D, c.N, c.H, c.B, c.k_strides);
    if (rc != FCR_OK) return rc;
    rc = make_tensor_map(&map_v, v_cache, c.dtype, c.D, c.N, c.H, c.B, c.v_strides);
    if (rc != FCR_OK) return rc;
  }
  if (mask) {
    const long long n_words = (long long)pl.mask_rows * t.M * pl.words;
    if (n_words > 0x7fffffffLL) return fail(FCR_ERR_UNSUPPORTED, "mask too large");
    uint32_t* packed = reinterpret_cast<uint32_t*>(ws + pl.off_mask);
    p.mask = packed;
    cudaError_t e = launch_kernel(tree_pack_mask_kernel, dim3((unsigned)((n_words + 7) / 8)), dim3(256), 0, stream, true,
                                  static_cast<const unsigned char*>(mask), (long long)t.mask_strides[0], (long long)t.mask_strides[1],
                                  (int)t.M, pl.words, (int)n_words, packed);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "mask packing launch");
  }
  return c.dtype == FCR_F16 ? launch_tree_d<__half>(pl.d_pad, c.format, map_k, map_v, p, pl, stream)
                            : launch_tree_d<__nv_bfloat16>(pl.d_pad, c.format, map_k, map_v, p, pl, stream);
}

}  // extern "C"
