// C entries of the serving operators: norm + rotation, the KV cache, attention of drafted tokens.
//
// Included by colreduce_sm100.cu after the other entry points (needs fail, cuda_fail, launch_kernel, device_info).
#pragma once

namespace fcr {

static bool kv_aligned(const void* ptr, const int64_t* strides, const int32_t* sizes, int dims, int elem_bytes, int bytes) {
  if (reinterpret_cast<uintptr_t>(ptr) % bytes) return false;
  for (int i = 0; i < dims; ++i)
    if (sizes[i] > 1 && (strides[i] * elem_bytes) % bytes) return false;
  return true;
}

static int check_cache(const fcr_kv_cache& c, const void* k, const void* v, const void* ks, const void* vs) {
  if (!k || !v) return fail(FCR_ERR_BAD_ARG, "null cache");
  if (c.B <= 0 || c.H <= 0 || c.N <= 0 || c.D <= 0) return fail(FCR_ERR_BAD_ARG, "cache sizes must be positive");
  if (c.D > 256) return fail(FCR_ERR_UNSUPPORTED, "head dimension " + std::to_string(c.D) + " exceeds 256");
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

static unsigned kv_blocks(long long rows, int group, int sms) {
  const long long per_block = 256 / group;
  return (unsigned)std::min<long long>((rows + per_block - 1) / per_block, (long long)sms * 32);
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

template <typename T>
static cudaError_t launch_tree(int format, const TreeParams& p, cudaStream_t stream) {
  const long long rows = (long long)p.B * p.Hq * p.M;
  const dim3 grid((unsigned)((rows + 3) / 4)), block(128);
  if (format == FCR_KV_FP8) return launch_kernel(tree_rows_kernel<T, FCR_KV_FP8>, grid, block, 0, stream, false, p);
  if (format == FCR_KV_INT8) return launch_kernel(tree_rows_kernel<T, FCR_KV_INT8>, grid, block, 0, stream, false, p);
  return launch_kernel(tree_rows_kernel<T, FCR_KV_16BIT>, grid, block, 0, stream, false, p);
}

static int check_tree(const fcr_kv_cache& c, const fcr_tree& t) {
  if (c.B <= 0 || c.H <= 0 || c.N <= 0 || c.D <= 0 || t.Hq <= 0 || t.M <= 0)
    return fail(FCR_ERR_BAD_ARG, "attention sizes must be positive");
  if (t.Hq % c.H) return fail(FCR_ERR_BAD_ARG, "query heads must be a multiple of the cache's heads");
  if (t.M > 256) return fail(FCR_ERR_UNSUPPORTED, std::to_string(t.M) + " drafted tokens exceed 256");
  if (c.D > 128 || c.D % (c.format == FCR_KV_16BIT ? 8 : 16))
    return fail(FCR_ERR_UNSUPPORTED, "attention takes head dimensions up to 128, multiples of 8 for a 16-bit cache and of 16 for an 8-bit one");
  if (t.index_bits != 32 && t.index_bits != 64) return fail(FCR_ERR_BAD_ARG, "index_bits must be 32 or 64");
  if (t.q_strides[3] != 1) return fail(FCR_ERR_UNSUPPORTED, "innermost stride of the queries must be 1");
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

}  // namespace fcr

extern "C" {

int fcr_qk_norm_rope(const fcr_rope* problem, const void* q, const void* k, const void* positions,
                     const float* inv_freq, const void* q_weight, const void* k_weight, void* q_out,
                     void* k_out, void* stream_v) {
  if (!problem) return fail(FCR_ERR_BAD_ARG, "null argument");
  const fcr_rope& r = *problem;
  if (r.B <= 0 || r.M <= 0 || r.D <= 0 || r.Hq < 0 || r.Hk < 0 || r.Hq + r.Hk <= 0)
    return fail(FCR_ERR_BAD_ARG, "sizes must be positive");
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
  const long long rows = (long long)r.B * r.M * (r.Hq + r.Hk);
  const dim3 grid((unsigned)std::min<long long>((rows + 7) / 8, (long long)sms * 64)), block(256);
  cudaError_t e;
  if (r.dtype == FCR_F16)
    e = launch_kernel(rope_rows_kernel<__half>, grid, block, 0, stream, false, p);
  else if (r.dtype == FCR_BF16)
    e = launch_kernel(rope_rows_kernel<__nv_bfloat16>, grid, block, 0, stream, false, p);
  else
    e = launch_kernel(rope_rows_kernel<float>, grid, block, 0, stream, false, p);
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
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != FCR_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const unsigned blocks = kv_blocks(2LL * c.B * c.H * M, p.group, sms);
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
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != FCR_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const unsigned blocks = kv_blocks(2LL * c.B * c.H * n, p.group, sms);
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
  (void)num_sms;
  return 256;
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
  TreeParams p;
  memset(&p, 0, sizeof(p));
  p.q = q;
  p.cache[0] = k_cache;
  p.cache[1] = v_cache;
  p.scales[0] = static_cast<const unsigned char*>(k_scales);
  p.scales[1] = static_cast<const unsigned char*>(v_scales);
  p.lengths = lengths;
  p.mask = static_cast<const unsigned char*>(mask);
  p.out = out;
  p.lse = lse;
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
  p.mask_b = t.mask_strides[0];
  p.mask_m = t.mask_strides[1];
  p.B = c.B;
  p.Hq = t.Hq;
  p.Hk = c.H;
  p.M = t.M;
  p.N = c.N;
  p.D = c.D;
  p.G = t.Hq / c.H;
  p.index_bits = t.index_bits;
  p.scale2 = t.scale * 1.4426950408889634f;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  if (!workspace || workspace_bytes < 256) return fail(FCR_ERR_WORKSPACE, "workspace missing or too small");
  cudaError_t e = cudaMemsetAsync(workspace, 0, 256, stream);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync");
  e = c.dtype == FCR_F16 ? launch_tree<__half>(c.format, p, stream) : launch_tree<__nv_bfloat16>(c.format, p, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree attention launch");
  return FCR_OK;
}

}  // extern "C"
