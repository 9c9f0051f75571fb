// Dynamic int8 quantisation of K and V into the paged cache, and the way back out of it.
#include "paged_cache.cuh"
#include "tma_pipe.cuh"

namespace mcop {
namespace {

// ---------------------------------------------------------------------------------------------
// Store: per (token, head) row  s = max|x| / 127 (one IEEE fp32 division),  code = nearest integer of the REAL quotient
// x / s, ties to even.  The quotient is never formed: n = rint(x * rn(1/s)) is off by one at most (|x * rn(1/s)| <= 127.5
// and carries two roundings, 2^-16 in absolute terms), and the sign of the residual fma(-(n +- 1/2), s, x), which one rounding
// cannot change, says on which side of the midpoint x lies.  Only lanes within 2^-12 of a midpoint look.
// A row of zeros has s = 0 and codes 0; a row that holds a NaN or an infinity has s = NaN and codes 0, so that it reads
// back as NaN instead of as plausible values.
//
// Bound: HBM bytes (2 * head_size read, head_size + 4 written per row).  A row sits on LANES lanes of 16 elements: two
// 16-byte loads and one 16-byte store per lane; a thread does one row slice, so 64 KB of loads are in flight per SM.
// ---------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  float a[8], b[8];
  Vec8<T>::load_nc(p, a);
  Vec8<T>::load_nc(p + 8, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) { v[i] = a[i]; v[8 + i] = b[i]; }
}

// Smallest normal scale for which 1/s is finite and the residuals are exact enough; smaller ones take the division.
constexpr float kTinyScale = 0x1p-100f;

__device__ __forceinline__ int nearest_code(float x, float s, float inv) {
  float n;
  if (s < kTinyScale) {  // subnormal territory (1/s may overflow): the quotient in double is exact enough to round once
    n = (float)rint((double)x / (double)s);
  } else {
    const float t = __fmul_rn(x, inv);
    n = rintf(t);
    if (fabsf(__fsub_rn(t, n)) > 0.5f - 0x1p-12f) {
      const float up = __fmaf_rn(-(n + 0.5f), s, x), down = __fmaf_rn(-(n - 0.5f), s, x);
      const bool odd = ((int)n) & 1;
      if (up > 0.f || (up == 0.f && odd)) n += 1.f;
      else if (down < 0.f || (down == 0.f && odd)) n -= 1.f;
    }
  }
  return max(-127, min(127, (int)n));
}

template <typename T, int LANES>
__global__ void __launch_bounds__(256) kv_quant_store_kernel(const T* __restrict__ key, const T* __restrict__ value, int64_t key_stride,
                                                             int64_t value_stride, int8_t* __restrict__ key_cache,
                                                             int8_t* __restrict__ value_cache, int64_t block_stride, int64_t page_stride,
                                                             int64_t head_stride, float* __restrict__ k_scale, float* __restrict__ v_scale,
                                                             const int64_t* __restrict__ slots, int64_t rows, int kv_heads, int head_size,
                                                             int block_size, int64_t capacity, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;  // (token, K or V, head)
  const int lane = threadIdx.x % LANES, d0 = lane * 16;
  const bool live = row < rows && d0 < head_size;
  const int64_t token = row / (2 * kv_heads);
  const int rest = (int)(row - token * (2 * kv_heads));
  const bool is_v = rest >= kv_heads;
  const int head = is_v ? rest - kv_heads : rest;
  const int64_t slot = row < rows ? slots[token] : -1;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  if (live) load16((is_v ? value + token * value_stride : key + token * key_stride) + head * head_size + d0, x);
  float m = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    m = fmaxf(m, fabsf(x[i]));
    bad |= !(fabsf(x[i]) <= FLT_MAX);
  }
  if (bad) m = INFINITY;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (!live || slot < 0) return;
  if (slot >= capacity) {
    if (lane == 0) report(err, MCOP_DEVERR_SLOT);
    return;
  }
  const int64_t block = slot / block_size;
  const int64_t at = block * block_stride + (slot - block * block_size) * page_stride + head * head_stride + d0;
  const bool finite = m <= FLT_MAX;
  const float s = finite ? __fdiv_rn(m, 127.f) : __int_as_float(0x7fc00000);
  uint32_t w[4] = {0, 0, 0, 0};
  if (finite && s > 0.f) {
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i / 4] |= (uint32_t)(nearest_code(x[i], s, inv) & 0xff) << (8 * (i % 4));
  }
  st_u4((is_v ? value_cache : key_cache) + at, make_uint4(w[0], w[1], w[2], w[3]));
  if (lane == 0) (is_v ? v_scale : k_scale)[slot * kv_heads + head] = s;
}

// ---------------------------------------------------------------------------------------------
// Read-back: row t of sequence b (cu[b] <= t < cu[b + 1]) = T(cached row * scale), one rounding.  One warp per token.
// The sequence is found by a 32-way search (one ballot per level: a batch of up to 31 needs one load), then the warp walks
// the token's kv_heads * head_size elements of K and V, 16 per lane.
// Rows behind cu[batch] are left as they were; a row whose page is not in the table or not in the cache likewise, and
// it is reported.
// ---------------------------------------------------------------------------------------------
template <typename T, bool I8>
__global__ void __launch_bounds__(256) kv_gather_kernel(T* __restrict__ key_out, T* __restrict__ value_out, PagedCache c, int scale_mode,
                                                        const int32_t* __restrict__ cu, int batch, int64_t tokens, int head_size, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens || t < cu[0] || t >= cu[batch]) return;
  const int b = find_sequence(cu, batch, t);
  const int64_t pos = t - cu[b];
  if (pos < 0) {  // the bounds are not ascending
    if (lane == 0) report(err, MCOP_DEVERR_SEQUENCE);
    return;
  }
  const int64_t page = pos / c.block_size;
  const int64_t block = page < c.max_blocks ? c.tables[b * c.table_stride + page] : -1;
  if (block < 0 || block >= c.num_blocks) {
    if (lane == 0) report(err, page < c.max_blocks ? MCOP_DEVERR_SLOT : MCOP_DEVERR_KV_INDEX);
    return;
  }
  const int64_t off = pos - page * c.block_size;
  const int64_t base = block * c.block_stride + off * c.page_stride, slot = block * c.block_size + off;
  const int per_head = head_size / 16, chunks = c.kv_heads * per_head;
  const int64_t out0 = t * (int64_t)c.kv_heads * head_size;
  for (int i = lane; i < 2 * chunks; i += 32) {
    const bool is_v = i >= chunks;
    const int j = is_v ? i - chunks : i;
    const int head = j / per_head, d0 = (j - head * per_head) * 16;
    const int64_t at = base + head * c.head_stride + d0;
    T* o = (is_v ? value_out : key_out) + out0 + j * 16;
    if constexpr (I8) {
      const uint4 u = ld_nc_u4(static_cast<const int8_t*>(is_v ? c.v : c.k) + at);
      const float* sp = is_v ? c.v_scale : c.k_scale;
      const float s = scale_mode == kScaleToken ? sp[slot * c.kv_heads + head] : sp[head];
      float v[8], w[8];
      unpack_i8x8(make_uint2(u.x, u.y), v);
      unpack_i8x8(make_uint2(u.z, u.w), w);
#pragma unroll
      for (int k = 0; k < 8; ++k) { v[k] = __fmul_rn(v[k], s); w[k] = __fmul_rn(w[k], s); }
      Vec8<T>::store(o, v);
      Vec8<T>::store(o + 8, w);
    } else {
      const T* p = static_cast<const T*>(is_v ? c.v : c.k) + at;
      const uint4 u = ld_nc_u4(p), w = ld_nc_u4(p + 8);
      st_u4(o, u);
      st_u4(o + 8, w);
    }
  }
}

template <typename T>
int launch_store(const void* key, const void* value, int64_t ks, int64_t vs, int8_t* kc, int8_t* vc, int64_t bs, int64_t ps, int64_t hs,
                 float* k_scale, float* v_scale, const int64_t* slots, int64_t tokens, int kv_heads, int head_size, int block_size,
                 int64_t num_blocks, cudaStream_t st) {
  const int64_t rows = tokens * 2 * kv_heads;
  int lanes = 1;
  while (lanes * 16 < head_size) lanes *= 2;
  const int64_t ctas = (rows * lanes + 255) / 256;
  MCOP_REQUIRE(ctas <= INT32_MAX, MCOP_ERR_UNSUPPORTED, "reshape_and_cache_dynamic_int8: too many rows");
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3((unsigned)ctas), dim3(256), 0, st, static_cast<const T*>(key), static_cast<const T*>(value), ks, vs, kc, vc, bs,
               ps, hs, k_scale, v_scale, slots, rows, kv_heads, head_size, block_size, num_blocks * block_size, pipe_error_ptr());
    return check_launch("reshape_and_cache_dynamic_int8");
  };
  switch (lanes) {
    case 1: return go(kv_quant_store_kernel<T, 1>);
    case 2: return go(kv_quant_store_kernel<T, 2>);
    case 4: return go(kv_quant_store_kernel<T, 4>);
    case 8: return go(kv_quant_store_kernel<T, 8>);
    default: return go(kv_quant_store_kernel<T, 16>);
  }
}

}  // namespace
}  // namespace mcop

using namespace mcop;

extern "C" int mcop_reshape_and_cache_dynamic_i8(const void* key, const void* value, int64_t key_stride, int64_t value_stride,
                                                 int8_t* key_cache, int8_t* value_cache, int64_t block_stride, int64_t page_stride,
                                                 int64_t head_stride, float* k_scale, float* v_scale, const int64_t* slot_mapping,
                                                 int64_t tokens, int kv_heads, int head_size, int block_size, int64_t num_blocks, int dtype,
                                                 mcop_stream_t stream) {
  const char* what = "reshape_and_cache_dynamic_int8";
  MCOP_REQUIRE(tokens >= 0, MCOP_ERR_ARGUMENT, "%s: negative token count", what);
  if (tokens == 0) return MCOP_OK;
  MCOP_REQUIRE(key && value && key_cache && value_cache && k_scale && v_scale && slot_mapping, MCOP_ERR_ARGUMENT, "%s: null pointer", what);
  if (int rc = bad_cache_layout(what, key_cache, value_cache, block_stride, page_stride, head_stride, 1, kv_heads, head_size, block_size, num_blocks))
    return rc;
  MCOP_REQUIRE(dtype == MCOP_F32 || dtype == MCOP_BF16 || dtype == MCOP_F16, MCOP_ERR_UNSUPPORTED, "%s: unknown element type", what);
  const int elem = dtype == MCOP_F32 ? 4 : 2;
  MCOP_REQUIRE(aligned16(key) && aligned16(value) && key_stride * elem % 16 == 0 && value_stride * elem % 16 == 0, MCOP_ERR_ARGUMENT,
               "%s: key / value rows must be 16-byte aligned", what);
  MCOP_REQUIRE(key_stride >= 0 && value_stride >= 0 && block_stride >= 0 && page_stride >= 0 && head_stride >= 0, MCOP_ERR_ARGUMENT,
               "%s: negative stride", what);
  cudaStream_t st = (cudaStream_t)stream;
#define MCOP_STORE(T)                                                                                                                    \
  launch_store<T>(key, value, key_stride, value_stride, key_cache, value_cache, block_stride, page_stride, head_stride, k_scale, v_scale, \
                  slot_mapping, tokens, kv_heads, head_size, block_size, num_blocks, st)
  if (dtype == MCOP_F32) return MCOP_STORE(float);
  return dtype == MCOP_BF16 ? MCOP_STORE(__nv_bfloat16) : MCOP_STORE(__half);
#undef MCOP_STORE
}

extern "C" int mcop_gather_and_dequant_cache(void* key_out, void* value_out, const void* key_cache, const void* value_cache,
                                             int64_t block_stride, int64_t page_stride, int64_t head_stride, const float* k_scale,
                                             const float* v_scale, int scale_mode, const int32_t* block_tables, int64_t table_stride,
                                             int max_blocks, const int32_t* cu_seq_lens, int batch, int64_t tokens, int kv_heads,
                                             int head_size, int block_size, int64_t num_blocks, int dtype, mcop_stream_t stream) {
  const char* what = "gather_and_dequant_cache";
  MCOP_REQUIRE(tokens >= 0 && batch >= 0, MCOP_ERR_ARGUMENT, "%s: negative size", what);
  if (tokens == 0 || batch == 0) return MCOP_OK;
  MCOP_REQUIRE(key_out && value_out && key_cache && value_cache && block_tables && cu_seq_lens, MCOP_ERR_ARGUMENT, "%s: null pointer", what);
  MCOP_REQUIRE(scale_mode >= kScaleNone && scale_mode <= kScaleToken && (scale_mode == kScaleNone || (k_scale && v_scale)), MCOP_ERR_ARGUMENT,
               "%s: scales missing", what);
  const bool i8 = scale_mode != kScaleNone;
  if (int rc = bad_cache_layout(what, key_cache, value_cache, block_stride, page_stride, head_stride, i8 ? 1 : 2, kv_heads, head_size,
                                block_size, num_blocks))
    return rc;
  MCOP_REQUIRE(dtype == MCOP_BF16 || dtype == MCOP_F16 || (dtype == MCOP_F32 && i8), MCOP_ERR_UNSUPPORTED, "%s: unsupported output type", what);
  MCOP_REQUIRE(aligned16(key_out) && aligned16(value_out), MCOP_ERR_ARGUMENT, "%s: outputs must be 16-byte aligned", what);
  MCOP_REQUIRE(max_blocks >= 0 && table_stride >= 0 && block_stride >= 0 && page_stride >= 0 && head_stride >= 0, MCOP_ERR_ARGUMENT,
               "%s: bad stride", what);
  const int64_t ctas = (tokens + 7) / 8;
  MCOP_REQUIRE(ctas <= INT32_MAX, MCOP_ERR_UNSUPPORTED, "%s: too many tokens", what);
  PagedCache c{key_cache, value_cache, k_scale, v_scale, block_stride, page_stride, head_stride, block_tables, table_stride, max_blocks,
               block_size, num_blocks, kv_heads};
  auto go = [&](auto kernel, auto* ko, auto* vo) {
    launch_pdl(kernel, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, ko, vo, c, scale_mode, cu_seq_lens, batch, tokens, head_size,
               pipe_error_ptr());
    return check_launch(what);
  };
  using bf = __nv_bfloat16;
  if (dtype == MCOP_F32) return go(kv_gather_kernel<float, true>, (float*)key_out, (float*)value_out);
  if (dtype == MCOP_BF16) return i8 ? go(kv_gather_kernel<bf, true>, (bf*)key_out, (bf*)value_out) : go(kv_gather_kernel<bf, false>, (bf*)key_out, (bf*)value_out);
  return i8 ? go(kv_gather_kernel<__half, true>, (__half*)key_out, (__half*)value_out) : go(kv_gather_kernel<__half, false>, (__half*)key_out, (__half*)value_out);
}
