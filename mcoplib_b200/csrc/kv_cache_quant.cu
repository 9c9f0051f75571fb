// Dynamic int8 quantisation of K and V into the paged cache, and the way back out of it.
#include "paged_cache.cuh"
#include "tma_pipe.cuh"

namespace mcop {
namespace {

// ---------------------------------------------------------------------------------------------
// Store: per (token, head) row  s = max|x| / 127 (one IEEE fp32 division),  code = nearest integer of the REAL quotient
// x / s, ties to even.  The quotient is never formed: n = rint(x * rn(1/s)) is off by one at most (|x * rn(1/s)| <= 127.5
// and carries two roundings, 2^-16 in absolute terms), and the sign of the residual fma(-(n +- 1/2), s, x), which one rounding
// cannot change, says on which side of the midpoint x lies.  Only threads with an element within 2^-15 of a midpoint look.
// A row of zeros has s = 0 and codes 0; a row that holds a NaN or an infinity has s = NaN and codes 0, so that it reads
// back as NaN instead of as plausible values.
//
// Bound: HBM bytes (2 * head_size read, head_size + 4 written per row).  A row sits on LANES lanes, each with 8 elements of its
// first and 8 of its second half, so that every load and store of a warp covers whole sectors (16 neighbouring elements per
// lane fetched each sector twice).
// ---------------------------------------------------------------------------------------------
// Smallest scale for which 1/s is finite and the residuals are exact enough; smaller ones take the division.
constexpr float kTinyScale = 0x1p-100f;

template <typename T, int LANES>
__global__ void __launch_bounds__(256) kv_quant_store_kernel(const T* __restrict__ key, const T* __restrict__ value, int64_t key_stride,
                                                             int64_t value_stride, int8_t* __restrict__ key_cache,
                                                             int8_t* __restrict__ value_cache, int64_t block_stride, int64_t page_stride,
                                                             int64_t head_stride, float* __restrict__ k_scale, float* __restrict__ v_scale,
                                                             const int64_t* __restrict__ slots, uint32_t rows, uint32_t kv_heads, int head_size,
                                                             uint32_t block_size, int64_t capacity, Divisor by_rows, Divisor by_block, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;  // (token, K or V, head)
  const int lane = threadIdx.x % LANES, d0 = lane * 8, d1 = d0 + LANES * 8;
  const bool live = row < rows;
  const uint32_t token = live ? by_rows.of(row) : 0, rest = row - token * (2 * kv_heads);
  const bool is_v = rest >= kv_heads;
  const uint32_t head = is_v ? rest - kv_heads : rest;
  const int64_t slot = live ? slots[token] : -1;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  if (live) {
    const T* p = (is_v ? value + token * value_stride : key + token * key_stride) + head * head_size;
    float a[8], b[8];
    if (d0 < head_size) {
      Vec8<T>::load_nc(p + d0, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = a[i];
    }
    if (d1 < head_size) {
      Vec8<T>::load_nc(p + d1, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 + i] = b[i];
    }
  }
  float m = 0.f;  // a NaN stays one
#pragma unroll
  for (int i = 0; i < 16; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x[i]), "f"(x[i + 1]));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, m, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(other));
  }
  if (!live || slot < 0) return;
  if (slot >= capacity) {
    if (lane == 0) report(err, MCOP_DEVERR_SLOT);
    return;
  }
  const uint32_t block = by_block.of((uint32_t)slot);
  int8_t* out = (is_v ? value_cache : key_cache) + block * block_stride + ((uint32_t)slot - block * block_size) * page_stride + head * head_stride;
  const bool finite = m <= FLT_MAX;
  const float s = finite ? __fdiv_rn(m, 127.f) : __int_as_float(0x7fc00000);
  uint32_t q[16];
  const float inv = finite && s > 0.f ? __frcp_rn(s) : 0.f;
  const float2 inv2 = make_float2(inv, inv);
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    // 1.5 * 2^23: the low byte of the sum is x * inv rounded to an integer, ties to even
    const float2 v = make_float2(x[i], x[i + 1]), u = __ffma2_rn(v, inv2, make_float2(12582912.f, 12582912.f));
    const float2 minus_n = __ffma2_rn(u, make_float2(-1.f, -1.f), make_float2(12582912.f, 12582912.f)), d = __ffma2_rn(v, inv2, minus_n);
    q[i] = __float_as_uint(u.x);
    q[i + 1] = __float_as_uint(u.y);
    far = max3_abs(far, d.x, d.y);
  }
  if (finite && s > 0.f) {
    if (s < kTinyScale) {  // subnormal territory (1/s may overflow): the quotient in double is exact enough to round once
#pragma unroll
      for (int i = 0; i < 16; ++i) q[i] = (uint32_t)max(-127, min(127, (int)rint((double)x[i] / (double)s)));
    } else if (far > 0.5f - 0x1p-15f) {  // (half of the largest value is the midpoint 63.5: common, so this is branch-free)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float n = __fsub_rn(__uint_as_float(q[i]), 12582912.f), d = __fmaf_rn(x[i], inv, -n);
        const float beyond = copysignf(1.f, d), r = __fmaf_rn(-__fmaf_rn(0.5f, beyond, n), s, x[i]) * beyond;
        if (r > 0.f || (r == 0.f && (q[i] & 1))) q[i] += d < 0.f ? ~0u : 1u;
      }
    }
  }
  if (!finite) {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = 0;
  }
  if (d0 < head_size) *reinterpret_cast<uint2*>(out + d0) = make_uint2(pack4_low_bytes(q[0], q[1], q[2], q[3]), pack4_low_bytes(q[4], q[5], q[6], q[7]));
  if (d1 < head_size) *reinterpret_cast<uint2*>(out + d1) = make_uint2(pack4_low_bytes(q[8], q[9], q[10], q[11]), pack4_low_bytes(q[12], q[13], q[14], q[15]));
  if (lane == 0) (is_v ? v_scale : k_scale)[slot * kv_heads + head] = s;
}

// ---------------------------------------------------------------------------------------------
// Read-back: row t of sequence b (cu[b] <= t < cu[b + 1]) = T(fp32(cached row * scale)): the product has up to 31 bits, is rounded to fp32
// and then to T, as the same expression on fp32 tensors is.  One warp per token.
// The sequence is found by a 32-way search (one ballot per level: a batch of up to 31 needs one load), then the warp walks
// the token's kv_heads * head_size elements of K and V, 16 per lane.
// Rows behind cu[batch] are left as they were; a row whose page is not in the table or not in the cache likewise, and
// it is reported.  So are the rows of a sequence that leaves the buffer.  One CTA behind the others looks all bounds over and reports
// those that descend or leave the buffer (a sequence without rows leads no warp to its bounds).
// ---------------------------------------------------------------------------------------------
template <typename T, bool I8>
__global__ void __launch_bounds__(256) kv_gather_kernel(T* __restrict__ key_out, T* __restrict__ value_out, PagedCache c, int scale_mode,
                                                        const int32_t* __restrict__ cu, int batch, int64_t tokens, int head_size, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == gridDim.x - 1) {
    for (int b = threadIdx.x; b < batch; b += 256)
      if (cu[b] < 0 || cu[b + 1] < cu[b] || cu[b + 1] > tokens) report(err, MCOP_DEVERR_SEQUENCE);
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens || t < cu[0] || t >= cu[batch]) return;
  const int b = find_sequence(cu, batch, t);  // cu[b] <= t < cu[b + 1], whatever the others are
  const int64_t pos = t - cu[b];
  if (pos > t || cu[b + 1] > tokens) return;  // the sequence leaves the buffer
  const int64_t page = pos / c.block_size;
  const int64_t block = page < c.max_blocks ? c.tables[b * c.table_stride + page] : -1;
  if (block < 0 || block >= c.num_blocks) {
    if (lane == 0) report(err, page < c.max_blocks ? MCOP_DEVERR_SLOT : MCOP_DEVERR_KV_INDEX);
    return;
  }
  const int64_t off = pos - page * c.block_size;
  const int64_t base = block * c.block_stride + off * c.page_stride, slot = block * c.block_size + off;
  // pieces of 8 elements, 4 to 8 of them in flight per lane: every load and store of the warp covers whole sectors
  const int per_head = head_size / 8, pieces = c.kv_heads * per_head;
  const int64_t out0 = t * (int64_t)pieces * 8;
  constexpr int N = 4;
  for (int i0 = lane; i0 < pieces; i0 += 32 * N) {
    uint2 k8[N], v8[N];
    uint4 k16[N], v16[N];
    float ks[N], vs[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + 32 * n;
      if (i < pieces) {
        const int head = i / per_head;
        const int64_t at = base + head * c.head_stride + (i - head * per_head) * 8;
        if constexpr (I8) {
          k8[n] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(c.k) + at);
          v8[n] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(c.v) + at);
          const int64_t si = scale_mode == kScaleToken ? slot * c.kv_heads + head : head;
          ks[n] = c.k_scale[si];
          vs[n] = c.v_scale[si];
        } else {
          k16[n] = ld_nc_u4(static_cast<const T*>(c.k) + at);
          v16[n] = ld_nc_u4(static_cast<const T*>(c.v) + at);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + 32 * n;
      if (i < pieces) {
        if constexpr (I8) {
          float v[8];
          unpack_i8x8(k8[n], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], ks[n]);
          Vec8<T>::store(key_out + out0 + i * 8, v);
          unpack_i8x8(v8[n], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], vs[n]);
          Vec8<T>::store(value_out + out0 + i * 8, v);
        } else {
          st_u4(key_out + out0 + i * 8, k16[n]);
          st_u4(value_out + out0 + i * 8, v16[n]);
        }
      }
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
  MCOP_REQUIRE(rows < INT32_MAX / 2, MCOP_ERR_UNSUPPORTED, "reshape_and_cache_dynamic_int8: too many rows");
  const int64_t ctas = (rows * lanes + 255) / 256;
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3((unsigned)ctas), dim3(256), 0, st, static_cast<const T*>(key), static_cast<const T*>(value), ks, vs, kc, vc, bs,
               ps, hs, k_scale, v_scale, slots, (uint32_t)rows, (uint32_t)kv_heads, head_size, (uint32_t)block_size, num_blocks * block_size,
               Divisor(2u * (uint32_t)kv_heads), Divisor((uint32_t)block_size), pipe_error_ptr());
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
  MCOP_REQUIRE(key_out && value_out && key_cache && value_cache && (block_tables || max_blocks == 0) && cu_seq_lens, MCOP_ERR_ARGUMENT, "%s: null pointer", what);
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
  const int64_t ctas = (tokens + 7) / 8 + 1;
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
