// Attention over the paged cache: the entry points, and the chunk kernel for large heads.
#include "paged_attention.cuh"

namespace mcop {
namespace {

// ---------------------------------------------------------------------------------------------
// Chunks at head sizes from 144 to 256, where two tiles of S and of O do not fit tensor memory: one warp per (new token, query
// head), 32 positions at a time.  A lane forms the whole logit of one position (q from shared memory), the warp turns the 32 logits
// into weights with a running maximum and sum, and each lane adds up its own elements of the output.  Every warp reads all rows
// that its token sees, one after another: far from any floor (2 x 512 new tokens after 7680, 32 query and 8 KV heads of 256, bf16: 101 ms).
// ---------------------------------------------------------------------------------------------
template <typename T, bool I8>
__global__ void __launch_bounds__(128) attention_rows_kernel(AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float qs[4][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  if (blockIdx.x == 0)  // reports bounds that no token of its own leads to
    for (int b = threadIdx.x; b < a.batch; b += 128) (void)sequence(a, b);
  if (item >= (int64_t)a.tokens * a.q_heads) return;
  const int token = (int)(item / a.q_heads), head = (int)(item - (int64_t)token * a.q_heads);
  if (token < a.cu[0] || token >= a.cu[a.batch]) return;
  const int b = find_sequence(a.cu, a.batch, token);
  const Seq s = sequence(a, b);
  if (token < s.q0 || token >= s.q0 + s.qn) return;
  int lo, hi;
  span(a, s, token - s.q0, lo, hi);
  const int kv_head = head / (a.q_heads / a.c.kv_heads), D = a.head_size;
  const T* q = static_cast<const T*>(a.q) + token * a.q_token + head * a.q_head;
  for (int d = lane; d < D; d += 32) qs[warp][d] = ElemTraits<T>::to_float(q[d]);
  __syncwarp();
  float acc[8] = {}, m = -INFINITY, l = 0.f;
  for (int base = lo; base < hi; base += 32) {
    const int pos = base + lane;
    const int slot = pos < hi ? slot_of(a, b, pos) : -1;
    float x = -INFINITY, vs = 1.f;
    if (slot >= 0) {
      const int64_t at = row_of(a.c, slot, kv_head);
      float dot = 0.f;
      for (int d = 0; d < D; d += 8) {
        float k[8];
        if constexpr (I8) unpack_i8x8(*reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.c.k) + at + d), k);
        else Vec8<T>::load_nc(static_cast<const T*>(a.c.k) + at + d, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = __fmaf_rn(qs[warp][d + i], k[i], dot);
      }
      float c = a.scale;
      if constexpr (I8) {
        const int64_t si = a.scale_mode == kScaleToken ? (int64_t)slot * a.c.kv_heads + kv_head : kv_head;
        c *= a.c.k_scale[si];
        vs = a.c.v_scale[si];
      }
      x = dot * c;
    }
    const float top = fmaxf(m, warp_max(x));
    const bool nan = __any_sync(0xffffffffu, x != x);
    const float safe = top == -INFINITY ? 0.f : top;
    const float keep = m == -INFINITY ? 0.f : expf(m - safe);
    const float p = nan ? (slot >= 0 ? NAN : 0.f) : x == -INFINITY ? 0.f : expf(x - safe);
    l = l * keep + warp_sum(p);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= keep;
    for (int j = 0; j < 32; ++j) {
      const int sj = __shfl_sync(0xffffffffu, slot, j);
      const float w = __shfl_sync(0xffffffffu, p * vs, j);
      if (sj < 0) continue;
      const int64_t at = row_of(a.c, sj, kv_head);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d >= D) break;
        float v;
        if constexpr (I8) v = (float)static_cast<const int8_t*>(a.c.v)[at + d];
        else v = ElemTraits<T>::to_float(static_cast<const T*>(a.c.v)[at + d]);
        acc[i] = __fmaf_rn(w, v, acc[i]);
      }
    }
  }
  T* o = static_cast<T*>(a.out) + token * a.o_token + head * a.o_head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < D) o[lane + 32 * i] = ElemTraits<T>::from_float(acc[i] * inv);
  if (a.lse && lane == 0) a.lse[(int64_t)token * a.q_heads + head] = l == 0.f ? -INFINITY : m + logf(l);
}

int check_args(const char* what, const AttnArgs& a, int64_t tokens, int dtype) {
  MCOP_REQUIRE(a.q && a.out && a.c.k && a.c.v && (a.c.tables || a.c.max_blocks == 0) && a.seq_lens, MCOP_ERR_ARGUMENT, "%s: null pointer", what);
  MCOP_REQUIRE(tokens <= INT32_MAX, MCOP_ERR_UNSUPPORTED, "%s: too many tokens", what);
  MCOP_REQUIRE(dtype == MCOP_BF16 || dtype == MCOP_F16, MCOP_ERR_UNSUPPORTED, "%s: query must be bf16 or f16", what);
  MCOP_REQUIRE(a.scale_mode >= kScaleNone && a.scale_mode <= kScaleToken && (a.scale_mode == kScaleNone || (a.c.k_scale && a.c.v_scale)),
               MCOP_ERR_ARGUMENT, "%s: scales missing", what);
  if (int rc = bad_cache_layout(what, a.c.k, a.c.v, a.c.block_stride, a.c.page_stride, a.c.head_stride, a.scale_mode ? 1 : 2, a.c.kv_heads,
                                a.head_size, a.c.block_size, a.c.num_blocks))
    return rc;
  MCOP_REQUIRE(a.q_heads > 0 && a.q_heads % a.c.kv_heads == 0, MCOP_ERR_ARGUMENT, "%s: q_heads must be a multiple of kv_heads", what);
  MCOP_REQUIRE(aligned16(a.q) && aligned16(a.out) && a.q_token % 8 == 0 && a.q_head % 8 == 0 && a.o_token % 8 == 0 && a.o_head % 8 == 0,
               MCOP_ERR_ARGUMENT, "%s: query and output rows must be 16-byte aligned", what);
  // positions and (token, query head) rows are ints, also rounded up to a tile of up to 256
  constexpr int64_t kMost = INT32_MAX - 255;
  MCOP_REQUIRE(a.c.max_blocks >= 0 && a.c.table_stride >= 0 && (int64_t)a.c.max_blocks * a.c.block_size <= kMost, MCOP_ERR_ARGUMENT,
               "%s: block table too wide", what);
  MCOP_REQUIRE(tokens * a.q_heads <= kMost, MCOP_ERR_UNSUPPORTED, "%s: more than 2^31 - 256 query rows", what);
  // rows are addressed in units of 16 bytes with 32 bits
  const double span = (double)a.c.num_blocks * a.c.block_stride + (double)a.c.block_size * a.c.page_stride + (double)a.c.kv_heads * a.c.head_stride;
  MCOP_REQUIRE(a.c.block_stride >= 0 && a.c.page_stride >= 0 && a.c.head_stride >= 0 && span * (a.scale_mode ? 1 : 2) < 0x1p36, MCOP_ERR_UNSUPPORTED,
               "%s: a cache may span at most 64 GB, with strides >= 0", what);
  MCOP_REQUIRE(a.window >= 0, MCOP_ERR_ARGUMENT, "%s: negative window", what);
  MCOP_REQUIRE(a.scale > 0.f && a.scale <= FLT_MAX, MCOP_ERR_ARGUMENT, "%s: the scale must be positive", what);
  return MCOP_OK;
}

int launch_rows(const char* what, const AttnArgs& a, int dtype, cudaStream_t st) {
  const int64_t ctas = ((int64_t)a.tokens * a.q_heads + 3) / 4;
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3((unsigned)ctas), dim3(128), 0, st, a);
    return check_launch(what);
  };
  const bool i8 = a.scale_mode != kScaleNone;
  if (dtype == MCOP_BF16) return i8 ? go(attention_rows_kernel<__nv_bfloat16, true>) : go(attention_rows_kernel<__nv_bfloat16, false>);
  return i8 ? go(attention_rows_kernel<__half, true>) : go(attention_rows_kernel<__half, false>);
}

}  // namespace
}  // namespace mcop

using namespace mcop;

extern "C" size_t mcop_paged_attention_decode_workspace_bytes(int batch, int q_heads, int kv_heads, int head_size) {
  return batch > 0 && kv_heads > 0 && q_heads >= kv_heads && head_size > 0 ? decode_workspace(q_heads, kv_heads, head_size) : 0;
}
extern "C" size_t mcop_paged_attention_chunk_workspace_bytes(int64_t tokens, int batch, int q_heads, int kv_heads, int head_size) {
  const bool any = tokens > 0 && batch > 0 && kv_heads > 0 && q_heads >= kv_heads && head_size > 0 && head_size <= kChunkHead;
  return any ? chunk_workspace(tokens, batch, q_heads, kv_heads, head_size) : 0;
}

extern "C" int mcop_paged_attention_decode(void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, const void* query,
                                           int64_t query_token_stride, int64_t query_head_stride, const void* key_cache,
                                           const void* value_cache, int64_t block_stride, int64_t page_stride, int64_t head_stride,
                                           const float* k_scale, const float* v_scale, int scale_mode, const int32_t* block_tables,
                                           int64_t table_stride, int max_blocks, const int32_t* seq_lens, int batch, int q_heads,
                                           int kv_heads, int head_size, int block_size, int64_t num_blocks, float scale, int window,
                                           int dtype, void* workspace, size_t workspace_bytes, mcop_stream_t stream) {
  const char* what = "paged_attention_decode";
  MCOP_REQUIRE(batch >= 0, MCOP_ERR_ARGUMENT, "%s: negative batch", what);
  if (batch == 0) return MCOP_OK;
  AttnArgs a{{key_cache, value_cache, k_scale, v_scale, block_stride, page_stride, head_stride, block_tables, table_stride, max_blocks,
              block_size, num_blocks, kv_heads},
             query, out, lse, query_token_stride, query_head_stride, out_token_stride, out_head_stride, seq_lens, nullptr, batch, batch, q_heads,
             head_size, scale_mode, scale, 1, window, pipe_error_ptr()};
  if (int rc = check_args(what, a, batch, dtype)) return rc;
  a.c.prepare();
  return launch_decode(a, dtype, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int mcop_paged_attention_chunk(void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, const void* query,
                                          int64_t query_token_stride, int64_t query_head_stride, const void* key_cache,
                                          const void* value_cache, int64_t block_stride, int64_t page_stride, int64_t head_stride,
                                          const float* k_scale, const float* v_scale, int scale_mode, const int32_t* block_tables,
                                          int64_t table_stride, int max_blocks, const int32_t* seq_lens, const int32_t* cu_seqlens_q,
                                          int batch, int64_t tokens, int q_heads, int kv_heads, int head_size, int block_size,
                                          int64_t num_blocks, float scale, int causal, int window, int dtype, void* workspace,
                                          size_t workspace_bytes, mcop_stream_t stream) {
  const char* what = "paged_attention_chunk";
  MCOP_REQUIRE(batch >= 0 && tokens >= 0, MCOP_ERR_ARGUMENT, "%s: negative size", what);
  if (batch == 0 || tokens == 0) return MCOP_OK;
  MCOP_REQUIRE(cu_seqlens_q, MCOP_ERR_ARGUMENT, "%s: null pointer", what);
  AttnArgs a{{key_cache, value_cache, k_scale, v_scale, block_stride, page_stride, head_stride, block_tables, table_stride, max_blocks,
              block_size, num_blocks, kv_heads},
             query, out, lse, query_token_stride, query_head_stride, out_token_stride, out_head_stride, seq_lens, cu_seqlens_q, batch, (int)tokens,
             q_heads, head_size, scale_mode, scale, causal, window, pipe_error_ptr()};
  if (int rc = check_args(what, a, tokens, dtype)) return rc;
  a.c.prepare();
  if (a.head_size <= kChunkHead) return launch_chunk(a, dtype, workspace, workspace_bytes, (cudaStream_t)stream);
  return launch_rows(what, a, dtype, (cudaStream_t)stream);
}
