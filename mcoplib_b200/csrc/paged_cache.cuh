// The paged KV cache as the kernels that quantise into it, read it back and attend over it see it.
//
// Layout [num_blocks, block_size, kv_heads, head_size] with free strides for block, in-block position and head (in
// elements, shared by the K and the V cache) and contiguous heads.  Rows are int8 or a 2-byte type; int8 rows have a
// dequantisation scale per head (kScaleHead) or per (slot, head) (kScaleToken: fp32 [num_blocks, block_size, kv_heads]).
#pragma once

#include "common.cuh"

namespace mcop {

enum ScaleMode { kScaleNone = 0, kScaleHead = 1, kScaleToken = 2 };

// Division of p < 2^31 by a fixed d as a multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31 + s) / d) < 2^32,
// floor(p * m / 2^(31 + s)) = floor(p / d), since m exceeds 2^(31 + s) / d by less than 2^s / d.
struct Divisor {
  uint32_t mul = 0, shift = 0;
  Divisor() = default;
  __host__ explicit Divisor(uint32_t d) {
    while ((uint64_t(1) << shift) < d) ++shift;
    mul = (uint32_t)(((uint64_t(1) << (31 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t of(uint32_t p) const { return __umulhi(2u * p, mul) >> shift; }
};

struct PagedCache {
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
  int64_t block_stride, page_stride, head_stride;
  const int32_t* tables;  // [batch, table_stride], the first max_blocks entries of a row are used
  int64_t table_stride;
  int max_blocks;
  int block_size;
  int64_t num_blocks;
  int kv_heads;
  Divisor by_block;  // the division by block_size

  __host__ void prepare() { by_block = Divisor((uint32_t)block_size); }
  __device__ __forceinline__ int page_of(int p) const { return (int)by_block.of((uint32_t)p); }
};

__device__ __forceinline__ void report(int* err, int code) {
  if (err) atomicCAS(err, 0, code);
}

// Largest b in [0, batch) with cu[b] <= t, given cu[0] <= t < cu[batch] (all lanes take part, same t).
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, i < hi && (int64_t)cu[i] <= t);  // lane 0: always
    const int last = 31 - __clz(le | 1u);
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Eight int8 codes (two words) as floats.
__device__ __forceinline__ void unpack_i8x8(uint2 u, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)(int8_t)(u.x >> (8 * i));
    v[4 + i] = (float)(int8_t)(u.y >> (8 * i));
  }
}

// Host side: refuses a cache that the kernels cannot address (MCOP_OK otherwise).
inline int bad_cache_layout(const char* what, const void* k, const void* v, int64_t block_stride, int64_t page_stride, int64_t head_stride,
                     int elem, int kv_heads, int head_size, int block_size, int64_t num_blocks) {
  MCOP_REQUIRE(kv_heads > 0 && block_size > 0 && num_blocks > 0, MCOP_ERR_ARGUMENT, "%s: empty cache", what);
  MCOP_REQUIRE(head_size > 0 && head_size % 16 == 0 && head_size <= 256, MCOP_ERR_UNSUPPORTED,
               "%s: head_size must be a multiple of 16 of at most 256", what);
  MCOP_REQUIRE(num_blocks <= INT32_MAX && num_blocks * block_size <= INT32_MAX, MCOP_ERR_UNSUPPORTED, "%s: more than 2^31 slots", what);
  MCOP_REQUIRE(aligned16(k) && aligned16(v) && block_stride * elem % 16 == 0 && page_stride * elem % 16 == 0 && head_stride * elem % 16 == 0,
               MCOP_ERR_ARGUMENT, "%s: cache rows must be 16-byte aligned", what);
  return MCOP_OK;
}

}  // namespace mcop
