// Attention of new tokens over the paged KV cache.
//
// New token i of a sequence with q_len new tokens and len cached ones (the new ones are cached already) stands at
// position  pos = len - q_len + i  and sees the positions
//     [max(0, window ? pos - window + 1 : 0), causal ? pos + 1 : len)  clipped to [0, len).
// Over those, with s_j = scale * (q . k_j):   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   lse = m + ln sum_j exp(s_j - m).
// A token that sees nothing gets out = 0 and lse = -inf.  The scales of an int8 cache never touch the codes: the K scale multiplies
// the logit, the V scale the weight, both in fp32.
#pragma once

#include "paged_cache.cuh"
#include "tma_pipe.cuh"

namespace mcop {

struct AttnArgs {
  PagedCache c;
  const void* q;
  void* out;
  float* lse;  // [tokens, q_heads] or null
  int64_t q_token, q_head, o_token, o_head;
  const int32_t* seq_lens;
  const int32_t* cu;  // null: one new token per sequence
  int batch, tokens, q_heads, head_size, scale_mode;
  float scale;
  int causal, window;
  int* err;
};

struct Seq {
  int q0, qn, len;  // first new token, number of new tokens, cached tokens
};

// Bounds of sequence b, checked: what the caller's tensors say is never turned into an address beyond the buffers.
// REPORT: whether this call records what it finds wrong (once per launch is enough).
template <bool REPORT = true> __device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  s.q0 = a.cu ? a.cu[b] : b;
  const int q1 = a.cu ? a.cu[b + 1] : b + 1;
  s.qn = q1 - s.q0;
  if (s.q0 < 0 || q1 < s.q0 || q1 > a.tokens) {
    if (REPORT) report(a.err, MCOP_DEVERR_SEQUENCE);
    s.q0 = s.qn = 0;
  }
  s.len = a.seq_lens[b];
  const int64_t room = (int64_t)a.c.max_blocks * a.c.block_size;
  if (s.len < 0 || s.len > room) {
    if (REPORT) report(a.err, MCOP_DEVERR_KV_INDEX);
    s.len = s.len < 0 ? 0 : (int)room;
  }
  return s;
}

// Positions [lo, hi) that new token i of a sequence sees.
__device__ __forceinline__ void span(const AttnArgs& a, const Seq& s, int i, int& lo, int& hi) {
  const int pos = s.len - s.qn + i;
  hi = a.causal ? min(s.len, max(0, pos + 1)) : s.len;
  lo = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
}

// Slot of position `pos` of sequence b, or -1 (reported) where the table names a page that the cache does not have.
__device__ __forceinline__ int slot_of(const AttnArgs& a, int b, int pos) {
  const int page = pos / a.c.block_size;
  const int block = a.c.tables[b * a.c.table_stride + page];
  if (block < 0 || block >= a.c.num_blocks) {
    report(a.err, MCOP_DEVERR_SLOT);
    return -1;
  }
  return block * a.c.block_size + (pos - page * a.c.block_size);
}
__device__ __forceinline__ int64_t row_of(const PagedCache& c, int slot, int head) {
  const int block = slot / c.block_size;
  return block * c.block_stride + (slot - block * c.block_size) * c.page_stride + head * c.head_stride;
}

// Weights are formed as powers of two of logits in units of log2: x = scale * log2(e) * (q . k).
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A running maximum is moved only when a logit passes it by more than this (in log2 units): weights then stay below 2^8, and
// the accumulators are rescaled a few times per row instead of once per tile.
constexpr float kMaxSlack = 8.f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes to shared memory, or 16 zeros (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// Two floats rounded to T, lo in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (ElemTraits<T>::code == MCOP_BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Decode (paged_decode.cu): one new token per sequence, head sizes up to 256.
size_t decode_workspace(int q_heads, int kv_heads, int head_size);
int launch_decode(const AttnArgs& a, int dtype, void* ws, size_t ws_bytes, cudaStream_t st);

// Chunk (paged_chunk.cu): head sizes up to 128.
constexpr int kChunkHead = 128;
size_t chunk_workspace(int64_t tokens, int batch, int q_heads, int kv_heads, int head_size);
int launch_chunk(const AttnArgs& a, int dtype, void* ws, size_t ws_bytes, cudaStream_t st);

}  // namespace mcop
