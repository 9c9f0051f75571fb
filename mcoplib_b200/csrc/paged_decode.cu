// Decode attention: one new token per sequence over its cached tokens.
//
// Bound: HBM bytes of the cached rows (all query heads of a KV head share its rows).  16 * head_size flops per row byte
// (int8, 8 query heads per KV head) is more than the fp32 pipes give at the memory's rate, so both products run on the
// tensor cores with TOKENS as the M dimension: m16n8k16 takes 16 cached tokens against 8 query heads, which wastes nothing at
// 8 heads per KV head.  (tcgen05.mma could take 128 tokens against 8 heads as well; it would want K and V, converted, in swizzled
// shared memory, where mma.sync takes them from registers as they arrive.  Not built.)
//   S^T[16 tokens x 8 heads] = K[16 x D] Q^T[D x 8]         O^T[D x 8] += V^T[D x 16] P^T[16 x 8]
// The order of the contracted index is free as long as both operands agree, and so is the order of O's rows: a lane's
// fragments are 16-byte pieces of cached rows as they lie, int8 codes become f16 in registers (exactly), and the only
// exchange of computed values is one 8x8 transpose of P per 8 tokens (movmatrix).
//
// Work split: the units (32 or 16 tokens of one sequence and head tile for each of 4 warps) of ALL sequences form one line, cut
// into equal ranges, one per CTA, whatever the lengths.  The lengths are read on the device: a captured graph serves any.  A
// warp's copies run on across sequence borders.  An item that crosses a CTA border leaves one partial result per CTA in the
// workspace (two slots per CTA are enough: the item it starts in and the item it ends in), joined by a second launch in a
// fixed order: the same bits every time, no atomics.
#include "paged_attention.cuh"

namespace mcop {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kMaxCtasPerSm = 3;

struct Rec {
  int b, tile, count, pad;
};

__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// T: type of query and output; MODE: the cache's scales; DP: head size the fragments are laid out for; NT: n8 tiles of query
// heads (8 * NT heads of one KV head per work item).
template <typename T, int MODE, int DP, int NT> struct Cfg {
  static constexpr bool I8 = MODE != kScaleNone;
  static constexpr int ELEM = I8 ? 1 : 2;
  static constexpr int RB = DP * ELEM;                   // bytes of a (padded) cached row
  static constexpr int TOK = !I8 && RB >= 256 ? 16 : 32;  // tokens of a warp's step: 8 KB of K and V keep the set-up of a step small beside it
  static constexpr uint32_t ALL = TOK == 32 ? 0xffffffffu : 0xffffu;
  static constexpr int HALVES = TOK / 16;
  static constexpr int UNIT = TOK * kWarps;
  static constexpr int KCH = RB / 64;                    // 16-byte pieces of a K row per lane
  static constexpr int VCH = RB >= 128 ? RB / 128 : 1;   // pieces of a V row per lane (8 bytes when RB == 64)
  static constexpr int VPIECE = RB >= 128 ? 16 : 8;
  static constexpr int MT = DP / 16;                     // m16 tiles of O^T
  static constexpr int HEADS = 8 * NT;
  static constexpr int ROW16 = RB / 16;                  // pieces of a row
  static constexpr int V_HALF = 4 * VCH * VPIECE * 32;   // bytes per 16 tokens
  static constexpr int K_BYTES = TOK * RB, V_BYTES = HALVES * V_HALF;
  static constexpr int S_BYTES = MODE == kScaleToken ? TOK * 8 : 0;
  static constexpr int ST = 3;                           // steps of K and of V a warp holds
  static constexpr int WARP = ST * (K_BYTES + V_BYTES + S_BYTES), SMEM = kWarps * WARP;
  // Two CTAs of 4 warps and up to 255 registers: a warp's step is a chain of conversions and products, and the registers that let
  // it overlap with itself are worth more than a third CTA (537 MB of int8 rows: 125 us against 148 with three CTAs at 168).
  static constexpr int CTAS = SMEM <= 56 * 1024 ? 3 : SMEM <= 112 * 1024 ? 2 : 1;
  static constexpr int SLOT = HEADS * (DP + 2);          // floats of a partial result: O, then maximum and sum of every head
  static_assert(MT * 512 <= V_BYTES, "the warps' O are joined where the last V was");
};

// int8 codes (the bytes 0 and 2 of x) as a pair of f16, exactly: 1024 + (code + 128) has ulp 1.  One logic operation with both
// masks in registers (as immediates they would be two), one subtraction.
struct Codes {
  uint32_t mask = 0x00ff00ffu, bias = 0x64806480u;  // bias: 1024 + 128 twice
  __device__ __forceinline__ Codes() { asm("" : "+r"(mask), "+r"(bias)); }
  __device__ __forceinline__ uint32_t f16(uint32_t x) const {
    uint32_t u;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(u) : "r"(x), "r"(mask), "r"(bias));  // (x & mask) ^ bias
    __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<uint32_t*>(&r);
  }
};

// Where a warp is in the line of units.
struct Cursor {
  int u, b, tile, k, n, first, lo, hi;
  template <int UNIT> __device__ __forceinline__ void load(const AttnArgs& a) {
    const Seq s = sequence(a, b);
    span(a, s, 0, lo, hi);
    first = lo / UNIT;
    n = max(1, (hi + UNIT - 1) / UNIT - first);
  }
  template <int UNIT> __device__ __forceinline__ void next(const AttnArgs& a, int tiles) {
    ++u;
    if (++k < n) return;
    k = 0;
    if (++tile < tiles) return;
    tile = 0;
    if (++b < a.batch) load<UNIT>(a);
  }
};

// FULL: the head size is DP itself.
template <typename T, int MODE, int DP, int NT, bool FULL>
__global__ void __launch_bounds__(kThreads, Cfg<T, MODE, DP, NT>::CTAS) decode_kernel(AttnArgs a, float* __restrict__ parts, Rec* __restrict__ recs) {
  using C = Cfg<T, MODE, DP, NT>;
  // Types of the two products.  int8 codes are exact in f16: there the queries are scaled by a power of two per head to fit it, and
  // a weight is rounded to 11 bits instead of bf16's 8.  With one scale per token the running maximum follows the weight
  // TIMES the scale, so that the largest product is near 1 whatever the scales.
  using QT = typename std::conditional<C::I8, __half, T>::type;
  using W = QT;
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int64_t scan[kWarps];
  __shared__ int start[3];
  __shared__ uint32_t valid[kWarps][C::ST];
  __shared__ float ml[kWarps][2][C::HEADS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.q_heads / a.c.kv_heads, head_tiles = (G + C::HEADS - 1) / C::HEADS, tiles = a.c.kv_heads * head_tiles;

  // --- this CTA's range of the line of units
  int64_t mine = 0;
  const int share = (a.batch + kThreads - 1) / kThreads, b0 = min(a.batch, tid * share), b1 = min(a.batch, b0 + share);
  Cursor q;
  for (q.b = b0; q.b < b1; ++q.b) {
    q.load<C::UNIT>(a);
    mine += (int64_t)q.n * tiles;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += scan[w];
    total += scan[w];
  }
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t u0 = per * blockIdx.x, u1 = min(total, u0 + per);
  if (u0 >= u1) {  // nothing left for this CTA
    if (tid == 0) recs[blockIdx.x].count = 0;
    return;
  }
  if (incl - mine <= u0 && u0 < incl) {
    int64_t at = incl - mine;
    for (q.b = b0;; ++q.b) {
      q.load<C::UNIT>(a);
      if (u0 < at + (int64_t)q.n * tiles) break;
      at += (int64_t)q.n * tiles;
    }
    start[0] = q.b;
    start[1] = (int)((u0 - at) / q.n);
    start[2] = (int)((u0 - at) % q.n);
  }
  __syncthreads();
  const int units = (int)(u1 - u0);
  Cursor in;  // the unit whose copies are issued next
  in.u = 0; in.b = start[0]; in.tile = start[1]; in.k = start[2];
  in.load<C::UNIT>(a);
  Cursor cur = in;  // the unit that is consumed

  const Codes codes;
  // a warp's memory: ST steps of K, of V, of scales
  unsigned char* const kring = smem + warp * C::WARP;
  unsigned char* const vring = kring + C::ST * C::K_BYTES;
  float* const sring = reinterpret_cast<float*>(vring + C::ST * C::V_BYTES);
  const int row_bytes = a.head_size * C::ELEM;
  const char* kbase = static_cast<const char*>(a.c.k);
  const char* vbase = static_cast<const char*>(a.c.v);
  const uint32_t block16 = (uint32_t)(a.c.block_stride * C::ELEM / 16), page16 = (uint32_t)(a.c.page_stride * C::ELEM / 16),
                 head16 = (uint32_t)(a.c.head_stride * C::ELEM / 16);
  // Where a lane's pieces of a V row begin.  With FULL these are constants; otherwise pieces behind a row's end read its last
  // one again: those rows of O are never written.  (K is filled up with zeros there: an infinity times the query's zero would be NaN.)
  auto v_piece = [&](int c) { return FULL ? 8 * C::VPIECE * c + C::VPIECE * g : min(8 * C::VPIECE * c + C::VPIECE * g, row_bytes - C::VPIECE); };

  // Page and offset of token `lane` of the step at `in`, fetched a step before the copies need them.
  int block = 0, off = -1;  // off -1: outside the span
  auto look_up = [&]() {
    off = -1;
    if (in.u >= units) return;
    const int pos = (in.first + in.k) * C::UNIT + warp * C::TOK + (lane & (C::TOK - 1));
    if (pos >= in.lo && pos < in.hi) {
      const int page = a.c.page_of(pos);
      off = pos - page * a.c.block_size;
      block = a.c.tables[in.b * a.c.table_stride + page];
    }
  };
  look_up();

  // The copies of a step's K (all rows, 512 / RB of them at once) and V (a lane's own fragments: tokens 2t, 2t + 1, 2t + 8, 2t + 9 of
  // each half).  ALL: every token of the step is there.
  auto copy_k = [&](auto all, uint32_t dst, uint32_t row, uint32_t ok) {
#pragma unroll
    for (int i = 0; i < C::K_BYTES / 512; ++i) {
      const int tok = i * (512 / C::RB > 0 ? 512 / C::RB : 1) + lane / C::ROW16, piece = lane % C::ROW16;
      const char* p = kbase + (uint64_t)__shfl_sync(0xffffffffu, row, tok) * 16;
      cp_async16(dst + tok * C::RB + 16 * (piece ^ (C::RB >= 128 ? (tok & 1) * 4 : 0)), p + (FULL ? 16 * piece : min(16 * piece, row_bytes - 16)),
                 (decltype(all)::value || (ok >> tok & 1)) && (FULL || 16 * piece < row_bytes));
    }
  };
  auto copy_v = [&](auto all, uint32_t dst, uint32_t row, uint32_t ok) {
#pragma unroll
    for (int hf = 0; hf < C::HALVES; ++hf) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = 16 * hf + 2 * t + (j & 1) + 8 * (j >> 1);
        const char* p = vbase + (uint64_t)__shfl_sync(0xffffffffu, row, tok) * 16;
        const bool live = decltype(all)::value || (ok >> tok & 1);
#pragma unroll
        for (int c = 0; c < C::VCH; ++c) {
          const uint32_t to = dst + hf * C::V_HALF + ((j * C::VCH + c) * 32 + lane) * C::VPIECE;
          if constexpr (C::VPIECE == 16) cp_async16(to, p + v_piece(c), live);
          else cp_async8(to, p + v_piece(c), live);
        }
      }
    }
  };

  uint32_t row = 0, there = 0;  // row of token `lane` of the step whose K was fetched last (in units of 16 bytes), which tokens of it are there
  auto fetch_k = [&](int st) {
    there = 0;
    if (in.u < units) {
      const int kv_head = head_tiles == 1 ? in.tile : in.tile / head_tiles;
      const bool known = (uint32_t)block < (uint32_t)a.c.num_blocks, here = off >= 0 && known;
      if (off >= 0 && !known) report(a.err, MCOP_DEVERR_SLOT);
      // a token that is not there is copied as zeros: nothing is read for it (reading some other row in its place made that row's
      // L2 slice the bottleneck), its logit is replaced and its weight, 0, meets no NaN of a float cache
      row = here ? (uint32_t)block * block16 + (uint32_t)off * page16 + (uint32_t)kv_head * head16 : 0u;
      there = __ballot_sync(0xffffffffu, here) & C::ALL;
      if (lane == 0) valid[warp][st] = there;
      if (there) {
        const uint32_t dst = smem_addr(kring + st * C::K_BYTES);
        if (there == C::ALL) copy_k(std::true_type{}, dst, row, there);
        else copy_k(std::false_type{}, dst, row, there);
        if constexpr (MODE == kScaleToken) {  // 0 where there is no token
          const int64_t at = here ? ((int64_t)block * a.c.block_size + off) * a.c.kv_heads + kv_head : 0;
          const uint32_t to = smem_addr(sring + st * 2 * C::TOK + (lane & (C::TOK - 1)));
          if (C::TOK == 32 || lane < 16) cp_async4(to, a.c.k_scale + at, here);
          if (C::TOK == 32 || lane >= 16) cp_async4(to + C::TOK * 4, a.c.v_scale + at, here);
        }
      }
      in.next<C::UNIT>(a, tiles);
      look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto fetch_v = [&](int st) {
    const uint32_t dst = smem_addr(vring + st * C::V_BYTES);
    if (there == C::ALL) copy_v(std::true_type{}, dst, row, there);
    else if (there) copy_v(std::false_type{}, dst, row, there);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // K and V of ST steps are on their way or in use at any time: K's place is refilled as soon as the logits are formed, V's as
  // soon as it is added up.  Of the 2 ST copies in flight the oldest is waited for.
  auto wait_oldest = [&]() {
    asm volatile("cp.async.wait_group %0;" ::"n"(2 * C::ST - 1) : "memory");
    __syncwarp();
  };

#pragma unroll
  for (int s = 0; s < C::ST; ++s) {
    fetch_k(s);
    fetch_v(s);
  }

  float o[NT][C::MT][4], m[NT][2], l[NT][2], kf[NT][2];
  uint32_t qf[NT][C::MT][2];
  bool fresh = true;
  int stage = 0;
  bool began_here = cur.k == 0;

  for (int u = 0; u < units; ++u) {
    const int kv_head = head_tiles == 1 ? cur.tile : cur.tile / head_tiles, h0 = (cur.tile - kv_head * head_tiles) * C::HEADS;
    if (fresh) {
      fresh = false;
      const Seq s = sequence(a, cur.b);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = h0 + nt * 8 + g;
        const T* qp = static_cast<const T*>(a.q) + (int64_t)s.q0 * a.q_token + (int64_t)(kv_head * G + min(h, G - 1)) * a.q_head;
        float unscale = 1.f;
        if constexpr (C::I8) {
          // k16 step i: word i % 4 of K piece i / 4; its first register holds the bytes 0 and 2, its second the bytes 1 and 3.
          // The largest |q| of a head goes to [2^14, 2^15): what f16 then loses below 2^-14 is 2^-40 of it.
          float x[C::MT][4], top = 0.f;
#pragma unroll
          for (int i = 0; i < C::MT; ++i) {
            const int d = 64 * (i / 4) + 16 * t + 4 * (i % 4);
            uint2 w = make_uint2(0, 0);
            if (h < G && d < a.head_size && s.qn > 0) w = *reinterpret_cast<const uint2*>(qp + d);
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              x[i][c] = ElemTraits<T>::to_float(e[c]);
              top = fmaxf(top, fabsf(x[i][c]));
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = max((int)(__float_as_uint(top) >> 23) - 127, -86);
          const float up = top <= FLT_MAX ? __uint_as_float((uint32_t)(127 + 14 - e) << 23) : 1.f;
          unscale = top <= FLT_MAX ? __uint_as_float((uint32_t)(127 + e - 14) << 23) : 1.f;
#pragma unroll
          for (int i = 0; i < C::MT; ++i) {
            qf[nt][i][0] = pack2<QT>(x[i][0] * up, x[i][2] * up);
            qf[nt][i][1] = pack2<QT>(x[i][1] * up, x[i][3] * up);
          }
        } else {
#pragma unroll
          for (int i = 0; i < C::MT; ++i) {  // k16 step i: half i % 2 of K piece i / 2
            const int d = 32 * (i / 2) + 8 * t + 4 * (i % 2);
            uint2 w = make_uint2(0, 0);
            if (h < G && d < a.head_size && s.qn > 0) w = *reinterpret_cast<const uint2*>(qp + d);
            qf[nt][i][0] = w.x;
            qf[nt][i][1] = w.y;
          }
        }
        // the factors of this lane's columns, heads 2t and 2t + 1 of the tile
        const float u0 = __shfl_sync(0xffffffffu, unscale, 8 * t), u1 = __shfl_sync(0xffffffffu, unscale, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          m[nt][c] = -INFINITY;
          l[nt][c] = 0.f;
          kf[nt][c] = a.scale * kLog2e * (MODE == kScaleHead ? a.c.k_scale[kv_head] : 1.f) * (c ? u1 : u0);
        }
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
      }
    }
    wait_oldest();
    const uint32_t ok = valid[warp][stage];
    uint32_t p[C::HALVES][NT][2];
    if (ok) {
      const unsigned char* src = kring + stage * C::K_BYTES;
      float s[C::HALVES][NT][4];
#pragma unroll
      for (int hf = 0; hf < C::HALVES; ++hf) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[hf][nt][0] = s[hf][nt][1] = s[hf][nt][2] = s[hf][nt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < C::KCH; ++c) {
          const unsigned char* at = src + (16 * hf + g) * C::RB + 16 * ((4 * c + t) ^ (C::RB >= 128 ? (g & 1) * 4 : 0));
          const uint4 x = *reinterpret_cast<const uint4*>(at), y = *reinterpret_cast<const uint4*>(at + 8 * C::RB);
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
          if constexpr (C::I8) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t a0 = codes.f16(xw[w]), a1 = codes.f16(yw[w]), a2 = codes.f16(xw[w] >> 8), a3 = codes.f16(yw[w] >> 8);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<QT>(s[hf][nt], a0, a1, a2, a3, qf[nt][4 * c + w][0], qf[nt][4 * c + w][1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<QT>(s[hf][nt], xw[2 * e], yw[2 * e], xw[2 * e + 1], yw[2 * e + 1], qf[nt][2 * c + e][0], qf[nt][2 * c + e][1]);
          }
        }
      }
      // s[hf][nt][2 r + c]: token g + 8 r of half hf, head 2t + c of tile nt
      const float* scales = sring + stage * 2 * C::TOK;
      float ref[C::HALVES][2], vs[C::HALVES][2];
      bool grown = false;
#pragma unroll
      for (int hf = 0; hf < C::HALVES; ++hf) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int tok = 16 * hf + 8 * r + g;
          const bool here = ok == C::ALL || (ok >> tok & 1);
          float ks = 1.f;
          ref[hf][r] = 0.f;
          vs[hf][r] = 1.f;
          if constexpr (MODE == kScaleToken) {
            ks = scales[tok];
            vs[hf][r] = scales[C::TOK + tok];
            // what a token's scale adds to its logit where the maximum is concerned (bounded, so that fp32 holds the weights and their
            // sum: 2^29 weights of 2^(90 + 8), and weights down to 2^-26 of the largest beside a scale of 2^100)
            ref[hf][r] = __log2f(fminf(fmaxf(fabsf(vs[hf][r]), 0x1p-90f), 0x1p100f));
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float& x = s[hf][nt][2 * r + c];
              x = here ? x * (MODE == kScaleToken ? kf[nt][c] * ks : kf[nt][c]) : -INFINITY;
              grown |= x + ref[hf][r] > m[nt][c] + kMaxSlack;
            }
          }
        }
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = m[nt][c];
#pragma unroll
            for (int hf = 0; hf < C::HALVES; ++hf) top = fmaxf(top, fmaxf(s[hf][nt][c] + ref[hf][0], s[hf][nt][2 + c] + ref[hf][1]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float keep = m[nt][c] == -INFINITY ? 0.f : exp2_approx(m[nt][c] - top);
            m[nt][c] = top;
            l[nt][c] *= keep;
#pragma unroll
            for (int i = 0; i < C::MT; ++i) {
              o[nt][i][c] *= keep;
              o[nt][i][2 + c] *= keep;
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float safe[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) safe[c] = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
#pragma unroll
        for (int hf = 0; hf < C::HALVES; ++hf)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float w0 = exp2_approx(s[hf][nt][2 * r] - safe[0]), w1 = exp2_approx(s[hf][nt][2 * r + 1] - safe[1]);
            l[nt][0] += w0;
            l[nt][1] += w1;
            p[hf][nt][r] = transpose8x8(MODE == kScaleToken ? pack2<W>(w0 * vs[hf][r], w1 * vs[hf][r]) : pack2<W>(w0, w1));
          }
      }
    }
    __syncwarp();
    fetch_k(stage);
    wait_oldest();
    if (ok) {
      const unsigned char* src = vring + stage * C::V_BYTES;
#pragma unroll
      for (int hf = 0; hf < C::HALVES; ++hf)
#pragma unroll
        for (int c = 0; c < C::VCH; ++c) {
          constexpr int WORDS = C::VPIECE / 4;
          uint32_t v[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned char* at = src + hf * C::V_HALF + ((j * C::VCH + c) * 32 + lane) * C::VPIECE;
            if constexpr (C::VPIECE == 16) {
              const uint4 x = *reinterpret_cast<const uint4*>(at);
              v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2*>(at);
              v[j][0] = x.x; v[j][1] = x.y;
            }
          }
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            if constexpr (C::I8) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {  // elements 2e, 2e + 1 of the word, each with the two tokens of a register
                const uint32_t s0 = e ? 0x0602 : 0x0400, s1 = e ? 0x0703 : 0x0501;
                const uint32_t a0 = codes.f16(__byte_perm(v[0][w], v[1][w], s0)), a1 = codes.f16(__byte_perm(v[0][w], v[1][w], s1));
                const uint32_t a2 = codes.f16(__byte_perm(v[2][w], v[3][w], s0)), a3 = codes.f16(__byte_perm(v[2][w], v[3][w], s1));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<W>(o[nt][(c * WORDS + w) * 2 + e], a0, a1, a2, a3, p[hf][nt][0], p[hf][nt][1]);
              }
            } else {
              const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5410), a1 = __byte_perm(v[0][w], v[1][w], 0x7632);
              const uint32_t a2 = __byte_perm(v[2][w], v[3][w], 0x5410), a3 = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<W>(o[nt][c * 4 + w], a0, a1, a2, a3, p[hf][nt][0], p[hf][nt][1]);
            }
          }
        }
    }


    const bool ends = cur.k == cur.n - 1;
    if (ends || u == units - 1) {
      // --- join the warps: every warp has its own maximum, sum and O (put where the V was that the warp added up last)
      auto merge = [&](int w) { return reinterpret_cast<float*>(smem + w * C::WARP + C::ST * C::K_BYTES + stage * C::V_BYTES); };
      __syncwarp();
      const bool whole = began_here && ends;
      const Seq s = sequence(a, cur.b);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
          if (g == 0) {
            ml[warp][0][nt * 8 + 2 * t + c] = m[nt][c];
            ml[warp][1][nt * 8 + 2 * t + c] = l[nt][c];
          }
        }
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) merge(warp)[i * 128 + c * 32 + lane] = o[nt][i][c];
        __syncthreads();
        const int par = warp & 1, hh = nt * 8 + 2 * t + par, h = h0 + hh;  // this thread's head; rows d, d + 1 of its tiles
        float top = ml[0][0][hh], scale[kWarps], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ml[w][0][hh]);
        const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          scale[w] = ml[w][0][hh] == -INFINITY ? (ml[w][1][hh] == 0.f ? 0.f : 1.f) : exp2_approx(ml[w][0][hh] - safe);
          sum += ml[w][1][hh] * scale[w];
        }
        if (h < G) {
          float* part = parts + (int64_t)(2 * blockIdx.x + (began_here ? 1 : 0)) * C::SLOT;
          const int head = kv_head * G + h;
          float f = sum == 0.f ? 0.f : 1.f / sum;
          if (MODE == kScaleHead) f *= a.c.v_scale[kv_head];
          T* out = static_cast<T*>(a.out) + (int64_t)s.q0 * a.o_token + (int64_t)head * a.o_head;
#pragma unroll
          for (int ii = 0; ii < C::MT / 2; ++ii) {
            const int i = 2 * ii + (warp >> 1);
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float* r = merge(w) + i * 128 + lane;
              x = __fmaf_rn(scale[w], r[par * 32], x);
              y = __fmaf_rn(scale[w], r[(par + 2) * 32], y);
            }
            const int d = C::I8 ? (C::RB >= 128 ? 128 * (i / 8) + 16 * g + 2 * (i % 8) : 8 * g + 2 * i) : 64 * (i / 4) + 8 * g + 2 * (i % 4);
            if (!whole) *reinterpret_cast<float2*>(part + hh * DP + d) = make_float2(x, y);
            else if (d < a.head_size && s.qn > 0) *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(x * f, y * f);
          }
          if (g == 0 && warp < 2) {
            if (!whole) *reinterpret_cast<float2*>(part + C::HEADS * DP + 2 * hh) = make_float2(top, sum);
            else if (a.lse && s.qn > 0) a.lse[(int64_t)s.q0 * a.q_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
          }
        }
        __syncthreads();
      }
      if (u == units - 1 && tid == 0) {
        Rec r{cur.b, cur.tile, 0, 0};
        if (!ends && began_here) {
          const int64_t last = (u1 - 1 + (cur.n - 1 - cur.k)) / per;
          r.count = (int)(last - blockIdx.x) + 1;
        }
        recs[blockIdx.x] = r;
      }
      fresh = true;
      began_here = true;
    }
    __syncwarp();
    fetch_v(stage);
    stage = stage + 1 == C::ST ? 0 : stage + 1;
    cur.next<C::UNIT>(a, tiles);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins the partial results of the items that cross CTA borders: CTA c of the kernel above holds the first part of at most
// one such item, the CTAs behind it one part each.  A thread takes four elements of one head, and every GROUPS-th part: the parts
// come from L2, and it is the number of loads on their way that counts (one long sequence has 16 parts or more per head).
template <int DP, int NT> struct Join {
  static constexpr int SPAN = 2 * NT * DP;               // threads that cover all heads of an item
  static constexpr int GROUPS = SPAN <= 256 ? 4 : 2;
};
template <typename T, int MODE, int DP, int NT>
__global__ void __launch_bounds__(Join<DP, NT>::SPAN * Join<DP, NT>::GROUPS) decode_join_kernel(AttnArgs a, const float* __restrict__ parts,
                                                                                               const Rec* __restrict__ recs) {
  using C = Cfg<T, MODE, DP, NT>;
  using J = Join<DP, NT>;
  __shared__ int tops[C::HEADS];
  __shared__ float4 part_x[J::GROUPS - 1][J::SPAN];
  __shared__ float part_sum[J::GROUPS - 1][J::SPAN];
  pdl_launch_dependents();
  pdl_wait();
  const Rec r = recs[blockIdx.x];
  if (r.count == 0) return;
  const int G = a.q_heads / a.c.kv_heads, head_tiles = (G + C::HEADS - 1) / C::HEADS;
  const int group = threadIdx.x / J::SPAN, me = threadIdx.x % J::SPAN, hh = me / (DP / 4), d = me % (DP / 4) * 4;
  auto part = [&](int i) { return parts + (int64_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * C::SLOT; };
  // the largest maximum of each head, as an integer of the same order
  auto ordered = [](float x) { const int i = __float_as_int(x); return i < 0 ? i ^ 0x7fffffff : i; };
  if (threadIdx.x < C::HEADS) tops[threadIdx.x] = ordered(-INFINITY);
  __syncthreads();
  int mine = ordered(-INFINITY);
  for (int i = group * (DP / 4) + me % (DP / 4); i < r.count; i += J::GROUPS * (DP / 4)) mine = max(mine, ordered(part(i)[C::HEADS * DP + 2 * hh]));
  if (mine != ordered(-INFINITY)) atomicMax(&tops[hh], mine);
  __syncthreads();
  const int ti = tops[hh];
  const float top = __int_as_float(ti < 0 ? ti ^ 0x7fffffff : ti), safe = top == -INFINITY ? 0.f : top;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = group; i < r.count; i += J::GROUPS) {
    const float2 ml = *reinterpret_cast<const float2*>(part(i) + C::HEADS * DP + 2 * hh);
    const float4 v = *reinterpret_cast<const float4*>(part(i) + hh * DP + d);
    const float w = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_approx(ml.x - safe);
    sum = __fmaf_rn(w, ml.y, sum);
    x.x = __fmaf_rn(w, v.x, x.x);
    x.y = __fmaf_rn(w, v.y, x.y);
    x.z = __fmaf_rn(w, v.z, x.z);
    x.w = __fmaf_rn(w, v.w, x.w);
  }
  if (group > 0) {
    part_x[group - 1][me] = x;
    part_sum[group - 1][me] = sum;
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int g = 0; g < J::GROUPS - 1; ++g) {
    const float4 y = part_x[g][me];
    x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
    sum += part_sum[g][me];
  }
  const int kv_head = r.tile / head_tiles, h = (r.tile - kv_head * head_tiles) * C::HEADS + hh;
  if (h >= G) return;
  float f = sum == 0.f ? 0.f : 1.f / sum;
  if (MODE == kScaleHead) f *= a.c.v_scale[kv_head];
  const int head = kv_head * G + h;
  if (d < a.head_size)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)r.b * a.o_token + (int64_t)head * a.o_head + d) =
        make_uint2(pack2<T>(x.x * f, x.y * f), pack2<T>(x.z * f, x.w * f));
  if (a.lse && d == 0) a.lse[(int64_t)r.b * a.q_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

template <typename T, int MODE, int DP, int NT, bool FULL> int launch_one(const AttnArgs& a, void* ws, cudaStream_t st) {
  using C = Cfg<T, MODE, DP, NT>;
  auto kernel = decode_kernel<T, MODE, DP, NT, FULL>;
  if (cudaError_t e = ensure_dynamic_smem((const void*)kernel, C::SMEM); e != cudaSuccess)
    return set_error(MCOP_ERR_CUDA, "paged_attention_decode: %s", cudaGetErrorString(e));
  const int grid = sm_count() * C::CTAS;
  float* parts = static_cast<float*>(ws);
  Rec* recs = reinterpret_cast<Rec*>(parts + (int64_t)grid * 2 * C::SLOT);
  launch_pdl(kernel, dim3(grid), dim3(kThreads), C::SMEM, st, a, parts, recs);
  if (int rc = check_launch("paged_attention_decode")) return rc;
  launch_pdl(decode_join_kernel<T, MODE, DP, NT>, dim3(grid), dim3(Join<DP, NT>::SPAN * Join<DP, NT>::GROUPS), 0, st, a, (const float*)parts, (const Rec*)recs);
  return check_launch("paged_attention_decode");
}

// Two n8 tiles share a read of the rows where a KV head has more than 8 query heads (at head size 256 they would need 128
// accumulators a lane beside 64 registers of Q).
bool two_tiles(int q_heads, int kv_heads, int head_size) { return q_heads / kv_heads > 8 && (head_size == 64 || head_size == 128); }

template <typename T, int MODE> int launch_mode(const AttnArgs& a, void* ws, cudaStream_t st) {
  const bool two = two_tiles(a.q_heads, a.c.kv_heads, a.head_size);
  if (a.head_size == 64) return two ? launch_one<T, MODE, 64, 2, true>(a, ws, st) : launch_one<T, MODE, 64, 1, true>(a, ws, st);
  if (a.head_size == 128) return two ? launch_one<T, MODE, 128, 2, true>(a, ws, st) : launch_one<T, MODE, 128, 1, true>(a, ws, st);
  if (a.head_size < 64) return launch_one<T, MODE, 64, 1, false>(a, ws, st);
  return a.head_size < 128 ? launch_one<T, MODE, 128, 1, false>(a, ws, st) : launch_one<T, MODE, 256, 1, false>(a, ws, st);
}

}  // namespace

size_t decode_workspace(int q_heads, int kv_heads, int head_size) {
  const int heads = two_tiles(q_heads, kv_heads, head_size) ? 16 : 8, dp = head_size <= 64 ? 64 : head_size <= 128 ? 128 : 256;
  const size_t ctas = (size_t)sm_count() * kMaxCtasPerSm;
  return ctas * (2 * heads * (dp + 2) * sizeof(float) + sizeof(Rec));
}

int launch_decode(const AttnArgs& a, int dtype, void* ws, size_t ws_bytes, cudaStream_t st) {
  MCOP_REQUIRE(ws && aligned16(ws) && ws_bytes >= decode_workspace(a.q_heads, a.c.kv_heads, a.head_size), MCOP_ERR_WORKSPACE,
               "paged_attention_decode: workspace missing, misaligned or too small");
  if (dtype == MCOP_BF16) {
    if (a.scale_mode == kScaleNone) return launch_mode<__nv_bfloat16, kScaleNone>(a, ws, st);
    return a.scale_mode == kScaleHead ? launch_mode<__nv_bfloat16, kScaleHead>(a, ws, st) : launch_mode<__nv_bfloat16, kScaleToken>(a, ws, st);
  }
  if (a.scale_mode == kScaleNone) return launch_mode<__half, kScaleNone>(a, ws, st);
  return a.scale_mode == kScaleHead ? launch_mode<__half, kScaleHead>(a, ws, st) : launch_mode<__half, kScaleToken>(a, ws, st);
}

}  // namespace mcop
