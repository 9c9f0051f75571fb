// Chunk attention on the fifth-generation tensor cores: a run of new tokens per sequence over its cached tokens.
//
// The rows of a work item are (new token, query head) pairs of one sequence and one KV head, in that order: all query heads of a
// KV head share the tiles of K and V, and a short chunk still fills a tile.  256 rows make an item: two M = 128 tiles, so that the
// tensor cores form the logits of one tile while the other tile's softmax runs.
//   S[128 x 128] = Q[128 x D] K^T        (both operands in shared memory, S in tensor memory)
//   P = exp2(S * c - m)                  (a thread owns a row: no shuffles; P goes back to tensor memory over S, in 16 bits)
//   O[128 x D]  += P[128 x 128] V        (P from tensor memory, V in shared memory as it lies: MN-major)
// Roles (16 warps, registers dealt by setmaxnreg): 2 x 4 warps of softmax, 4 warps that bring Q, K and V into shared memory, one
// thread that issues the MMAs.  K and V pass through a ring of 16-bit tiles of 128 tokens; rows are gathered from their pages, and int8
// codes become bf16 (K, beside bf16 queries) or f16 on the way, exactly: their scales multiply logits and weights in fp32.  The
// running maximum is moved (and O rescaled) only when a logit passes it by 2^8.
//
// Work split: the (item, 128-token tile) pairs of the whole call form one line, cut into equal ranges, one per CTA and SM; a first
// launch of one CTA lays the line out from the lengths on the device (so a captured graph serves any), a third joins the items
// that cross a border, in a fixed order.
//
// Bound: per pair of 256 x 128 logits 2 x 256 x 128 x D x 2 flops of MMA (2048 cycles at D = 128) and 32,768 exponentials (2048
// cycles of the SM's 16 per cycle): the two are equal, and everything else has to hide behind them.
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace mcop {
namespace {

constexpr int kRows = 256, kTile = 128, kThreads = 512;
// Fewer tiles than this per CTA are not worth a partial result of their own.
constexpr int kMinTiles = 2;
constexpr uint32_t kSpin = 1u << 20, kPolls = 1u << 26;  // tries of a wait, of a poll that does not suspend the thread
constexpr int kWaitSoftmax = 8, kWaitLoad = 9, kWaitMma = 10;  // codes of the error word

// The line of work, in the workspace.  A query tile: 256 rows of one sequence, and the tokens that they see between them.
struct alignas(16) PlanTile {
  int b, t, rows, q0;      // sequence, tile of it, rows of the tile that are there, first new token of the sequence
  int qn, len, first, n;   // new tokens, cached tokens; tiles [first, first + n) of 128 tokens reach from lo to hi
  int lo, hi, pad[2];
};
// Where a CTA begins: `left` tiles of 128 tokens from tile k of query tile `tile` and KV head `head` on.
struct alignas(16) Start {
  int left, tile, head, k;
};
struct Plan {
  int64_t share, pad;  // tiles of 128 tokens per CTA
};
struct Rec {
  int b, t, head, count;
};
struct Layout {  // of the workspace
  Plan* plan;
  Start* starts;        // [ctas]
  int64_t* prefix;      // [max_tiles + 1]: tiles of 128 tokens (of one KV head) in front of a query tile
  PlanTile* tile;       // [max_tiles]
  int64_t* seq_tiles;   // [batch + 1]
  Rec* recs;            // [ctas]
  float* parts;         // [2 * ctas] slots: O [256][DP], then (maximum, sum) [256][2]
};
__host__ __device__ inline int64_t max_tiles(int64_t tokens, int batch, int group) { return tokens * group / kRows + batch; }
__host__ __device__ inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }
__host__ inline size_t layout(char* ws, int64_t tokens, int batch, int group, int dp, int ctas, Layout* l) {
  const int64_t mt = max_tiles(tokens, batch, group);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t was = at; at += up16(bytes); return ws + was; };
  Layout x;
  x.plan = (Plan*)take(sizeof(Plan));
  x.starts = (Start*)take(ctas * sizeof(Start));
  x.prefix = (int64_t*)take((mt + 1) * 8);
  x.tile = (PlanTile*)take(mt * sizeof(PlanTile));
  x.seq_tiles = (int64_t*)take((batch + 1) * 8);
  x.recs = (Rec*)take(ctas * sizeof(Rec));
  x.parts = (float*)take((size_t)ctas * 2 * kRows * (dp + 2) * 4);
  if (l) *l = x;
  return at;
}

// Tiles [first, first + n) of 128 tokens that the rows of query tile t of a sequence see between them; tokens [lo, hi).
struct Reach {
  int first, n, lo, hi;
};
__device__ __forceinline__ Reach reach(const AttnArgs& a, const Seq& s, int t, int group) {
  const int i0 = t * kRows / group, i1 = min(s.qn - 1, (t * kRows + kRows - 1) / group);
  Reach r;
  int other;
  span(a, s, i0, r.lo, other);
  span(a, s, i1, other, r.hi);
  r.lo = min(r.lo, r.hi);
  r.first = r.lo / kTile;
  r.n = max(1, (r.hi + kTile - 1) / kTile - r.first);
  return r;
}

// Tokens [lo, hi) that all rows of a query tile see: 128 tokens inside need no care for what a row must not see.
struct Common {
  int lo, hi;
  __device__ __forceinline__ bool whole(int base) const { return base >= lo && base + kTile <= hi; }
};
__device__ __forceinline__ Common seen_by_all(const AttnArgs& a, const PlanTile& pt, int group) {
  const Seq s{pt.q0, pt.qn, pt.len};
  Common c;
  int other;
  span(a, s, (pt.t * kRows + pt.rows - 1) / group, c.lo, other);
  span(a, s, pt.t * kRows / group, other, c.hi);
  return c;
}

__global__ void __launch_bounds__(1024) chunk_plan_kernel(AttnArgs a, Layout w, int64_t limit, int ctas) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int64_t sums[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.q_heads / a.c.kv_heads;
  auto scan = [&](int64_t v) {  // inclusive over the CTA; sums[32] = total
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
      int64_t u = sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) u += x;
      }
      sums[lane] = u;
      if (lane == 31) sums[32] = u;
    }
    __syncthreads();
    if (warp) v += sums[warp - 1];
    const int64_t total = sums[32];
    __syncthreads();
    return make_longlong2(v, total);
  };
  auto count = [&](int b) { return (int64_t)((int64_t)sequence(a, b).qn * G + kRows - 1) / kRows; };
  int64_t base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 1024) {
    const int b = b0 + tid;
    const int64_t n = b < a.batch ? count(b) : 0;
    const longlong2 s = scan(n);
    if (b < a.batch) w.seq_tiles[b] = base + s.x - n;
    base += s.y;
  }
  // sequences that overlap (reported as descending bounds) could add up to more than there is room for
  const int64_t tiles = min(base, limit);
  if (tid == 0) {
    w.seq_tiles[a.batch] = base;
  }
  __syncthreads();
  int64_t front = 0;
  for (int64_t i0 = 0; i0 < tiles; i0 += 1024) {
    const int64_t i = i0 + tid;
    int64_t n = 0;
    if (i < tiles) {
      int lo = 0, hi = a.batch;  // seq_tiles[lo] <= i < seq_tiles[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (w.seq_tiles[mid] <= i) lo = mid;
        else hi = mid;
      }
      const int t = (int)(i - w.seq_tiles[lo]);
      const Seq s = sequence<false>(a, lo);
      const Reach r = reach(a, s, t, G);
      n = r.n;
      w.tile[i] = PlanTile{lo, t, (int)min((int64_t)kRows, (int64_t)s.qn * G - (int64_t)t * kRows), s.q0, s.qn, s.len, r.first, r.n, r.lo, r.hi, {0, 0}};
    }
    const longlong2 s = scan(n);
    if (i < tiles) w.prefix[i] = front + s.x - n;
    front += s.y;
  }
  if (tid == 0) w.prefix[tiles] = front;
  __syncthreads();
  // equal shares of the line
  const int64_t heads = a.c.kv_heads, total = front * heads, share = max((int64_t)kMinTiles, (total + ctas - 1) / ctas);
  if (tid == 0) w.plan->share = share;
  for (int c = tid; c < ctas; c += 1024) {
    const int64_t u = share * c;
    Start s{(int)max((int64_t)0, min(total - u, share)), 0, 0, 0};
    if (s.left > 0) {
      int lo = 0, hi = (int)tiles;  // prefix[lo] * heads <= u < prefix[hi] * heads
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (w.prefix[mid] * heads <= u) lo = mid;
        else hi = mid;
      }
      const int64_t off = u - w.prefix[lo] * heads, n = w.prefix[lo + 1] - w.prefix[lo];
      s.tile = lo;
      s.head = (int)(off / n);
      s.k = (int)(off - s.head * n);
    }
    w.starts[c] = s;
  }
}

// A piece of work of a CTA: a query tile of the plan against tiles [k0, k1) of the n of its reach, for one KV head.
struct WorkLine {
  Start at;
  int head, k0, k1;
  __device__ __forceinline__ bool next(const Layout& w, int kv_heads, PlanTile& pt) {
    if (at.left <= 0) return false;
    pt = w.tile[at.tile];
    head = at.head;
    k0 = at.k;
    k1 = min(pt.n, at.k + at.left);
    at.left -= k1 - k0;
    at.k = 0;
    if (++at.head == kv_heads) { at.head = 0; ++at.tile; }
    return true;
  }
};

__device__ __forceinline__ void sts_u4(uint32_t dst, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ float4 lds4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
// Whether the phase is complete, without waiting for it (try_wait may suspend the thread for microseconds).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(smem_addr(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Two codes (bytes 0 and 2 of x, the others ignored) as a pair of T, exactly: 128 + seven bits minus 128 or 256 in bf16, 1024 +
// (code + 128) in f16.  The masks stay in registers: as immediates each would cost an instruction of its own.
struct Codes {
  uint32_t m7 = 0x007f007fu, m1 = 0x00800080u, one = 0x43004300u, m8 = 0x00ff00ffu, bias = 0x64806480u;
  __device__ __forceinline__ Codes() { asm volatile("" : "+r"(m7), "+r"(m1), "+r"(one), "+r"(m8), "+r"(bias)); }
  template <typename T> __device__ __forceinline__ uint32_t two(uint32_t x) const {
    uint32_t lo, hi;
    if constexpr (ElemTraits<T>::code == MCOP_BF16) {
      asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(lo) : "r"(x), "r"(m7), "r"(one));  // (x & mask) | one
      asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(hi) : "r"(x), "r"(m1), "r"(one));
      __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi));
      return *reinterpret_cast<uint32_t*>(&r);
    } else {
      asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(lo) : "r"(x), "r"(m8), "r"(bias));  // (x & mask) ^ bias
      __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&bias));
      return *reinterpret_cast<uint32_t*>(&r);
    }
  }
};
// Whether one of the eight 16-bit floats is a NaN or an infinity; `clean` gets them with those replaced by 0.
template <typename T> __device__ __forceinline__ bool not_finite(uint4& u) {
  constexpr uint32_t E = ElemTraits<T>::code == MCOP_BF16 ? 0x7f80u : 0x7c00u;
  bool bad = false;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & E) == E) { bad = true; w[i] &= 0xffff0000u; }
    if ((w[i] >> 16 & E) == E) { bad = true; w[i] &= 0x0000ffffu; }
  }
  return bad;
}

template <int ST, int NI> struct Bars {
  uint64_t full[ST], empty[ST], q_full, q_empty, s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2], info_full[NI], drain;
};
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int n) {
    if (++s == n) { s = 0; phase ^= 1u; }
  }
};
// What the softmax has to know of a tile's tokens beside the logits.
struct alignas(16) TileInfo {
  float ks[kTile], vs[kTile];  // kScaleToken: K scale times the logit factor, V scale
  uint32_t here[4];            // which tokens are there (their page is in the cache)
  int all;                     // all of those inside the reach are
  float power;                 // scale_power of the largest finite V scale
  int wild, odd;               // a V scale is not finite; a K scale is not, or is negative
  float kmax, pad[3];          // the largest factor
};
struct TileBits {
  uint32_t here[4];
  int all;
};
// With a scale per token the running maximum follows, tile by tile, the largest logit plus the power of two above the largest V
// scale that the row sees there: weight times scale then lies below 2^kMaxSlack and fits f16.  Hidden tokens have no say: a tile's
// own power would let them take bits from the rows of an item that do not see them.  Scales count within 2^-90 and 2^100, so that
// fp32 holds the weights and their sum.
__device__ __forceinline__ float scale_power(float largest) { return (float)min(100, max(-90, (int)(__float_as_uint(largest) >> 23) - 126)); }

template <typename Info, int ST, int NI> struct Control {
  Info info[NI];
  Bars<ST, NI> bars;
  uint32_t row_at[2][kTile];  // cached rows of a tile, in units of 16 bytes
  uint32_t q_at[kRows];       // rows of a query tile, in units of 8 elements (0xffffffff: none)
  float vmax[2][4], kmax[2][4];
  int poison[8];              // items whose masked tiles hold a NaN or an infinity in V
  uint32_t tmem_at;
  alignas(16) float ones[std::is_same<Info, TileInfo>::value ? kTile : 4];
};

template <typename T, int MODE, int DP> struct Cfg {
  static constexpr bool I8 = MODE != kScaleNone;
  static constexpr int HALF = kTile * 128;               // 64 columns of 128 rows, 128-byte swizzle
  static constexpr int TILE = HALF * (DP / 64);          // a 16-bit tile of 128 rows
  static constexpr int RAW = I8 ? 2 * kTile * DP : 0;     // two int8 tiles on their way
  static constexpr int ST = DP == 128 ? (MODE == kScaleToken ? 3 : I8 ? 4 : 5) : 8;
  static constexpr int NI = ST < 4 ? 4 : ST;             // tiles whose information is kept
  using Info = typename std::conditional<MODE == kScaleToken, TileInfo, TileBits>::type;
  static constexpr int SMEM = (2 + ST) * TILE + RAW + (int)sizeof(Control<Info, ST, NI>);
  static_assert(SMEM <= 227 * 1024, "shared memory of an SM");
  static constexpr int PIECES = DP / 8;                  // 16-byte pieces of a row in shared memory
};

template <typename T, int MODE, int DP>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(AttnArgs a, Layout w) {
  using C = Cfg<T, MODE, DP>;
  using VT = typename std::conditional<C::I8, __half, T>::type;  // type of P and V
  using Info = typename C::Info;
  constexpr int ST = C::ST;
  using Ctl = Control<Info, C::ST, C::NI>;
  extern __shared__ __align__(1024) unsigned char raw[];  // Q: two tiles; the ring of K and V; control
  Ctl& ctl = *reinterpret_cast<Ctl*>(raw + (2 + ST) * C::TILE + C::RAW);
  auto& bars = ctl.bars;
  auto& info = ctl.info;
  auto& row_at = ctl.row_at;
  auto& q_at = ctl.q_at;
  auto& vmax = ctl.vmax;
  auto& kmax = ctl.kmax;
  auto& poison = ctl.poison;
  uint32_t& tmem_at = ctl.tmem_at;
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = warp >> 2;
  const uint32_t smem = smem_addr(raw);
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&bars.full[i], 4);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < C::NI; ++i) mbar_init(&bars.info_full[i], 4);
    mbar_init(&bars.q_full, 4);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_half[i], 4);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_empty[i], 4);
    }
    mbar_init(&bars.drain, 1);
    mbar_init_fence();
  }
  if (MODE == kScaleToken && tid >= 384) ctl.ones[tid - 384] = 1.f;
  if (warp == 12) tmem_alloc_all(&tmem_at);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = tmem_at;
  const int G = a.q_heads / a.c.kv_heads;
  WorkLine x;
  PlanTile pt;
  x.at = w.starts[blockIdx.x];
  if (tid == 0) w.recs[blockIdx.x].count = 0;
  if (smem & 1023) {  // (never seen: the window starts on such a boundary) the swizzle would not match
    if (tid == 0) report(a.err, kWaitMma);
    x.at.left = 0;
  }

  if (group < 2) {
    // ------------------------------------------------------------------------------------------ softmax of tile `group`
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const int r = tid & 127;  // row of the tile
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t s_addr = tmem + lanes + group * 128, o_addr = tmem + lanes + 256 + group * DP;
    Ring inf;
    uint32_t s_phase = 0, o_phase = 0;
    int item = 0;
    bool ok = true;
    while (ok && x.next(w, a.c.kv_heads, pt)) {
      const bool idle = group == 1 && pt.rows <= 128;
      const int row = group * 128 + r;
      const bool mine = row < pt.rows;
      const int flat = pt.t * kRows + row, token = flat / G, head = x.head * G + flat - token * G;
      int lo = 0, hi = INT_MAX;
      if (mine) span(a, Seq{pt.q0, pt.qn, pt.len}, token, lo, hi);
      float c = a.scale * kLog2e;
      if (MODE == kScaleHead) c *= a.c.k_scale[x.head];
      const bool flip = c < 0.f;  // a negative scale: the largest logit is the smallest product
      c = c == 0.f ? 1e-37f : fabsf(c);  // (0 times the -inf of a hidden column would be NaN)
      float m = -INFINITY, l = 0.f;
      if (idle) {  // no rows: keep in step with the item
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.o_full[group], o_phase, a.err, kWaitSoftmax, kSpin)))) break;
        o_phase ^= 1;
        for (int k = x.k0; k < x.k1; ++k) inf.advance(C::NI);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.o_empty[group]);
        ++item;
        continue;
      }
      for (int k = x.k0; k < x.k1 && ok; ++k) {
        const Info& in = info[inf.s];
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.info_full[inf.s], inf.phase, a.err, kWaitSoftmax, kSpin)))) break;
        inf.advance(C::NI);
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.s_full[group], s_phase, a.err, kWaitSoftmax, kSpin)))) break;
        s_phase ^= 1;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(s_addr + 32 * i, s + 32 * i);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_loaded32(s + 32 * i);
        if (MODE == kScaleHead && flip) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = -s[i];
        }
        const int base = (pt.first + k) * kTile;
        const bool masked = __any_sync(0xffffffffu, base < lo || base + kTile > hi) || !in.all;
        auto seen_of = [&](int i) {  // columns [lo - base, hi - base) of [32 i, 32 i + 32) that are there
          const int f = min(32, max(0, lo - base - 32 * i)), e = min(32, max(0, hi - base - 32 * i));
          return (uint32_t)((1ull << e) - 1) & ~(uint32_t)((1ull << f) - 1) & in.here[i];
        };
        // factors of the columns; where columns are hidden, the products with them are formed here
        uint32_t factor = 0, vfactor = 0;
        bool wild = false;
        if constexpr (MODE == kScaleToken) {
          factor = smem_addr(masked ? ctl.ones : in.ks);
          vfactor = smem_addr(in.vs);
          wild = in.wild;
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t seen = seen_of(i);
#pragma unroll
            for (int d = 0; d < 32; ++d) {
              float v = s[32 * i + d];
              if constexpr (MODE == kScaleToken) v *= in.ks[32 * i + d];
              s[32 * i + d] = seen & 1u << d ? v : -INFINITY;
            }
          }
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) asm("max.f32 %0, %0, %1, %2;" : "+f"(tops[j]) : "f"(s[i + j]), "f"(s[i + j + 4]));
        }
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        [[maybe_unused]] float logit = top;
        if constexpr (MODE == kScaleToken) {
          // The largest product, times the largest factor, bounds the logits; they are looked at one by one only where the
          // bound would move the maximum.
          if (masked) {
            top += in.power;
          } else {
            top = fmaxf(top, 0.f) * in.kmax + in.power;
            if (__any_sync(0xffffffffu, top > m + kMaxSlack) || in.odd) {
              float2 best = make_float2(-INFINITY, -INFINITY);
#pragma unroll
              for (int i = 0; i < 128; i += 4) {
                if (i % 32 == 0) asm volatile("" ::: "memory");  // (not all 128 factors in registers at once)
                const float4 f = lds4(factor + 4 * i);
                const float2 u = __fmul2_rn(make_float2(s[i], s[i + 1]), make_float2(f.x, f.y)), v = __fmul2_rn(make_float2(s[i + 2], s[i + 3]), make_float2(f.z, f.w));
                asm("max.f32 %0, %0, %1, %2;" : "+f"(best.x) : "f"(u.x), "f"(u.y));
                asm("max.f32 %0, %0, %1, %2;" : "+f"(best.y) : "f"(v.x), "f"(v.y));
              }
              top = fmaxf(best.x, best.y) + in.power;
            }
          }
        } else {
          top *= c;
        }
        bool grown = top > m + kMaxSlack;
        if (__any_sync(0xffffffffu, grown)) {
          if constexpr (MODE == kScaleToken) {
            if (masked) {  // by what this row sees
              float largest = 0.f;
#pragma unroll 1
              for (int i = 0; i < 4; ++i) {
                const uint32_t seen = seen_of(i);
#pragma unroll
                for (int d = 0; d < 32; d += 4) {
                  const float4 f = lds4(vfactor + 128 * i + 4 * d);
                  largest = fmaxf(fmaxf(largest, seen & 1u << d ? fabsf(f.x) : 0.f), seen & 2u << d ? fabsf(f.y) : 0.f);
                  largest = fmaxf(fmaxf(largest, seen & 4u << d ? fabsf(f.z) : 0.f), seen & 8u << d ? fabsf(f.w) : 0.f);
                }
              }
              top = logit + scale_power(largest);
              grown = top > m + kMaxSlack;
            }
          }
          const float to = grown ? top : m;
          float keep = m == -INFINITY ? 0.f : exp2_approx(m - to);
          m = to;
          l *= keep;
          if (k > x.k0) {
            // (S of this tile was issued behind the previous tile's P V: that product is complete.  8 columns at a time: the logits
            // stay in registers meanwhile)
#pragma unroll 1
            for (int i = 0; i < DP; i += 8) {
              float o[8];
              tmem_ld8(o_addr + i, o);
              tmem_wait_ld();
              tmem_loaded8(o);
#pragma unroll
              for (int d = 0; d < 8; ++d) o[d] *= keep;
              tmem_st8(o_addr + i, o);
            }
          }
        }
        const float safe = m == -INFINITY ? 0.f : m;
        float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
        // 32 weights: summed, times their tokens' scales, rounded.  FIX: a scale that is not finite reaches only the rows that see its token.
        auto weights = [&](auto FIX, int i, uint32_t* p) {
          const float2 shift = make_float2(-safe, -safe);
#pragma unroll
          for (int d = 0; d < 16; d += 2) {
            float2 u = make_float2(s[32 * i + 2 * d], s[32 * i + 2 * d + 1]), v = make_float2(s[32 * i + 2 * d + 2], s[32 * i + 2 * d + 3]);
            if constexpr (MODE == kScaleToken) {
              const float4 f = lds4(factor + 4 * (32 * i + 2 * d));
              u = __ffma2_rn(u, make_float2(f.x, f.y), shift);
              v = __ffma2_rn(v, make_float2(f.z, f.w), shift);
            } else {
              u = __ffma2_rn(u, make_float2(c, c), shift);
              v = __ffma2_rn(v, make_float2(c, c), shift);
            }
            u.x = exp2_approx(u.x); u.y = exp2_approx(u.y);
            v.x = exp2_approx(v.x); v.y = exp2_approx(v.y);
            sum0 = __fadd2_rn(sum0, u);
            sum1 = __fadd2_rn(sum1, v);
            if constexpr (MODE == kScaleToken) {
              const float4 f = lds4(vfactor + 4 * (32 * i + 2 * d));
              const float2 y = __fmul2_rn(u, make_float2(f.x, f.y)), z = __fmul2_rn(v, make_float2(f.z, f.w));
              if constexpr (decltype(FIX)::value) {
                u.x = u.x == 0.f ? 0.f : y.x; u.y = u.y == 0.f ? 0.f : y.y;
                v.x = v.x == 0.f ? 0.f : z.x; v.y = v.y == 0.f ? 0.f : z.y;
              } else {
                u = y;
                v = z;
              }
            }
            p[d] = pack2<VT>(u.x, u.y);
            p[d + 1] = pack2<VT>(v.x, v.y);
          }
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
          if (MODE == kScaleToken && wild) weights(std::true_type{}, i, p);
          else weights(std::false_type{}, i, p);
          tmem_st16(s_addr + 16 * i, p);
          if (i == 1) {  // the product with the first 64 tokens can start
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_half[group]);
          }
        }
        l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[group]);
      }
      if (ok) {
        // O of the item
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.o_full[group], o_phase, a.err, kWaitSoftmax, kSpin)))) break;
        o_phase ^= 1;
        tc_fence_after();
        const bool whole = x.k1 - x.k0 == pt.n;
        float f = 1.f;
        if (MODE == kScaleHead) f = a.c.v_scale[x.head];
        const float norm = whole ? (l == 0.f ? 0.f : f / l) : f;
        float* part = w.parts + (int64_t)(2 * blockIdx.x + (x.k0 == 0 ? 1 : 0)) * (kRows * (DP + 2));
        T* out = static_cast<T*>(a.out) + (int64_t)(pt.q0 + token) * a.o_token + (int64_t)head * a.o_head;
        const bool sick = !C::I8 && *(volatile int*)&poison[item & 7];
#pragma unroll 1
        for (int i = 0; i < DP / 32; ++i) {
          float o[32];
          __syncwarp();
          tmem_ld32(o_addr + 32 * i, o);
          tmem_wait_ld();
          tmem_loaded32(o);
          if (i == DP / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.o_empty[group]);
          }
          if constexpr (!C::I8) {
            if (sick && mine) {  // the tiles that some rows see in part were added up without their NaNs and infinities: add those that this row sees
              const Common common = seen_by_all(a, pt, G);
              for (int k = x.k0; k < x.k1; ++k) {
                const int base = (pt.first + k) * kTile;
                if (common.whole(base)) continue;
                for (int j = max(lo, base); j < min(hi, base + kTile); ++j) {
                  const int slot = slot_of(a, pt.b, j);
                  if (slot < 0) continue;
                  const T* v = static_cast<const T*>(a.c.v) + row_of(a.c, slot, x.head) + 32 * i;
#pragma unroll
                  for (int d = 0; d < 32; d += 8) {
                    if (32 * i + d >= a.head_size) break;
                    const uint4 u = *reinterpret_cast<const uint4*>(v + d);
                    uint4 clean = u;
                    if (!not_finite<T>(clean)) continue;
                    const T* y = reinterpret_cast<const T*>(&u);
#pragma unroll
                    for (int z = 0; z < 8; ++z) {
                      const float x = ElemTraits<T>::to_float(y[z]);
                      if (!(fabsf(x) <= FLT_MAX)) o[d + z] += x;
                    }
                  }
                }
              }
            }
          }
#pragma unroll
          for (int d = 0; d < 32; ++d) o[d] *= norm;
          if (!mine) {
          } else if (whole) {
#pragma unroll
            for (int d = 0; d < 32; d += 8)
              if (32 * i + d < a.head_size)
                *reinterpret_cast<uint4*>(out + 32 * i + d) = make_uint4(pack2<T>(o[d], o[d + 1]), pack2<T>(o[d + 2], o[d + 3]), pack2<T>(o[d + 4], o[d + 5]),
                                                                         pack2<T>(o[d + 6], o[d + 7]));
          } else {
#pragma unroll
            for (int d = 0; d < 32; d += 4) *reinterpret_cast<float4*>(part + row * DP + 32 * i + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          }
        }
        if (mine) {
          if (!whole) *reinterpret_cast<float2*>(part + kRows * DP + 2 * row) = make_float2(m, l);
          else if (a.lse) a.lse[(int64_t)(pt.q0 + token) * a.q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      if (tid == 0 && x.at.left == 0 && x.k0 == 0 && x.k1 < pt.n) {  // the item that begins here and goes on in the next CTA
        const int64_t share = w.plan->share, last = share * (blockIdx.x + 1) - 1 + (pt.n - x.k1);
        w.recs[blockIdx.x] = Rec{pt.b, pt.t, x.head, (int)(last / share - blockIdx.x) + 1};
      }
      ++item;
    }
  } else if (group == 2) {
    // ------------------------------------------------------------------------------------------ Q, K and V into shared memory
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int lt = tid & 127, lwarp = warp & 3;
    uint32_t q_smem = smem;
    asm volatile("" : "+r"(q_smem));  // (keeps what the roles derive from it out of the code in front of them)
    const uint32_t ring = q_smem + 2 * C::TILE;
    const int row_pieces = a.head_size * (C::I8 ? 1 : 2) / 16;  // 16-byte pieces of a cached row
    const uint32_t block16 = (uint32_t)(a.c.block_stride * (C::I8 ? 1 : 2) / 16), page16 = (uint32_t)(a.c.page_stride * (C::I8 ? 1 : 2) / 16),
                   head16 = (uint32_t)(a.c.head_stride * (C::I8 ? 1 : 2) / 16);
    const char* kbase = static_cast<const char*>(a.c.k);
    const char* vbase = static_cast<const char*>(a.c.v);
    auto sync = [&]() { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    auto sync_and = [&](bool v) {
      uint32_t r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(r)
          : "r"((uint32_t)v)
          : "memory");
      return r != 0;
    };
    Ring st, done, inf;       // stage to fill next, stage to hand over next, tile information to fill next
    const uint32_t rawbuf = ring + ST * C::TILE;
    const Codes codes;
    uint32_t q_phase = 0;
    int pending = 0;          // copies issued and not handed over (float caches)
    uint32_t with_q = 0, scan_v = 0;  // one bit per pending copy, the oldest in bit pending - 1: Q came with it; V of a masked tile
    uint32_t scan_item = 0;
    // Once a wait has run out (ok false) a warp copies nothing more, but walks on to the end: the four meet at barriers.
    bool ok = true;
    int item = 0, buf = 0;

    // hands over the oldest pending copy
    auto hand_over = [&]() {
      const uint32_t bit = 1u << (pending - 1);
      if constexpr (!C::I8) {
        if (scan_v & bit) {  // a NaN or an infinity times the weight 0 of a row that does not see it would be NaN
          const int c = lt % C::PIECES;
          bool bad = false;
          for (int row = lt / C::PIECES; row < kTile; row += 128 / C::PIECES) {
            const uint32_t p = ring + done.s * C::TILE + (c / 8) * C::HALF + row * 128 + ((c % 8) ^ (row % 8)) * 16;
            uint4 u;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(p) : "memory");
            if (not_finite<T>(u)) { sts_u4(p, u.x, u.y, u.z, u.w); bad = true; }
          }
          if (bad) *(volatile int*)&poison[scan_item >> (4 * (pending - 1)) & 7] = 1;
        }
      }
      async_proxy_fence();
      __syncwarp();
      if (lane == 0) {
        if (with_q & bit) mbar_arrive(&bars.q_full);
        mbar_arrive(&bars.full[done.s]);
      }
      with_q &= ~bit;
      scan_v &= ~bit;
      --pending;
      done.advance(ST);
    };
    constexpr int kDepth = 3;  // copies in flight while the next one is issued
    auto committed = [&](bool q, bool scan) {
      asm volatile("cp.async.commit_group;" ::: "memory");
      with_q = with_q << 1 | (q ? 1u : 0u);
      scan_v = scan_v << 1 | (scan ? 1u : 0u);
      scan_item = scan_item << 4 | (uint32_t)(item & 7);
      ++pending;
      if (pending > kDepth) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth) : "memory");
        hand_over();
      }
    };

    // Waits for a barrier; copies that have arrived meanwhile are handed over first, since what frees the barrier may need them.
    auto acquire = [&](uint64_t* bar, uint32_t phase) {
      while (pending > 0 && !__any_sync(0xffffffffu, mbar_test(bar, phase))) {
        switch (pending) {
          case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
          case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
          default: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        }
        hand_over();
      }
      return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase, a.err, kWaitLoad, kSpin));
    };

    while (x.next(w, a.c.kv_heads, pt)) {
      if (lt == 0) *(volatile int*)&poison[item & 7] = 0;
      // rows of Q
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = lt + 128 * i, flat = pt.t * kRows + row, token = flat / G;
        q_at[row] = row < pt.rows ? (uint32_t)(((int64_t)(pt.q0 + token) * a.q_token + (int64_t)(x.head * G + flat - token * G) * a.q_head) / 8) : 0xffffffffu;
      }
      if (item > 0) {
        ok = ok && acquire(&bars.q_empty, q_phase);
        q_phase ^= 1;
      }
      sync();
      if (ok) {
        const int c = lt % C::PIECES;
        for (int row = lt / C::PIECES; row < (pt.rows + 127) / 128 * 128; row += 128 / C::PIECES) {
          const uint32_t at = q_at[row];
          const bool live = at != 0xffffffffu && c * 8 < a.head_size;
          cp_async16(q_smem + (row / 128) * C::TILE + (c / 8) * C::HALF + (row % 128) * 128 + ((c % 8) ^ (row % 8)) * 16,
                     live ? static_cast<const T*>(a.q) + (int64_t)at * 8 + c * 8 : static_cast<const T*>(a.q), live);
        }
      }
      // page of token `lt` of a tile, fetched a tile ahead
      int block = -1, off = -1;
      auto look_up = [&](int k) {
        off = -1;
        if (k >= x.k1) return;
        const int pos = (pt.first + k) * kTile + lt;
        if (pos < pt.lo || pos >= pt.hi) return;
        const int page = a.c.page_of(pos);
        off = pos - page * a.c.block_size;
        block = a.c.tables[pt.b * a.c.table_stride + page];
      };
      look_up(x.k0);
      // its scales, fetched a conversion ahead of their use
      float ks = 0.f, vs = 0.f;
      auto look_scales = [&]() {
        ks = vs = 0.f;
        if (MODE == kScaleToken && off >= 0 && (uint32_t)block < (uint32_t)a.c.num_blocks) {
          const int64_t at = ((int64_t)block * a.c.block_size + off) * a.c.kv_heads + x.head;
          ks = a.c.k_scale[at];
          vs = a.c.v_scale[at];
        }
      };
      // where the rows of tile k are, and what the softmax needs to know of them
      auto prepare = [&](int k) {
        const bool known = (uint32_t)block < (uint32_t)a.c.num_blocks, here = off >= 0 && known;
        if (off >= 0 && !known) report(a.err, MCOP_DEVERR_SLOT);
        row_at[buf][lt] = here ? (uint32_t)block * block16 + (uint32_t)off * page16 + (uint32_t)x.head * head16 : 0xffffffffu;
        Info& in = info[inf.s];
        const uint32_t word = __ballot_sync(0xffffffffu, here);
        if constexpr (MODE == kScaleToken) {
          const float top = warp_max(fabsf(vs) <= FLT_MAX ? fabsf(vs) : 0.f);
          const bool wild = __any_sync(0xffffffffu, !(fabsf(vs) <= FLT_MAX));
          const bool odd = __any_sync(0xffffffffu, !(ks >= 0.f && ks <= FLT_MAX));
          const float ktop = warp_max(ks >= 0.f && ks <= FLT_MAX ? ks : 0.f);
          if (lane == 0) {
            vmax[buf][lwarp] = wild ? -1.f - top : top;
            kmax[buf][lwarp] = odd ? -1.f : ktop;
          }
        }
        const bool sound = sync_and(off < 0 || known);
        if constexpr (MODE == kScaleToken) {
          float top = 0.f;
          bool wild = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = vmax[buf][i];
            wild |= v < 0.f;
            top = fmaxf(top, v < 0.f ? -1.f - v : v);
          }
          const float ktop = fmaxf(fmaxf(kmax[buf][0], kmax[buf][1]), fmaxf(kmax[buf][2], kmax[buf][3])), klow = fminf(fminf(kmax[buf][0], kmax[buf][1]), fminf(kmax[buf][2], kmax[buf][3]));
          if (lt == 0) {
            in.wild = wild;
            in.odd = klow < 0.f;
            in.kmax = ktop * (a.scale * kLog2e) * (1.f + 0x1p-20f);
            in.power = scale_power(top);
          }
          in.ks[lt] = ks * (a.scale * kLog2e);
          in.vs[lt] = vs;
        }
        if (lane == 0) {
          in.here[lwarp] = word;
          if (lwarp == 0) in.all = sound ? 1 : 0;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.info_full[inf.s]);
        inf.advance(C::NI);
        look_up(k + 1);
      };
      if constexpr (!C::I8) {
        const Common common = seen_by_all(a, pt, G);
        for (int k = x.k0; k < x.k1; ++k) {
          prepare(k);
          const int base = (pt.first + k) * kTile;
          const bool scan = !common.whole(base);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const char* src = kv ? vbase : kbase;
            ok = ok && acquire(&bars.empty[st.s], st.phase ^ 1);
            if (!ok) continue;
            const uint32_t dst = ring + st.s * C::TILE;
            const int c = lt % C::PIECES;
#pragma unroll
            for (int i = 0; i < kTile * C::PIECES / 128; ++i) {
              const int row = lt / C::PIECES + i * (128 / C::PIECES);
              const uint32_t at = row_at[buf][row];
              const bool live = at != 0xffffffffu && c < row_pieces;
              cp_async16(dst + (c / 8) * C::HALF + row * 128 + ((c % 8) ^ (row % 8)) * 16, live ? src + (uint64_t)at * 16 + c * 16 : src, live);
            }
            st.advance(ST);
            committed(kv == 0 && k == x.k0, kv == 1 && scan);
          }
          buf ^= 1;
        }
      } else {
        // int8 rows come by asynchronous copy, a tile ahead of the conversion; a thread converts the pieces that it has copied
        constexpr int IP = DP / 16, N = kTile * IP / 128;  // 16-byte pieces of a row; pieces per thread
        const int c = lt % IP;
        auto fetch = [&](int kv) {  // K (0) or V (1) of the tile prepared last
          const char* src = kv ? vbase : kbase;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t at = row_at[buf][lt / IP + i * (128 / IP)];
            const bool live = at != 0xffffffffu && c < row_pieces;
            cp_async16(rawbuf + kv * (kTile * DP) + (i * 128 + lt) * 16, live ? src + (uint64_t)at * 16 + c * 16 : src, live);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto convert = [&](auto which, bool with_q) {
          constexpr int kv = decltype(which)::value;
          ok = ok && acquire(&bars.empty[st.s], st.phase ^ 1);
          if (!ok) return;
          const uint32_t dst = ring + st.s * C::TILE, from = rawbuf + kv * (kTile * DP) + lt * 16;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int row = lt / IP + i * (128 / IP);
            uint32_t wd[4], y[8];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(wd[0]), "=r"(wd[1]), "=r"(wd[2]), "=r"(wd[3]) : "r"(from + i * 2048) : "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t p = __byte_perm(wd[j], 0, 0x4140), q = __byte_perm(wd[j], 0, 0x4342);
              y[2 * j] = kv ? codes.template two<VT>(p) : codes.template two<T>(p);
              y[2 * j + 1] = kv ? codes.template two<VT>(q) : codes.template two<T>(q);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int piece = 2 * c + h;
              sts_u4(dst + (piece / 8) * C::HALF + row * 128 + ((piece % 8) ^ (row % 8)) * 16, y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]);
            }
          }
          async_proxy_fence();
          __syncwarp();
          if (lane == 0) {
            if (with_q) mbar_arrive(&bars.q_full);
            mbar_arrive(&bars.full[st.s]);
          }
          st.advance(ST);
        };
        look_scales();
        prepare(x.k0);
        if (ok) {
          fetch(0);  // (Q is in the same group)
          fetch(1);
        }
        for (int k = x.k0; k < x.k1; ++k) {
          const bool more = k + 1 < x.k1;
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          look_scales();
          convert(std::integral_constant<int, 0>{}, k == x.k0);
          buf ^= 1;
          if (more) {
            prepare(k + 1);
            if (ok) fetch(0);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
          } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
          }
          convert(std::integral_constant<int, 1>{}, false);
          if (more && ok) fetch(1);
        }
      }
      ++item;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (!C::I8) {
      while (pending > 0) hand_over();
    }
  } else {
    // ------------------------------------------------------------------------------------------ the MMAs
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 12) {
      // The whole warp walks the loop and one elected thread issues: in uniform code the descriptors live in uniform registers, which
      // the instruction takes (from a single thread's registers it took 100 cycles to issue a product of 64).
      constexpr uint32_t kAll = 0xffffffffu;
      uint32_t q_smem = smem;
      asm volatile("" : "+r"(q_smem));
      q_smem = __reduce_max_sync(kAll, q_smem);
      const uint32_t at = __reduce_max_sync(kAll, tmem), ring = q_smem + 2 * C::TILE;
      constexpr uint32_t QK = f16_idesc(ElemTraits<T>::code == MCOP_BF16, 128, kTile, false);
      constexpr uint32_t PV = f16_idesc(ElemTraits<VT>::code == MCOP_BF16, 128, DP, true);
      Ring st;
      uint32_t q_phase = 0, p_phase[2] = {0, 0}, oe_phase[2] = {1, 1};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t phase) {
        // (polled: a suspended thread wakes late, and everything waits for this one)
        uint32_t tries = 0;
        while (ok && !__all_sync(kAll, mbar_test(bar, phase))) {
          if (++tries == kPolls) {
            report(a.err, kWaitMma);
            ok = false;
          }
        }
        tc_fence_after();
        return ok;
      };
      const uint32_t q_low = desc_low(q_smem, 16), k_low = desc_low(ring, 16), v_low = desc_low(ring, C::HALF);
      auto logits = [&](int tile, int stage) {
        const uint32_t q = q_low + tile * (C::TILE / 16), k = k_low + stage * (C::TILE / 16);
        static_for<DP / 16>([&](auto i) {
          constexpr uint32_t off = (i.value / 4) * C::HALF + (i.value % 4) * 32;
          tc_mma_ss<QK, off, off>(at + tile * 128, q, k, i.value > 0);
        });
        tc_commit(&bars.s_full[tile]);
      };
      auto values = [&](auto half, int tile, int stage, bool more) {
        const uint32_t v = v_low + stage * (C::TILE / 16);
        static_for<kTile / 32>([&](auto j) {
          constexpr int i = half.value * (kTile / 32) + j.value;
          tc_mma_ts<PV, 8 * i, 2048 * i>(at + 256 + tile * DP, at + tile * 128, v, more || i > 0);
        });
      };
      while (ok && __any_sync(kAll, x.next(w, a.c.kv_heads, pt))) {
        const int two = 1 + (int)__reduce_max_sync(kAll, pt.rows > 128), n = __reduce_max_sync(kAll, x.k1 - x.k0);
        if (!wait(&bars.q_full, q_phase)) break;
        q_phase ^= 1;
        if (!wait(&bars.full[st.s], st.phase)) break;
        for (int t = 0; t < two; ++t) logits(t, st.s);
        tc_commit(&bars.empty[st.s]);
        if (n == 1) tc_commit(&bars.q_empty);
        st.advance(ST);
        for (int k = 0; k < n && ok; ++k) {
          Ring v = st;
          st.advance(ST);
          const bool last = k + 1 == n;
          if (!wait(&bars.full[v.s], v.phase)) break;
          for (int t = 0; t < two && ok; ++t) {
            if (!wait(&bars.p_half[t], p_phase[t])) break;
            if (k == 0) {  // the item before has left O
              if (!wait(&bars.o_empty[t], oe_phase[t])) break;
              oe_phase[t] ^= 1;
            }
            values(std::integral_constant<int, 0>{}, t, v.s, k > 0);
            if (!wait(&bars.p_full[t], p_phase[t])) break;
            p_phase[t] ^= 1;
            values(std::integral_constant<int, 1>{}, t, v.s, true);
            if (last) tc_commit(&bars.o_full[t]);
            else {
              if (t == 0 && !wait(&bars.full[st.s], st.phase)) break;
              logits(t, st.s);
            }
          }
          if (!ok) break;
          if (last && two == 1) {  // the other tile has no rows in this item: its warps only hear that it is over
            if (!wait(&bars.o_empty[1], oe_phase[1])) break;
            oe_phase[1] ^= 1;
            tc_commit(&bars.o_full[1]);
          }
          tc_commit(&bars.empty[v.s]);
          if (!last) {
            tc_commit(&bars.empty[st.s]);
            if (k + 2 == n) tc_commit(&bars.q_empty);
            st.advance(ST);
          }
        }
      }
      // whatever is still running must not outlive the CTA's tensor memory
      tc_commit(&bars.drain);
      (void)mbar_wait_bounded(&bars.drain, 0, a.err, kWaitMma, kSpin);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_free_all(tmem);
}

// Joins the partial results of the items that cross CTA borders: CTA c of the kernel above holds the first part of at most one such
// item, the CTAs behind it one part each.  blockIdx.y: 16 rows; a thread takes four elements of one row at a time.
template <typename T, int DP> __global__ void __launch_bounds__(512) chunk_join_kernel(AttnArgs a, Layout w) {
  pdl_launch_dependents();
  pdl_wait();
  const Rec rec = w.recs[blockIdx.x];
  if (rec.count == 0) return;
  const int G = a.q_heads / a.c.kv_heads, d = threadIdx.x % (DP / 4) * 4;
  const Seq s = sequence(a, rec.b);
  auto part = [&](int i) { return w.parts + (int64_t)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * (kRows * (DP + 2)); };
  for (int i = threadIdx.x / (DP / 4); i < 16; i += 2048 / DP) {
    const int row = blockIdx.y * 16 + i, flat = rec.t * kRows + row, token = flat / G, head = rec.head * G + flat - token * G;
    if (token >= s.qn) return;
    float top = -INFINITY;
#pragma unroll 4
    for (int p = 0; p < rec.count; ++p) top = fmaxf(top, part(p)[kRows * DP + 2 * row]);
    const float safe = top == -INFINITY ? 0.f : top;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int p = 0; p < rec.count; ++p) {
      const float2 ml = *reinterpret_cast<const float2*>(part(p) + kRows * DP + 2 * row);
      const float4 v = *reinterpret_cast<const float4*>(part(p) + row * DP + d);
      const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_approx(ml.x - safe);
      sum = __fmaf_rn(f, ml.y, sum);
      x.x = __fmaf_rn(f, v.x, x.x);
      x.y = __fmaf_rn(f, v.y, x.y);
      x.z = __fmaf_rn(f, v.z, x.z);
      x.w = __fmaf_rn(f, v.w, x.w);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    if (d < a.head_size)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.q0 + token) * a.o_token + (int64_t)head * a.o_head + d) =
          make_uint2(pack2<T>(x.x * f, x.y * f), pack2<T>(x.z * f, x.w * f));
    if (a.lse && d == 0) a.lse[(int64_t)(s.q0 + token) * a.q_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
}

template <typename T, int MODE, int DP> int launch_one(const AttnArgs& a, void* ws, cudaStream_t st) {
  using C = Cfg<T, MODE, DP>;
  const char* what = "paged_attention_chunk";
  auto kernel = chunk_kernel<T, MODE, DP>;
  if (cudaError_t e = ensure_dynamic_smem((const void*)kernel, C::SMEM); e != cudaSuccess) return set_error(MCOP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  const int grid = sm_count(), G = a.q_heads / a.c.kv_heads;
  Layout w;
  layout((char*)ws, a.tokens, a.batch, G, DP, grid, &w);
  launch_pdl(chunk_plan_kernel, dim3(1), dim3(1024), 0, st, a, w, max_tiles(a.tokens, a.batch, G), grid);
  if (int rc = check_launch(what)) return rc;
  launch_pdl(kernel, dim3(grid), dim3(kThreads), C::SMEM, st, a, w);
  if (int rc = check_launch(what)) return rc;
  launch_pdl(chunk_join_kernel<T, DP>, dim3(grid, kRows / 16), dim3(512), 0, st, a, w);
  return check_launch(what);
}

template <typename T, int MODE> int launch_mode(const AttnArgs& a, void* ws, cudaStream_t st) {
  return a.head_size <= 64 ? launch_one<T, MODE, 64>(a, ws, st) : launch_one<T, MODE, 128>(a, ws, st);
}
template <typename T> int launch_type(const AttnArgs& a, void* ws, cudaStream_t st) {
  if (a.scale_mode == kScaleNone) return launch_mode<T, kScaleNone>(a, ws, st);
  return a.scale_mode == kScaleHead ? launch_mode<T, kScaleHead>(a, ws, st) : launch_mode<T, kScaleToken>(a, ws, st);
}

}  // namespace

size_t chunk_workspace(int64_t tokens, int batch, int q_heads, int kv_heads, int head_size) {
  return layout(nullptr, tokens, batch, q_heads / kv_heads, head_size <= 64 ? 64 : 128, sm_count(), nullptr);
}

int launch_chunk(const AttnArgs& a, int dtype, void* ws, size_t ws_bytes, cudaStream_t st) {
  const char* what = "paged_attention_chunk";
  MCOP_REQUIRE(ws && aligned16(ws) && ws_bytes >= chunk_workspace(a.tokens, a.batch, a.q_heads, a.c.kv_heads, a.head_size), MCOP_ERR_WORKSPACE,
               "%s: workspace missing, misaligned or too small", what);
  const double span = (double)a.tokens * a.q_token + (double)a.q_heads * a.q_head;
  MCOP_REQUIRE(a.q_token >= 0 && a.q_head >= 0 && span < 0x1p34, MCOP_ERR_UNSUPPORTED, "%s: a query that spans more than 2^34 elements", what);
  return dtype == MCOP_BF16 ? launch_type<__nv_bfloat16>(a, ws, st) : launch_type<__half>(a, ws, st);
}

}  // namespace mcop
