// Decode attention over the 4-bit paged KV cache (format: kv4.cuh).
//
//   out[b][h] = sum_t softmax_t(scale q.k_t) v_t,  k_t = s n (4 groups of 32 dims)
//
// The floor is 144 bytes per (token, kv head) from HBM.  At that rate an SM
// has about 400 cycles per 64 tokens, in which it expands 16384 codes: that,
// not the memory, is what bounds the kernel (with the arithmetic taken out
// 256 rows take 110 us).
//
// Measured (B200, bf16 q, replayed from a graph; floor at a copy's 6.45 TB/s):
// 256 rows of 512..4096 tokens at 16/8 heads 120 us (5.7 TB/s, floor 106; called
// one by one over changing inputs 131); 256 of 1024..2047 at 64/8 heads 96 us
// (floor 71); 40 of 1..3001 at 64/8 heads 28.4 us (floor 10); 1 row of 40960 at
// 32/8 heads 20 us (floor 7.3), of 333 at 16/8 6.2 us: a launch, the plan and the
// merge are about 6 us of each.
//
// Work: the kernel is persistent, one CTA per SM of 8 warps that compute and 8
// that load, grouped into teams of T = 1, 2, 4 or 8.  An item is one (row, kv
// head), a unit a round of T tiles of 64 tokens of an item, one for each warp
// of a team.  Every CTA counts the batch's units itself from seqlens and takes
// the T of the least estimated time (large T: few partials to merge; small T:
// no round that is not full, no waiting); the units are cut into equal runs,
// one per team, whatever the rows' lengths are.  A run that ends inside an
// item leaves an fp32 partial (max, sum, O); the last team of the item to
// arrive merges the partials in order.
//
// Tiles: each computing warp has a loading warp and two stages of a K and a V
// record, filled by bulk copies: warps never wait for one another but at the
// end of a team's item.  The tiles' block ids are fetched by the loading
// warps, 32 at a time; with their registers handed over (216 and 40 of the 128
// at launch) the whole tile is straight-line code without spills.  Where this
// took 131 us for 256 rows, others took: 16 warps that load for themselves and
// work on halves of a tile in a rolled loop 141; 8 that load for themselves
// 138; 12 that compute and 4 that load 157, with three records each and 152
// registers; a third stage 131; Q.K of the next tile between P.V of this one
// 156.
//
// Q.K: the tokens are the rows of m16n8k16's A operand, the G <= 8 query heads
// its 8 columns.  Fewer heads share the columns out: with a column each, a lane
// would take the exponentials of two columns, empty or not, for all tokens
// (256 rows at two heads 130 us, against 124 with four columns a head).  m16n8k32
// on e4m3, where codes are operands as they are, is no way: it takes four times
// as long as this one.  With all else masked off, four bits at the foot of an fp16
// are the subnormal 2^-24 u, or 2^-20 u one nibble higher, and the tensor
// cores take subnormals as they are: an AND makes two operands.  The 2^24 is
// put right in the softmax scale, the 16 in q, and the offset of 8 through the
// accumulator's start, -8 sum(q) of the group; the group's scale multiplies
// the fp32 sum.  q is scaled by a power of two per head to a largest element
// in [2^14, 2^15), so that bf16 values go into fp16 unrounded down to 2^-27 of
// the largest.  Items with smaller ones, or with q or a softmax scale for which
// fp32 has no room, take the second path below.
// P.V: O^T = V^T P^T with V^T (dims x tokens) as the A operand.  Here the sum
// over thousands of tokens would cancel against its offset, so u - 8 is made
// exactly, by one more fp16x2 add or fma.  P^T is 2^kUp p in fp16, p <= 2^kLag,
// transposed in registers and multiplied by the V scales of its two tokens in
// fp16: two roundings of 2^-11, a quarter of what one to bf16 costs.  The
// scales are held relative to 2^(e + 1), the largest so far being in
// [2^e, 2^(e + 1)), and are exact down to 2^-kSpan of that.  Once per tile each
// lane turns the scales of its two tokens into such pairs.
//
// fp16 ends 2^-40 below its largest number: in P, and in the product with a
// scale, up to 2^-25 is lost, 2^-(24 + kUp) 2^(e + 1) of a token's p s.  That
// matters where the tokens of most of the probability have the small scales.
// When the softmax reference was set, its token had p = 1 and a scale of at
// least 2^low, the smallest in that tile, so that D = sum p s >= 2^low from then
// on, and n tiles of 64 tokens lose at most 2^-16 D while
// n <= 2^(kUp + 1 + low - e): 2^7 tiles, 8192 tokens of one warp, for scales
// within 2^6 of one another.  Later tiles, and tiles with a scale below
// 2^-kSpan of the largest (zero among others) or a NaN, take a second path:
// codes and q in bf16, no product rounded; p s in fp32, cut into two bf16 that
// two MMAs add up.  O is held relative to the largest scale and q to its
// largest element, so that what lies 2^-100 below them still counts in full.  A
// tile takes 3.6 times as long on it, in loops that are rolled so that the first
// path keeps its registers (256 rows with one token in 16 at 2^-20 of the
// others: 433 us, without 119; with the loops unrolled, or in a function of its
// own, 256 x 1500 at 64/8 heads take 99 or 105 us on the first path, and so 96).
#include <cuda_fp16.h>

#include <type_traits>

#include "host.h"
#include "kv4.cuh"

namespace aacc {

constexpr int kAttWarps = 8;
constexpr int kSizes = 4;   // team sizes: 1, 2, 4, 8 warps
constexpr int kStages = 2;  // tiles of K and V that a warp has in hand or in flight
constexpr int kAttThreads = 2 * kAttWarps * 32;  // as many warps again load
constexpr int kPlanWarps = kAttThreads / 32;
constexpr int kLag = 3;           // the softmax reference follows a score that passes it by more than 2^kLag
constexpr int kUp = 15 - kLag;    // P is held times 2^kUp: at most 2^15 in fp16
constexpr int kSpan = 16;         // powers of two that V scales in fp16 may lie below the largest
constexpr int kRoom = kUp + 1;    // see kv4_room
constexpr int kNone = -512;       // instead of an exponent: no tile has room
// less `from` and a scale: bits 15 and 31 where the scale is below 2^(ev + 1)
constexpr uint32_t kUpTo = (0x807fu + 0x8000u + (kSpan << 7)) * 0x10001u;

// A run of tiles [t0, t1) of item (b, h), whose row has n tiles; u is the unit number of t0.
struct Kv4Seg {
  uint32_t u;
  int b, row, h, n, t0, t1, ctx;
};

template <int G>
struct Kv4Smem {
  uint8_t kv[kAttWarps][kStages][2][kKv4Record];
  uint4 vpair[kAttWarps][32];  // V scales of tokens 2 i and 2 i + 1, fp16 pairs of groups 0..3
  float red_o[kAttWarps][G][128];
  float red_ml[kAttWarps][G][2];
  int first_b[kAttWarps];       // per team: the first row of the thread that holds its first unit,
  uint32_t first_u[kAttWarps];  // and the unit that row starts at
  int row[kAttThreads];       // of batches up to kAttThreads rows
  int ctx[kAttThreads];
  uint32_t wsum[kSizes + 1][kPlanWarps];
  uint32_t sum[kSizes + 1];
  uint32_t plan[3];  // log2 T, units, units per run
  uint64_t full[kAttWarps][kStages];
  uint64_t empty[kAttWarps][kStages];
  uint32_t merge_k[kAttWarps][2];  // per team and shared item: first run, and
  int merge_n[kAttWarps][2];       // the number of runs if this one came last, else 0
  int abort;
};

struct Kv4Args {
  const bf16* q;
  bf16* out;
  const uint8_t* kc;
  const uint8_t* vc;
  const int32_t* bt;
  const int64_t* rows;
  const int32_t* seqlens;
  unsigned* cnt;  // [teams], zero between calls
  float* ws_o;    // [2 * teams][G][128]
  float* ws_ml;   // [2 * teams][G][2]
  unsigned* err;
  int64_t max_blocks;
  int num_blocks, num_rows, batch, max_ctx, ctx_add, Hkv, tpb;  // tpb: tiles per block
  float scale;
};

// Tokens of batch row b (0: padding, outside the tables, or empty).
__device__ __forceinline__ int kv4_ctx(const Kv4Args& a, int b, int* row, unsigned* err = nullptr) {
  const int64_t r = a.rows[b];
  *row = (int)r;
  if (r < 0 || r >= a.num_rows) {
    if (r >= 0) report(err, ERR_SLOT_OOB);
    return 0;
  }
  const int64_t c = (int64_t)a.seqlens[r] + a.ctx_add;
  if (c > a.max_ctx) report(err, ERR_CTX_OOB);
  return (int)max((int64_t)0, min(c, (int64_t)a.max_ctx));
}

__device__ __forceinline__ int tiles_of(int ctx) { return (int)(((unsigned)ctx + kKv4Tile - 1) / kKv4Tile); }

template <int G>
__device__ __forceinline__ void kv4_row(const Kv4Args& a, const Kv4Smem<G>& sm, Kv4Seg& s) {
  if (a.batch <= kAttThreads) {
    s.ctx = sm.ctx[s.b];
    s.row = sm.row[s.b];
  } else {
    s.ctx = kv4_ctx(a, s.b, &s.row);
  }
  s.n = tiles_of(s.ctx);
}

// Tiles of a segment that starts at t0 with `units` units left in its run.
__device__ __forceinline__ int seg_end(int n, int t0, uint32_t units, int tsh) {
  return (int)min((uint64_t)n, (uint64_t)t0 + ((uint64_t)units << tsh));
}

// The run's next segment; false when the run is over.
template <int G>
__device__ __forceinline__ bool kv4_next(const Kv4Args& a, const Kv4Smem<G>& sm, Kv4Seg& s, uint32_t uend, int tsh) {
  s.u += (uint32_t)(s.t1 - s.t0 + (1 << tsh) - 1) >> tsh;
  if (s.u >= uend) return false;
  if (++s.h == a.Hkv) {  // within a run only its end cuts an item short
    s.h = 0;
    do {
      ++s.b;
      kv4_row(a, sm, s);
    } while (s.n == 0);
  }
  s.t0 = 0;
  s.t1 = seg_end(s.n, 0, uend - s.u, tsh);
  return true;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// 8x8 transpose of b16 values over the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// d = a b + c, where c holds for both rows of a column pair.
__device__ __forceinline__ void mma_f16_16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                                   float c0, float c1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t mul_f16(uint32_t x, uint32_t y) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Bits 0-3 (HI: 4-7) of both halves of x, a code u each: as fp16 subnormals 2^-24 u (HI: 2^-20 u).
template <bool HI>
__device__ __forceinline__ uint32_t code_sub(uint32_t x) {
  return x & (HI ? 0x00f000f0u : 0x000f000fu);
}

// The same as the fp16 pair (u - 8, u' - 8), through 1024 + u or 1024 + 16 u.
template <bool HI>
__device__ __forceinline__ uint32_t code(uint32_t x) {
  const uint32_t y = and_or<HI ? 0x00f000f0u : 0x000f000fu>(x, 0x64006400u);
  const __half2 h = *reinterpret_cast<const __half2*>(&y);
  const __half2 r = HI ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-72.f))
                       : __hadd2(h, __float2half2_rn(-1032.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Bits 0-3 of both halves of x as the bf16 pair (u - 8, u' - 8), through 128 + u.
__device__ __forceinline__ uint32_t code_bf16(uint32_t x) {
  const uint32_t y = and_or<0x000f000fu>(x, 0x43004300u);
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&y), __float2bfloat162_rn(-136.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Power of two by which the second path multiplies q: the softmax scale's if that is below 1, and less where q's
// largest element (bf16 bits mx) would pass 2^101.
__device__ __forceinline__ int kv4_q_exp(float scale, uint32_t mx) {
  const int e = (int)(__float_as_uint(fabsf(scale) * kLog2e) >> 23) - 127;
  return min(min(max(e, -120), 0), 227 - (int)(mx >> 7));
}

// Tiles that may hold p s in fp16 (see the head of the file) for the largest V scale in [2^ev, 2^(ev + 1)) and none
// below 2^low where the softmax reference was set.
__device__ __forceinline__ int kv4_room(int ev, int low) {
  const int d = ev - low;
  return d > kRoom ? 0 : 1 << (kRoom - max(d, 0));
}

// bf16 pair W / 2 of `p`, member W % 2, as fp32.
template <int W>
__device__ __forceinline__ float scale_of(uint2 p) {
  const uint32_t x = W < 2 ? p.x : p.y;
  return __uint_as_float((W & 1) ? x & 0xffff0000u : x << 16);
}

// All lanes' bounded wait; the first try is the common case.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* err, volatile int* abort) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, abort));
}

__device__ __forceinline__ void team_sync(int team, int tsh) {
  if (tsh == 0)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(32 << tsh) : "memory");
}

// How a warp shares out sums of partial results: VW dims a lane, 4 at a time, so GS lanes to a head.
// Several heads to a warp (VW 8, 16) have their loads in flight together.
template <int VW>
struct Kv4Share {
  static constexpr int GS = 128 / VW;
  static constexpr int P = VW / 4;  // pieces
  int hd, d;                        // head; the first piece's first dim
  __device__ __forceinline__ Kv4Share(int i, int lane) : hd(i * (32 / GS) + lane / GS), d(lane % GS * 4) {}
  template <class Load>
  __device__ __forceinline__ void read(const float* head, float (&y)[VW], Load load) const {
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const float4 v = load(reinterpret_cast<const float4*>(head + d + q * GS * 4));
      y[4 * q] = v.x, y[4 * q + 1] = v.y, y[4 * q + 2] = v.z, y[4 * q + 3] = v.w;
    }
  }
  __device__ __forceinline__ void write(float* head, const float (&y)[VW]) const {
#pragma unroll
    for (int q = 0; q < P; ++q)
      *reinterpret_cast<float4*>(head + d + q * GS * 4) =
          make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
  }
  __device__ __forceinline__ void write(bf16* head, const float (&y)[VW], float l) const {
    const float inv = 1.f / l;
#pragma unroll
    for (int q = 0; q < P; ++q)
      *reinterpret_cast<uint2*>(head + d + q * GS * 4) =
          make_uint2(pack_bf16(y[4 * q] * inv, y[4 * q + 1] * inv), pack_bf16(y[4 * q + 2] * inv, y[4 * q + 3] * inv));
  }
};

// Sum of `count` partial results (max, sum, O) of this lane's head, weighted 2^max: ml(p) gives (max, sum),
// o(p, y) this lane's dims.  Each of the head's lanes weighs one part, so all loads are independent.
template <int VW, class ML, class OF>
__device__ __forceinline__ void kv4_combine(int count, int lane, ML ml, OF o, float& M, float& L, float (&O)[VW]) {
  constexpr int GS = Kv4Share<VW>::GS;
  const int gl = lane % GS, g0 = lane - gl;
  M = -INFINITY;
  L = 0.f;
#pragma unroll
  for (int i = 0; i < VW; ++i) O[i] = 0.f;
  for (int p0 = 0; p0 < count; p0 += GS) {
    const int n = min(GS, count - p0);
    float2 x = make_float2(-INFINITY, 0.f);
    if (gl < n) x = ml(p0 + gl);
    float y0[2][VW];  // the first two parts' O set out with the weights
    o(p0, y0[0]);
    o(p0 + min(1, n - 1), y0[1]);
    float top = x.x;
#pragma unroll
    for (int d = 1; d < GS; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    top = fmaxf(M, top);
    const float u = top == -INFINITY ? 0.f : top;
    const float f = ex2(x.x - u), keep = ex2(M - u);
    M = top;
    float l = x.y * f;
#pragma unroll
    for (int d = 1; d < GS; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    L = L * keep + l;
#pragma unroll
    for (int i = 0; i < VW; ++i) O[i] *= keep;
    const float w0 = __shfl_sync(0xffffffffu, f, g0), w1 = __shfl_sync(0xffffffffu, f, g0 + 1);
#pragma unroll
    for (int i = 0; i < VW; ++i) O[i] = fmaf(w0, y0[0][i], n > 1 ? fmaf(w1, y0[1][i], O[i]) : O[i]);
#pragma unroll(32 / VW)
    for (int p = 2; p < n; ++p) {
      const float w = __shfl_sync(0xffffffffu, f, g0 + p);
      float y[VW];
      o(p0 + p, y);
#pragma unroll
      for (int i = 0; i < VW; ++i) O[i] = fmaf(w, y[i], O[i]);
    }
  }
}

// f(VW) for a team of T warps and G heads: a head to a warp, or as many as it takes.  (A head cut over several
// warps was slower: every warp has to fetch all the parts' weights, 16 rows of 40960 at 8/8 heads 131 -> 124 us.)
template <int G, class F>
__device__ __forceinline__ void kv4_share(int T, F f) {
  if (T >= G)
    f(std::integral_constant<int, 4>{});
  else if (2 * T == G || G == 2)
    f(std::integral_constant<int, G >= 2 ? 8 : 4>{});
  else
    f(std::integral_constant<int, G >= 4 ? 16 : 4>{});
}

template <int G>
__global__ void __launch_bounds__(kAttThreads, 1) kv4_decode_kernel(const Kv4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Kv4Smem<G>& sm = *reinterpret_cast<Kv4Smem<G>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  if (lane == 0 && warp < kAttWarps) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[warp][i], 1);
      mbar_init(&sm.empty[warp][i], 1);
    }
    fence_mbar_init();
  }
  if (threadIdx.x <= kSizes) sm.sum[threadIdx.x] = 0;
  if (threadIdx.x == 0) sm.abort = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch();

  // ---- count the batch's units for every team size: each thread sums a run of rows, then the CTA
  const int per = (a.batch + kAttThreads - 1) / kAttThreads;
  const int b_lo = min(a.batch, (int)threadIdx.x * per), b_hi = min(a.batch, b_lo + per);
  uint32_t cnt[kSizes + 1] = {};  // [kSizes]: rows with tokens
  for (int b = b_lo; b < b_hi; ++b) {
    int row;
    const int ctx = kv4_ctx(a, b, &row, blockIdx.x == 0 ? a.err : nullptr);
    if (per == 1) {
      sm.ctx[b] = ctx;
      sm.row[b] = row;
    }
#pragma unroll
    for (int i = 0; i < kSizes; ++i) cnt[i] += (uint32_t)(tiles_of(ctx) + (1 << i) - 1) >> i;
    cnt[kSizes] += ctx > 0;
  }
  if (warp * 32 * per < a.batch) {
    uint32_t x = 0;  // lane i: counter i over the warp
#pragma unroll
    for (int i = 0; i <= kSizes; ++i) {
      const uint32_t y = __reduce_add_sync(0xffffffffu, cnt[i]);
      x = lane == i ? y : x;
    }
    if (lane <= kSizes) {
      sm.wsum[lane][warp] = x;
      if (x) atomicAdd(&sm.sum[lane], x);
    }
  }
  __syncthreads();
  // Lane i weighs T = 2^i, in units of a model fitted to runs of 24 shapes with each T (B200; on average within 2 %
  // of the best T, at most 11 %; T = 1, 2, 4 or 8 for all would cost 112, 28, 13 or 19 % on average): 3 for a round of
  // tiles; for each segment of a run 0.14 per head and warp that meets the first; where items are shared, 1.2, and
  // for each part of an item 0.93 and 0.25 for each of the heads that a warp adds.
  if (warp == 0) {
    const int opt = min(lane, kSizes - 1);
    const uint32_t n = sm.sum[opt] * a.Hkv, teams = gridDim.x * (kAttWarps >> opt);
    const uint32_t c = max((n + teams - 1) / teams, 1u);
    const float t = (float)(1 << opt), ch = (float)c;
    const float per_item = __fdividef((float)n, (float)max(sm.sum[kSizes] * a.Hkv, 1u));
    float cost = 3.f * ch + 0.14f * G * (t - 1.f) * (1.f + __fdividef(ch, fmaxf(per_item, 1.f)));
    if (per_item > ch) cost += 1.2f + __fdividef(per_item, ch) * (0.93f + __fdividef(0.25f * G, fminf(t, (float)G)));
    const uint32_t best = __reduce_min_sync(0xffffffffu, (__float_as_uint(cost) & ~7u) | opt) & 7u;
    if (lane == best) {
      sm.plan[0] = best;
      sm.plan[1] = n;
      sm.plan[2] = c;
    }
  }
  __syncthreads();
  const int tsh = (int)sm.plan[0];
  const uint32_t N = sm.plan[1], chunk = sm.plan[2];
  if (warp * 32 * per < a.batch) {
    uint32_t mine = cnt[0];
#pragma unroll
    for (int i = 1; i < kSizes; ++i) mine = tsh == i ? cnt[i] : mine;
    uint32_t inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    // The thread whose rows hold a team's first unit tells it where they start.
    const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.wsum[tsh][lane % kPlanWarps] : 0);
    const uint32_t s0 = (before + inc - mine) * a.Hkv, s1 = s0 + mine * a.Hkv;
    if (mine)
      for (int i = 0; i < kAttWarps >> tsh; ++i) {
        const uint32_t u = ((uint32_t)i * gridDim.x + blockIdx.x) * chunk;  // at most N + teams
        if (u >= s0 && u < s1) {
          sm.first_b[i] = b_lo;
          sm.first_u[i] = s0;
        }
      }
  }
  __syncthreads();

  // ---- this team's run of units
  const int wc = warp % kAttWarps;  // the consumer warp that this one is, or loads for
  const int team = wc >> tsh, wt = wc & ((1 << tsh) - 1), T = 1 << tsh;
  const uint32_t k = (uint32_t)team * gridDim.x + blockIdx.x;  // runs go round the SMs: few runs use many of them
  const uint32_t u0 = min(k * chunk, N), uend = min(u0 + chunk, N);
  volatile int* abort = &sm.abort;
  Kv4Seg cs;
  if (u0 < uend) {
    uint32_t u = sm.first_u[team];
    cs.b = sm.first_b[team];
    kv4_row(a, sm, cs);
    uint32_t rounds = (uint32_t)(cs.n + T - 1) >> tsh;
    while (u + rounds * a.Hkv <= u0) {
      u += rounds * a.Hkv;
      ++cs.b;
      kv4_row(a, sm, cs);
      rounds = (uint32_t)(cs.n + T - 1) >> tsh;
    }
    cs.u = u0;
    cs.h = (int)((u0 - u) / rounds);
    cs.t0 = (int)((u0 - u) - (uint32_t)cs.h * rounds) << tsh;
    cs.t1 = seg_end(cs.n, cs.t0, uend - u0, tsh);
  }

  if (warp >= kAttWarps) {
    // ---- a loading warp: the tiles of its consumer, in order, up to kStages ahead.  It lists up to 32 of them at
    // a time, a tile per lane: the block ids arrive together.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (u0 >= uend) return;
    uint32_t issued = 0;
    bool ok = true, more = true;
    int t = cs.t0 + wt;
    while (ok && more) {
      const int n = min(32, (cs.t1 - t + T - 1) >> tsh);  // <= 0: no tile of this segment for this warp
      if (n > 0) {
        const int my = min(t + (lane << tsh), cs.t1 - 1), bi = my / a.tpb;
        uint32_t rec = (uint32_t)a.bt[cs.row * a.max_blocks + bi];
        if (rec >= (uint32_t)a.num_blocks) {
          report(a.err, ERR_BLOCK_OOB);
          rec = 0;  // a valid address keeps the pipeline going; the result is flagged
        }
        rec = (rec * (uint32_t)a.Hkv + (uint32_t)cs.h) * (uint32_t)a.tpb + (uint32_t)(my - bi * a.tpb);
        for (int i = 0; ok && i < n; ++i, ++issued) {
          const uint32_t st = issued % kStages;
          const int64_t at = (int64_t)__shfl_sync(0xffffffffu, rec, i) * kKv4Record;
          if (issued >= kStages) ok = warp_wait(&sm.empty[wc][st], (issued / kStages - 1) & 1, a.err, abort);
          if (!ok) break;
          if (lane == 0) {
            uint64_t* bar = &sm.full[wc][st];
            mbar_arrive_expect_tx(bar, 2 * kKv4Record);
            bulk_load(sm.kv[wc][st][0], a.kc + at, kKv4Record, bar);
            bulk_load(sm.kv[wc][st][1], a.vc + at, kKv4Record, bar);
          }
          __syncwarp();
        }
        t += n << tsh;
      }
      if (ok && t >= cs.t1) {
        more = kv4_next(a, sm, cs, uend, tsh);
        t = cs.t0 + wt;
      }
    }
    // Every copy has landed (or has run out of time) before the warp, and with it the CTA, may end.
    for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
      mbar_wait(&sm.full[wc][i % kStages], i / kStages & 1, a.err, nullptr);
    return;
  }
  asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");

  if (u0 < uend) {
    // The 8 columns of an MMA are kCols to a head.  A lane (g, c) looks at columns 2 c and 2 c + 1: with kCols = 1 it
    // holds the scores of two heads for tokens g and g + 8 of 16, with 2 those of one head, and with 4 those of one
    // head for one of the tokens (columns 4 h and 4 h + 2 are the same, so one lane takes g, its neighbour g + 8).
    constexpr int kCols = G == 8 ? 1 : G == 4 ? 2 : 4;
    constexpr int HV = kCols == 1 ? 2 : 1;  // heads per lane
    constexpr int NV = 4 / kCols;           // scores per lane of 16 tokens: [token][head]
    constexpr int kLow = kCols == 4 ? 1 : 4;  // a head's lanes: all g, and with kCols = 4 both of c / 2's
    const int tok = kCols == 4 ? g + 8 * (c & 1) : g;  // the first's token; the second's is 8 further
    // Queries of a segment: raw, as loaded; the dims 32 w + 8 c .. + 7 of the head of column g.
    const int qh = g / kCols;
    uint4 xq[4];
    auto load_q = [&](const Kv4Seg& s) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        xq[w] = qh < G ? *reinterpret_cast<const uint4*>(a.q + (((int64_t)s.b * a.Hkv + s.h) * G + qh) * 128 +
                                                         32 * w + 8 * c)
                       : make_uint4(0, 0, 0, 0);
    };
    load_q(cs);
    uint32_t used = 0;  // tiles; tile i lies in stage i % kStages
    bool dead = false;  // a copy did not come in time: no more tiles

    // Items that this run holds a part of, not the whole: first query head, first and last unit.
    int parts = 0;
    int64_t part_q[2] = {0, 0};
    uint32_t part_first[2] = {0, 0}, part_last[2] = {0, 0};

    while (true) {
      // ---- queries of the item: B operand (columns without a head are zero)
      const int64_t qh0 = ((int64_t)cs.b * a.Hkv + cs.h) * G;
      uint32_t qf[4][4];
      float sl[HV];       // log2 softmax scale of the raw scores of this lane's heads
      float corr[4][HV];  // -8 times 2^-24 times the sum of their q over group w
      bool fits;          // q into fp16
      {
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns q's sign
        uint32_t hi = 0, lo = 0x7fff7fffu;  // in pairs: largest |q|; smallest above zero, plus 0x7fff
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          qf[w][0] = xq[w].x ^ flip;
          qf[w][1] = xq[w].y ^ flip;
          qf[w][2] = xq[w].z ^ flip;
          qf[w][3] = xq[w].w ^ flip;
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const uint32_t y = qf[w][r] & 0x7fff7fffu, z = qf[w][r + 1] & 0x7fff7fffu;
            hi = __vimax3_u16x2(hi, y, z);
            lo = __vimin3_s16x2(lo, y + 0x7fff7fffu, z + 0x7fff7fffu);
          }
        }
        // largest, and 2^16 less the smallest above zero (0: there is none)
        uint32_t both = max(hi & 0xffffu, hi >> 16) |
                        (uint32_t)(0x7fff - min((int)(int16_t)lo, (int)lo >> 16)) << 16;
        both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 1));
        both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 2));
        const uint32_t mx = both & 0xffffu, mn = 0x10000u - (both >> 16);
        // If not, or if fp32 has no room for the raw scores, the second path takes all of the item.
        fits = !__any_sync(0xffffffffu, mx >> 7 > 200 || (int)(mx >> 7) - (int)(mn >> 7) > (mn < 0x80u ? 20 : 27) ||
                                                   !(fabsf(a.scale) < 0x1p40f));
        // 2^(14 - e) for a largest element in [2^e, 2^(e + 1)), as far as fp32 goes
        const int f = min(268 - (int)(mx >> 7), 254);
        const float up = __uint_as_float((uint32_t)f << 23);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float2 y = unpack_bf16(qf[w][r]);
            const float f16 = r & 1 ? 0.0625f * up : up;  // registers 1 and 3 meet the codes that weigh 16
            qf[w][r] = pack_f16(y.x * f16, y.y * f16);
            sum[w] += (y.x + y.y) * up;
          }
        const float down = fabsf(a.scale) * (0x1p24f * kLog2e) *
                           (f == 254 ? 0x1p-127f : __uint_as_float((uint32_t)(254 - f) << 23));
#pragma unroll
        for (int e = 0; e < HV; ++e) sl[e] = __shfl_sync(0xffffffffu, down, 8 * c + 4 * e);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
          sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
#pragma unroll
          for (int e = 0; e < HV; ++e) corr[w][e] = -0x1p-21f * __shfl_sync(0xffffffffu, sum[w], 8 * c + 4 * e);
        }
      }
      float o[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m[HV], l[HV];
#pragma unroll
      for (int e = 0; e < HV; ++e) m[e] = -INFINITY, l[e] = 0.f;
      // Biased exponents of the largest V scale so far (at least this) and of the smallest in the tiles that set the
      // softmax reference; tiles from `room` on are left to the second path.  O is kept times 2^(kUp + 126 - ev).
      int ev = kSpan + 1, low = 255, room = fits ? 0 : -1;
      uint32_t from = 0;  // and a scale: bits 15 and 31 where the scale is at least 2^(ev - kSpan); 0: not set

      for (int t = cs.t0 + wt;; t += T) {
        for (; t < cs.t1 && !dead; t += T) {
          const uint32_t st = used % kStages;
          if (!warp_wait(&sm.full[warp][st], used / kStages & 1, a.err, abort)) {
            dead = true;
            break;
          }
          if (room < 0) break;
          const uint8_t* kb = sm.kv[warp][st][0];
          const uint8_t* vb = sm.kv[warp][st][1];
          const int lim = cs.ctx - t * kKv4Tile;  // tokens from here to the end of the context

          // ---- S = K Q^T
          float s[4][NV];
#pragma unroll
          for (int sb = 0; sb < 4; ++sb) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + lane * 16);        // token g
            const uint4 y4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + 512 + lane * 16);  // token g + 8
            const uint2 sx = *reinterpret_cast<const uint2*>(kb + kKv4Codes + (16 * sb + tok) * 8);
            const uint2 sy =
                kCols == 4 ? sx : *reinterpret_cast<const uint2*>(kb + kKv4Codes + (16 * sb + tok + 8) * 8);
            auto group = [&](auto W, uint32_t x, uint32_t y) {
              constexpr int w = decltype(W)::value;
              float acc[4];
              const uint32_t a0[4] = {code_sub<false>(x), code_sub<false>(y), code_sub<true>(x), code_sub<true>(y)};
              mma_f16_16816_from(acc, a0, qf[w][0], qf[w][1], corr[w][0], corr[w][HV - 1]);
              x >>= 8;
              y >>= 8;
              const uint32_t a1[4] = {code_sub<false>(x), code_sub<false>(y), code_sub<true>(x), code_sub<true>(y)};
              mma_f16_16816(acc, a1, qf[w][2], qf[w][3]);
              const float fx = scale_of<w>(sx), fy = scale_of<w>(sy);
#pragma unroll
              for (int i = 0; i < NV; ++i) {
                const float v = kCols == 1 ? acc[i] : kCols == 2 ? acc[2 * i] : c & 1 ? acc[2] : acc[0];
                const float f = i < HV ? fx : fy;
                s[sb][i] = w == 0 ? v * f : fmaf(v, f, s[sb][i]);
              }
            };
            group(std::integral_constant<int, 0>{}, x4.x, y4.x);
            group(std::integral_constant<int, 1>{}, x4.y, y4.y);
            group(std::integral_constant<int, 2>{}, x4.z, y4.z);
            group(std::integral_constant<int, 3>{}, x4.w, y4.w);
          }

          // ---- the tile's V scales; lane: tokens 2 lane and 2 lane + 1.  Behind the context a scale may be anything:
          // it becomes that of the tile's first token, and p zero.
          uint4 vs = *(reinterpret_cast<const uint4*>(vb + kKv4Codes) + lane);
          if (lim < kKv4Tile) {
            const uint2 first = *reinterpret_cast<const uint2*>(vb + kKv4Codes);
            if (2 * lane >= lim) vs.x = first.x, vs.y = first.y;
            if (2 * lane + 1 >= lim) vs.z = first.x, vs.w = first.y;
#pragma unroll
            for (int sb = 0; sb < 4; ++sb)
#pragma unroll
              for (int i = 0; i < NV; ++i)
                if (16 * sb + tok + i / HV * 8 >= lim) s[sb][i] = -INFINITY;
          }
          // Scales are not negative, so their bits order as they do: bits 15 and 31 stay where all are in range.
          const uint32_t hi = __vmaxu2(__vimax3_u16x2(vs.x, vs.y, vs.z), vs.w);
          const uint32_t lo = __vminu2(__vimin3_u16x2(vs.x, vs.y, vs.z), vs.w);
          const bool odd = ~((lo + from) & (kUpTo - from - hi)) & 0x80008000u;

          // ---- online softmax in the log2 domain.  The reference of the exponentials follows the maximum only when a
          // score passes it by 2^kLag: p stays below that, and most tiles need no shuffles and no rescaling.
          float x[HV];
          bool above = false;
#pragma unroll
          for (int e = 0; e < HV; ++e) {
            x[e] = s[0][e];
#pragma unroll
            for (int i = 1; i < 4 * NV / HV; ++i) x[e] = fmaxf(x[e], s[i % 4][i / 4 * HV + e]);
            x[e] *= sl[e];
            above |= x[e] > m[e] + (float)kLag;
          }
          if (__any_sync(0xffffffffu, above || odd) || t >= room) {
            const uint32_t big = __reduce_max_sync(0xffffffffu, max(hi & 0xffffu, hi >> 16));
            const uint32_t least = __reduce_min_sync(0xffffffffu, min(lo & 0xffffu, lo >> 16));
            const bool set = __any_sync(0xffffffffu, above);
            const int e0 = ev;
            if (big < 253u << 7) ev = max(ev, (int)(big >> 7));  // else the second path does
            const uint32_t from_v = (uint32_t)(ev - kSpan) << 7;
            const bool wide = big >= 253u << 7 || least < from_v;
            from = (0x8000u - from_v) * 0x10001u;
            const float up = ex2((float)(e0 - ev));
            if (set) low = min(low, least < 0x80u ? kNone : (int)(least >> 7));
            float al[HV];
#pragma unroll
            for (int e = 0; e < HV; ++e) {
#pragma unroll
              for (int d = kLow; d < 32; d += d == 1 ? 3 : d) x[e] = fmaxf(x[e], __shfl_xor_sync(0xffffffffu, x[e], d));
              x[e] = set ? fmaxf(m[e], x[e]) : m[e];
              const float f = ex2(m[e] - x[e]);
              m[e] = x[e];
              al[e] = set ? f * up : up;
              l[e] *= set ? f : 1.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[j][i] *= al[i % HV];
            room = cs.t0 + wt + (kv4_room(ev, low) << tsh);
            if ((wide || t >= room) && big) break;  // fp16 loses nothing of zeros
          }
          {
            const float cv = __uint_as_float((uint32_t)(253 - ev) << 23);
            const uint2 ta = make_uint2(vs.x, vs.y), tb = make_uint2(vs.z, vs.w);
            sm.vpair[warp][lane] = make_uint4(pack_f16(scale_of<0>(ta) * cv, scale_of<0>(tb) * cv),
                                              pack_f16(scale_of<1>(ta) * cv, scale_of<1>(tb) * cv),
                                              pack_f16(scale_of<2>(ta) * cv, scale_of<2>(tb) * cv),
                                              pack_f16(scale_of<3>(ta) * cv, scale_of<3>(tb) * cv));
          }
#pragma unroll
          for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < NV; ++i) s[sb][i] = ex2(fmaf(s[sb][i], sl[i % HV], (float)kUp - m[i % HV]));  // 2^kUp p
          if (lim < kKv4Tile) {  // also where a scale of 0 makes -inf * 0 a NaN
#pragma unroll
            for (int sb = 0; sb < 4; ++sb)
#pragma unroll
              for (int i = 0; i < NV; ++i)
                if (16 * sb + tok + i / HV * 8 >= lim) s[sb][i] = 0.f;
          }
#pragma unroll
          for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < NV; ++i) l[i % HV] += s[sb][i];
          __syncwarp();  // vpair is written

          // ---- O^T += V^T P^T
          uint32_t pt = 0;
#pragma unroll
          for (int sb = 0; sb < 4; ++sb) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + lane * 16);        // tokens 2c, 2c + 1
            const uint4 y4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + 512 + lane * 16);  // ... + 8
            const uint4 sx = sm.vpair[warp][sb * 8 + c], sy = sm.vpair[warp][sb * 8 + 4 + c];
            uint32_t px, py;  // column g: its head's tokens 2c, 2c + 1 and ... + 8
            if constexpr (kCols == 1) {
              px = movmatrix_trans(pack_f16(s[sb][0], s[sb][1]));
              py = movmatrix_trans(pack_f16(s[sb][NV - 2], s[sb][NV - 1]));
            } else if constexpr (kCols == 2) {
              // A head's even column takes tokens 0 .. 7, its odd one 8 .. 15: one transpose for both.
              const uint32_t y = movmatrix_trans(pack_f16(s[sb][0], s[sb][NV - 1]));
              px = g & 1 ? 0u : y;
              py = g & 1 ? y : 0u;
            } else {
              // Columns 4 h and 4 h + 1 take tokens 0 .. 7 of even and of odd sb, + 2 and + 3 tokens 8 .. 15.
              if (sb % 2 == 0) pt = movmatrix_trans(pack_f16(s[sb][0], s[(sb + 1) % 4][0]));
              px = (g & 3) == sb % 2 ? pt : 0u;
              py = (g & 3) == sb % 2 + 2 ? pt : 0u;
            }
            auto group = [&](auto W) {  // 32 dims: j = 2w and 2w + 1
              constexpr int w = decltype(W)::value;
              const uint32_t b0 = mul_f16(px, w == 0 ? sx.x : w == 1 ? sx.y : w == 2 ? sx.z : sx.w);
              const uint32_t b1 = mul_f16(py, w == 0 ? sy.x : w == 1 ? sy.y : w == 2 ? sy.z : sy.w);
              // 16 bits of tokens 2c | 2c + 1 each: four nibbles = dims 16 j + 2g, + 1 of j = 2w, 2w + 1
              constexpr uint32_t sel = (w & 1) ? 0x7632u : 0x5410u;
              uint32_t x = w < 2 ? __byte_perm(x4.x, x4.z, sel) : __byte_perm(x4.y, x4.w, sel);
              uint32_t y = w < 2 ? __byte_perm(y4.x, y4.z, sel) : __byte_perm(y4.y, y4.w, sel);
              const uint32_t a0[4] = {code<false>(x), code<true>(x), code<false>(y), code<true>(y)};
              mma_f16_16816(o[2 * w], a0, b0, b1);
              x >>= 8;
              y >>= 8;
              const uint32_t a1[4] = {code<false>(x), code<true>(x), code<false>(y), code<true>(y)};
              mma_f16_16816(o[2 * w + 1], a1, b0, b1);
            };
            group(std::integral_constant<int, 0>{});
            group(std::integral_constant<int, 1>{});
            group(std::integral_constant<int, 2>{});
            group(std::integral_constant<int, 3>{});
          }
          __syncwarp();  // every lane has read the stage
          if (lane == 0) mbar_arrive(&sm.empty[warp][st]);
          ++used;
        }
        if (t >= cs.t1 || dead) break;
        // ---- this tile on the second path: the scores first
        const uint32_t st = used % kStages;
        const uint8_t* kb = sm.kv[warp][st][0];
        const uint8_t* vb = sm.kv[warp][st][1];
        const int lim = cs.ctx - t * kKv4Tile;
        float* mine = &sm.red_o[warp][0][lane];  // free until the segment ends: this lane's scores
        float x[HV];
#pragma unroll
        for (int e = 0; e < HV; ++e) x[e] = -INFINITY;
        {
          const uint4* qp = reinterpret_cast<const uint4*>(a.q + (qh0 + min(qh, G - 1)) * 128 + 8 * c);
          uint32_t mx = 0;
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {
            const uint4 y = qp[4 * w];
            mx = __vimax3_u16x2(mx, __vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu),
                                __vmaxu2(y.z & 0x7fff7fffu, y.w & 0x7fff7fffu));
          }
          mx = max(mx & 0xffffu, mx >> 16);
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const int by = kv4_q_exp(a.scale, mx);
          const float up = copysignf(exp2i(by), a.scale);
          float sw[HV];
#pragma unroll
          for (int e = 0; e < HV; ++e)
            sw[e] = __shfl_sync(0xffffffffu, fabsf(a.scale) * kLog2e * exp2i(-by), 8 * c + 4 * e);
#pragma unroll 1
          for (int sb = 0; sb < 4; ++sb) {
            float y[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) y[i] = 0.f;
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              const uint32_t u = *reinterpret_cast<const uint32_t*>(kb + sb * 1024 + lane * 16 + 4 * w);
              const uint32_t v = *reinterpret_cast<const uint32_t*>(kb + sb * 1024 + 512 + lane * 16 + 4 * w);
              const uint8_t* sp = kb + kKv4Codes + (16 * sb + tok) * 8 + 2 * w;
              const float fx = bf16_bits(*reinterpret_cast<const uint16_t*>(sp));
              const float fy = kCols == 4 ? fx : bf16_bits(*reinterpret_cast<const uint16_t*>(sp + 64));
              const uint4 qw = qp[4 * w];
              auto pair = [&](uint32_t z) {
                const float2 f = unpack_bf16(z);
                return pack_bf16(f.x * up, f.y * up);
              };
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              const uint32_t a0[4] = {code_bf16(u), code_bf16(v), code_bf16(u >> 4), code_bf16(v >> 4)};
              mma_bf16_16816(acc, a0, pair(qw.x), pair(qw.y));
              const uint32_t a1[4] = {code_bf16(u >> 8), code_bf16(v >> 8), code_bf16(u >> 12), code_bf16(v >> 12)};
              mma_bf16_16816(acc, a1, pair(qw.z), pair(qw.w));
#pragma unroll
              for (int i = 0; i < NV; ++i) {
                const float z = kCols == 1 ? acc[i] : kCols == 2 ? acc[2 * i] : c & 1 ? acc[2] : acc[0];
                y[i] = fmaf(z, i < HV ? fx : fy, y[i]);
              }
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
              const float z = 16 * sb + tok + i / HV * 8 < lim ? y[i] * sw[i % HV] : -INFINITY;
              mine[32 * (sb * NV + i)] = z;
              x[i % HV] = fmaxf(x[i % HV], z);
            }
          }
        }
        // the reference of the softmax, and the largest finite V scale
        bool above = false;
#pragma unroll
        for (int e = 0; e < HV; ++e) above |= x[e] > m[e] + (float)kLag;
        const bool set = __any_sync(0xffffffffu, above);
        if (set) low = kNone;
        uint32_t top = 0;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const uint32_t u = *reinterpret_cast<const uint16_t*>(vb + kKv4Codes + 2 * (32 * i + lane)) & 0x7fffu;
          if (u < 0x7f80u && 8 * i + lane / 4 < lim) top = max(top, u);
        }
        const int e0 = ev;
        ev = max(ev, min((int)(__reduce_max_sync(0xffffffffu, top) >> 7), 252));
        if (ev > e0) from = 0;  // the next tile sets its limits
        const float up = ex2((float)(e0 - ev));
        float al[HV];
#pragma unroll
        for (int e = 0; e < HV; ++e) {
#pragma unroll
          for (int d = kLow; d < 32; d += d == 1 ? 3 : d) x[e] = fmaxf(x[e], __shfl_xor_sync(0xffffffffu, x[e], d));
          x[e] = set ? fmaxf(m[e], x[e]) : m[e];
          const float f = set ? ex2(m[e] - x[e]) : 1.f;
          m[e] = x[e];
          al[e] = f * up;
          l[e] *= f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] *= al[i % HV];
        // p s as a sum of two bf16: 2^-17 of itself off, over all of fp32's range.  A column's B is zero at the places
        // of tokens that are another's.
        const float cw = __uint_as_float((uint32_t)(253 - ev) << 23);
#pragma unroll 1
        for (int sb = 0; sb < 4; ++sb) {
          const uint4 x4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + lane * 16);
          const uint4 y4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + 512 + lane * 16);
          const int t0 = 16 * sb + tok;
          float p[NV];
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            p[i] = t0 + i / HV * 8 < lim ? ex2(mine[32 * (sb * NV + i)] + ((float)kUp - m[i % HV])) : 0.f;
            l[i % HV] += p[i];
          }
          uint2 sx = *reinterpret_cast<const uint2*>(vb + kKv4Codes + t0 * 8), sy = make_uint2(0, 0);
          if constexpr (kCols < 4) sy = *reinterpret_cast<const uint2*>(vb + kKv4Codes + (t0 + 8) * 8);
          if (t0 >= lim) sx = make_uint2(0, 0);
          if (t0 + 8 >= lim) sy = make_uint2(0, 0);
          auto group = [&](auto W) {
            constexpr int w = decltype(W)::value;
            const float fx = scale_of<w>(sx) * cw, fy = scale_of<w>(sy) * cw;
            float v[4];
            if constexpr (kCols == 1)
              v[0] = p[0] * fx, v[1] = p[1] * fx, v[2] = p[NV - 2] * fy, v[3] = p[NV - 1] * fy;
            else if constexpr (kCols == 2)
              v[0] = p[0] * fx, v[1] = p[NV - 1] * fy, v[2] = v[3] = 0.f;
            else
              v[0] = v[1] = p[0] * fx, v[2] = v[3] = 0.f;
            constexpr uint32_t sel = (w & 1) ? 0x7632u : 0x5410u;
            const uint32_t y = w < 2 ? __byte_perm(x4.x, x4.z, sel) : __byte_perm(x4.y, x4.w, sel);
            const uint32_t z = w < 2 ? __byte_perm(y4.x, y4.z, sel) : __byte_perm(y4.y, y4.w, sel);
            const uint32_t a0[4] = {code_bf16(y), code_bf16(y >> 4), code_bf16(z), code_bf16(z >> 4)};
            const uint32_t a1[4] = {code_bf16(y >> 8), code_bf16(y >> 12), code_bf16(z >> 8), code_bf16(z >> 12)};
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
              const uint32_t u0 = pack_bf16(v[0], v[1]), u1 = pack_bf16(v[2], v[3]);
              const float2 r0 = unpack_bf16(u0), r1 = unpack_bf16(u1);
              v[0] -= r0.x, v[1] -= r0.y, v[2] -= r1.x, v[3] -= r1.y;
              const uint32_t u = movmatrix_trans(u0);
              uint32_t b0 = u, b1 = u;
              if constexpr (kCols == 1)
                b1 = movmatrix_trans(u1);
              else if constexpr (kCols == 2)
                b0 = g & 1 ? 0u : u, b1 = g & 1 ? u : 0u;
              else
                b0 = (g & 3) == 0 ? u : 0u, b1 = (g & 3) == 2 ? u : 0u;
              mma_bf16_16816(o[2 * w], a0, b0, b1);
              mma_bf16_16816(o[2 * w + 1], a1, b0, b1);
            }
          };
          group(std::integral_constant<int, 0>{});
          group(std::integral_constant<int, 1>{});
          group(std::integral_constant<int, 2>{});
          group(std::integral_constant<int, 3>{});
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[warp][st]);
        ++used;
      }

      // ---- end of the segment: the team's warps meet in shared memory
      Kv4Seg nx = cs;
      const bool more = kv4_next(a, sm, nx, uend, tsh);
      if (more) load_q(nx);
      const float down = __uint_as_float((uint32_t)(ev + 1) << 23) * (1.f / (1 << kUp));
#pragma unroll
      for (int e = 0; e < HV; ++e) {  // dims 16 j + 2g and + 1: o[j][e], o[j][2 + e], summed over a head's columns
        const int hd = (2 * c + e) / kCols;
#pragma unroll
        for (int d = kLow; d < 32; d += d == 1 ? 3 : d) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float y0 = o[j][e], y1 = o[j][2 + e];
          if constexpr (kCols > 1) y0 += o[j][1], y1 += o[j][3];
          if constexpr (kCols > 2) {
            y0 += __shfl_xor_sync(0xffffffffu, y0, 1);
            y1 += __shfl_xor_sync(0xffffffffu, y1, 1);
          }
          if (hd < G && (kCols < 4 || (c & 1) == (j & 1)))
            *reinterpret_cast<float2*>(&sm.red_o[warp][hd][16 * j + 2 * g]) = make_float2(y0 * down, y1 * down);
        }
        if (hd < G && g == 0 && (kCols < 4 || (c & 1) == 0))
          *reinterpret_cast<float2*>(sm.red_ml[warp][hd]) = make_float2(m[e], l[e] * (1.f / (1 << kUp)));
      }
      team_sync(team, tsh);
      const bool whole = cs.t0 == 0 && cs.t1 == cs.n;
      const uint32_t slot = 2 * k + (cs.t0 == 0);
      kv4_share<G>(T, [&](auto V) {
        constexpr int VW = decltype(V)::value;
        for (int i = wt; i < G * 4 / VW; i += T) {
          const Kv4Share<VW> sh(i, lane);
          float M, L, O[VW];
          kv4_combine<VW>(
              T, lane, [&](int w) { return *reinterpret_cast<const float2*>(sm.red_ml[(team << tsh) + w][sh.hd]); },
              [&](int w, float(&y)[VW]) {
                sh.read(sm.red_o[(team << tsh) + w][sh.hd], y, [](auto* p) { return *p; });
              },
              M, L, O);
          if (whole) {
            sh.write(a.out + (qh0 + sh.hd) * 128, O, L);
          } else {
            const int64_t at = (int64_t)slot * G + sh.hd;
            sh.write(a.ws_o + at * 128, O);
            if (sh.d == 0) reinterpret_cast<float2*>(a.ws_ml)[at] = make_float2(M, L);
          }
        }
      });
      if (!whole) {  // at most twice: where the run begins and where it ends
        const uint32_t first = cs.u - (cs.t0 >> tsh);
        const uint32_t end = first + ((uint32_t)(cs.n + T - 1) >> tsh) - 1;
        if (parts == 0) {  // (no indexing: they stay in registers)
          part_q[0] = qh0, part_first[0] = first, part_last[0] = end;
        } else {
          part_q[1] = qh0, part_first[1] = first, part_last[1] = end;
        }
        ++parts;
      }
      team_sync(team, tsh);  // the team's shared buffers are read
      if (!more) break;
      cs = nx;
    }
    if (parts) {
      // Of the runs k0 .. k0 + n - 1 that share an item, the last to get here sums their parts: run k0's tail
      // (slot 2 k0 + 1), then the heads of the others (slots 2 k), in this order whichever run it is.
      __threadfence();
      team_sync(team, tsh);
      if (wt == 0 && lane < parts) {
        const uint32_t k0 = (lane ? part_first[1] : part_first[0]) / chunk;
        const uint32_t n = (lane ? part_last[1] : part_last[0]) / chunk - k0 + 1;
        sm.merge_k[team][lane] = k0;
        sm.merge_n[team][lane] = atomicInc(a.cnt + k0, n - 1) == n - 1 ? (int)n : 0;
      }
      team_sync(team, tsh);
#pragma unroll 1
      for (int q = 0; q < parts; ++q) {
        const int n = sm.merge_n[team][q];
        if (n == 0) continue;
        __threadfence();
        const int64_t k0 = sm.merge_k[team][q];
        bf16* out = a.out + (q ? part_q[1] : part_q[0]) * 128;
        kv4_share<G>(T, [&](auto V) {
          constexpr int VW = decltype(V)::value;
          for (int i = wt; i < G * 4 / VW; i += T) {
            const Kv4Share<VW> sh(i, lane);
            auto at = [&](int p) { return (2 * (k0 + p) + (p == 0)) * G + sh.hd; };
            float M, L, O[VW];
            kv4_combine<VW>(
                n, lane, [&](int p) { return __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + at(p)); },
                [&](int p, float(&y)[VW]) { sh.read(a.ws_o + at(p) * 128, y, [](auto* x) { return __ldcg(x); }); },
                M, L, O);
            sh.write(out + sh.hd * 128, O, L);
          }
        });
      }
    }
  }

  // ---- rows without tokens are zero
  for (int b = blockIdx.x + warp * gridDim.x; b < a.batch; b += kAttWarps * gridDim.x) {
    int row;
    if ((per == 1 ? sm.ctx[b] : kv4_ctx(a, b, &row)) == 0)
      for (int i = lane; i < a.Hkv * G * 16; i += 32)
        reinterpret_cast<uint4*>(a.out + (int64_t)b * a.Hkv * G * 128)[i] = make_uint4(0, 0, 0, 0);
  }
}

// Workspace: counters of every team a device can have (T = 1), then two partials per team.
static int64_t kv4_teams() { return (int64_t)sm_count() * kAttWarps; }
static int64_t kv4_counter_bytes() { return (kv4_teams() * 4 + 255) / 256 * 256; }

template <int G>
static cudaError_t kv4_launch(const Kv4Args& a, cudaStream_t stream) {
  const size_t smem = sizeof(Kv4Smem<G>);
  set_smem_once<kv4_decode_kernel<G>>((int)smem);
  return launch_k(kv4_decode_kernel<G>, dim3(sm_count()), dim3(kAttThreads), smem, stream, a);
}

}  // namespace aacc

using namespace aacc;

extern "C" {

int64_t aacc_kv4_decode_workspace_bytes(int num_q_heads, int num_kv_heads) {
  if (num_kv_heads <= 0 || num_q_heads <= 0) return 0;
  const int64_t G = (num_q_heads + num_kv_heads - 1) / num_kv_heads;
  return kv4_counter_bytes() + 2 * kv4_teams() * G * (128 + 2) * (int64_t)sizeof(float);
}

int aacc_kv4_decode_attention(const void* q, void* out, const void* k_cache, const void* v_cache, int64_t num_blocks,
                              const int32_t* block_tables, int64_t num_rows, int64_t max_blocks,
                              const int64_t* slot_indices, const int32_t* seqlens, int ctx_add, int64_t batch,
                              int num_q_heads, int num_kv_heads, int block_size, float scale, int64_t max_context,
                              void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  if (batch < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || block_size <= 0 ||
      block_size % kKv4Tile || num_blocks <= 0 || num_rows < 0 || max_blocks <= 0 || max_context <= 0)
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: bad sizes");
  const int G = num_q_heads / num_kv_heads;
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_decode_attention: q/kv head ratio %d not in {1,2,4,8}", G);
  if (batch == 0) return AACC_OK;
  if (max_context > max_blocks * block_size) max_context = max_blocks * block_size;
  if (max_context > 0x7fffffc0) max_context = 0x7fffffc0;
  // Units are counted in 32 bits.
  if (batch > 0x7fffffff || num_rows > 0x7ffffffe ||
      (double)batch * num_kv_heads * (double)((max_context + kKv4Tile - 1) / kKv4Tile) > 2147483647.0)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_decode_attention: %lld rows of up to %lld tokens are too many",
                     (long long)batch, (long long)max_context);
  if (!q || !out || !k_cache || !v_cache || !block_tables || !slot_indices || !seqlens)
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: null pointer");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: pointers must be 16-byte aligned");
  const int64_t need = aacc_kv4_decode_workspace_bytes(num_q_heads, num_kv_heads);
  if (!workspace || workspace_bytes < need)
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: workspace %lld < %lld bytes", (long long)workspace_bytes,
                     (long long)need);
  Kv4Args a;
  a.q = (const bf16*)q;
  a.out = (bf16*)out;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.bt = block_tables;
  a.rows = slot_indices;
  a.seqlens = seqlens;
  a.cnt = (unsigned*)workspace;
  a.ws_o = reinterpret_cast<float*>((uint8_t*)workspace + kv4_counter_bytes());
  a.ws_ml = a.ws_o + 2 * kv4_teams() * G * 128;
  a.err = device_error_ptr();
  a.num_blocks = (int)(num_blocks < 0x7fffffff ? num_blocks : 0x7fffffff);  // ids are 32-bit
  a.num_rows = (int)num_rows;
  a.max_blocks = max_blocks;
  a.batch = (int)batch;
  a.max_ctx = (int)max_context;
  a.ctx_add = ctx_add;
  a.Hkv = num_kv_heads;
  a.tpb = block_size / kKv4Tile;
  a.scale = scale;
  cudaError_t le;
  switch (G) {
    case 1: le = kv4_launch<1>(a, stream); break;
    case 2: le = kv4_launch<2>(a, stream); break;
    case 4: le = kv4_launch<4>(a, stream); break;
    default: le = kv4_launch<8>(a, stream); break;
  }
  return check_launch("kv4_decode_kernel", le);
}

}  // extern "C"
