// Decode attention over the 4-bit paged KV cache (format: kv4.cuh).
//
//   out[b][h] = sum_t softmax_t(scale q.k_t) v_t,  k_t = s n (4 groups of 32 dims)
//
// The floor is 144 bytes per (token, kv head) from HBM.  At that rate an SM
// has about 400 cycles per 64 tokens, so the expansion of the codes has to
// stay near one instruction a value, and there is no time for barriers.
//
// Work: the kernel is persistent, one CTA of 16 warps per SM, grouped into
// teams of T = 1, 2, 4, 8 or 16 warps.  An item is one (row, kv head), a unit
// a round of T tiles of 64 tokens of an item, one for each warp of a team.
// Every CTA counts the batch's units itself from seqlens and takes the T of
// the least estimated time (large T: few partials to merge; small T: no round
// that is not full, no waiting); the units are cut into equal runs, one per
// team, whatever the rows' lengths are.  A run that ends inside an item leaves an fp32 partial (max, sum, O);
// the last team of the item to arrive merges the partials in order.
//
// Tiles: each warp streams its own tiles through one K and one V buffer with
// bulk copies (lane 0 issues; the next K is fetched during softmax and P.V,
// the next V during the next Q.K), so warps never wait for one another but at
// the end of a team's item.  A tile is worked on in halves of 32 tokens, in a
// rolled loop: straight-line code for whole tiles spent a fifth of a small
// call on instruction fetches.
//
// Q.K: the tokens are the rows of m16n8k16's A operand, the G <= 8 query heads
// its 8 columns.  With all else masked off, four bits at the foot of an fp16
// are the subnormal 2^-24 u, or 2^-20 u one nibble higher, and the tensor
// cores take subnormals as they are: an AND makes two operands.  The 2^24 is
// put right in the softmax scale, the 16 in q, and the offset of 8 through the
// accumulator's start, -8 sum(q) of the group; the group's scale multiplies
// the fp32 sum.  q is scaled by a power of two per head to a largest element
// in [2^14, 2^15), so that bf16 values go into fp16 unrounded down to 2^-24 of
// the largest.
// P.V: O^T = V^T P^T with V^T (dims x tokens) as the A operand.  Here the sum
// over thousands of tokens would cancel against its offset, so u - 8 is made
// exactly, by one more fp16x2 add or fma.  P^T is 2^4 p in fp16 (the 2^4 also
// in the sum it is divided by), p < 2^6, transposed in registers and multiplied
// by the V scales of its two tokens in fp16: two roundings of 2^-12, a quarter
// of what one to bf16 costs.  The scales are held relative to the largest so
// far, at [2^4, 2^5): products reach 2^15, and a p down to 2^-18 and a scale
// down to 2^-21 of the largest have no other rounding than those two.
// Once per tile each lane turns the scales of its two tokens into such pairs.
#include <cuda_fp16.h>

#include <type_traits>

#include "host.h"
#include "kv4.cuh"

namespace aacc {

constexpr int kAttWarps = 16;
constexpr int kAttThreads = kAttWarps * 32;

// A run of tiles [t0, t1) of item (b, h), whose row has n tiles; u is the unit number of t0.
struct Kv4Seg {
  uint32_t u;
  int b, row, h, n, t0, t1, ctx;
};

template <int G>
struct Kv4Smem {
  uint8_t k[kAttWarps][kKv4Record];
  uint8_t v[kAttWarps][kKv4Record];
  uint4 vpair[kAttWarps][32];  // V scales of tokens 2 i and 2 i + 1, fp16 pairs of groups 0..3
  float red_o[kAttWarps][G][128];
  float red_ml[kAttWarps][G][2];
  uint32_t pre[kAttThreads];  // units before thread i's rows, per kv head
  int row[kAttThreads];       // of batches up to kAttThreads rows
  int ctx[kAttThreads];
  uint32_t wsum[6][kAttWarps];
  uint32_t sum[6];
  uint64_t kfull[kAttWarps];
  uint64_t vfull[kAttWarps];
  Kv4Seg ahead[kAttWarps];  // where each warp's loads are: segment, and
  int ahead_t[kAttWarps];          // its next tile there that is not in the warp's list
  int last[kAttWarps];
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
                                                   const float (&c)[2]) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]));
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

// Running (max, sum, O) of partial results that are weighted 2^max.
struct Kv4Acc {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float pm, float pl, float4 po) {
    const float n = fmaxf(m, pm);
    const float u = n == -INFINITY ? 0.f : n;
    const float f = ex2(m - u), g = ex2(pm - u);
    m = n;
    l = l * f + pl * g;
    o.x = o.x * f + po.x * g;
    o.y = o.y * f + po.y * g;
    o.z = o.z * f + po.z * g;
    o.w = o.w * f + po.w * g;
  }
  __device__ __forceinline__ uint2 result() const {
    const float inv = 1.f / l;
    return make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  }
};

template <int G>
__global__ void __launch_bounds__(kAttThreads, 1) kv4_decode_kernel(const Kv4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Kv4Smem<G>& sm = *reinterpret_cast<Kv4Smem<G>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  if (lane == 0) {
    mbar_init(&sm.kfull[warp], 1);
    mbar_init(&sm.vfull[warp], 1);
    fence_mbar_init();
  }
  if (threadIdx.x < 6) sm.sum[threadIdx.x] = 0;
  if (threadIdx.x == 0) sm.abort = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch();

  // ---- count the batch's units for every team size: each thread sums a run of rows, then the CTA
  const int per = (a.batch + kAttThreads - 1) / kAttThreads;
  const int b_lo = min(a.batch, (int)threadIdx.x * per), b_hi = min(a.batch, b_lo + per);
  uint32_t cnt[6] = {0, 0, 0, 0, 0, 0};  // [5]: rows with tokens
  for (int b = b_lo; b < b_hi; ++b) {
    int row;
    const int ctx = kv4_ctx(a, b, &row, blockIdx.x == 0 ? a.err : nullptr);
    if (per == 1) {
      sm.ctx[b] = ctx;
      sm.row[b] = row;
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) cnt[i] += (uint32_t)(tiles_of(ctx) + (1 << i) - 1) >> i;
    cnt[5] += ctx > 0;
  }
  {
    uint32_t x = 0;  // lane i < 6: counter i over the warp
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const uint32_t y = __reduce_add_sync(0xffffffffu, cnt[i]);
      x = lane == i ? y : x;
    }
    if (lane < 6) {
      sm.wsum[lane][warp] = x;
      if (x) atomicAdd(&sm.sum[lane], x);
    }
  }
  __syncthreads();
  // Lane i weighs T = 2^i, in microseconds of a model fitted to runs of 17 shapes with each T (B200; within 2 %
  // of the best T on average): a round of tiles takes 0.26 us per warp at work on the SM, but 2.5 us at least;
  // a partial costs 0.1 us for each of the G / T heads that a warp merges; the end of a segment 0.2 us for each.
  const int opt = min(lane, 4);
  const uint32_t n_opt = sm.sum[opt] * a.Hkv, teams = gridDim.x * (kAttWarps >> opt);
  const uint32_t c_opt = max((n_opt + teams - 1) / teams, 1u);
  uint32_t key;
  {
    const float t = (float)(1 << opt), ch = (float)c_opt;
    const float per_item = __fdividef((float)n_opt, (float)max(sm.sum[5] * a.Hkv, 1u));
    const float busy = t * ceilf(__fdividef(ceilf(__fdividef((float)n_opt, ch)), (float)gridDim.x));
    float cost = ch * fmaxf(2.5f, 0.26f * busy) +
                 0.2f * (1.f + __fdividef(ch, fmaxf(per_item, 1.f))) * fmaxf(1.f, __fdividef(G, t));
    if (per_item > 1.f) cost += 0.1f * G * __fdividef(per_item, ch * t);
    key = (__float_as_uint(cost) & ~7u) | opt;
  }
  const int tsh = (int)(__reduce_min_sync(0xffffffffu, key) & 7u);
  const uint32_t N = __shfl_sync(0xffffffffu, n_opt, tsh), chunk = __shfl_sync(0xffffffffu, c_opt, tsh);
  const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.wsum[tsh][lane & 15] : 0);
  uint32_t mine = cnt[0];
#pragma unroll
  for (int i = 1; i < 5; ++i) mine = tsh == i ? cnt[i] : mine;
  uint32_t inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  sm.pre[threadIdx.x] = before + inc - mine;
  __syncthreads();

  // ---- this team's run of units
  const int team = warp >> tsh, wt = warp & ((1 << tsh) - 1), T = 1 << tsh;
  const uint32_t k = (uint32_t)team * gridDim.x + blockIdx.x;  // runs go round the SMs: few runs use many of them
  const uint32_t u0 = (uint32_t)min((uint64_t)k * chunk, (uint64_t)N), uend = min(u0 + chunk, N);
  volatile int* abort = &sm.abort;

  if (u0 < uend) {
    Kv4Seg cs;
    {
      int lo = 0, hi = kAttThreads;  // the last thread whose rows start at or before u0
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sm.pre[mid] * a.Hkv <= u0)
          lo = mid;
        else
          hi = mid;
      }
      uint32_t u = sm.pre[lo] * a.Hkv;
      cs.b = lo * per;
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
    // The loads run one tile ahead of the arithmetic, across segments.  The warp lists up to 32 of its tiles
    // at a time, a tile per lane: block id `ids` and, within the block's records, `sub`; entry li of ln is next.
    // The segment they come from rests in shared memory.
    sm.ahead[warp] = cs;
    sm.ahead_t[warp] = cs.t0 + wt;
    __syncwarp();
    int32_t ids = 0;
    int sub = 0, li = 0, ln = 0;
    auto list_tiles = [&]() {
      Kv4Seg s = sm.ahead[warp];
      int t = sm.ahead_t[warp];
      li = 0;
      ln = 0;
      while (t >= s.t1) {
        if (!kv4_next(a, sm, s, uend, tsh)) return;
        t = s.t0 + wt;
      }
      ln = min(32, (s.t1 - t + T - 1) >> tsh);
      const int mine = min(t + (lane << tsh), s.t1 - 1), bi = mine / a.tpb;
      ids = a.bt[s.row * a.max_blocks + bi];
      sub = s.h * a.tpb + (mine - bi * a.tpb);
      __syncwarp();
      sm.ahead[warp] = s;
      sm.ahead_t[warp] = t + (ln << tsh);
      __syncwarp();
    };
    auto record = [&]() -> int64_t {
      int32_t id = __shfl_sync(0xffffffffu, ids, li);
      const int at = __shfl_sync(0xffffffffu, sub, li);
      if ((uint32_t)id >= (uint32_t)a.num_blocks) {
        if (lane == 0) report(a.err, ERR_BLOCK_OOB);
        id = 0;  // a valid address keeps the pipeline going; the result is flagged
      }
      return ((int64_t)id * (a.Hkv * a.tpb) + at) * kKv4Record;
    };
    auto load_k = [&](int64_t rec) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.kfull[warp], kKv4Record);
        bulk_load(sm.k[warp], a.kc + rec, kKv4Record, &sm.kfull[warp]);
      }
    };
    auto load_v = [&](int64_t rec) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.vfull[warp], kKv4Record);
        bulk_load(sm.v[warp], a.vc + rec, kKv4Record, &sm.vfull[warp]);
      }
    };
    list_tiles();
    bool lhas = ln > 0;  // there is a tile to load
    if (lhas) {
      const int64_t rec = record();
      load_k(rec);
      load_v(rec);
    }
    uint32_t ph = 0;    // parity of the tile in hand, for both buffers
    bool dead = false;  // a copy did not come in time: no more loads, no more tiles
    uint32_t kph = 0;   // then: the parity that the K buffer still waits for

    while (true) {
      // ---- queries of the item: B operand, column g = query head (columns >= G are zero)
      const int64_t qh0 = ((int64_t)cs.b * a.Hkv + cs.h) * G;
      uint32_t qf[4][4];
      float sl0, sl1;     // log2 softmax scale of the raw scores of heads 2c and 2c + 1
      float corr[4][2];  // -8 times 2^-24 times the sum of their q over group w
      {
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns q's sign
        uint32_t mx = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (g < G) x = *reinterpret_cast<const uint4*>(a.q + (qh0 + g) * 128 + 32 * w + 8 * c);
          qf[w][0] = x.x ^ flip;
          qf[w][1] = x.y ^ flip;
          qf[w][2] = x.z ^ flip;
          qf[w][3] = x.w ^ flip;
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = max(mx, max(qf[w][r] & 0x7fffu, (qf[w][r] >> 16) & 0x7fffu));
        }
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
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
        const float down = fabsf(a.scale) * (0x1p24f * kLog2e) * (f == 254 ? 0x1p-127f : __uint_as_float((uint32_t)(254 - f) << 23));
        sl0 = __shfl_sync(0xffffffffu, down, 8 * c);
        sl1 = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
          sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
          corr[w][0] = -0x1p-21f * __shfl_sync(0xffffffffu, sum[w], 8 * c);
          corr[w][1] = -0x1p-21f * __shfl_sync(0xffffffffu, sum[w], 8 * c + 4);
        }
      }
      float o[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      int ev = 4;  // biased exponent of the largest V scale so far (at least 4): O is kept times 2^(131 - ev)

      for (int t = cs.t0 + wt; t < cs.t1 && !dead; t += T) {
        if (lhas && ++li == ln) {  // the next block ids are in flight during Q.K
          list_tiles();
          lhas = ln > 0;
        }
        if (!warp_wait(&sm.kfull[warp], ph, a.err, abort)) {
          dead = true;
          kph = ph;
          lhas = false;
          break;
        }
        int64_t next_rec = 0;
        int lim = cs.ctx - t * kKv4Tile;  // tokens from here to the end of the context
#pragma unroll 1
        for (int half = 0; half < 2; ++half, lim -= 32) {
          // ---- S = K Q^T for 32 tokens; lane (g, c): tokens 16 sb + g (+ 8), heads 2c and 2c + 1
          const uint8_t* kb = sm.k[warp] + half * 2048;
          const uint8_t* ksc = sm.k[warp] + kKv4Codes + half * 256;
          float s[2][4];
#pragma unroll
          for (int sb = 0; sb < 2; ++sb) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + lane * 16);        // token g
            const uint4 y4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + 512 + lane * 16);  // token g + 8
            const uint2 sx = *reinterpret_cast<const uint2*>(ksc + (16 * sb + g) * 8);
            const uint2 sy = *reinterpret_cast<const uint2*>(ksc + (16 * sb + g + 8) * 8);
            auto group = [&](auto W, uint32_t x, uint32_t y) {
              constexpr int w = decltype(W)::value;
              float acc[4];
              const uint32_t a0[4] = {code_sub<false>(x), code_sub<false>(y), code_sub<true>(x), code_sub<true>(y)};
              mma_f16_16816_from(acc, a0, qf[w][0], qf[w][1], corr[w]);
              x >>= 8;
              y >>= 8;
              const uint32_t a1[4] = {code_sub<false>(x), code_sub<false>(y), code_sub<true>(x), code_sub<true>(y)};
              mma_f16_16816(acc, a1, qf[w][2], qf[w][3]);
              const float fx = scale_of<w>(sx), fy = scale_of<w>(sy);
              s[sb][0] = w == 0 ? acc[0] * fx : fmaf(acc[0], fx, s[sb][0]);
              s[sb][1] = w == 0 ? acc[1] * fx : fmaf(acc[1], fx, s[sb][1]);
              s[sb][2] = w == 0 ? acc[2] * fy : fmaf(acc[2], fy, s[sb][2]);
              s[sb][3] = w == 0 ? acc[3] * fy : fmaf(acc[3], fy, s[sb][3]);
            };
            group(std::integral_constant<int, 0>{}, x4.x, y4.x);
            group(std::integral_constant<int, 1>{}, x4.y, y4.y);
            group(std::integral_constant<int, 2>{}, x4.z, y4.z);
            group(std::integral_constant<int, 3>{}, x4.w, y4.w);
          }
          const bool done = half == 1 || lim <= 32;  // no more tokens in this tile
          if (done) {
            __syncwarp();  // every lane has read the K buffer
            if (lhas) {
              next_rec = record();
              load_k(next_rec);
            }
          }

          // ---- online softmax in the log2 domain
          if (lim < 32) {
#pragma unroll
            for (int sb = 0; sb < 2; ++sb) {
              if (16 * sb + g >= lim) s[sb][0] = s[sb][1] = -INFINITY;
              if (16 * sb + g + 8 >= lim) s[sb][2] = s[sb][3] = -INFINITY;
            }
          }
          // The reference of the exponentials follows the maximum only when a score passes it by 2^6: p stays
          // below 2^6, and most halves need no shuffles and no rescaling.
          const float x0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])) * sl0;
          const float x1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3])) * sl1;
          float a0 = 1.f, a1 = 1.f;
          bool grow = __any_sync(0xffffffffu, x0 > m0 + 6.f || x1 > m1 + 6.f);
          if (grow) {
            float n0 = x0, n1 = x1;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
              n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
            }
            n0 = fmaxf(m0, n0);
            n1 = fmaxf(m1, n1);
            a0 = ex2(m0 - n0);
            a1 = ex2(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= a0;
            l1 *= a1;
          }
          const float r0 = 4.f - m0, r1 = 4.f - m1;  // 2^4 p
#pragma unroll
          for (int sb = 0; sb < 2; ++sb) {
            s[sb][0] = ex2(fmaf(s[sb][0], sl0, r0));
            s[sb][1] = ex2(fmaf(s[sb][1], sl1, r1));
            s[sb][2] = ex2(fmaf(s[sb][2], sl0, r0));
            s[sb][3] = ex2(fmaf(s[sb][3], sl1, r1));
          }
          if (lim < 32) {  // also where a scale of 0 makes -inf * 0 a NaN
#pragma unroll
            for (int sb = 0; sb < 2; ++sb) {
              if (16 * sb + g >= lim) s[sb][0] = s[sb][1] = 0.f;
              if (16 * sb + g + 8 >= lim) s[sb][2] = s[sb][3] = 0.f;
            }
          }
          l0 += (s[0][0] + s[0][2]) + (s[1][0] + s[1][2]);
          l1 += (s[0][1] + s[0][3]) + (s[1][1] + s[1][3]);

          if (half == 0) {
            if (!warp_wait(&sm.vfull[warp], ph, a.err, abort)) {
              dead = true;
              kph = lhas && done ? ph ^ 1 : ph;
              lhas = false;
              break;
            }
            // The tile's largest V scale (they are not negative: their bits order as they do); lane: tokens
            // 2 lane and 2 lane + 1.  Behind the context a scale may be anything: it becomes zero.
            uint4 x = *(reinterpret_cast<const uint4*>(sm.v[warp] + kKv4Codes) + lane);
            if (lim < kKv4Tile) {
              if (2 * lane >= lim) x.x = x.y = 0;
              if (2 * lane + 1 >= lim) x.z = x.w = 0;
            }
            const uint32_t big = max(max(max(x.x, x.y), max(x.z, x.w)),
                                     max(max(x.x << 16, x.y << 16), max(x.z << 16, x.w << 16)));
            const int e = (int)(__reduce_max_sync(0xffffffffu, big) >> 23);
            if (e > ev) {
              const float f = ex2((float)(ev - e));
              a0 *= f;
              a1 *= f;
              ev = e;
              grow = true;
            }
            const float cv = __uint_as_float((uint32_t)(258 - ev) << 23);
            const uint2 ta = make_uint2(x.x, x.y), tb = make_uint2(x.z, x.w);
            sm.vpair[warp][lane] = make_uint4(pack_f16(scale_of<0>(ta) * cv, scale_of<0>(tb) * cv),
                                              pack_f16(scale_of<1>(ta) * cv, scale_of<1>(tb) * cv),
                                              pack_f16(scale_of<2>(ta) * cv, scale_of<2>(tb) * cv),
                                              pack_f16(scale_of<3>(ta) * cv, scale_of<3>(tb) * cv));
            __syncwarp();
          }
          if (grow) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[j][0] *= a0;
              o[j][1] *= a1;
              o[j][2] *= a0;
              o[j][3] *= a1;
            }
          }

          // ---- O^T += V^T P^T
          const uint8_t* vb = sm.v[warp] + half * 2048;
#pragma unroll
          for (int sb = 0; sb < 2; ++sb) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + lane * 16);        // tokens 2c, 2c + 1
            const uint4 y4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + 512 + lane * 16);  // ... + 8
            const uint4 sx = sm.vpair[warp][(2 * half + sb) * 8 + c], sy = sm.vpair[warp][(2 * half + sb) * 8 + 4 + c];
            const uint32_t px = movmatrix_trans(pack_f16(s[sb][0], s[sb][1]));  // head g, tokens 2c, 2c + 1
            const uint32_t py = movmatrix_trans(pack_f16(s[sb][2], s[sb][3]));  // ... + 8
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
          if (done) break;
        }
        if (dead) break;
        ph ^= 1;
        __syncwarp();  // every lane has read the V buffer
        if (lhas) load_v(next_rec);
      }

      // ---- end of the segment: the team's warps meet in shared memory
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      const float down = __uint_as_float((uint32_t)(ev - 4) << 23) + (ev == 4 ? 0x1p-127f : 0.f);
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // o[j][e], o[j][2 + e]: dims 16 j + 2g and + 1 of head 2c + e
        const int hd = 2 * c + e;
        if (hd < G) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float2*>(&sm.red_o[warp][hd][16 * j + 2 * g]) =
                make_float2(o[j][e] * down, o[j][2 + e] * down);
          if (g == 0) *reinterpret_cast<float2*>(sm.red_ml[warp][hd]) = make_float2(e ? m1 : m0, e ? l1 : l0);
        }
      }
      team_sync(team, tsh);
      const bool whole = cs.t0 == 0 && cs.t1 == cs.n;
      const uint32_t slot = 2 * k + (cs.t0 == 0);
      for (int hd = wt; hd < G; hd += T) {
        Kv4Acc acc;
        for (int w = team << tsh; w < (team + 1) << tsh; ++w)
          acc.add(sm.red_ml[w][hd][0], sm.red_ml[w][hd][1], reinterpret_cast<const float4*>(sm.red_o[w][hd])[lane]);
        if (whole) {
          reinterpret_cast<uint2*>(a.out + (qh0 + hd) * 128)[lane] = acc.result();
        } else {
          reinterpret_cast<float4*>(a.ws_o)[((int64_t)slot * G + hd) * 32 + lane] = acc.o;
          if (lane == 0) reinterpret_cast<float2*>(a.ws_ml)[(int64_t)slot * G + hd] = make_float2(acc.m, acc.l);
        }
      }
      if (!whole) {
        // The item's first unit lies in run k0, its last in run k0 + parts - 1; the last of them to get
        // here merges: run k0's tail (slot 2 k0 + 1), then the heads of the others (2 k), in this order
        // within each of `sl` slices that the team's warps share out.
        const uint32_t first = cs.u - (cs.t0 >> tsh);
        const uint32_t k0 = first / chunk;
        const int parts = (int)((first + ((uint32_t)(cs.n + T - 1) >> tsh) - 1) / chunk - k0) + 1;
        __threadfence();
        team_sync(team, tsh);
        if (wt == 0 && lane == 0) sm.last[team] = atomicInc(a.cnt + k0, parts - 1) == (unsigned)(parts - 1);
        team_sync(team, tsh);
        if (sm.last[team]) {
          __threadfence();
          const int sl = max(T / G, 1);  // a power of two, as T and G are
          for (int hs = wt; hs < G * sl; hs += T) {
            const int hd = hs % G;
            Kv4Acc acc;
#pragma unroll 4
            for (int p = hs / G; p < parts; p += sl) {
              const int64_t at = (int64_t)(2 * (k0 + p) + (p == 0)) * G + hd;
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + at);
              acc.add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(a.ws_o) + at * 32 + lane));
            }
            if (sl == 1) {
              reinterpret_cast<uint2*>(a.out + (qh0 + hd) * 128)[lane] = acc.result();
            } else {
              reinterpret_cast<float4*>(sm.red_o[warp][0])[lane] = acc.o;
              if (lane == 0) *reinterpret_cast<float2*>(sm.red_ml[warp][0]) = make_float2(acc.m, acc.l);
            }
          }
          if (sl > 1) {
            team_sync(team, tsh);
            if (wt < G) {
              Kv4Acc acc;
              for (int i = 0; i < sl; ++i) {
                const int w = warp + i * G;
                acc.add(sm.red_ml[w][0][0], sm.red_ml[w][0][1], reinterpret_cast<const float4*>(sm.red_o[w][0])[lane]);
              }
              reinterpret_cast<uint2*>(a.out + (qh0 + wt) * 128)[lane] = acc.result();
            }
          }
        }
      }
      team_sync(team, tsh);  // the team's shared buffers are read
      if (!kv4_next(a, sm, cs, uend, tsh)) break;
    }
    if (dead) {  // copies in flight land (or run out of time once more) before the CTA ends
      mbar_wait(&sm.kfull[warp], kph, a.err, nullptr);
      mbar_wait(&sm.vfull[warp], ph, a.err, nullptr);
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
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: pointers must be 16-byte aligned");
  const int64_t need = aacc_kv4_decode_workspace_bytes(num_q_heads, num_kv_heads);
  if (!workspace || workspace_bytes < need)
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: workspace %lld < %lld bytes", (long long)workspace_bytes,
                     (long long)need);
  if (max_context > max_blocks * block_size) max_context = max_blocks * block_size;
  if (max_context > 0x7fffffc0) max_context = 0x7fffffc0;
  // Units are counted in 32 bits.
  if (batch > 0x7fffffff || num_rows > 0x7ffffffe ||
      (double)batch * num_kv_heads * (double)((max_context + kKv4Tile - 1) / kKv4Tile) > 2147483647.0)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_decode_attention: %lld rows of up to %lld tokens are too many",
                     (long long)batch, (long long)max_context);
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
