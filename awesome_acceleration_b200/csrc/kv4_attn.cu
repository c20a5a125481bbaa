// Decode attention over the 4-bit paged KV cache (format: kv4.cuh).
//
//   out[b][h] = sum_t softmax_t(scale q.k_t) v_t,  k_t = s n (4 groups of 32 dims)
//
// The floor is 144 bytes per (token, kv head) from HBM.  At that rate an SM
// has about 400 cycles per 64 tokens, so the expansion of the codes has to
// stay near one instruction a value, and there is no time for barriers.
//
// Work: the unit is a tile of 64 tokens of one (row, kv head), an item is all
// tiles of one (row, kv head).  The kernel is persistent: one CTA of 16 warps
// per SM, grouped into teams of TEAM warps; the N units of the batch, which
// every CTA counts itself from seqlens, are cut into equal runs, one per team,
// whatever the rows' lengths are.  A run that ends inside an item leaves an
// fp32 partial (max, sum, O); the last team of the item to arrive merges the
// partials in order.
//
// Tiles: each warp streams its own tiles through one K and one V buffer with
// bulk copies (lane 0 issues; the next K is fetched during softmax and P.V,
// the next V during the next Q.K), so warps never wait for one another.
//
// Q.K: the tile's tokens are the rows of m16n8k16's A operand, the G <= 8
// query heads its 8 columns.  A code u becomes the bf16 16 + u by one shift
// and one and-or; 24 sum(q) is taken off through the accumulator's start value,
// which leaves sum(q n) in fp32.  The group's scale multiplies the fp32 sum.
// P.V: O^T = V^T P^T with V^T (dims x tokens) as the A operand, whose values
// are 128 + u - 136, exact in bf16; the V scale of (token, group) multiplies p
// in fp32, and the product is rounded once to bf16, the only rounding before
// the output's (as P alone is in the bf16 kernels).
#include "host.h"
#include "kv4.cuh"

namespace aacc {

constexpr int kAttWarps = 16;
constexpr int kAttThreads = kAttWarps * 32;

template <int G, int TEAM>
struct Kv4Smem {
  uint8_t k[kAttWarps][kKv4Record];
  uint8_t v[kAttWarps][kKv4Record];
  float red_o[TEAM > 1 ? kAttWarps : 1][G][128];
  float red_ml[TEAM > 1 ? kAttWarps : 1][G][2];
  int64_t pre[kAttThreads];
  int64_t wsum[kAttWarps];
  uint64_t kfull[kAttWarps];
  uint64_t vfull[kAttWarps];
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
  int64_t num_blocks, num_rows, max_blocks, batch;
  int max_ctx, ctx_add, Hkv, tpb;  // tpb: tiles per block
  float scale;
};

// A run of tiles [t0, t1) of item (b, h), whose row has n tiles; u is the unit number of t0.
struct Kv4Seg {
  int64_t u, b, row;
  int h, n, t0, t1, ctx;
};

// Tokens of batch row b (0: padding, outside the tables, or empty).
__device__ __forceinline__ int kv4_ctx(const Kv4Args& a, int64_t b, int64_t* row) {
  const int64_t r = a.rows[b];
  *row = r;
  if (r < 0 || r >= a.num_rows) return 0;
  const int64_t c = (int64_t)a.seqlens[r] + a.ctx_add;
  return (int)max((int64_t)0, min(c, (int64_t)a.max_ctx));
}

__device__ __forceinline__ void kv4_row(const Kv4Args& a, Kv4Seg& s) {
  s.ctx = kv4_ctx(a, s.b, &s.row);
  s.n = (s.ctx + kKv4Tile - 1) / kKv4Tile;
}

// The run's next segment; false when the run is over.
__device__ __forceinline__ bool kv4_next(const Kv4Args& a, Kv4Seg& s, int64_t uend) {
  s.u += s.t1 - s.t0;
  if (s.u >= uend) return false;
  s.t0 = 0;  // within a run only its end cuts an item short
  if (++s.h == a.Hkv) {
    s.h = 0;
    do {
      ++s.b;
      kv4_row(a, s);
    } while (s.n == 0);
  }
  s.t1 = (int)min((int64_t)s.n, uend - s.u);
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
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Nibbles R and R + 4 of x as the bf16 pair (16 + u, 16 + u').
template <int R>
__device__ __forceinline__ uint32_t code16(uint32_t x) {
  const uint32_t y = R == 0 ? x << 3 : x >> (4 * R - 3);
  return (y & 0x00780078u) | 0x41804180u;
}

// Nibbles R and R + 4 of x as the bf16 pair (u - 8, u' - 8).
template <int R>
__device__ __forceinline__ uint32_t code_exact(uint32_t x) {
  const uint32_t y = ((x >> (4 * R)) & 0x000f000fu) | 0x43004300u;  // 128 + u
  const __nv_bfloat162 off = __float2bfloat162_rn(-136.f);
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&y), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int TEAM>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (TEAM == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM * 32) : "memory");
}

// Merge the parts of an item (team k0's tail, then the heads of k0 + 1 .. k0 + parts - 1) in order.
template <int G, int TEAM>
__device__ __forceinline__ void kv4_merge(const Kv4Args& a, int64_t k0, int parts, int64_t qh0, int tid) {
  for (int i = tid; i < G * 32; i += TEAM * 32) {
    const int g = i >> 5, d4 = i & 31;
    float M = -INFINITY;
    for (int p = 0; p < parts; ++p) {
      const int64_t slot = 2 * (k0 + p) + (p == 0);
      M = fmaxf(M, __ldcg(a.ws_ml + (slot * G + g) * 2));
    }
    const float mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < parts; ++p) {
      const int64_t slot = 2 * (k0 + p) + (p == 0);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + slot * G + g);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(a.ws_o) + (slot * G + g) * 32 + d4);
      const float f = ex2(ml.x - mu);
      L += f * ml.y;
      O.x += f * o.x;
      O.y += f * o.y;
      O.z += f * o.z;
      O.w += f * o.w;
    }
    const float inv = 1.f / L;
    reinterpret_cast<uint2*>(a.out + (qh0 + g) * 128)[d4] =
        make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
  }
}

template <int G, int TEAM>
__global__ void __launch_bounds__(kAttThreads, 1) kv4_decode_kernel(const Kv4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Smem = Kv4Smem<G, TEAM>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int team = warp / TEAM, wt = warp % TEAM;
  if (lane == 0) {
    mbar_init(&sm.kfull[warp], 1);
    mbar_init(&sm.vfull[warp], 1);
    if (warp == 0) sm.abort = 0;
    fence_mbar_init();
  }
  griddep_wait();
  griddep_launch();

  // ---- count the batch's units: every thread sums a run of rows, then a scan over the CTA
  const int64_t per = (a.batch + kAttThreads - 1) / kAttThreads;
  int64_t mine = 0;
  for (int64_t b = threadIdx.x * per; b < min(a.batch, (threadIdx.x + 1) * per); ++b) {
    int64_t row;
    mine += (kv4_ctx(a, b, &row) + kKv4Tile - 1) / kKv4Tile;
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sm.wsum[warp] = inc;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kAttWarps; ++w) {
    const int64_t x = sm.wsum[w];
    if (w < warp) before += x;
    total += x;
  }
  sm.pre[threadIdx.x] = before + inc - mine;
  __syncthreads();

  // ---- this team's run of units
  constexpr int kTeams = kAttWarps / TEAM;
  const int64_t N = total * a.Hkv;
  const int64_t teams = (int64_t)gridDim.x * kTeams;
  const int64_t chunk = max((N + teams - 1) / teams, (int64_t)TEAM);
  const int64_t k = (int64_t)team * gridDim.x + blockIdx.x;  // runs go round the SMs, so few runs use many of them
  const int64_t u0 = k * chunk, uend = min(u0 + chunk, N);
  uint32_t ph = 0;                 // parity of the tile in hand, for both buffers
  bool dead = false;               // a copy did not come in time: no more loads, no more tiles
  uint32_t kph = 0;                // then: the parity that the K buffer still waits for
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
      int64_t u = sm.pre[lo] * a.Hkv;
      cs.b = lo * per;
      kv4_row(a, cs);
      while (u + (int64_t)cs.n * a.Hkv <= u0) {
        u += (int64_t)cs.n * a.Hkv;
        ++cs.b;
        kv4_row(a, cs);
      }
      cs.u = u0;
      cs.h = (int)((u0 - u) / cs.n);
      cs.t0 = (int)((u0 - u) - (int64_t)cs.h * cs.n);
      cs.t1 = (int)min((int64_t)cs.n, cs.t0 + (uend - u0));
    }
    // The loads run one tile ahead of the arithmetic, across segments.
    Kv4Seg ls = cs;
    int lt = ls.t0 + wt;
    bool lhas = true;
    while (lhas && lt >= ls.t1) {
      lhas = kv4_next(a, ls, uend);
      lt = ls.t0 + wt;
    }
    auto record = [&](int32_t id) -> int64_t {
      int64_t blk = id;
      if (blk < 0 || blk >= a.num_blocks) {
        if (lane == 0) report(a.err, ERR_BLOCK_OOB);
        blk = 0;  // a valid address keeps the pipeline going; the result is flagged
      }
      return kv4_record(blk, ls.h, lt % a.tpb, a.Hkv, a.tpb);
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
    if (lhas) {
      const int64_t rec = record(a.bt[ls.row * a.max_blocks + lt / a.tpb]);
      load_k(rec);
      load_v(rec);
    }
    const float sl = fabsf(a.scale) * kLog2e;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns q's sign

    while (true) {
      // ---- queries of the item: B operand, column g = query head (columns >= G are zero)
      const int64_t qh0 = (cs.b * a.Hkv + cs.h) * G;
      uint32_t qf[4][4];
      float corr[4][2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (g < G) x = *reinterpret_cast<const uint4*>(a.q + (qh0 + g) * 128 + 32 * w + 8 * c);
        qf[w][0] = x.x ^ flip;
        qf[w][1] = x.y ^ flip;
        qf[w][2] = x.z ^ flip;
        qf[w][3] = x.w ^ flip;
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 f = unpack_bf16(qf[w][r]);
          s += f.x + f.y;
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        corr[w][0] = -24.f * __shfl_sync(0xffffffffu, s, 8 * c);      // head 2c
        corr[w][1] = -24.f * __shfl_sync(0xffffffffu, s, 8 * c + 4);  // head 2c + 1
      }
      float o[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

      for (int t = cs.t0 + wt; t < cs.t1 && !dead; t += TEAM) {
        // the next tile's block id, in flight during Q.K
        lt += TEAM;
        while (lhas && lt >= ls.t1) {
          lhas = kv4_next(a, ls, uend);
          lt = ls.t0 + wt;
        }
        const int32_t next_id = lhas ? a.bt[ls.row * a.max_blocks + lt / a.tpb] : 0;

        // ---- S = K Q^T
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.kfull[warp], ph, a.err, abort))) {
          dead = true;
          kph = ph;
          lhas = false;
          break;
        }
        const uint8_t* kb = sm.k[warp];
        float s[4][4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
          const uint4 x4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + lane * 16);        // token g
          const uint4 y4 = *reinterpret_cast<const uint4*>(kb + sb * 1024 + 512 + lane * 16);  // token g + 8
          const uint2 sx = *reinterpret_cast<const uint2*>(kb + kKv4Codes + (16 * sb + g) * 8);
          const uint2 sy = *reinterpret_cast<const uint2*>(kb + kKv4Codes + (16 * sb + g + 8) * 8);
          const uint32_t xw[4] = {x4.x, x4.y, x4.z, x4.w}, yw[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float acc[4] = {corr[w][0], corr[w][1], corr[w][0], corr[w][1]};
            const uint32_t a0[4] = {code16<0>(xw[w]), code16<0>(yw[w]), code16<1>(xw[w]), code16<1>(yw[w])};
            mma_bf16_16816(acc, a0, qf[w][0], qf[w][1]);
            const uint32_t a1[4] = {code16<2>(xw[w]), code16<2>(yw[w]), code16<3>(xw[w]), code16<3>(yw[w])};
            mma_bf16_16816(acc, a1, qf[w][2], qf[w][3]);
            const uint32_t px = w < 2 ? sx.x : sx.y, py = w < 2 ? sy.x : sy.y;
            const float fx = __uint_as_float((w & 1) ? px & 0xffff0000u : px << 16);
            const float fy = __uint_as_float((w & 1) ? py & 0xffff0000u : py << 16);
            if (w == 0) {
              s[sb][0] = acc[0] * fx;
              s[sb][1] = acc[1] * fx;
              s[sb][2] = acc[2] * fy;
              s[sb][3] = acc[3] * fy;
            } else {
              s[sb][0] += acc[0] * fx;
              s[sb][1] += acc[1] * fx;
              s[sb][2] += acc[2] * fy;
              s[sb][3] += acc[3] * fy;
            }
          }
        }
        __syncwarp();  // every lane has read the K buffer
        int64_t next_rec = 0;
        if (lhas) {
          next_rec = record(next_id);
          load_k(next_rec);
        }

        // ---- online softmax, log2 domain; lane (g, c): tokens 16 sb + g (+ 8), heads 2c and 2c + 1
        const int lim = cs.ctx - t * kKv4Tile;
        if (lim < kKv4Tile) {
#pragma unroll
          for (int sb = 0; sb < 4; ++sb) {
            if (16 * sb + g >= lim) s[sb][0] = s[sb][1] = -INFINITY;
            if (16 * sb + g + 8 >= lim) s[sb][2] = s[sb][3] = -INFINITY;
          }
        }
        float x0 = s[0][0], x1 = s[0][1];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
          x0 = fmaxf(x0, fmaxf(s[sb][0], s[sb][2]));
          x1 = fmaxf(x1, fmaxf(s[sb][1], s[sb][3]));
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        const float n0 = fmaxf(m0, x0 * sl), n1 = fmaxf(m1, x1 * sl);  // a tile has a token: finite
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
          const float a0 = ex2(m0 - n0), a1 = ex2(m1 - n1);
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[j][0] *= a0;
            o[j][1] *= a1;
            o[j][2] *= a0;
            o[j][3] *= a1;
          }
          m0 = n0;
          m1 = n1;
        }
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
          s[sb][0] = ex2(fmaf(s[sb][0], sl, -m0));
          s[sb][1] = ex2(fmaf(s[sb][1], sl, -m1));
          s[sb][2] = ex2(fmaf(s[sb][2], sl, -m0));
          s[sb][3] = ex2(fmaf(s[sb][3], sl, -m1));
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.vfull[warp], ph, a.err, abort))) {
          dead = true;
          kph = lhas ? ph ^ 1 : ph;
          lhas = false;
          break;
        }
        ph ^= 1;
        if (lim < kKv4Tile) {
          // Behind the context: no weight (also where sl = 0 makes -inf * sl a NaN), and no V scale,
          // which may be anything there.
#pragma unroll
          for (int sb = 0; sb < 4; ++sb) {
            if (16 * sb + g >= lim) s[sb][0] = s[sb][1] = 0.f;
            if (16 * sb + g + 8 >= lim) s[sb][2] = s[sb][3] = 0.f;
          }
          for (int i = lane; i < kKv4Tile; i += 32)
            if (i >= lim) *reinterpret_cast<uint2*>(sm.v[warp] + kKv4Codes + 8 * i) = make_uint2(0, 0);
          fence_proxy_async();  // before the bulk copy that overwrites the buffer
          __syncwarp();
        }
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
          l0 += s[sb][0] + s[sb][2];
          l1 += s[sb][1] + s[sb][3];
        }

        // ---- O^T += V^T P^T
        const uint8_t* vb = sm.v[warp];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
          const uint4 x4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + lane * 16);        // tokens 2c, 2c + 1
          const uint4 y4 = *reinterpret_cast<const uint4*>(vb + sb * 1024 + 512 + lane * 16);  // ... + 8
          const uint2 sx = *reinterpret_cast<const uint2*>(vb + kKv4Codes + (16 * sb + g) * 8);
          const uint2 sy = *reinterpret_cast<const uint2*>(vb + kKv4Codes + (16 * sb + g + 8) * 8);
#pragma unroll
          for (int w = 0; w < 4; ++w) {  // 32 dims: j = 2w and 2w + 1
            const uint32_t px = w < 2 ? sx.x : sx.y, py = w < 2 ? sy.x : sy.y;
            const float fx = __uint_as_float((w & 1) ? px & 0xffff0000u : px << 16);
            const float fy = __uint_as_float((w & 1) ? py & 0xffff0000u : py << 16);
            const uint32_t b0 = movmatrix_trans(pack_bf16(s[sb][0] * fx, s[sb][1] * fx));
            const uint32_t b1 = movmatrix_trans(pack_bf16(s[sb][2] * fy, s[sb][3] * fy));
            // the words' 16 bits of tokens 2c | 2c + 1: four nibbles = dims 16 j + 2g, + 1 of j = 2w, 2w + 1
            const uint32_t sel = (w & 1) ? 0x7632u : 0x5410u;
            const uint32_t lo = w < 2 ? __byte_perm(x4.x, x4.z, sel) : __byte_perm(x4.y, x4.w, sel);
            const uint32_t hi = w < 2 ? __byte_perm(y4.x, y4.z, sel) : __byte_perm(y4.y, y4.w, sel);
            const uint32_t a0[4] = {code_exact<0>(lo), code_exact<1>(lo), code_exact<0>(hi), code_exact<1>(hi)};
            mma_bf16_16816(o[2 * w], a0, b0, b1);
            const uint32_t a1[4] = {code_exact<2>(lo), code_exact<3>(lo), code_exact<2>(hi), code_exact<3>(hi)};
            mma_bf16_16816(o[2 * w + 1], a1, b0, b1);
          }
        }
        __syncwarp();  // every lane has read the V buffer
        if (lhas) load_v(next_rec);
      }

      // ---- end of the segment
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      const bool whole = cs.t0 == 0 && cs.t1 == cs.n;
      const int64_t slot = 2 * k + (cs.t0 == 0);
      if constexpr (TEAM == 1) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // heads 2c and 2c + 1; o[j][e], o[j][2 + e] are dims 16 j + 2g, + 1
          const int hd = 2 * c + e;
          if (hd < G) {
            const float inv = 1.f / (e ? l1 : l0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int d = 16 * j + 2 * g;
              if (whole)
                *reinterpret_cast<uint32_t*>(a.out + (qh0 + hd) * 128 + d) = pack_bf16(o[j][e] * inv, o[j][2 + e] * inv);
              else
                *reinterpret_cast<float2*>(a.ws_o + (slot * G + hd) * 128 + d) = make_float2(o[j][e], o[j][2 + e]);
            }
            if (!whole && g == 0)
              reinterpret_cast<float2*>(a.ws_ml)[slot * G + hd] = make_float2(e ? m1 : m0, e ? l1 : l0);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int hd = 2 * c + e;
          if (hd < G) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float2*>(&sm.red_o[warp][hd][16 * j + 2 * g]) = make_float2(o[j][e], o[j][2 + e]);
            if (g == 0) {
              sm.red_ml[warp][hd][0] = e ? m1 : m0;
              sm.red_ml[warp][hd][1] = e ? l1 : l0;
            }
          }
        }
        team_sync<TEAM>(team);
        for (int i = wt * 32 + lane; i < G * 32; i += TEAM * 32) {
          const int hd = i >> 5, d4 = i & 31;
          float M = -INFINITY;
#pragma unroll
          for (int w = 0; w < TEAM; ++w) M = fmaxf(M, sm.red_ml[team * TEAM + w][hd][0]);
          const float mu = M == -INFINITY ? 0.f : M;
          float L = 0.f;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < TEAM; ++w) {
            const float f = ex2(sm.red_ml[team * TEAM + w][hd][0] - mu);
            const float4 x = reinterpret_cast<const float4*>(sm.red_o[team * TEAM + w][hd])[d4];
            L += f * sm.red_ml[team * TEAM + w][hd][1];
            O.x += f * x.x;
            O.y += f * x.y;
            O.z += f * x.z;
            O.w += f * x.w;
          }
          if (whole) {
            const float inv = 1.f / L;
            reinterpret_cast<uint2*>(a.out + (qh0 + hd) * 128)[d4] =
                make_uint2(pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv));
          } else {
            reinterpret_cast<float4*>(a.ws_o)[(slot * G + hd) * 32 + d4] = O;
            if (d4 == 0) reinterpret_cast<float2*>(a.ws_ml)[slot * G + hd] = make_float2(M, L);
          }
        }
      }
      if (!whole) {
        // The item's first unit lies in run k0, its last in run k1; the last of them to get here merges.
        const int64_t first = cs.u - cs.t0;
        const int64_t k0 = first / chunk;
        const int parts = (int)((first + cs.n - 1) / chunk - k0) + 1;
        __threadfence();
        team_sync<TEAM>(team);
        if (wt == 0 && lane == 0) sm.last[warp] = atomicInc(a.cnt + k0, parts - 1) == (unsigned)(parts - 1);
        team_sync<TEAM>(team);
        if (sm.last[team * TEAM]) {
          __threadfence();
          kv4_merge<G, TEAM>(a, k0, parts, qh0, wt * 32 + lane);
        }
      }
      team_sync<TEAM>(team);  // the team's shared buffers are read
      if (!kv4_next(a, cs, uend)) break;
    }
    if (dead) {  // copies in flight land (or run out of time once more) before the CTA ends
      mbar_wait(&sm.kfull[warp], kph, a.err, nullptr);
      mbar_wait(&sm.vfull[warp], ph, a.err, nullptr);
    }
  }

  // ---- rows without tokens are zero; rows out of bounds are reported
  for (int64_t b = blockIdx.x + (int64_t)warp * gridDim.x; b < a.batch; b += (int64_t)kAttWarps * gridDim.x) {
    int64_t row;
    const int ctx = kv4_ctx(a, b, &row);
    if (lane == 0 && row >= a.num_rows) report(a.err, ERR_SLOT_OOB);
    if (lane == 0 && ctx > 0 && (int64_t)a.seqlens[row] + a.ctx_add > a.max_ctx) report(a.err, ERR_CTX_OOB);
    if (ctx == 0)
      for (int i = lane; i < a.Hkv * G * 16; i += 32)
        reinterpret_cast<uint4*>(a.out + b * a.Hkv * G * 128)[i] = make_uint4(0, 0, 0, 0);
  }
}

// Workspace: counters of every team a device can have (TEAM = 1), then two partials per team.
static int64_t kv4_teams() { return (int64_t)sm_count() * kAttWarps; }
static int64_t kv4_counter_bytes() { return (kv4_teams() * 4 + 255) / 256 * 256; }

template <int G, int TEAM>
static cudaError_t kv4_launch(const Kv4Args& a, cudaStream_t stream) {
  const size_t smem = sizeof(Kv4Smem<G, TEAM>);
  set_smem_once<kv4_decode_kernel<G, TEAM>>((int)smem);
  return launch_k(kv4_decode_kernel<G, TEAM>, dim3(sm_count()), dim3(kAttThreads), smem, stream, a);
}

template <int G>
static cudaError_t kv4_pick(const Kv4Args& a, cudaStream_t stream) {
  const int64_t items = a.batch * a.Hkv;
  if (items >= 256) return kv4_launch<G, 1>(a, stream);
  if (items >= 64) return kv4_launch<G, 4>(a, stream);
  return kv4_launch<G, 16>(a, stream);
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
  a.num_blocks = num_blocks;
  a.num_rows = num_rows;
  a.max_blocks = max_blocks;
  a.batch = batch;
  a.max_ctx = (int)max_context;
  a.ctx_add = ctx_add;
  a.Hkv = num_kv_heads;
  a.tpb = block_size / kKv4Tile;
  a.scale = scale;
  cudaError_t le;
  switch (G) {
    case 1: le = kv4_pick<1>(a, stream); break;
    case 2: le = kv4_pick<2>(a, stream); break;
    case 4: le = kv4_pick<4>(a, stream); break;
    default: le = kv4_pick<8>(a, stream); break;
  }
  return check_launch("kv4_decode_kernel", le);
}

}  // extern "C"
