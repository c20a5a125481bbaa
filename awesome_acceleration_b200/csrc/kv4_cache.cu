// Storing into and loading from the 4-bit paged KV cache (format: kv4.cuh).
//
// Both move each byte once: per (token, kv head) 512 bytes of bf16 K and V on
// one side, 144 bytes of codes and scales on the other.
#include "host.h"
#include "kv4.cuh"

namespace aacc {

// 4x4 byte transpose over the lanes {i, i^2, i^4, i^6}: with b = (lane / 2) % 4,
// lane b's byte k becomes byte b of lane k.  Its own inverse.
__device__ __forceinline__ uint32_t transpose4(uint32_t w, int lane) {
  uint32_t y = __shfl_xor_sync(0xffffffffu, w, 4);
  w = (lane & 4) ? __byte_perm(w, y, 0x3276) : __byte_perm(w, y, 0x5410);
  y = __shfl_xor_sync(0xffffffffu, w, 2);
  return (lane & 2) ? __byte_perm(w, y, 0x3715) : __byte_perm(w, y, 0x6240);
}

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994): with 2^(L-1) < d <= 2^L and
// m = ceil(2^(31+L) / d), floor(n / d) = floor(n m / 2^(31+L)).
struct Divide {
  uint32_t d, m, sh;
  explicit Divide(uint32_t d_) : d(d_), m(0), sh(0) {
    if (d == 1) return;
    uint32_t L = 1;
    while ((uint64_t(1) << L) < d) ++L;
    m = (uint32_t)(((uint64_t(1) << (31 + L)) + d - 1) / d);
    sh = L - 1;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return m ? __umulhi(n, m) >> sh : n; }
};

// Work of both kernels: a warp takes two tokens, lanes 0-15 the first and
// 16-31 the second, and `hpw` heads of them, 8 dims a lane.  Two tokens that
// follow one another share the 16-byte pieces of V's layout, so each store
// instruction fills them whole.
//
// Measured, 32768 tokens of 8 heads (172 MB: 26.6 us at a copy's rate): store
// 34 us (5.1 TB/s), load 30 us (5.8 TB/s).  The load is bound by memory.  The
// store issues about 100 instructions per 8 values, in 70 % of all cycles,
// and needs warps behind them: 48 of 40 registers, one head at a time, beat
// 32 that load two heads together (37 us).  The load needs loads in flight:
// four heads together (one: 33 us).  CTAs of 4 warps leave finer holes than 8
// (35 and 30.5 us).
constexpr int kLoadHeads = 4;
constexpr int kMoveWarps = 4;
constexpr int kMoveThreads = kMoveWarps * 32;

struct Kv4Pair {
  int64_t t, rec0;  // token of this half warp; byte offset of its record for head 0
  int tt, h0, h1;
  bool on;
};

__device__ __forceinline__ Kv4Pair kv4_pair(int64_t T, int Hkv, int hpw, Divide groups, Divide bs,
                                            uint32_t num_slots, const int64_t* slots, unsigned* err) {
  Kv4Pair p;
  const uint32_t warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const uint32_t pair = groups(warp);
  p.h0 = (int)(warp - pair * groups.d) * hpw;
  p.h1 = min(p.h0 + hpw, Hkv);
  p.t = 2 * (int64_t)pair + ((threadIdx.x >> 4) & 1);
  int64_t slot = p.t < T ? slots[p.t] : -1;
  if (slot >= num_slots) {
    report(err, ERR_SLOT_OOB);
    slot = -1;
  }
  p.on = slot >= 0;
  const uint32_t u = p.on ? (uint32_t)slot : 0, blk = bs(u), off = u - blk * bs.d;
  p.rec0 = kv4_record(blk, 0, off / kKv4Tile, Hkv, bs.d / kKv4Tile);
  p.tt = off % kKv4Tile;
  return p;
}

// Offset of lane i's word of token tt: K word 4 (i % 4) + i / 4 (dims 8 i ..), V word i / 8 of octet
// 4 (i % 2) + (i / 2) % 4 (after transpose4: dims 8 i ..).
__device__ __forceinline__ int kv4_k_word(int tt, int i) { return 64 * tt + 4 * (4 * (i & 3) + (i >> 2)); }
__device__ __forceinline__ int kv4_v_word(int tt, int i) {
  return kv4_v_base(tt) + 64 * (4 * (i & 1) + ((i >> 1) & 3)) + 4 * (i >> 3);
}

// 8 bf16 of a group of 32 that four lanes hold together: the group's scale, and each value's code u as bits
// 0-3 of code[e] (higher bits: those of 12582912.0f).
__device__ __forceinline__ uint32_t kv4_quantise(uint4 x4, uint32_t (&code)[8]) {
  const uint32_t x2[4] = {x4.x, x4.y, x4.z, x4.w};
  // max |x|; a NaN stays one.
  const __nv_bfloat162* xh = reinterpret_cast<const __nv_bfloat162*>(x2);
  __nv_bfloat162 m2 = __hmax2_nan(__hmax2_nan(__habs2(xh[0]), __habs2(xh[1])),
                                  __hmax2_nan(__habs2(xh[2]), __habs2(xh[3])));
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&m2), d);
    m2 = __hmax2_nan(m2, *reinterpret_cast<const __nv_bfloat162*>(&y));
  }
  const float mx = bf(__hmax_nan(__low2bfloat16(m2), __high2bfloat16(m2)));
  const bool finite = mx < INFINITY;
  // max / 7 has 8 bits over 7: it is exact or at least 1/14 of bf16's step off a rounding border, so the
  // product with the rounded 1/7 rounds as the quotient does.
  const uint32_t sbits = finite ? (uint32_t)__bfloat16_as_ushort(tobf(mx * (1.f / 7.f))) : 0x7fc0u;
  const float s = bf16_bits(sbits);
  // n = rint(x / s) as exact arithmetic has it.  x and s have 8 significant bits, so x / s >= 1/2 is exactly
  // k + 1/2 or at least 1/510 off it.  x times the approximate 1 / s is within 2^-19 of x / s; rounded to
  // multiples of 2^-12 an exact k + 1/2 is back in place and no other value crosses one.  |x / s| <= 7 + 2^-5
  // needs no clamp.  A subnormal s (or none) has fewer bits: divide and clamp there.
  if (finite && sbits >= 0x80u) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));  // 2^-126 <= s < 2^126: within 1 ulp
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 y = __ffma2_rn(unpack_bf16(x2[e >> 1]), make_float2(r, r), make_float2(0x1.8p11f, 0x1.8p11f));
      constexpr float kTo = 0x1.8p23f - 0x1.8p11f + 8.f;  // exact; the sum is rounded once, to an integer
      const float2 z = __fadd2_rn(y, make_float2(kTo, kTo));
      code[e] = __float_as_uint(z.x);
      code[e + 1] = __float_as_uint(z.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __uint_as_float((e & 1) ? x2[e >> 1] & 0xffff0000u : x2[e >> 1] << 16);
      const float n = (finite && s > 0.f) ? fminf(fmaxf(rintf(__fdiv_rn(x, s)), -7.f), 7.f) : 0.f;
      code[e] = __float_as_uint(n + 12582920.f);
    }
  }
  return sbits;
}

__global__ void __launch_bounds__(kMoveThreads, 12)
    kv4_store_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t T, int64_t ks, int64_t kh,
                     int64_t vs, int64_t vh, const int64_t* __restrict__ slots, uint8_t* __restrict__ kc,
                     uint8_t* __restrict__ vc, uint32_t num_slots, int Hkv, int hpw, Divide groups, Divide bs,
                     unsigned* err) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, i = lane & 15;
  const Kv4Pair p = kv4_pair(T, Hkv, hpw, groups, bs, num_slots, slots, err);
  const int64_t head_bytes = (int64_t)(bs.d / kKv4Tile) * kKv4Record;
  const int scale_at = kKv4Codes + 8 * p.tt + (i >> 1);
  kc += p.rec0;
  vc += p.rec0;
  k += p.t * ks + 8 * i;
  v += p.t * vs + 8 * i;
  k += p.h0 * kh;
  v += p.h0 * vh;
  uint8_t* kw = kc + p.h0 * head_bytes + kv4_k_word(p.tt, i);
  uint8_t* vw = vc + p.h0 * head_bytes + kv4_v_word(p.tt, i);
  uint8_t* kq = kc + p.h0 * head_bytes + scale_at;
  uint8_t* vq = vc + p.h0 * head_bytes + scale_at;
#pragma unroll 1
  for (int h = p.h0; h < p.h1; ++h, k += kh, v += vh) {
    const uint4 xk = p.on ? *reinterpret_cast<const uint4*>(k) : make_uint4(0, 0, 0, 0);
    const uint4 xv = p.on ? *reinterpret_cast<const uint4*>(v) : make_uint4(0, 0, 0, 0);
    uint32_t code[8];
    // sum_e code[e] 16^place(e) carries 0x4b400000 16^0..7 along: take it off at the end
    constexpr uint32_t carried = 0x4b400000u * 0x11111111u;
    const uint32_t sk = kv4_quantise(xk, code);
    uint32_t w = 0;  // nibble n holds dim 8 i + 2 (n % 4) + n / 4
#pragma unroll
    for (int n = 7; n >= 0; --n) w = w * 16 + code[2 * (n & 3) + (n >> 2)];
    const uint32_t wk = w - carried;
    const uint32_t sv = kv4_quantise(xv, code);
    w = 0;  // byte b holds dims 8 i + 2 b and + 1
#pragma unroll
    for (int e = 7; e >= 0; --e) w = w * 16 + code[e];
    w = transpose4(w - carried, lane);
    if (p.on) {
      *reinterpret_cast<uint32_t*>(kw) = wk;
      *reinterpret_cast<uint32_t*>(vw) = w;
      if ((i & 3) == 0) {
        *reinterpret_cast<uint16_t*>(kq) = (uint16_t)sk;
        *reinterpret_cast<uint16_t*>(vq) = (uint16_t)sv;
      }
    }
    kw += head_bytes, vw += head_bytes, kq += head_bytes, vq += head_bytes;
  }
}

// Codes u in bits 0-3 and 16-19 of x times the bf16 pair `s`: 128 + u - 136 is exact in bf16, so
// the product is rounded once, to the bf16 that n s rounds to.
__device__ __forceinline__ uint32_t kv4_value(uint32_t x, uint32_t s) {
  const uint32_t u = and_or<0x000f000fu>(x, 0x43004300u);
  const __nv_bfloat162 n = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(-136.f));
  const __nv_bfloat162 y = __hmul2(n, *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&y);
}

__global__ void __launch_bounds__(kMoveThreads, 10)
    kv4_load_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, uint32_t num_slots, int Hkv,
                    int hpw, Divide groups, Divide bs, const int64_t* __restrict__ slots,
                    const int64_t* __restrict__ out_slots, int64_t T, bf16* __restrict__ ko, bf16* __restrict__ vo,
                    uint32_t out_total, Divide out_bs, unsigned* err) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, i = lane & 15;
  Kv4Pair p = kv4_pair(T, Hkv, hpw, groups, bs, num_slots, slots, err);
  int64_t dst = p.on ? (out_slots ? out_slots[p.t] : p.t) : -1;
  if (dst >= out_total) {
    report(err, ERR_SLOT_OOB);
    dst = -1;
  }
  p.on = dst >= 0;
  const uint32_t u = p.on ? (uint32_t)dst : 0, ob = out_bs(u), oo = u - ob * out_bs.d;
  const int64_t out0 = ((int64_t)ob * Hkv * out_bs.d + oo) * 16 + i;  // in 16-byte pieces
  const int64_t head_bytes = (int64_t)(bs.d / kKv4Tile) * kKv4Record;
  const int scale_at = kKv4Codes + 8 * p.tt + 2 * (i >> 2);
  const uint8_t* kr = kc + p.rec0;
  const uint8_t* vr = vc + p.rec0;
  uint4* ow = reinterpret_cast<uint4*>(ko) + out0;
  uint4* vw = reinterpret_cast<uint4*>(vo) + out0;
  for (int h0 = p.h0; h0 < p.h1; h0 += kLoadHeads) {
    uint32_t wk[kLoadHeads], wv[kLoadHeads], sk[kLoadHeads], sv[kLoadHeads];
#pragma unroll
    for (int q = 0; q < kLoadHeads; ++q) {
      wk[q] = wv[q] = sk[q] = sv[q] = 0;
      if (p.on && h0 + q < p.h1) {
        const int64_t rec = (h0 + q) * head_bytes;
        wk[q] = *reinterpret_cast<const uint32_t*>(kr + rec + kv4_k_word(p.tt, i));
        wv[q] = *reinterpret_cast<const uint32_t*>(vr + rec + kv4_v_word(p.tt, i));
        sk[q] = *reinterpret_cast<const uint16_t*>(kr + rec + scale_at);
        sv[q] = *reinterpret_cast<const uint16_t*>(vr + rec + scale_at);
      }
    }
#pragma unroll
    for (int q = 0; q < kLoadHeads; ++q) {
      const uint32_t x = transpose4(wv[q], lane);
      const uint32_t lo = x & 0x0f0f0f0fu, hi = (x >> 4) & 0x0f0f0f0fu;
      const uint32_t fk = __byte_perm(sk[q], 0, 0x1010), fv = __byte_perm(sv[q], 0, 0x1010);
      uint32_t yk[4], yv[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {  // dims 8 i + 2 b and + 1
        yk[b] = kv4_value(wk[q] >> (4 * b), fk);
        yv[b] = kv4_value(__byte_perm(lo, hi, b | (4 + b) << 8), fv);
      }
      if (p.on && h0 + q < p.h1) {
        const int64_t at = (int64_t)(h0 + q) * out_bs.d * 16;
        ow[at] = make_uint4(yk[0], yk[1], yk[2], yk[3]);
        vw[at] = make_uint4(yv[0], yv[1], yv[2], yv[3]);
      }
    }
  }
}

// Heads a warp walks, the slots looked up once for all: as many as leave every SM its fill of warps (64), up to 4.
// At 32768 tokens and 8 heads, store and load: 1 head 47 and 54 us, 2 heads 39 and 36, 4 heads 35 and 30, 8 heads 36
// and 30; at 32 tokens 4 heads a warp would leave most SMs without work.
static int kv4_heads_per_warp(int64_t T, int Hkv) {
  const int64_t rows = (T + 1) / 2 * Hkv, want = (int64_t)sm_count() * 64;
  return (int)(rows <= want ? 1 : rows / want < 4 ? rows / want : 4);
}

}  // namespace aacc

using namespace aacc;

extern "C" {

int aacc_kv4_store(const void* k, const void* v, int64_t num_tokens, int64_t k_row_stride, int64_t k_head_stride,
                   int64_t v_row_stride, int64_t v_head_stride, const int64_t* slot_mapping, void* k_cache,
                   void* v_cache, int64_t num_blocks, int num_kv_heads, int block_size, cudaStream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0 || block_size % kKv4Tile)
    return set_error(AACC_ERR_INVALID, "kv4_store: bad sizes");
  if (num_blocks > 0x7fffffff / block_size || num_tokens > 0x7fffffff / num_kv_heads)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_store: pool or token count too large");
  if (num_tokens == 0) return AACC_OK;
  if (!k || !v || !slot_mapping || !k_cache || !v_cache) return set_error(AACC_ERR_INVALID, "kv4_store: null pointer");
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (k_row_stride | k_head_stride | v_row_stride | v_head_stride) % 8)
    return set_error(AACC_ERR_INVALID, "kv4_store: pointers/strides must be 16-byte aligned");
  const int hpw = kv4_heads_per_warp(num_tokens, num_kv_heads);
  const int64_t warps = (num_tokens + 1) / 2 * ((num_kv_heads + hpw - 1) / hpw);
  const dim3 grid((unsigned)((warps + kMoveWarps - 1) / kMoveWarps));
  return check_launch("kv4_store",
                      launch_k(kv4_store_kernel, grid, dim3(kMoveThreads), 0, stream,
                               (const bf16*)k, (const bf16*)v, num_tokens, k_row_stride, k_head_stride, v_row_stride,
                               v_head_stride, slot_mapping, (uint8_t*)k_cache, (uint8_t*)v_cache,
                               (uint32_t)(num_blocks * block_size), num_kv_heads, hpw,
                               Divide((num_kv_heads + hpw - 1) / hpw), Divide(block_size), device_error_ptr()));
}

int aacc_kv4_load(const void* k_cache, const void* v_cache, int64_t num_blocks, int num_kv_heads, int block_size,
                  const int64_t* slots, const int64_t* out_slots, int64_t num_tokens, void* k_out, void* v_out,
                  int64_t out_blocks, int out_block_size, cudaStream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0 || block_size % kKv4Tile ||
      out_blocks < 0 || out_block_size <= 0)
    return set_error(AACC_ERR_INVALID, "kv4_load: bad sizes");
  if (num_blocks > 0x7fffffff / block_size || out_blocks > 0x7fffffff / out_block_size ||
      num_tokens > 0x7fffffff / num_kv_heads)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_load: pool or token count too large");
  if (num_tokens == 0) return AACC_OK;
  if (!k_cache || !v_cache || !slots || !k_out || !v_out)
    return set_error(AACC_ERR_INVALID, "kv4_load: null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return set_error(AACC_ERR_INVALID, "kv4_load: pointers must be 16-byte aligned");
  const int hpw = kv4_heads_per_warp(num_tokens, num_kv_heads);
  const int64_t warps = (num_tokens + 1) / 2 * ((num_kv_heads + hpw - 1) / hpw);
  const dim3 grid((unsigned)((warps + kMoveWarps - 1) / kMoveWarps));
  return check_launch(
      "kv4_load", launch_k(kv4_load_kernel, grid, dim3(kMoveThreads), 0, stream,
                           (const uint8_t*)k_cache, (const uint8_t*)v_cache, (uint32_t)(num_blocks * block_size),
                           num_kv_heads, hpw, Divide((num_kv_heads + hpw - 1) / hpw), Divide(block_size), slots,
                           out_slots, num_tokens, (bf16*)k_out, (bf16*)v_out, (uint32_t)(out_blocks * out_block_size),
                           Divide(out_block_size), device_error_ptr()));
}

}  // extern "C"
