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

// One warp per (token, kv head): lanes 0-15 quantise the K row, lanes 16-31
// the V row, 8 dims each; four lanes share a group of 32.
__global__ void kv4_store_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t T, int64_t ks,
                                 int64_t kh, int64_t vs, int64_t vh, const int64_t* __restrict__ slots,
                                 uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, int64_t num_slots, int Hkv, int bs,
                                 unsigned* err) {
  griddep_wait();
  griddep_launch();
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (warp >= T * Hkv) return;
  const int64_t t = warp / Hkv;
  const int h = (int)(warp % Hkv);
  const int64_t slot = slots[t];
  if (slot < 0) return;
  if (slot >= num_slots) {
    if (lane == 0) report(err, ERR_SLOT_OOB);
    return;
  }
  const bool is_v = lane >= 16;
  const int i = lane & 15;
  const bf16* src = is_v ? v + t * vs + h * vh : k + t * ks + h * kh;
  const uint4 x4 = reinterpret_cast<const uint4*>(src)[i];
  const uint32_t x2[4] = {x4.x, x4.y, x4.z, x4.w};
  // max |x| on the bit patterns: they order as the values do, infinities and NaN above every finite one.
  uint32_t mx = 0;
#pragma unroll
  for (int n = 0; n < 4; ++n) mx = max(mx, max(x2[n] & 0x7fffu, (x2[n] >> 16) & 0x7fffu));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const bool finite = mx < 0x7f80u;
  const uint32_t sbits = finite ? (uint32_t)__bfloat16_as_ushort(tobf(__fdiv_rn(bf16_bits(mx), 7.f))) : 0x7fc0u;
  const float s = bf16_bits(sbits);
  // x has 8 significant bits and s 8, so x / s is either exactly on a rounding border or at least 2^-9 off
  // it: the fp32 quotient rounds as the exact one does.
  uint32_t code[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = bf16_bits((e & 1) ? x2[e >> 1] >> 16 : x2[e >> 1] & 0xffffu);
    const float n = (finite && s > 0.f) ? fminf(fmaxf(rintf(__fdiv_rn(x, s)), -7.f), 7.f) : 0.f;
    code[e] = (uint32_t)((int)n + 8);
  }
  uint32_t w = 0;
  if (!is_v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code[e] << (4 * ((e >> 1) + 4 * (e & 1)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code[e] << (4 * e);
  }
  const uint32_t wt = transpose4(w, lane);
  const int64_t blk = slot / bs;
  const int off = (int)(slot - blk * bs);
  const int64_t rec = kv4_record(blk, h, off / kKv4Tile, Hkv, bs / kKv4Tile);
  const int tt = off % kKv4Tile;
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(kc + rec + 64 * tt + 4 * (4 * (i & 3) + (i >> 2))) = w;
  } else {
    const int g = 4 * (i & 1) + ((i >> 1) & 3), u = i >> 3;
    *reinterpret_cast<uint32_t*>(vc + rec + kv4_v_base(tt) + 64 * g + 4 * u) = wt;
  }
  if ((i & 3) == 0)
    *reinterpret_cast<uint16_t*>((is_v ? vc : kc) + rec + kKv4Codes + 8 * tt + 2 * (i >> 2)) = (uint16_t)sbits;
}

// One warp per (token, kv head): lanes 0-15 expand the K row, lanes 16-31 the V row, 8 dims each.
__global__ void kv4_load_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, int64_t num_slots,
                                int Hkv, int bs, const int64_t* __restrict__ slots,
                                const int64_t* __restrict__ out_slots, int64_t T, bf16* __restrict__ ko,
                                bf16* __restrict__ vo, int64_t out_total, int out_bs, unsigned* err) {
  griddep_wait();
  griddep_launch();
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (warp >= T * Hkv) return;
  const int64_t t = warp / Hkv;
  const int h = (int)(warp % Hkv);
  const int64_t slot = slots[t], dst = out_slots ? out_slots[t] : t;
  if (slot < 0 || dst < 0) return;
  if (slot >= num_slots || dst >= out_total) {
    if (lane == 0) report(err, ERR_SLOT_OOB);
    return;
  }
  const bool is_v = lane >= 16;
  const int i = lane & 15;
  const int64_t blk = slot / bs;
  const int off = (int)(slot - blk * bs);
  const int64_t rec = kv4_record(blk, h, off / kKv4Tile, Hkv, bs / kKv4Tile);
  const int tt = off % kKv4Tile;
  uint32_t w;
  if (!is_v) {
    w = *reinterpret_cast<const uint32_t*>(kc + rec + 64 * tt + 4 * (4 * (i & 3) + (i >> 2)));
  } else {
    const int g = 4 * (i & 1) + ((i >> 1) & 3), u = i >> 3;
    w = *reinterpret_cast<const uint32_t*>(vc + rec + kv4_v_base(tt) + 64 * g + 4 * u);
  }
  const uint32_t wt = transpose4(w, lane);
  const float s = bf16_bits(
      *reinterpret_cast<const uint16_t*>((is_v ? vc : kc) + rec + kKv4Codes + 8 * tt + 2 * (i >> 2)));
  uint32_t y[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {  // dims 8 i + 2 p and + 1
    const uint32_t lo = is_v ? wt >> (8 * p) : w >> (4 * p);
    const uint32_t hi = is_v ? wt >> (8 * p + 4) : w >> (4 * p + 16);
    y[p] = pack_bf16((float)((int)(lo & 15u) - 8) * s, (float)((int)(hi & 15u) - 8) * s);
  }
  const int64_t ob = dst / out_bs, oo = dst - ob * out_bs;
  bf16* out = (is_v ? vo : ko) + ((ob * Hkv + h) * out_bs + oo) * 128;
  reinterpret_cast<uint4*>(out)[i] = make_uint4(y[0], y[1], y[2], y[3]);
}

}  // namespace aacc

using namespace aacc;

extern "C" {

int aacc_kv4_store(const void* k, const void* v, int64_t num_tokens, int64_t k_row_stride, int64_t k_head_stride,
                   int64_t v_row_stride, int64_t v_head_stride, const int64_t* slot_mapping, void* k_cache,
                   void* v_cache, int64_t num_blocks, int num_kv_heads, int block_size, cudaStream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0 || block_size % kKv4Tile)
    return set_error(AACC_ERR_INVALID, "kv4_store: bad sizes");
  if (num_tokens == 0) return AACC_OK;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (k_row_stride | k_head_stride | v_row_stride | v_head_stride) % 8)
    return set_error(AACC_ERR_INVALID, "kv4_store: pointers/strides must be 16-byte aligned");
  const int64_t blocks = (num_tokens * num_kv_heads + 7) / 8;
  if (blocks > 0x7fffffff) return set_error(AACC_ERR_INVALID, "kv4_store: too many rows");
  return check_launch("kv4_store",
                      launch_k(kv4_store_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (const bf16*)k,
                               (const bf16*)v, num_tokens, k_row_stride, k_head_stride, v_row_stride, v_head_stride,
                               slot_mapping, (uint8_t*)k_cache, (uint8_t*)v_cache, num_blocks * block_size,
                               num_kv_heads, block_size, device_error_ptr()));
}

int aacc_kv4_load(const void* k_cache, const void* v_cache, int64_t num_blocks, int num_kv_heads, int block_size,
                  const int64_t* slots, const int64_t* out_slots, int64_t num_tokens, void* k_out, void* v_out,
                  int64_t out_blocks, int out_block_size, cudaStream_t stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0 || block_size % kKv4Tile ||
      out_blocks < 0 || out_block_size <= 0)
    return set_error(AACC_ERR_INVALID, "kv4_load: bad sizes");
  if (num_tokens == 0) return AACC_OK;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return set_error(AACC_ERR_INVALID, "kv4_load: pointers must be 16-byte aligned");
  const int64_t blocks = (num_tokens * num_kv_heads + 7) / 8;
  if (blocks > 0x7fffffff) return set_error(AACC_ERR_INVALID, "kv4_load: too many rows");
  return check_launch(
      "kv4_load", launch_k(kv4_load_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (const uint8_t*)k_cache,
                           (const uint8_t*)v_cache, num_blocks * block_size, num_kv_heads, block_size, slots, out_slots,
                           num_tokens, (bf16*)k_out, (bf16*)v_out, out_blocks * out_block_size, out_block_size,
                           device_error_ptr()));
}

}  // extern "C"
