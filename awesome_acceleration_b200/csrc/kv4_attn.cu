// Decode attention over the 4-bit paged KV cache (format: kv4.cuh).
//
// out[b][h] = sum_t softmax_t(scale q.k_t) v_t over the row's tokens, one
// query token per row, grouped queries.  One CTA per (kv head, row): a
// half-warp per token, 8 dims a lane, an online softmax per half-warp, the
// half-warps merged in shared memory.  Bound by instructions, not by HBM.
#include "host.h"
#include "kv4.cuh"

namespace aacc {

constexpr int kAttWarps = 8;
constexpr int kAttHalves = 2 * kAttWarps;

template <int G>
__global__ void __launch_bounds__(kAttWarps * 32)
    kv4_decode_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const uint8_t* __restrict__ kc,
                      const uint8_t* __restrict__ vc, int64_t num_blocks, const int32_t* __restrict__ bt,
                      int64_t num_rows, int64_t max_blocks, const int64_t* __restrict__ rows,
                      const int32_t* __restrict__ seqlens, int ctx_add, int Hkv, int bs, int64_t max_ctx, float scale_log2, unsigned* err) {
  __shared__ float red_m[kAttHalves][G], red_l[kAttHalves][G];
  __shared__ float red_o[kAttHalves][128];
  griddep_wait();
  griddep_launch();
  const int h = blockIdx.x;
  const int64_t b = blockIdx.y;
  int64_t row = rows[b];
  if (row >= num_rows) {
    if (threadIdx.x == 0) report(err, ERR_SLOT_OOB);
    row = -1;
  }
  int64_t ctx = row < 0 ? 0 : (int64_t)seqlens[row] + ctx_add;
  if (ctx > max_ctx) {
    if (threadIdx.x == 0) report(err, ERR_CTX_OOB);
    ctx = max_ctx;
  }
  const int half = threadIdx.x >> 4, i = threadIdx.x & 15;
  const int64_t q0 = (b * Hkv + h) * G;
  float qf[G][8], o[G][8], m[G], l[G];
  // lane i's K word holds dims 32 (i / 4) + 8 (i % 4) + e = 8 i + e
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[g][e] = bf(q[(q0 + g) * 128 + 8 * i + e]) * scale_log2;
      o[g][e] = 0.f;
    }
    m[g] = -INFINITY;
    l[g] = 0.f;
  }
  for (int64_t t0 = 0; t0 < ctx; t0 += kAttHalves) {
    const int64_t t = t0 + half;
    const bool in = t < ctx;
    int64_t blk = in ? bt[row * max_blocks + t / bs] : 0;
    if (blk < 0 || blk >= num_blocks) {
      if (i == 0) report(err, ERR_BLOCK_OOB);
      blk = 0;
    }
    const int off = in ? (int)(t % bs) : 0;
    const int64_t rec = kv4_record(blk, h, off / kKv4Tile, Hkv, bs / kKv4Tile);
    const int tt = off % kKv4Tile;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + rec + 64 * tt + 4 * (4 * (i & 3) + (i >> 2)));
    const float ks = bf16_bits(*reinterpret_cast<const uint16_t*>(kc + rec + kKv4Codes + 8 * tt + 2 * (i >> 2)));
    // lane i's V word: octet g = i / 2, bytes j = 4 (i % 2) + 0..3, dims 16 j + 2 g and + 1
    const uint32_t x = *reinterpret_cast<const uint32_t*>(vc + rec + kv4_v_base(tt) + 64 * (i >> 1) + 4 * (i & 1));
    const uint2 vs4 = *reinterpret_cast<const uint2*>(vc + rec + kKv4Codes + 8 * tt);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s += qf[g][e] * (float)((int)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - 8);
      s *= ks;
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (!in) s = -INFINITY;
      const float mn = fmaxf(m[g], s);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float a = exp2f(m[g] - mu), p = exp2f(s - mu);
      m[g] = mn;
      l[g] = l[g] * a + p;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = 4 * (i & 1) + (e >> 1);
        const uint32_t sw = (j >> 2) ? vs4.y : vs4.x;
        const float vsc = bf16_bits(((j >> 1) & 1) ? sw >> 16 : sw & 0xffffu);
        const float pv = in ? p * vsc * (float)((int)((x >> (4 * e)) & 15u) - 8) : 0.f;
        o[g][e] = o[g][e] * a + pv;
      }
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (i == 0) {
      red_m[half][g] = m[g];
      red_l[half][g] = l[g];
    }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) red_o[half][16 * (4 * (i & 1) + (e >> 1)) + 2 * (i >> 1) + (e & 1)] = o[g][e];
    __syncthreads();
    if (threadIdx.x < 128) {
      float M = -INFINITY;
      for (int w = 0; w < kAttHalves; ++w) M = fmaxf(M, red_m[w][g]);
      const float mu = M == -INFINITY ? 0.f : M;
      float L = 0.f, O = 0.f;
      for (int w = 0; w < kAttHalves; ++w) {
        const float f = exp2f(red_m[w][g] - mu);
        L += f * red_l[w][g];
        O += f * red_o[w][threadIdx.x];
      }
      out[(q0 + g) * 128 + threadIdx.x] = tobf(ctx > 0 ? O / L : 0.f);
    }
  }
}

}  // namespace aacc

using namespace aacc;

extern "C" {

int64_t aacc_kv4_decode_workspace_bytes(int num_q_heads, int num_kv_heads) {
  (void)num_q_heads;
  (void)num_kv_heads;
  return 0;
}

int aacc_kv4_decode_attention(const void* q, void* out, const void* k_cache, const void* v_cache, int64_t num_blocks,
                              const int32_t* block_tables, int64_t num_rows, int64_t max_blocks,
                              const int64_t* slot_indices, const int32_t* seqlens, int ctx_add, int64_t batch, int num_q_heads, int num_kv_heads,
                              int block_size, float scale, int64_t max_context, void* workspace,
                              int64_t workspace_bytes, cudaStream_t stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (batch < 0 || batch > 65535 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      block_size <= 0 || block_size % kKv4Tile || num_blocks <= 0 || num_rows < 0 || max_blocks <= 0 ||
      max_context <= 0)
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: bad sizes");
  const int G = num_q_heads / num_kv_heads;
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return set_error(AACC_ERR_UNSUPPORTED, "kv4_decode_attention: q/kv head ratio %d not in {1,2,4,8}", G);
  if (batch == 0) return AACC_OK;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache))
    return set_error(AACC_ERR_INVALID, "kv4_decode_attention: pointers must be 16-byte aligned");
  if (max_context > max_blocks * block_size) max_context = max_blocks * block_size;
  cudaError_t le;
  const dim3 grid(num_kv_heads, (unsigned)batch);
#define AACC_LAUNCH_KV4(GG)                                                                                        \
  le = launch_k(kv4_decode_kernel<GG>, grid, dim3(kAttWarps * 32), 0, stream, (const bf16*)q, (bf16*)out,          \
                (const uint8_t*)k_cache, (const uint8_t*)v_cache, num_blocks, block_tables, num_rows, max_blocks,     \
                slot_indices, seqlens, ctx_add, num_kv_heads, block_size, max_context, scale * kLog2e, device_error_ptr());
  switch (G) {
    case 1: AACC_LAUNCH_KV4(1) break;
    case 2: AACC_LAUNCH_KV4(2) break;
    case 4: AACC_LAUNCH_KV4(4) break;
    default: AACC_LAUNCH_KV4(8) break;
  }
#undef AACC_LAUNCH_KV4
  return check_launch("kv4_decode_kernel", le);
}

}  // extern "C"
