// Block tables and slot maps from request lengths, on the device.
//
// Both are prefix sums over the requests followed by a write per output
// element; the outputs are a few hundred KB at most, so launch latency and
// the dependent loads of the scan are the cost.  Every CTA scans the lengths
// itself (a few KB from L2) instead of waiting for another kernel or CTA.
//
// Measured (B200), a launch alone being 2.2 us: tables of 8 requests 2.4 us, of
// 2048 with 161 columns 5.5 us (2 MB moved; a CTA per request, each of
// which scans all lengths before it, 10.1 us); slot maps of 2 requests 2.6 us,
// of 256 prompts (262,144 tokens, 4.2 MB written) 5.2 us.  Bound by those
// launches and the scan's chain of dependent steps, not by bytes.
#include "common.cuh"
#include "host.h"

namespace aacc {

constexpr int kMapThreads = 256;
constexpr int kMapPer = 4;                             // requests a thread scans per chunk
constexpr int kMapChunk = kMapThreads * kMapPer;       // requests per chunk
constexpr int kMapTokens = 512;                        // packed tokens one CTA maps

__device__ __forceinline__ int64_t warp_scan_incl(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Exclusive prefix of every thread's `v` over the CTA; *total is the sum.
__device__ __forceinline__ int64_t block_scan_excl(int64_t v, int64_t* sh, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t inc = warp_scan_incl(v, lane);
  __syncthreads();  // sh of the previous call is read
  if (lane == 31) sh[warp] = inc;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kMapThreads / 32; ++w) {
    const int64_t x = sh[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return before + inc - v;
}

__device__ __forceinline__ int64_t blocks_of(int32_t len, int bs, int64_t max_blocks) {
  const int64_t need = len > 0 ? ((uint32_t)len - 1) / (uint32_t)bs + 1 : 0;  // 32-bit: a 64-bit division is a loop
  return min(need, max_blocks);
}

// One CTA per run of `per` requests: the first one's first block is the number
// of blocks that all requests before it take, the others' follow by a scan.
// A warp writes a row.
__global__ void __launch_bounds__(kMapThreads)
    build_block_tables_kernel(const int32_t* __restrict__ lengths, int64_t n, int64_t per, int bs,
                              const int32_t* __restrict__ free_blocks, int64_t num_free, int32_t* __restrict__ tables,
                              int64_t max_blocks, int32_t* __restrict__ used, unsigned* err) {
  __shared__ int64_t sh[kMapThreads / 32];
  __shared__ int64_t first[kMapThreads], count[kMapThreads];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i0 = blockIdx.x * per, i1 = min(n, i0 + per);
  int64_t part = 0, off;
  for (int64_t j = threadIdx.x; j < i0; j += kMapThreads) part += blocks_of(lengths[j], bs, max_blocks);
  block_scan_excl(part, sh, &off);
  for (int64_t r0 = i0; r0 < i1; r0 += kMapThreads) {
    const int64_t i = r0 + threadIdx.x;
    const int32_t len = i < i1 ? lengths[i] : 0;
    const int64_t need = blocks_of(len, bs, max_blocks);
    if ((int64_t)len > max_blocks * bs) report(err, ERR_CTX_OOB);
    int64_t total;
    first[threadIdx.x] = off + block_scan_excl(need, sh, &total);
    count[threadIdx.x] = need;
    off += total;
    __syncthreads();
    const int m = (int)min((int64_t)kMapThreads, i1 - r0);
    for (int r = warp; r < m; r += kMapThreads / 32) {
      const int64_t at0 = first[r], c = count[r];
      int32_t* row = tables + (r0 + r) * max_blocks;
      for (int64_t j = lane; j < max_blocks; j += 32) {
        int32_t b = -1;
        if (j < c) {
          if (at0 + j >= num_free)
            report(err, ERR_BLOCK_OOB);
          else
            b = free_blocks ? free_blocks[at0 + j] : (int32_t)(at0 + j);
        }
        row[j] = b;
      }
    }
    __syncthreads();  // first and count are rewritten
  }
  if (i1 == n && threadIdx.x == 0 && used) *used = (int32_t)min(off, (int64_t)0x7fffffff);
}

// One CTA per kMapTokens packed tokens.  It walks the requests in chunks; of
// the chunk whose tokens meet its own it keeps the prefix sums in shared
// memory, where every token finds its request by bisection.
__global__ void __launch_bounds__(kMapThreads)
    build_slot_maps_kernel(const int32_t* __restrict__ lengths, const int32_t* __restrict__ starts,
                           const int64_t* __restrict__ rows, int64_t n, const int32_t* __restrict__ bt,
                           int64_t num_rows, int64_t max_blocks, int bs, int64_t num_blocks, int32_t* __restrict__ cu,
                           int64_t* __restrict__ positions, int64_t* __restrict__ slots, int64_t num_tokens,
                           unsigned* err) {
  __shared__ int64_t sh[kMapThreads / 32];
  __shared__ int64_t pre[kMapChunk + 1];
  griddep_wait();
  griddep_launch();
  const int64_t t0 = (int64_t)blockIdx.x * kMapTokens;
  const int64_t t1 = min(t0 + kMapTokens, num_tokens);
  const bool first = blockIdx.x == 0;  // writes cu, so it walks every chunk
  int64_t base = 0;
  for (int64_t c0 = 0; c0 < n && (first || base < t1); c0 += kMapChunk) {
    int32_t len[kMapPer];
    int64_t mine = 0, total;
#pragma unroll
    for (int p = 0; p < kMapPer; ++p) {
      const int64_t j = c0 + threadIdx.x * kMapPer + p;
      len[p] = j < n ? max(lengths[j], 0) : 0;
      mine += len[p];
    }
    int64_t at = base + block_scan_excl(mine, sh, &total);
    const int m = (int)min((int64_t)kMapChunk, n - c0);
#pragma unroll
    for (int p = 0; p < kMapPer; ++p) {
      const int q = threadIdx.x * kMapPer + p;
      pre[q] = at;
      if (first && q < m) cu[c0 + q] = (int32_t)min(at, (int64_t)0x7fffffff);
      at += len[p];
    }
    if (threadIdx.x == 0) pre[kMapChunk] = base + total;
    __syncthreads();
    const int64_t lo = max(t0, base), hi = min(t1, base + total);
    for (int64_t t = lo + threadIdx.x; t < hi; t += kMapThreads) {
      int a = 0, b = m;  // the last request of the chunk that starts at or before t: pre[a] <= t < pre[b]
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (pre[mid] <= t)
          a = mid;
        else
          b = mid;
      }
      const int64_t req = c0 + a;
      const int64_t pos = t - pre[a] + (starts ? (int64_t)starts[req] : 0);
      const int64_t row = rows ? rows[req] : req;
      int64_t slot = -1;
      if (row >= num_rows) {
        report(err, ERR_SLOT_OOB);
      } else if (row >= 0) {  // negative rows are padding
        const int64_t j = (uint32_t)pos / (uint32_t)bs;
        if (pos < 0 || pos > 0x7fffffff || j >= max_blocks) {
          report(err, ERR_CTX_OOB);
        } else {
          const int64_t blk = bt[row * max_blocks + j];
          if (blk < 0 || blk >= num_blocks)
            report(err, ERR_BLOCK_OOB);
          else
            slot = blk * bs + (pos - j * bs);
        }
      }
      if (positions) positions[t] = pos;
      slots[t] = slot;
    }
    base += total;
    __syncthreads();  // pre is rewritten by the next chunk
  }
  if (first && threadIdx.x == 0) {
    cu[n] = (int32_t)min(base, (int64_t)0x7fffffff);
    if (base > num_tokens) report(err, ERR_CTX_OOB);
  }
  for (int64_t t = max(t0, base) + threadIdx.x; t < t1; t += kMapThreads) {  // behind the last request
    if (positions) positions[t] = 0;
    slots[t] = -1;
  }
}

}  // namespace aacc

using namespace aacc;

extern "C" {

int aacc_build_block_tables(const int32_t* lengths, int64_t num_requests, int block_size, const int32_t* free_blocks,
                            int64_t num_free, int32_t* block_tables, int64_t max_blocks, int32_t* used,
                            cudaStream_t stream) {
  if (num_requests < 0 || num_requests > 0x7fffffff || block_size <= 0 || max_blocks <= 0 || num_free < 0)
    return set_error(AACC_ERR_INVALID, "build_block_tables: bad sizes");
  if (num_requests == 0 && !used) return AACC_OK;
  if (num_requests > 0 && (!lengths || !block_tables))
    return set_error(AACC_ERR_INVALID, "build_block_tables: null pointer");
  // A CTA per SM at most twice over: each reads all the lengths before its own.
  const int64_t per = num_requests > 0 ? (num_requests + 2 * sm_count() - 1) / (2 * sm_count()) : 1;
  const int64_t ctas = num_requests > 0 ? (num_requests + per - 1) / per : 1;  // one writes *used
  return check_launch("build_block_tables",
                      launch_k(build_block_tables_kernel, dim3((unsigned)ctas), dim3(kMapThreads), 0, stream, lengths, num_requests, per, block_size, free_blocks,
                               num_free, block_tables, max_blocks, used, device_error_ptr()));
}

int aacc_build_slot_maps(const int32_t* lengths, const int32_t* starts, const int64_t* rows, int64_t num_requests,
                         const int32_t* block_tables, int64_t num_rows, int64_t max_blocks, int block_size,
                         int64_t num_blocks, int32_t* cu_seqlens, int64_t* positions, int64_t* slots,
                         int64_t num_tokens, cudaStream_t stream) {
  if (num_requests < 0 || num_rows < 0 || max_blocks <= 0 || block_size <= 0 || num_blocks <= 0 || num_tokens < 0 ||
      num_tokens > 0x7fffffff)
    return set_error(AACC_ERR_INVALID, "build_slot_maps: bad sizes");
  if (!cu_seqlens || (num_tokens > 0 && !slots) || (num_requests > 0 && (!lengths || !block_tables)))
    return set_error(AACC_ERR_INVALID, "build_slot_maps: null pointer");
  const int64_t ctas = num_tokens > 0 ? (num_tokens + kMapTokens - 1) / kMapTokens : 1;
  return check_launch("build_slot_maps",
                      launch_k(build_slot_maps_kernel, dim3((unsigned)ctas), dim3(kMapThreads), 0, stream, lengths,
                               starts, rows, num_requests, block_tables, num_rows, max_blocks, block_size, num_blocks,
                               cu_seqlens, positions, slots, num_tokens, device_error_ptr()));
}

}  // extern "C"
