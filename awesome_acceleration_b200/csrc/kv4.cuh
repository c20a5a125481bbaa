// The 4-bit KV cache's storage format.
//
// A pool holds K or V of one layer as uint8
//   [num_blocks][num_kv_heads][block_size / 64][4608]
// where a 4608-byte record is a tile of 64 tokens of one kv head: 4096 bytes
// of codes, then 64 x 4 bf16 scales.  Every 32 consecutive dims of a (token,
// kv head) share a scale s = bf16(max|x| / 7); a code u (4 bits) stands for
// (u - 8) * s with u - 8 = clamp(rint(x / s), -7, 7).  4.5 bits a value.
//
// The codes lie in the order in which the lanes of an m16n8k16 MMA need them
// (lane = 4 g + c, g in 0..7, c in 0..3), so that the attention reads its
// operands with 16-byte loads and no shuffles:
//   K  (A operand, rows = tokens): token t owns the 64 bytes at 64 t; the
//      16 bytes at 64 t + 16 c are lane c's, its word w (0..3) holds dims
//      32 w + 8 c + e, e in 0..7: nibble n holds e = 2 (n % 4) + n / 4, so
//      that nibbles n and n + 4 are the two halves of one operand register.
//   V  (transposed, A operand, rows = dims, depth = tokens): with r = t % 16,
//      base = 1024 (t / 16) + 512 (r / 8) + 16 ((r % 8) / 2) + 8 (r % 2),
//      byte base + 64 g + j (j in 0..7) holds dim 16 j + 2 g in its low
//      nibble and 16 j + 2 g + 1 in its high one: lane (g, c) finds tokens
//      2 c and 2 c + 1 in 16 adjacent bytes.
#pragma once

#include "common.cuh"

namespace aacc {

constexpr int kKv4Tile = 64;                        // tokens of a record
constexpr int kKv4Codes = kKv4Tile * 64;            // bytes of codes in a record
constexpr int kKv4Record = kKv4Codes + kKv4Tile * 8;

// Byte offset of record (blk, head, tile) of a pool.
__device__ __forceinline__ int64_t kv4_record(int64_t blk, int h, int tile, int Hkv, int tiles_per_block) {
  return ((blk * Hkv + h) * tiles_per_block + tile) * kKv4Record;
}

// Offset of the first of token t's eight V byte octets; octet g is 64 g further.
__device__ __forceinline__ int kv4_v_base(int t) {
  const int r = t & 15;
  return ((t >> 4) << 10) + ((r >> 3) << 9) + (((r & 7) >> 1) << 4) + ((r & 1) << 3);
}

// (x & M) | c in one operation; the compiler makes two of it.
template <uint32_t M>
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t c) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "n"(M), "r"(c));
  return y;
}

// bf16 pattern -> fp32.
__device__ __forceinline__ float bf16_bits(uint32_t u) { return __uint_as_float(u << 16); }

}  // namespace aacc
