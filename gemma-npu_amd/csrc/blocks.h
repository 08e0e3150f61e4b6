// The 8-bit key / value cache: whole blocks of 64 tokens as one-byte codes with one fp32 scale per block, KV head and
// operand, the newest two blocks' rows in bf16 beside them.
//
// Codes lie in the order in which the matrix instructions of the attention over them take them, 1 KiB fragments of
// 64 lanes x 16 bytes, lane 16 qq + qi:
//   keys, fragment (kt, jj) of a block, kt < 4, jj < D / 64: byte e is key 16 kt + qi, d = 64 jj + 16 qq + e;
//   values, fragment dt < D / 16: byte e is d = 16 dt + qi, key 32 (e / 8) + 16 (e / 4 % 2) + 4 qq + e % 4.
// The bf16 rows of block b lie in slot b % 2 of a ring, in the same order with 8 values a lane: keys (kt, 2 jj + h)
// holding e = 8 h .., values (dt, h) likewise.
#pragma once
#include "w8a8_common.h"

namespace w8a8 {

constexpr int BLK = 64;  // tokens of a block

struct BlockCache {
  uint8_t *k, *v;              // codes [KV][blocks][64 D]
  uint16_t *kt, *vt;           // bf16 ring [KV][2][64 D]
  float *ks, *vs;              // scales [KV][blocks]
  int KV, blocks, D;
};

// Element of a key's d (values: of d's key) within a block's bf16 ring slot.
__device__ __forceinline__ int ring_key(int r, int d, int D) {
  const int jj = d >> 6, qq = (d >> 4) & 3, h = (d >> 3) & 1;
  return ((((r >> 4) * (D >> 5) + 2 * jj + h) * 64) + 16 * qq + (r & 15)) * 8 + (d & 7);
}
__device__ __forceinline__ int ring_value(int r, int d) {
  const int h = r >> 5, qq = (r >> 2) & 3, e = 4 * ((r >> 4) & 1) + (r & 3);
  return ((((d >> 4) * 2 + h) * 64) + 16 * qq + (d & 15)) * 8 + e;
}

inline int64_t block_count(int64_t capacity) { return (capacity + BLK - 1) / BLK; }
inline bool block_shape_ok(int64_t KV, int64_t capacity, int64_t D) {
  return KV >= 1 && KV <= 65535 && capacity >= 1 && capacity <= INT32_MAX / 2 && (D == 128 || D == 256 || D == 512);
}
inline int64_t block_align(int64_t n) { return (n + 255) / 256 * 256; }
// Offsets of the parts in one allocation, and its size.
inline int64_t block_layout(void* data, int64_t KV, int64_t capacity, int64_t D, BlockCache& c) {
  const int64_t nb = block_count(capacity), codes = block_align(KV * nb * BLK * D), ring = KV * 2 * BLK * D * 2;
  const int64_t scales = block_align(KV * nb * 4);
  char* p = static_cast<char*>(data);
  c.k = reinterpret_cast<uint8_t*>(p);
  c.v = reinterpret_cast<uint8_t*>(p + codes);
  c.kt = reinterpret_cast<uint16_t*>(p + 2 * codes);
  c.vt = reinterpret_cast<uint16_t*>(p + 2 * codes + ring);
  c.ks = reinterpret_cast<float*>(p + 2 * codes + 2 * ring);
  c.vs = reinterpret_cast<float*>(p + 2 * codes + 2 * ring + scales);
  c.KV = int(KV);
  c.blocks = int(nb);
  c.D = int(D);
  return 2 * codes + 2 * ring + 2 * scales;
}

}  // namespace w8a8
