// Layout of the 4-bit key/value cache's blocks (sfx_kv4 in the header) and
// what its kernels share.
//
// Why this layout.  A wave computes K Q^T with tokens as the rows of a matrix
// instruction, so a lane needs consecutive channels of one token: keys lie
// token by token, and a channel group's scale is a power of two, which the
// conversion from 4 bits applies by itself.  It then computes V^T P^T, whose
// contraction runs over tokens, so a lane needs several tokens of one channel:
// values lie in words of 8 tokens of a channel, in the very order in which
// the first product leaves its results in the lanes, so the probabilities
// never cross lanes and neither operand goes through LDS.  A scale per token
// cannot be part of that operand; it is folded into the token's probability
// instead, which is why values have one scale a token (a float, as a sixth of
// the largest magnitude keeps the rounding steps as fine as they can be)
// where keys, whose channels differ more, have one for 32 channels.  A block
// is one stretch of memory: 32 (D + D/32 + 4) bytes, 4,352 for D = 128, in
// place of 16,384 in 16-bit types.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sfx_common.h"
#include "suffixgpu_amd.h"

namespace sfx {

constexpr int kKvBlock = 32;  // tokens

template <int D>
struct KvLayout {
  static constexpr int kScale = kKvBlock * (D / 2);
  static constexpr int kValue = kScale + kKvBlock * (D / 32);
  static constexpr int kVScale = kValue + kKvBlock * (D / 2);
  static constexpr int kBytes = kVScale + kKvBlock * 4;
  // Word of channel c and token t.
  __host__ __device__ static constexpr int word(int t, int c) {
    return ((c / 64 * 4 + 2 * (t / 16) + t / 4 % 2) * 16 + c % 16) * 4 +
           c / 16 % 4;
  }
};

// The cache as kernels take it.
struct KvView {
  char* pages;
  int64_t num_pages;
  const int32_t* table;
  int64_t table_stride;
  int64_t positions;   // table_width * page_size
  int heads;
  int page_shift;      // log2(page_size / 32)
};

// Place in the pool of block `blk` (32 positions) of row b and KV head h, or -1
// where the table holds no page.
__device__ __forceinline__ int64_t kv_place(const KvView& c, int64_t b, int h,
                                            int64_t blk) {
  // in blocks: a start next to 2^63 is past the table too
  if ((uint64_t)blk >= (uint64_t)c.positions / kKvBlock) return -1;
  const int64_t page = c.table[b * c.table_stride + (blk >> c.page_shift)];
  if (page < 0 || page >= c.num_pages) return -1;
  const int64_t in = blk & ((int64_t(1) << c.page_shift) - 1);
  return ((page * c.heads + h) << c.page_shift) + in;
}

// Its address, or NULL.
template <int D>
__device__ __forceinline__ char* kv_block(const KvView& c, int64_t b, int h,
                                          int64_t blk) {
  const int64_t at = kv_place(c, b, h, blk);
  return at < 0 ? nullptr : c.pages + at * (int64_t)KvLayout<D>::kBytes;
}

inline bool kv_view(const sfx_kv4* c, KvView* v) {
  if (!c || c->num_pages < 0 || c->heads < 1 || c->heads > 65535 ||
      c->table_width < 0 || c->page_size < kKvBlock || c->page_size > 65536 ||
      (c->page_size & (c->page_size - 1)) ||
      (c->dtype != SFX_BF16 && c->dtype != SFX_F16) ||
      (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256))
    return false;
  if (c->num_pages > 0 && (!c->pages || ((uintptr_t)c->pages & 15)))
    return false;
  if (c->table_width > 0 && !c->table) return false;
  // positions are counted in int32
  if (c->table_width > (int64_t(1) << 30) / c->page_size) return false;
  v->pages = (char*)c->pages;
  v->num_pages = c->num_pages;
  v->table = c->table;
  v->table_stride = c->table_stride;
  v->positions = c->table_width * c->page_size;
  v->heads = (int)c->heads;
  int s = 0;
  while ((int64_t(kKvBlock) << s) < c->page_size) ++s;
  v->page_shift = s;
  return true;
}

// Sixteen-bit types by their bits.
template <bool kHalf>
__device__ __forceinline__ float to_float16b(uint32_t bits) {
  if (kHalf)
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  return __uint_as_float(bits << 16);
}

template <bool kHalf>
__device__ __forceinline__ uint32_t from_float16b(float x) {
  if (kHalf) return __builtin_bit_cast(uint16_t, (_Float16)x);
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

}  // namespace sfx
