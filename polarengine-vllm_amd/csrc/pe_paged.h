// What the kernels over the paged 8-bit cache share.
#pragma once

#include "pe_internal.h"

namespace pe {

constexpr int kMinExp = -100;      // the smallest exponent of a block's scale
constexpr int64_t kPagedMaxBatch = 4096;
constexpr int64_t kPagedMaxRows = (int64_t)1 << 24;
constexpr int64_t kPagedMaxPositions = (int64_t)1 << 30;  // of a sequence
constexpr int64_t kPagedMaxWidth = kPagedMaxPositions / 128;

// One layer's cache.
struct PagedCache {
  uint8_t *k, *v;         // e4m3 [blocks][kv_heads][T][D] and [blocks][kv_heads][D][T]
  uint8_t *ks, *vs;       // e8m0 [blocks][kv_heads]
  int64_t k_b, v_b, s_b;  // bytes from block to block
  int64_t blocks;
  int kv_heads, log_t;
};

// Block size, pointers and strides of a cache; PE_OK or what is wrong with them.
inline int paged_cache(PagedCache& c, const void* k, int64_t k_b, const void* v, int64_t v_b,
                       const void* ks, const void* vs, int64_t s_b, int64_t blocks, int kv_heads,
                       int block_size, int head_dim) {
  if (!k || !v || !ks || !vs) return PE_ERR_NULL;
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return PE_ERR_DIMS;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return PE_ERR_DIMS;
  if (kv_heads < 1 || kv_heads > 4096 || blocks < 1 || blocks > INT32_MAX) return PE_ERR_DIMS;
  const int64_t part = (int64_t)kv_heads * block_size * head_dim;
  if (k_b < part || v_b < part || s_b < kv_heads) return PE_ERR_DIMS;
  if (k_b > INT32_MAX || v_b > INT32_MAX || s_b > INT32_MAX) return PE_ERR_DIMS;
  if (!aligned16(k) || !aligned16(v) || k_b % 16 || v_b % 16) return PE_ERR_ALIGN;
  c.k = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(k));
  c.v = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(v));
  c.ks = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(ks));
  c.vs = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(vs));
  c.k_b = k_b;
  c.v_b = v_b;
  c.s_b = s_b;
  c.blocks = blocks;
  c.kv_heads = kv_heads;
  c.log_t = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  return PE_OK;
}

// 2^(byte - 127) of an e8m0 scale (bytes from 1 on; 0 counts as 0, 255 as infinite)
__device__ __forceinline__ float e8m0(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

}  // namespace pe
