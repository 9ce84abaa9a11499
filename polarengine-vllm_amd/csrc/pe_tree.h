// What the kernels for drafted tokens share.
#pragma once

#include "pe_internal.h"

namespace pe {

constexpr int kTreeMax = 64;  // nodes of a tree: one bit each of a 64-bit mask, one lane each

constexpr int64_t kTreeMaxGrid = (1 << 24) - 1;          // workgroups of 256 along x
constexpr int64_t kTreeMaxStride = (int64_t)1 << 26;  // elements, of positions and dimensions

// Ancestor mask (itself among them) of node i = lane of a wave, from its parent:
// node 0 is the root, whatever its parent says; node i > 0 exists if 0 <= parent
// < i and the parent exists, else its mask is 0. All 64 lanes call. Pointer
// jumping: after round r a lane's mask holds its nearest 2^(r+1) ancestors.
__device__ __forceinline__ uint64_t tree_mask(int64_t parent, int i, int n) {
  const bool has = i > 0 && i < n && parent >= 0 && parent < i;
  uint64_t m = i < n ? 1ull << i : 0;
  int up = has ? (int)parent : i;  // a lane that points at itself is done
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    m |= (uint64_t)__shfl((unsigned long long)m, up, 64);
    up = __shfl(up, up, 64);
  }
  return m & 1 ? m : 0;  // absent: the chain of parents does not reach the root
}

// A cache of 16-bit rows: values by position (the dimension contiguous), keys by
// position or by dimension (the position contiguous). Rows are read and written
// 16 bytes at a time.
inline int cache_strides(const void* k, int64_t ks_b, int64_t ks_h, int64_t ks_l, int64_t ks_d,
                         const void* v, int64_t vs_b, int64_t vs_h, int64_t vs_l) {
  if (ks_b < 0 || ks_h < 0 || ks_l < 0 || ks_d < 0 || vs_b < 0 || vs_h < 0 || vs_l < 0)
    return PE_ERR_DIMS;
  if (ks_d != 1 && ks_l != 1) return PE_ERR_DIMS;
  // a workgroup's rows lie within 32-bit byte offsets of one another
  if (ks_l >= kTreeMaxStride || ks_d >= kTreeMaxStride || vs_l >= kTreeMaxStride) return PE_ERR_DIMS;
  if (!aligned16(v) || (vs_b | vs_h | vs_l) % 8) return PE_ERR_ALIGN;
  if (ks_d == 1 && (!aligned16(k) || (ks_b | ks_h | ks_l) % 8)) return PE_ERR_ALIGN;
  return PE_OK;
}

}  // namespace pe
