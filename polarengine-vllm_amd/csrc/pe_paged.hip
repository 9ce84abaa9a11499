// The paged 8-bit cache: block tables and slot maps of a step, blocks back to the
// pool, and the quantizing write of keys and values.

#include "pe_paged.h"

namespace pe {

typedef float float2v __attribute__((ext_vector_type(2)));

constexpr int kPlanThreads = 1024;

// Running sums over a workgroup of 1024 in order of thread; `total` in every thread.
// Values and sums stop at kPlanCap, which is past any number of rows or blocks.
constexpr uint32_t kPlanCap = 1u << 30;
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t* waves, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(v, off, 64);
    if (lane >= off) v = min(v + u, kPlanCap);
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before = min(before + waves[w], kPlanCap);
    total = min(total + waves[w], kPlanCap);
  }
  return min(before + v, kPlanCap);
}

// ---------------------------------------------------------------------------
// One workgroup: a thread a sequence, then a thread a row.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kPlanThreads) void plan_step_kernel(
    const int64_t* __restrict__ lengths, const int64_t* __restrict__ counts, int32_t* tables,
    int64_t t_b, int batch, int64_t width, const int32_t* __restrict__ free_blocks, int64_t free_cap,
    int64_t* free_count, int rows, int log_t, int64_t* starts, int64_t* __restrict__ positions,
    int64_t* __restrict__ slots, int64_t* out_lengths) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  __shared__ uint32_t used;
  const int tid = threadIdx.x;
  const int64_t have0 = *free_count;
  const uint32_t have = (uint32_t)max((int64_t)0, min(have0, free_cap));
  if (tid == 0) {
    starts[0] = 0;
    used = 0;
  }
  uint32_t row0 = 0, need0 = 0;  // of the sequences before this round's
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int64_t len = b < batch ? lengths[b] : -1;
    // a count past the rows is as good as one row more
    const uint32_t n = len >= 0 ? (uint32_t)max((int64_t)0, min(counts[b], (int64_t)rows + 1)) : 0;
    uint32_t total;
    const uint32_t end = min(row0 + plan_scan(n, waves, total), (uint32_t)rows + 1);
    row0 = min(row0 + total, (uint32_t)rows + 1);
    if (b < batch) starts[b + 1] = min(end, (uint32_t)rows);
    const bool fits = len >= 0 && len <= (width << log_t) - (int64_t)n && end <= (uint32_t)rows;
    uint32_t need = 0;
    const int64_t j0 = len >> log_t, j1 = fits && n ? (len + n - 1) >> log_t : j0 - 1;
    int32_t* row = tables + (int64_t)b * t_b;
    for (int64_t j = j0; j <= j1; ++j) need += row[j] < 0;
    const uint32_t cum = need0 + plan_scan(need, waves, total);
    need0 += total;
    const bool taken = fits && (need == 0 || cum <= have);
    if (b < batch) out_lengths[b] = taken ? len + n : -1;
    if (taken && need) {
      uint32_t at = cum - need;
      for (int64_t j = j0; j <= j1; ++j)
        if (row[j] < 0) row[j] = free_blocks[have - 1 - at++];
      atomicMax(&used, cum);
    }
  }
  __syncthreads();
  if (tid == 0) *free_count = (int64_t)have - used;
  for (int r = tid; r < rows; r += kPlanThreads) {
    int lo = 0, hi = batch;  // the first sequence that ends behind row r
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (starts[mid + 1] > r) hi = mid;
      else lo = mid + 1;
    }
    int64_t pos = -1, slot = -1;
    if (lo < batch && out_lengths[lo] >= 0) {
      pos = lengths[lo] + r - starts[lo];
      slot = ((int64_t)tables[lo * t_b + (pos >> log_t)] << log_t) + (pos & ((1 << log_t) - 1));
    }
    positions[r] = pos;
    slots[r] = slot;
  }
}

__global__ __launch_bounds__(kPlanThreads) void release_kernel(
    int32_t* __restrict__ tables, int64_t t_b, int batch, int64_t width,
    const int64_t* __restrict__ keep, int32_t* __restrict__ free_blocks, int64_t free_cap,
    int64_t* free_count, int log_t) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int64_t have = max((int64_t)0, min(*free_count, free_cap));
  uint32_t all = 0;
  auto count = [&](int b, int64_t& first) {
    uint32_t n = 0;
    first = width;
    const int64_t k = b < batch ? keep[b] : -1;
    if (k >= 0) {
      first = min(width, (k >> log_t) + ((k & ((1 << log_t) - 1)) != 0));
      while (first + n < width && tables[b * t_b + first + n] >= 0) ++n;
    }
    return n;
  };
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    int64_t first;
    uint32_t total;
    plan_scan(count(b0 + tid, first), waves, total);
    all += total;
  }
  if (have + all > free_cap) return;
  uint32_t before = 0;
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    int64_t first;
    uint32_t total;
    const uint32_t n = count(b0 + tid, first);
    const uint32_t at = before + plan_scan(n, waves, total) - n;
    before += total;
    for (uint32_t i = 0; i < n; ++i) {
      int32_t* e = tables + (b0 + tid) * t_b + first + i;
      free_blocks[have + all - 1 - (at + i)] = *e;
      *e = -1;
    }
  }
  if (tid == 0) *free_count = have + all;
}

// ---------------------------------------------------------------------------
// The write: one workgroup per row, KV head, and keys or values; it works if its
// row begins a run. The run's largest |x| gives the scale, codes go out one by one.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint8_t f8_code(float x) {
  if (!(fabsf(x) <= 3.4e38f)) return 0x7F;
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false);
}
// the smallest e with amax <= 448 2^e
__device__ __forceinline__ int f8_exp(float amax) {
  if (amax == 0.f) return kMinExp;
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  // amax = 1.m 2^x: x - 8, one more where 1.m passes 1.75
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
  return max(e, kMinExp);
}

struct WriteArgs {
  const uint16_t *k, *v;
  int64_t k_r, k_h, v_r, v_h;
  const int64_t* slots;
  PagedCache c;
  int rows;
};

template <int D, bool BF>
__global__ __launch_bounds__(256) void write_blocks_kernel(const WriteArgs a) {
  __shared__ float red[4];
  const int row = blockIdx.x, h = blockIdx.y;
  const bool val = blockIdx.z;
  const int T = 1 << a.c.log_t, tid = threadIdx.x;
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.c.blocks << a.c.log_t) return;
  const int off = (int)(slot & (T - 1));
  if (off && row && a.slots[row - 1] == slot - 1) return;  // within a run
  int n = 1;
  while (off + n < T && row + n < a.rows && a.slots[row + n] == slot + n) ++n;
  const int64_t block = slot >> a.c.log_t;
  const uint16_t* src = val ? a.v + row * a.v_r + h * a.v_h : a.k + row * a.k_r + h * a.k_h;
  const int64_t s_r = val ? a.v_r : a.k_r;
  uint8_t* dst = (val ? a.c.v + block * a.c.v_b : a.c.k + block * a.c.k_b) + (int64_t)h * T * D;
  uint8_t* scale = (val ? a.c.vs : a.c.ks) + block * a.c.s_b + h;
  float amax = 0.f;
  for (int i = tid; i < n * D; i += 256) {
    const float x = fabsf(f16or_bf(src[(i / D) * s_r + i % D], BF));
    if (x <= 3.4e38f) amax = fmaxf(amax, x);
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
  if ((tid & 63) == 0) red[tid >> 6] = amax;
  const int old = (int)*scale - 127;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int e = off ? max(old, f8_exp(amax)) : f8_exp(amax);
  if (off && e > old)
    for (int i = tid; i < T * D; i += 256) {
      const float f = __builtin_amdgcn_cvt_f32_fp8(dst[i], 0);
      dst[i] = f8_code(__builtin_ldexpf(f, old - e));
    }
  __syncthreads();
  if (tid == 0) *scale = (uint8_t)(e + 127);
  for (int i = tid; i < n * D; i += 256) {
    const int t = i / D, d = i % D;
    const uint8_t code = f8_code(__builtin_ldexpf(f16or_bf(src[t * s_r + d], BF), -e));
    dst[val ? d * T + off + t : (off + t) * D + d] = code;
  }
}

static bool plan_shape_ok(int64_t batch, int64_t width, int64_t t_b, int64_t free_cap,
                          int block_size) {
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return false;
  return batch >= 0 && batch <= kPagedMaxBatch && width >= 1 && width <= kPagedMaxWidth &&
         t_b >= width && free_cap >= 1 && free_cap <= INT32_MAX;
}
static int log2_of(int block_size) {
  return block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
}

}  // namespace pe

using namespace pe;

extern "C" int pe_plan_step(const int64_t* lengths, const int64_t* counts, int32_t* tables,
                            int64_t t_b, int64_t batch, int64_t width, const int32_t* free_blocks,
                            int64_t free_cap, int64_t* free_count, int64_t rows, int block_size,
                            int64_t* starts, int64_t* positions, int64_t* slots,
                            int64_t* out_lengths, void* stream) {
  if (!lengths || !counts || !tables || !free_blocks || !free_count || !starts || !out_lengths ||
      (rows > 0 && (!positions || !slots)))
    return PE_ERR_NULL;
  if (!plan_shape_ok(batch, width, t_b, free_cap, block_size) || rows < 0 || rows > kPagedMaxRows)
    return PE_ERR_DIMS;
  if (batch == 0) return PE_OK;
  plan_step_kernel<<<1, kPlanThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      lengths, counts, tables, t_b, (int)batch, width, free_blocks, free_cap, free_count, (int)rows,
      log2_of(block_size), starts, positions, slots, out_lengths);
  return launch_status();
}

extern "C" int pe_release_blocks(int32_t* tables, int64_t t_b, int64_t batch, int64_t width,
                                 const int64_t* keep, int32_t* free_blocks, int64_t free_cap,
                                 int64_t* free_count, int block_size, void* stream) {
  if (!tables || !keep || !free_blocks || !free_count) return PE_ERR_NULL;
  if (!plan_shape_ok(batch, width, t_b, free_cap, block_size)) return PE_ERR_DIMS;
  if (batch == 0) return PE_OK;
  release_kernel<<<1, kPlanThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      tables, t_b, (int)batch, width, keep, free_blocks, free_cap, free_count, log2_of(block_size));
  return launch_status();
}

extern "C" int pe_write_blocks(const void* k, const void* v, int dtype, int64_t rows, int64_t k_r,
                               int64_t k_h, int64_t v_r, int64_t v_h, const int64_t* slots,
                               void* k_codes, int64_t k_b, void* v_codes, int64_t v_b, void* k_scale,
                               void* v_scale, int64_t s_b, int64_t blocks, int kv_heads,
                               int block_size, int head_dim, void* stream) {
  if (!k || !v || !slots) return PE_ERR_NULL;
  const int bf = bf16_flag(dtype);
  if (bf < 0) return PE_ERR_DTYPE;
  WriteArgs a;
  const int ok = paged_cache(a.c, k_codes, k_b, v_codes, v_b, k_scale, v_scale, s_b, blocks, kv_heads,
                             block_size, head_dim);
  if (ok != PE_OK) return ok;
  if (rows < 0 || rows > kPagedMaxRows || k_r < 0 || k_h < 0 || v_r < 0 || v_h < 0) return PE_ERR_DIMS;
  if (!aligned16(k) || !aligned16(v) || (k_r | k_h | v_r | v_h) % 8) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  a.k = reinterpret_cast<const uint16_t*>(k);
  a.v = reinterpret_cast<const uint16_t*>(v);
  a.k_r = k_r;
  a.k_h = k_h;
  a.v_r = v_r;
  a.v_h = v_h;
  a.slots = slots;
  a.rows = (int)rows;
  const dim3 grid((unsigned)rows, (unsigned)kv_heads, 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim * 2 + bf) {
    case 128: write_blocks_kernel<64, false><<<grid, 256, 0, st>>>(a); break;
    case 129: write_blocks_kernel<64, true><<<grid, 256, 0, st>>>(a); break;
    case 256: write_blocks_kernel<128, false><<<grid, 256, 0, st>>>(a); break;
    case 257: write_blocks_kernel<128, true><<<grid, 256, 0, st>>>(a); break;
    case 512: write_blocks_kernel<256, false><<<grid, 256, 0, st>>>(a); break;
    default: write_blocks_kernel<256, true><<<grid, 256, 0, st>>>(a); break;
  }
  return launch_status();
}
