// Attention over the paged 8-bit cache: a wave per row and head, 64 positions a
// step, scores and sums in fp32.

#include "pe_paged.h"

namespace pe {

struct PagedAttnArgs {
  const uint16_t* q;
  int64_t q_r;
  PagedCache c;
  const int32_t* tables;
  int64_t t_b, width;
  const int64_t *starts, *lengths;
  uint16_t* out;
  int rows, batch, heads, group;
  int64_t window, sinks;
  float scale;
};

__device__ __forceinline__ float wave_max64(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

template <int D, bool BF>
__global__ __launch_bounds__(64) void paged_attn_kernel(const PagedAttnArgs a) {
  __shared__ float qs[D];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int T = 1 << a.c.log_t;
  int lo = 0, hi = a.batch;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid + 1] > row) hi = mid;
    else lo = mid + 1;
  }
  uint16_t* out = a.out + ((int64_t)row * a.heads + h) * D;
  float o[D / 64] = {};
  float m = -__builtin_inff(), l = 0.f;
  int64_t p = -1;
  const int b = lo;
  if (b < a.batch && row >= a.starts[b] && a.lengths[b] >= 0)
    p = a.lengths[b] - (a.starts[b + 1] - row);
  const uint16_t* q = a.q + row * a.q_r + (int64_t)h * D;
  for (int d = lane; d < D; d += 64) qs[d] = f16or_bf(q[d], BF) * a.scale;
  __syncthreads();
  const int kvh = h / a.group;
  const int64_t end = min(p + 1, a.width << a.c.log_t);
  for (int64_t j0 = 0; j0 < end; j0 += 64) {
    if (a.window && j0 + 63 <= p - a.window && j0 >= a.sinks) continue;
    const int64_t j = j0 + lane;
    bool seen = j < end && (!a.window || j > p - a.window || j < a.sinks);
    const int64_t block = seen ? a.tables[b * a.t_b + (j >> a.c.log_t)] : -1;
    seen = block >= 0 && block < a.c.blocks;
    float s = -__builtin_inff();
    if (seen) {
      const uint8_t* k = a.c.k + block * a.c.k_b + ((int64_t)kvh * T + (j & (T - 1))) * D;
      s = 0.f;
      for (int d = 0; d < D; ++d) s += qs[d] * __builtin_amdgcn_cvt_f32_fp8(k[d], 0);
      s *= e8m0(a.c.ks[block * a.c.s_b + kvh]);
    }
    const float top = fmaxf(m, wave_max64(s));
    const float base = top == -__builtin_inff() ? 0.f : top;
    const float al = expf(m - base);
    const float w = expf(s - base);
    m = top;
    l = l * al + wave_sum(w);
    for (int i = 0; i < D / 64; ++i) o[i] *= al;
    for (int i = 0; i < 64; ++i) {
      const int64_t blk = __shfl(seen ? (int)block : -1, i, 64);
      if (blk < 0) continue;
      const float pw = __shfl(w, i, 64) * e8m0(a.c.vs[blk * a.c.s_b + kvh]);
      const uint8_t* v = a.c.v + blk * a.c.v_b + (int64_t)kvh * T * D + ((j0 + i) & (T - 1));
      for (int u = 0; u < D / 64; ++u)
        o[u] += pw * __builtin_amdgcn_cvt_f32_fp8(v[(lane + 64 * u) * T], 0);
    }
  }
  for (int u = 0; u < D / 64; ++u)
    out[lane + 64 * u] = to16(l > 0.f || l != l ? o[u] / l : 0.f, BF);
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_paged_attention_workspace_size(int64_t rows, int64_t batch, int heads,
                                                    int kv_heads, int head_dim, int64_t positions) {
  return 0;
}

extern "C" int pe_paged_attention(const void* q, int dtype, int64_t q_r, int64_t rows, int heads,
                                  const void* k_codes, int64_t k_b, const void* v_codes, int64_t v_b,
                                  const void* k_scale, const void* v_scale, int64_t s_b,
                                  int64_t blocks, int kv_heads, int block_size, int head_dim,
                                  const int32_t* tables, int64_t t_b, int64_t batch, int64_t width,
                                  const int64_t* starts, const int64_t* lengths, int64_t window,
                                  int64_t sinks, float scale, void* out, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (!q || !tables || !starts || !lengths || !out) return PE_ERR_NULL;
  const int bf = bf16_flag(dtype);
  if (bf < 0) return PE_ERR_DTYPE;
  PagedAttnArgs a;
  const int ok = paged_cache(a.c, k_codes, k_b, v_codes, v_b, k_scale, v_scale, s_b, blocks, kv_heads,
                             block_size, head_dim);
  if (ok != PE_OK) return ok;
  if (rows < 0 || rows > kPagedMaxRows || batch < 0 || batch > kPagedMaxBatch || width < 1 ||
      width > INT32_MAX / 128 || t_b < width || heads < 1 || heads > 65535 || heads % kv_heads ||
      q_r < 0 || window < 0 || sinks < 0 || !(scale >= 0.f && scale <= 3e38f))
    return PE_ERR_DIMS;
  if (!aligned16(q) || q_r % 8 || !aligned16(out)) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  a.q = reinterpret_cast<const uint16_t*>(q);
  a.q_r = q_r;
  a.tables = tables;
  a.t_b = t_b;
  a.width = width;
  a.starts = starts;
  a.lengths = lengths;
  a.out = reinterpret_cast<uint16_t*>(out);
  a.rows = (int)rows;
  a.batch = (int)batch;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.window = window;
  a.sinks = sinks;
  a.scale = scale;
  const dim3 grid((unsigned)rows, (unsigned)heads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim * 2 + bf) {
    case 128: paged_attn_kernel<64, false><<<grid, 64, 0, st>>>(a); break;
    case 129: paged_attn_kernel<64, true><<<grid, 64, 0, st>>>(a); break;
    case 256: paged_attn_kernel<128, false><<<grid, 64, 0, st>>>(a); break;
    case 257: paged_attn_kernel<128, true><<<grid, 64, 0, st>>>(a); break;
    case 512: paged_attn_kernel<256, false><<<grid, 64, 0, st>>>(a); break;
    default: paged_attn_kernel<256, true><<<grid, 64, 0, st>>>(a); break;
  }
  return launch_status();
}
