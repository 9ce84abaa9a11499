// Attention of the drafted tokens of a step over a cache: every token of a
// sequence sees the sequence's cached positions and, of the drafted ones behind
// them, those that its mask names (itself and its ancestors).

#include "pe_tree.h"

namespace pe {

struct TreeAttnArgs {
  const uint16_t* q;
  int64_t q_b, q_n;
  const uint16_t *k, *v;
  int64_t ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l;
  const int64_t *lengths, *masks;
  int64_t m_b;
  uint16_t* out;
  int n, heads, kv_heads;
  int64_t cap;
  float scale;
};

// one wave per (sequence, drafted token, query head): lane = position for the
// scores, lane = dimensions for the values
template <int D, bool BF>
__global__ __launch_bounds__(64) void tree_attn_kernel(const TreeAttnArgs a) {
  __shared__ float qs[D];
  const int lane = threadIdx.x;
  const int64_t item = blockIdx.x;
  const int h = (int)(item % a.heads);
  const int i = (int)(item / a.heads % a.n);
  const int64_t b = item / a.heads / a.n;
  const int64_t len = a.lengths[b];
  uint16_t* out = a.out + item * D;
  if (len < 0 || len > a.cap - a.n) {
    for (int d = lane; d < D; d += 64) out[d] = 0;
    return;
  }
  const uint64_t mask = (uint64_t)a.masks[b * a.m_b + i];
  const uint16_t* q = a.q + b * a.q_b + i * a.q_n + (int64_t)h * D;
  for (int d = lane; d < D; d += 64) qs[d] = f16or_bf(q[d], BF);
  __syncthreads();
  const int kvh = h / (a.heads / a.kv_heads);
  const uint16_t* k = a.k + b * a.ks_b + kvh * a.ks_h;
  const uint16_t* v = a.v + b * a.vs_b + kvh * a.vs_h;
  float m = -__builtin_inff(), l = 0.f, o[D / 64] = {};
  const int64_t end = len + a.n;
  for (int64_t p0 = 0; p0 < end; p0 += 64) {
    const int64_t p = p0 + lane;
    const bool seen = p < len || (p < end && (mask >> (p - len) & 1));
    float s = -__builtin_inff();
    if (seen) {
      s = 0.f;
      for (int d = 0; d < D; ++d)
        s = __builtin_fmaf(qs[d], f16or_bf(k[p * a.ks_l + d * a.ks_d], BF), s);
      s *= a.scale;
    }
    float mn = s;
    for (int off = 32; off >= 1; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
    mn = fmaxf(mn, m);
    const float base = mn == -__builtin_inff() ? 0.f : mn;
    const float e = seen ? expf(s - base) : 0.f, al = expf(m - base);
    m = mn;
    l = l * al + wave_sum(e);
    for (int c = 0; c < D / 64; ++c) o[c] *= al;
    uint64_t live = __ballot(seen);
    while (live) {
      const int j = __builtin_ctzll(live);
      live &= live - 1;
      const float w = __shfl(e, j, 64);
      for (int c = 0; c < D / 64; ++c)
        o[c] = __builtin_fmaf(w, f16or_bf(v[(p0 + j) * a.vs_l + c * 64 + lane], BF), o[c]);
    }
  }
  for (int c = 0; c < D / 64; ++c) out[c * 64 + lane] = to16(l > 0.f ? o[c] / l : 0.f, BF);
}

template <bool BF>
static int launch_tree_attn(int dim, const TreeAttnArgs& a, int64_t batch, hipStream_t st) {
  const unsigned grid = (unsigned)(batch * a.n * a.heads);
  if (dim == 64) tree_attn_kernel<64, BF><<<grid, 64, 0, st>>>(a);
  else if (dim == 128) tree_attn_kernel<128, BF><<<grid, 64, 0, st>>>(a);
  else tree_attn_kernel<256, BF><<<grid, 64, 0, st>>>(a);
  return launch_status();
}

static bool tree_attn_shape_ok(int64_t batch, int n, int heads, int kv_heads, int dim, int64_t cap) {
  return batch >= 1 && batch <= 65535 && n >= 1 && n <= kTreeMax && kv_heads >= 1 && heads >= 1 &&
         heads <= 65536 && heads % kv_heads == 0 && (dim == 64 || dim == 128 || dim == 256) &&
         cap >= 1 && batch * n * heads <= INT32_MAX;
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_tree_attention_workspace_size(int64_t batch, int n, int heads, int kv_heads,
                                                   int head_dim, int64_t cap) {
  (void)batch, (void)n, (void)heads, (void)kv_heads, (void)head_dim, (void)cap;
  return 0;
}

extern "C" int pe_tree_attention(const void* q, int dtype, int64_t q_b, int64_t q_n,
                                 const void* k_cache, int64_t ks_b, int64_t ks_h, int64_t ks_l,
                                 int64_t ks_d, const void* v_cache, int64_t vs_b, int64_t vs_h,
                                 int64_t vs_l, const int64_t* lengths, const int64_t* masks,
                                 int64_t m_b, void* out, int64_t batch, int n, int heads,
                                 int kv_heads, int head_dim, int64_t cap, float scale,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !lengths || !masks || !out) return PE_ERR_NULL;
  const int bf = bf16_flag(dtype);
  if (bf < 0) return PE_ERR_DTYPE;
  if (batch == 0) return PE_OK;
  if (!tree_attn_shape_ok(batch, n, heads, kv_heads, head_dim, cap) || q_b < 0 || q_n < 0 || m_b < 0)
    return PE_ERR_DIMS;
  if (!aligned16(q) || (q_b | q_n) % 8 || !aligned16(out)) return PE_ERR_ALIGN;
  const int ok = cache_strides(k_cache, ks_b, ks_h, ks_l, ks_d, v_cache, vs_b, vs_h, vs_l);
  if (ok != PE_OK) return ok;
  TreeAttnArgs a{reinterpret_cast<const uint16_t*>(q), q_b, q_n,
                 reinterpret_cast<const uint16_t*>(k_cache),
                 reinterpret_cast<const uint16_t*>(v_cache), ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l,
                 lengths, masks, m_b, reinterpret_cast<uint16_t*>(out), n, heads, kv_heads, cap, scale};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return bf ? launch_tree_attn<true>(head_dim, a, batch, st)
            : launch_tree_attn<false>(head_dim, a, batch, st);
}
