// A step with several drafted tokens per sequence (a chain or a tree of them):
// the plan of the trees, the per-head norms of queries and keys with the rotary
// embedding and the cache write, and the accepted tokens' rows of the cache
// moved to their places. The attention is in pe_tree_attn.hip, the verification
// in pe_verify.hip.

#include "pe_tree.h"

namespace pe {

// ---------------------------------------------------------------------------
// positions and ancestor masks: one wave per sequence, lane = node
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(64) void tree_plan_kernel(const int64_t* __restrict__ parents,
                                                       int64_t stride,
                                                       const int64_t* __restrict__ lengths, int n,
                                                       int64_t* __restrict__ positions,
                                                       int64_t* __restrict__ masks) {
  const int i = threadIdx.x;
  const int64_t b = blockIdx.x;
  const int64_t p = i < n ? parents[b * stride + i] : -1;
  const uint64_t m = tree_mask(p, i, n);
  if (i >= n) return;
  const int64_t len = lengths[b];
  positions[b * n + i] = m && len >= 0 ? len + __popcll(m) - 1 : -1;
  masks[b * n + i] = (int64_t)m;
}

// ---------------------------------------------------------------------------
// y = x / sqrt(mean(x^2) + eps) * w per head, then pairs (j, j + rot / 2) turned
// by the position's angles; values pass as they are. D / 8 lanes a head, one
// 16-byte load each, so a row is read once and the norm, the rotation and the one
// rounding happen in registers. Bound by bytes: rows of 16-bit values read and
// written once.
// ---------------------------------------------------------------------------
struct RopeArgs {
  const uint16_t* qkv;
  int64_t ld, items;
  int heads, kv_heads, per_row, rot;
  const float* rope;
  int64_t rope_rows;
  const int64_t* positions;
  const uint16_t *qw, *kw;
  float eps;
  uint16_t *q_out, *k_out;
  // cache form
  uint16_t *kc, *vc;
  int64_t ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l;
  const int64_t* lengths;
  int64_t n, cap;
};

template <int D, bool BF, bool CACHE>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const RopeArgs a) {
  constexpr int LPG = D / 8;  // lanes per head
  const int lane = threadIdx.x & (LPG - 1);
  const int64_t item = (int64_t)blockIdx.x * (256 / LPG) + threadIdx.x / LPG;
  const bool live = item < a.items;  // the others take part in the exchanges
  const int64_t row = live ? item / a.per_row : 0;
  const int head = live ? (int)(item - row * a.per_row) : 0;
  const int H = a.heads, KVH = a.kv_heads;
  float v[8];
  load8<BF ? PE_DTYPE_BF16 : PE_DTYPE_F16>(a.qkv + row * a.ld + (int64_t)head * D + 8 * lane, v);
  const int64_t pos = a.positions[row];
  const bool inside = pos >= 0 && pos < a.rope_rows;
  if (head < H + KVH) {
    const uint16_t* w = head < H ? a.qw : a.kw;
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
#pragma unroll
      for (int off = LPG / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
      const float r = 1.f / __builtin_sqrtf(ss * (1.f / D) + a.eps);
      float g[8];
      load8<BF ? PE_DTYPE_BF16 : PE_DTYPE_F16>(w + 8 * lane, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= r * g[i];
    }
    const int hl = a.rot / 16;  // lanes of half the rotary dimensions
    const bool lo = lane < hl, in = lane < 2 * hl;
    const int me = (int)(threadIdx.x & 63);
    const int other = lo ? me + hl : in ? me - hl : me;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl(v[i], other, 64);
    if (in && inside) {
      const float* t = a.rope + pos * a.rot + 8 * (lo ? lane : lane - hl);
      float c[8], s[8];
      load8<PE_DTYPE_F32>(t, c);
      load8<PE_DTYPE_F32>(t + a.rot / 2, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * c[i] + (lo ? -o[i] : o[i]) * s[i];
    }
  }
  if (!live) return;
  uint4 out;
  out.x = pack16x2(v[0], v[1], BF);
  out.y = pack16x2(v[2], v[3], BF);
  out.z = pack16x2(v[4], v[5], BF);
  out.w = pack16x2(v[6], v[7], BF);
  if (!inside) out = make_uint4(0, 0, 0, 0);
  if (head < H) {
    *reinterpret_cast<uint4*>(a.q_out + (row * H + head) * D + 8 * lane) = out;
    return;
  }
  if constexpr (!CACHE) {
    *reinterpret_cast<uint4*>(a.k_out + (row * KVH + head - H) * D + 8 * lane) = out;
  } else {
    const int64_t b = row / a.n, slot = a.lengths[b] + (row - b * a.n);
    if (!inside || a.lengths[b] < 0 || a.lengths[b] > a.cap - a.n) return;
    if (head >= H + KVH) {
      *reinterpret_cast<uint4*>(a.vc + b * a.vs_b + (head - H - KVH) * a.vs_h + slot * a.vs_l +
                                8 * lane) = out;
    } else {
      uint16_t* k = a.kc + b * a.ks_b + (head - H) * a.ks_h + slot * a.ks_l;
      if (a.ks_d == 1) {
        *reinterpret_cast<uint4*>(k + 8 * lane) = out;
      } else {
        const uint32_t u[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          k[(8 * lane + i) * a.ks_d] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// cache rows of the accepted path to the front: slot len + j takes slot len +
// path[j]. Paths ascend, so path[j] >= j and no source lies before a later
// destination: a thread that goes through its own column in order of j never
// reads what it has written.
// ---------------------------------------------------------------------------
struct KeepArgs {
  uint16_t* c;
  int64_t s_layer, s_b, s_h, s_l, s_d;
  int heads, n, dim;
  int64_t cap;
  const int64_t *lengths, *path, *count;
};

// how many leading entries of the path are moved: those of an ascending path
// inside the n slots
__device__ __forceinline__ int keep_count(const KeepArgs& a, int64_t b, int lane) {
  const int64_t len = a.lengths[b];
  const int64_t c = a.count[b];
  if (len < 0 || len > a.cap - a.n || c <= 0) return 0;
  const int64_t p = lane < a.n ? a.path[b * a.n + lane] : -1;
  const int64_t before = __shfl_up(p, 1, 64);
  const bool ok = lane < c && p < a.n && p >= lane && (lane == 0 || p > before);
  const uint64_t bad = ~__ballot(ok);
  return bad ? __builtin_ctzll(bad) : 64;
}

// rows of 16-bit values, 16 bytes a thread (s_d = 1)
__global__ __launch_bounds__(256) void keep_rows_kernel(const KeepArgs a) {
  const int64_t b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int count = keep_count(a, b, lane);
  const int per = a.dim / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // (head, 8 dimensions)
  if (i >= (int64_t)a.heads * per) return;
  const int64_t len = a.lengths[b];
  uint16_t* c = a.c + blockIdx.z * a.s_layer + b * a.s_b + (i / per) * a.s_h + (i % per) * 8 +
                len * a.s_l;
  for (int j = 0; j < count; ++j) {
    const int64_t p = a.path[b * a.n + j];
    if (p != j)
      *reinterpret_cast<uint4*>(c + j * a.s_l) = *reinterpret_cast<const uint4*>(c + p * a.s_l);
  }
}

// columns (s_l = 1): a wave moves the slots of one dimension, lane = j; every
// lane's load comes before any lane's store
__global__ __launch_bounds__(256) void keep_cols_kernel(const KeepArgs a) {
  const int64_t b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int count = keep_count(a, b, lane);
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (head, dimension)
  if (i >= (int64_t)a.heads * a.dim || lane >= count) return;
  uint16_t* c = a.c + blockIdx.z * a.s_layer + b * a.s_b + (i / a.dim) * a.s_h +
                (i % a.dim) * a.s_d + a.lengths[b];
  const uint16_t v = c[a.path[b * a.n + lane]];
  c[lane] = v;
}

template <bool BF, bool CACHE>
static int launch_rope(int dim, const RopeArgs& a, hipStream_t st) {
  const int64_t per = 256 / (dim / 8);
  const int64_t grid = (a.items + per - 1) / per;
  if (grid > INT32_MAX) return PE_ERR_DIMS;
  if (dim == 64) qk_norm_rope_kernel<64, BF, CACHE><<<(unsigned)grid, 256, 0, st>>>(a);
  else if (dim == 128) qk_norm_rope_kernel<128, BF, CACHE><<<(unsigned)grid, 256, 0, st>>>(a);
  else qk_norm_rope_kernel<256, BF, CACHE><<<(unsigned)grid, 256, 0, st>>>(a);
  return launch_status();
}

// what both forms check and set
static int rope_args(const void* qkv, int dtype, int64_t rows, int64_t ld, int heads, int kv_heads,
                     int head_dim, const float* rope, int64_t rope_rows, int rot,
                     const int64_t* positions, const void* q_weight, const void* k_weight, float eps,
                     void* q_out, bool cache, RopeArgs& a) {
  if (!qkv || !rope || !positions || !q_out) return PE_ERR_NULL;
  if (bf16_flag(dtype) < 0) return PE_ERR_DTYPE;
  if (rows < 0 || heads < 1 || kv_heads < 1 || heads > 65536 || kv_heads > 65536 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || rope_rows < 1 || rot < 16 ||
      rot % 16 || rot > head_dim || ld < (int64_t)(heads + 2 * kv_heads) * head_dim)
    return PE_ERR_DIMS;
  if (!aligned16(qkv) || ld % 8 || !aligned16(rope) || !aligned16(q_out) ||
      (q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)))
    return PE_ERR_ALIGN;
  a = RopeArgs{};
  a.qkv = reinterpret_cast<const uint16_t*>(qkv);
  a.ld = ld;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.per_row = heads + (cache ? 2 : 1) * kv_heads;
  if (rows > INT64_MAX / 4 / a.per_row) return PE_ERR_DIMS;
  a.items = rows * a.per_row;
  a.rot = rot;
  a.rope = rope;
  a.rope_rows = rope_rows;
  a.positions = positions;
  a.qw = reinterpret_cast<const uint16_t*>(q_weight);
  a.kw = reinterpret_cast<const uint16_t*>(k_weight);
  a.eps = eps;
  a.q_out = reinterpret_cast<uint16_t*>(q_out);
  return PE_OK;
}

}  // namespace pe

using namespace pe;

extern "C" int pe_tree_plan(const int64_t* parents, int64_t parents_stride, const int64_t* lengths,
                            int64_t batch, int n, int64_t* positions, int64_t* masks, void* stream) {
  if (!parents || !lengths || !positions || !masks) return PE_ERR_NULL;
  if (batch < 0 || batch > INT32_MAX || n < 1 || n > kTreeMax || parents_stride < 0)
    return PE_ERR_DIMS;
  if (batch == 0) return PE_OK;
  tree_plan_kernel<<<(unsigned)batch, 64, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      parents, parents_stride, lengths, n, positions, masks);
  return launch_status();
}

extern "C" int pe_qk_norm_rope(const void* qkv, int dtype, int64_t rows, int64_t ld, int heads,
                               int kv_heads, int head_dim, const float* rope, int64_t rope_rows,
                               int rot, const int64_t* positions, const void* q_weight,
                               const void* k_weight, float eps, void* q_out, void* k_out,
                               void* stream) {
  RopeArgs a;
  const int rc = rope_args(qkv, dtype, rows, ld, heads, kv_heads, head_dim, rope, rope_rows, rot,
                           positions, q_weight, k_weight, eps, q_out, false, a);
  if (rc != PE_OK) return rc;
  if (!k_out) return PE_ERR_NULL;
  if (!aligned16(k_out)) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  a.k_out = reinterpret_cast<uint16_t*>(k_out);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return bf16_flag(dtype) ? launch_rope<true, false>(head_dim, a, st)
                          : launch_rope<false, false>(head_dim, a, st);
}

extern "C" int pe_qk_norm_rope_write(const void* qkv, int dtype, int64_t batch, int64_t n, int64_t ld,
                                     int heads, int kv_heads, int head_dim, const float* rope,
                                     int64_t rope_rows, int rot, const int64_t* positions,
                                     const void* q_weight, const void* k_weight, float eps,
                                     void* q_out, void* k_cache, int64_t ks_b, int64_t ks_h,
                                     int64_t ks_l, int64_t ks_d, void* v_cache, int64_t vs_b,
                                     int64_t vs_h, int64_t vs_l, const int64_t* lengths, int64_t cap,
                                     void* stream) {
  if (!k_cache || !v_cache || !lengths) return PE_ERR_NULL;
  if (batch < 0 || n < 1 || batch > INT64_MAX / 8 / n || cap < 1) return PE_ERR_DIMS;
  RopeArgs a;
  const int rc = rope_args(qkv, dtype, batch * n, ld, heads, kv_heads, head_dim, rope, rope_rows, rot,
                           positions, q_weight, k_weight, eps, q_out, true, a);
  if (rc != PE_OK) return rc;
  const int ok = cache_strides(k_cache, ks_b, ks_h, ks_l, ks_d, v_cache, vs_b, vs_h, vs_l);
  if (ok != PE_OK) return ok;
  if (batch == 0) return PE_OK;
  a.kc = reinterpret_cast<uint16_t*>(k_cache);
  a.vc = reinterpret_cast<uint16_t*>(v_cache);
  a.ks_b = ks_b, a.ks_h = ks_h, a.ks_l = ks_l, a.ks_d = ks_d;
  a.vs_b = vs_b, a.vs_h = vs_h, a.vs_l = vs_l;
  a.lengths = lengths;
  a.n = n;
  a.cap = cap;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return bf16_flag(dtype) ? launch_rope<true, true>(head_dim, a, st)
                          : launch_rope<false, true>(head_dim, a, st);
}

extern "C" int pe_keep_accepted(void* cache, int64_t layers, int64_t batch, int heads, int64_t cap,
                                int dim, int64_t s_layer, int64_t s_b, int64_t s_h, int64_t s_l,
                                int64_t s_d, const int64_t* lengths, const int64_t* path,
                                const int64_t* count, int n, void* stream) {
  if (!cache || !lengths || !path || !count) return PE_ERR_NULL;
  if (layers < 0 || layers > 65535 || batch < 0 || batch > 65535 || heads < 1 || heads > 65536 ||
      cap < 1 || dim < 8 || dim % 8 || dim > 4096 || n < 1 || n > kTreeMax || (s_d != 1 && s_l != 1))
    return PE_ERR_DIMS;
  if (s_d == 1 && (!aligned16(cache) || (s_layer | s_b | s_h | s_l) % 8)) return PE_ERR_ALIGN;
  if (layers == 0 || batch == 0) return PE_OK;
  KeepArgs a{reinterpret_cast<uint16_t*>(cache), s_layer, s_b, s_h, s_l, s_d,
             heads, n, dim, cap, lengths, path, count};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t items = (int64_t)heads * (s_d == 1 ? dim / 8 : dim);
  const int64_t per = s_d == 1 ? 256 : 4;
  const dim3 grid((unsigned)((items + per - 1) / per), (unsigned)batch, (unsigned)layers);
  if (s_d == 1) keep_rows_kernel<<<grid, 256, 0, st>>>(a);
  else keep_cols_kernel<<<grid, 256, 0, st>>>(a);
  return launch_status();
}
