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
// written once. The arithmetic behind the products of two 16-bit values (exact in 32
// bits) is in 64 and its result is rounded once, so that a value is the exact one rounded
// (but for one within 2^-45 of the middle between two): keys do not depend on the order
// of a sum or on which call wrote them. In 32 bits one fp16 value in 5,500 and one bf16
// value in 53,000 rounds the other way; rounded to 32 bits before the 16, one in 18,000
// and in 170,000. It is about half of the vector instructions, which now take as long as
// the bytes: 8192 rows of 48 heads of 128 to a cache 55 to 57 us (3.6 TB/s; with two
// roundings 53), keys by position 51; 16 rows 4.2 us.
//
// A workgroup takes a row (or several of a model with few heads), its heads four
// loads a lane at a time, the row's angles once. Keys that the cache stores by
// dimension go through LDS instead, 64 rows of a head a workgroup, and leave as 16
// bytes of eight consecutive positions (as 2-byte stores the 8192 rows took 101 us).
// ---------------------------------------------------------------------------
constexpr int kRopeTile = 64;

struct RopeArgs {
  const uint16_t* qkv;
  int64_t ld, rows;
  int heads, kv_heads, rot;
  int per_row;        // heads of a row that the row form takes
  int rows_per_wg;    // of the row form,
  int parts, part;    // or workgroups per row and heads of each
  int64_t col_wgs;    // workgroups that take keys by dimension, before those of the row form
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

// cosines and sines of a lane's eight dimensions (sines of the lower half negated);
// lanes past the rotary dimensions have 1 and 0
struct RopeAngles {
  double c[8], s[8];
};
__device__ __forceinline__ RopeAngles rope_angles(const RopeArgs& a, int64_t pos, int lane) {
  RopeAngles r;
  const int hl = a.rot / 16;  // lanes of half the rotary dimensions
  float c[8] = {1, 1, 1, 1, 1, 1, 1, 1}, s[8] = {};
  if (lane < 2 * hl && pos >= 0 && pos < a.rope_rows) {
    const float* t = a.rope + pos * a.rot + 8 * (lane < hl ? lane : lane - hl);
    load8<PE_DTYPE_F32>(t, c);
    load8<PE_DTYPE_F32>(t + a.rot / 2, s);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r.c[i] = c[i];
    r.s[i] = lane < hl ? -s[i] : s[i];
  }
  return r;
}

// 64-bit lane move by a DPP control word
template <int CTRL>
__device__ __forceinline__ double dpp_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// sum over the D / 8 lanes of a head, in each of them
template <int D>
__device__ __forceinline__ double head_sum(double v) {
  v += dpp_move<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v += dpp_move<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v += dpp_move<0x141>(v);  // row_half_mirror: the other quad of eight
  if constexpr (D >= 128) v += dpp_move<0x140>(v);  // row_mirror: the other eight of 16
  if constexpr (D == 256) v += __shfl_xor(v, 16, 64);
  return v;
}

// fp32 that rounds to 16 bits as v does: v's first 20 fraction bits, the last of them set
// where anything follows (a bf16 result below 2^-126 is rounded twice all the same)
__device__ __forceinline__ float to_odd_f32(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t hi = (uint32_t)(u >> 32) | min((uint32_t)u, 1u);
  return (float)__builtin_bit_cast(double, (uint64_t)hi << 32);
}

// one head: u (eight 16-bit values of the lane) normed with w, turned, rounded
template <int D, bool BF>
__device__ __forceinline__ u32x4v rope_head(const RopeArgs& a, u32x4v u, const uint16_t* w,
                                            const RopeAngles& r, int lane) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t two = u[i / 2];
    v[i] = f16or_bf((uint16_t)(two >> (16 * (i & 1))), BF);
  }
  double y = 1.0;
  if (w) {
    float g[8];
    double ss = 0.0;
    load8<BF ? PE_DTYPE_BF16 : PE_DTYPE_F16>(w + 8 * lane, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)v[i], (double)v[i], ss);
    const double x = head_sum<D>(ss) * (1.0 / D) + (double)a.eps;
    // 1 / sqrt(x): the instruction's value (relative error below 2^-26) and a Newton step
    y = __builtin_amdgcn_rsq(x);
    const double z = y * __builtin_fma(-0.5 * x * y, y, 1.5);
    y = x < 1e300 ? z : y;  // an infinite square: 0
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= g[i];  // exact: two 16-bit values
  }
  float o[8], f[8];
  if (a.rot == D && D == 128) {  // lane ^ 8
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = lane_xor<8>(v[i]);
  } else {
    const int hl = a.rot / 16, me = (int)(threadIdx.x & 63);
    const int other = lane < hl ? me + hl : lane < 2 * hl ? me - hl : me;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl(v[i], other, 64);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double t = v[i];
    // dimensions past the rotary ones keep their value, whatever the other lane holds
    if (lane < a.rot / 8) t = __builtin_fma(t, r.c[i], (double)o[i] * r.s[i]);
    f[i] = to_odd_f32(t * y);
    // kept in 32 bits: the direct conversion to 16 takes a dozen instructions more
    asm("" : "+v"(f[i]));
  }
  return u32x4v{pack16x2(f[0], f[1], BF), pack16x2(f[2], f[3], BF), pack16x2(f[4], f[5], BF),
                pack16x2(f[6], f[7], BF)};
}

// where row `row` of the step goes in the cache: its sequence and slot, -1 if nowhere
__device__ __forceinline__ int64_t rope_slot(const RopeArgs& a, int64_t row, int64_t pos, int64_t& b) {
  b = (uint32_t)row / (uint32_t)a.n;  // below 2^31 both
  const int64_t len = a.lengths[b];
  if (pos < 0 || pos >= a.rope_rows || len < 0 || len > a.cap - a.n) return -1;
  return len + (row - b * a.n);
}

// ONE: a workgroup takes one row, so that what follows from the row is uniform. Five waves
// a SIMD where the registers allow it: heads of 256 take more, and several rows to a cache
// would spill two to six of them (4 x 2048 rows of 8 heads of 128, keys by dimension: 20.1
// us, with four waves 18.2; by position 16.3 and 16.2).
template <int D, bool BF, bool CACHE, bool COL, bool ONE>
__global__ __launch_bounds__(256, D == 256 || (CACHE && !ONE) ? 4 : 5) void qk_norm_rope_kernel(const RopeArgs a) {
  constexpr int LPG = D / 8;      // lanes per head
  constexpr int G = 256 / LPG;    // heads at a time
  constexpr int U = 4;            // loads of a lane on their way
  const int lane = threadIdx.x % LPG, grp = threadIdx.x / LPG;
  const int H = a.heads, KVH = a.kv_heads;
  if constexpr (COL) {
    constexpr int PITCH = kRopeTile + 2;  // 16-bit values
    __shared__ uint16_t tile[D * PITCH];
    __shared__ int64_t slots[kRopeTile];
    if ((int64_t)blockIdx.x < a.col_wgs) {  // first: they take longest
      // keys of one head, rows i0 .. of one sequence
      constexpr int P = kRopeTile / G;  // passes, their loads all out at once
      const int per_seq = (int)((a.n + kRopeTile - 1) / kRopeTile);
      const int kvh = (int)blockIdx.x % KVH, rest = (int)blockIdx.x / KVH;
      const int64_t b = rest / per_seq, i0 = (int64_t)(rest % per_seq) * kRopeTile;
      const int count = (int)(a.n - i0 < kRopeTile ? a.n - i0 : kRopeTile);
      const int64_t first = b * a.n + i0;
      u32x4v u[P];
      int64_t pos[P];
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int64_t row = first + min(k * G + grp, count - 1);
        pos[k] = a.positions[row];
        u[k] = *reinterpret_cast<const u32x4v*>(a.qkv + row * a.ld + (int64_t)(H + kvh) * D + 8 * lane);
      }
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int r = k * G + grp;
        if (k * G >= count) break;
        const RopeAngles ang = rope_angles(a, pos[k], lane);
        const u32x4v out = rope_head<D, BF>(a, u[k], a.kw, ang, lane);
        if (r < count) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t two = out[i / 2];
            tile[(8 * lane + i) * PITCH + r] = (uint16_t)(two >> (16 * (i & 1)));
          }
          int64_t seq;
          if (lane == 0) slots[r] = rope_slot(a, first + r, pos[k], seq);
        }
      }
      __syncthreads();
      uint16_t* k = a.kc + b * a.ks_b + kvh * a.ks_h;
      const int chunks = (count + 7) / 8;
      for (int t = threadIdx.x; t < D * chunks; t += 256) {
        const int d = t / chunks, c = t - d * chunks;
        bool whole = 8 * c + 8 <= count;
        for (int e = 0; e < 8 && whole; ++e) whole = slots[8 * c + e] >= 0;
        uint16_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[d * PITCH + 8 * c + e];
        uint16_t* dst = k + d * a.ks_d;
        if (whole) {
          __builtin_memcpy(dst + slots[8 * c], v, 16);  // any alignment
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * c + e < count && slots[8 * c + e] >= 0) dst[slots[8 * c + e]] = v[e];
        }
      }
      return;
    }
  }
  const int wg = blockIdx.x - (COL ? (int)a.col_wgs : 0);
  const int64_t row0 = ONE ? wg / a.parts : (int64_t)wg * a.rows_per_wg;
  const int head0 = ONE ? (wg - (int)row0 * a.parts) * a.part : 0;
  const int here = (int)(a.rows - row0 < a.rows_per_wg ? a.rows - row0 : a.rows_per_wg);
  const int items = ONE ? min(a.part, a.per_row - head0) : here * a.per_row;
  RopeAngles ang;
  int64_t pos = 0, b = 0, slot = 0;
  if constexpr (ONE) {
    pos = a.positions[row0];
    if constexpr (CACHE) slot = rope_slot(a, row0, pos, b);
  }
  for (int i0 = 0; i0 < items; i0 += U * G) {
    u32x4v u[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int item = min(i0 + k * G + grp, items - 1);
      const int local = ONE ? 0 : item / a.per_row;
      int head = head0 + item - local * a.per_row;
      if (COL && head >= H) head += KVH;
      u[k] = *reinterpret_cast<const u32x4v*>(a.qkv + (row0 + local) * a.ld + head * D + 8 * lane);
    }
    if (ONE && i0 == 0) ang = rope_angles(a, pos, lane);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int item = i0 + k * G + grp;
      if (i0 + k * G >= items) break;
      const bool live = item < items;  // the others take part in the exchanges
      const int at = live ? item : items - 1;
      const int local = ONE ? 0 : at / a.per_row;
      int head = head0 + at - local * a.per_row;
      if (COL && head >= H) head += KVH;
      const int64_t row = row0 + local;
      if constexpr (!ONE) {
        pos = a.positions[row];
        if constexpr (CACHE) slot = rope_slot(a, row, pos, b);
        ang = rope_angles(a, pos, lane);
      }
      u32x4v out = u[k];
      if (__any(head < H + KVH)) {  // a wave of values alone passes them
        const u32x4v turned = rope_head<D, BF>(a, u[k], head < H ? a.qw : a.kw, ang, lane);
        if (head < H + KVH) out = turned;
      }
      if (!live) continue;
      if (head < H || !CACHE) {
        if (pos < 0 || pos >= a.rope_rows) out = u32x4v{0, 0, 0, 0};
        uint16_t* dst = head < H ? a.q_out + (row * H + head) * D : a.k_out + (row * KVH + head - H) * D;
        *reinterpret_cast<u32x4v*>(dst + 8 * lane) = out;
      } else if (slot >= 0) {
        uint16_t* dst = head < H + KVH
                            ? a.kc + b * a.ks_b + slot * a.ks_l + (head - H) * a.ks_h
                            : a.vc + b * a.vs_b + slot * a.vs_l + (head - H - KVH) * a.vs_h;
        *reinterpret_cast<u32x4v*>(dst + 8 * lane) = out;
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

template <int D, bool BF, bool ONE>
static int launch_rope(const RopeArgs& a, bool cache, bool col, int64_t grid, hipStream_t st) {
  if (!cache) qk_norm_rope_kernel<D, BF, false, false, ONE><<<(unsigned)grid, 256, 0, st>>>(a);
  else if (col) qk_norm_rope_kernel<D, BF, true, true, ONE><<<(unsigned)grid, 256, 0, st>>>(a);
  else qk_norm_rope_kernel<D, BF, true, false, ONE><<<(unsigned)grid, 256, 0, st>>>(a);
  return launch_status();
}
template <int D, bool BF>
static int launch_rope(RopeArgs a, bool cache, hipStream_t st) {
  const bool col = cache && a.ks_d != 1;
  a.per_row = a.heads + (!cache ? 1 : col ? 1 : 2) * a.kv_heads;
  const int at_once = 256 / (D / 8);
  a.rows_per_wg = a.per_row >= at_once ? 1 : at_once / a.per_row;
  // few rows: a workgroup a pass, so that no pass waits for another
  const int passes = (a.per_row + at_once - 1) / at_once;
  a.parts = a.rows * passes <= 8 * (int64_t)num_cus() ? passes : 1;
  a.part = a.parts > 1 ? at_once : a.per_row;
  a.col_wgs = col ? a.rows / a.n * a.kv_heads * ((a.n + kRopeTile - 1) / kRopeTile) : 0;
  const int64_t grid = a.col_wgs + (a.parts > 1 ? a.rows * a.parts
                                                : (a.rows + a.rows_per_wg - 1) / a.rows_per_wg);
  if (grid > kTreeMaxGrid) return PE_ERR_DIMS;
  return a.rows_per_wg == 1 ? launch_rope<D, BF, true>(a, cache, col, grid, st)
                            : launch_rope<D, BF, false>(a, cache, col, grid, st);
}
template <bool BF>
static int launch_rope(int dim, const RopeArgs& a, bool cache, hipStream_t st) {
  return dim == 64 ? launch_rope<64, BF>(a, cache, st)
         : dim == 128 ? launch_rope<128, BF>(a, cache, st) : launch_rope<256, BF>(a, cache, st);
}

// what both forms check and set
static int rope_args(const void* qkv, int dtype, int64_t rows, int64_t ld, int heads, int kv_heads,
                     int head_dim, const float* rope, int64_t rope_rows, int rot,
                     const int64_t* positions, const void* q_weight, const void* k_weight, float eps,
                     void* q_out, RopeArgs& a) {
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
  if (rows > INT32_MAX) return PE_ERR_DIMS;
  a.rows = rows;
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
  if (batch < 0 || batch > kTreeMaxGrid || n < 1 || n > kTreeMax || parents_stride < 0)
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
                           positions, q_weight, k_weight, eps, q_out, a);
  if (rc != PE_OK) return rc;
  if (!k_out) return PE_ERR_NULL;
  if (!aligned16(k_out)) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  a.k_out = reinterpret_cast<uint16_t*>(k_out);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return bf16_flag(dtype) ? launch_rope<true>(head_dim, a, false, st)
                          : launch_rope<false>(head_dim, a, false, st);
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
  if (batch < 0 || n < 1 || n > INT32_MAX || batch > INT64_MAX / 8 / n || cap < 1) return PE_ERR_DIMS;
  RopeArgs a;
  const int rc = rope_args(qkv, dtype, batch * n, ld, heads, kv_heads, head_dim, rope, rope_rows, rot,
                           positions, q_weight, k_weight, eps, q_out, a);
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
  return bf16_flag(dtype) ? launch_rope<true>(head_dim, a, true, st)
                          : launch_rope<false>(head_dim, a, true, st);
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
  if ((items + per - 1) / per > kTreeMaxGrid) return PE_ERR_DIMS;
  const dim3 grid((unsigned)((items + per - 1) / per), (unsigned)batch, (unsigned)layers);
  if (s_d == 1) keep_rows_kernel<<<grid, 256, 0, st>>>(a);
  else keep_cols_kernel<<<grid, 256, 0, st>>>(a);
  return launch_status();
}
