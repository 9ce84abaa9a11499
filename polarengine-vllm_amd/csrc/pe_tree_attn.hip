// Attention of the drafted tokens of a step over a cache: every token of a
// sequence sees the sequence's cached positions and, of the drafted ones behind
// them, those that its mask names (itself and its ancestors).
//
// The rows of one KV head (n nodes x group query heads) go through the matrix
// cores together, so a key or value is read from memory once for all of them.
// A workgroup of four waves takes RB = 16 RT WR rows and a run of tiles of 64
// positions:
//  * a tile of keys and values is staged in LDS, the next one in registers;
//  * scores S^T = K Q^T (v_mfma_f32_16x16x32, keys as A, so a lane holds four
//    keys of one row and the row's maximum needs two exchanges), Q in registers;
//  * one pass with running maximum and sum in fp32; the probabilities, rounded to
//    the cache's 16-bit type, are the B operand of O^T = V^T P^T just as S^T left
//    them (the order of a product's keys is free as long as V^T has the same);
//  * V^T, and K where it is stored by dimension, come out of LDS through
//    ds_read_b64_tr_b16: within 16 lanes, lane i gives the address of 8 bytes of
//    row i / 4 and gets column i of the 4 x 16 block.
// WR waves share a tile's keys and differ in their rows, 4 / WR differ in their
// keys (few rows): those join their sums in LDS at the end.
// Tiles are divided over workgroups by the lengths, read on the device; a second
// launch joins the parts of a sequence.

#include "pe_tree.h"

namespace pe {

constexpr int kTile = 64;          // positions of a tile
constexpr int kTreeTarget = 512;   // workgroups wanted
constexpr int kTreeMinTiles = 2;   // least tiles of a part
constexpr float kTreeLog2e = 1.4426950408889634f;

struct TreeAttnArgs {
  const uint16_t* q;
  int64_t q_b, q_n;
  const uint16_t *k, *v;
  int64_t ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l;
  const int64_t *lengths, *masks;
  int64_t m_b;
  uint16_t* out;
  int batch, n, group, kv_heads, rows;  // rows: n * group of one KV head
  int blocks;                           // row blocks of one KV head
  int64_t cap;
  float scale;
  float* parts;  // null: no sequence is divided
};

// fp32 words of one part: RB x D sums, RB maxima, RB sums
__host__ __device__ inline int64_t part_words(int rb, int dim) { return (int64_t)rb * (dim + 2); }

// ---------------------------------------------------------------------------
// Division of the tiles, from the lengths alone, so that both launches and every
// workgroup arrive at the same one. A sequence of t tiles is cut into ceil(t / C)
// equal parts, C such that all parts together give about kTreeTarget workgroups;
// a unit is one part of one KV head. Every wave does this for itself.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int wave_sum_i32(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ bool tree_active(const TreeAttnArgs& a, int64_t len) {
  return len >= 0 && len <= a.cap - a.n;
}
__device__ __forceinline__ int tree_tiles(const TreeAttnArgs& a, int b) {
  const int64_t len = b < a.batch ? a.lengths[b] : -1;
  return tree_active(a, len) ? (int)((len + a.n + kTile - 1) / kTile) : 0;
}
__device__ __forceinline__ int tree_part_tiles(const TreeAttnArgs& a, int lane) {
  int total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) total += tree_tiles(a, b0 + lane);
  total = wave_sum_i32(total) * a.kv_heads * a.blocks;
  return max(kTreeMinTiles, (total + kTreeTarget - 1) / kTreeTarget);
}
__device__ __forceinline__ int tree_parts(int tiles, int part) {
  return tiles > part ? (tiles + part - 1) / part : 1;
}

// MFMA and conversions of the 16-bit type
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
template <bool BF>
__device__ __forceinline__ float4v mfma32(u32x4v a, u32x4v b, float4v c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a),
                                                   __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a),
                                                  __builtin_bit_cast(half8v, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ float4v mfma16(u32x2v a, u32x2v b, float4v c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4v, a),
                                                     __builtin_bit_cast(s16x4v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4v, a),
                                                 __builtin_bit_cast(half4v, b), c, 0, 0, 0);
}
typedef __attribute__((address_space(3))) s16x4v lds_s16x4;
typedef __attribute__((address_space(3))) unsigned char lds_byte;
__device__ __forceinline__ u32x2v lds_tr(const lds_byte* p) {
  return __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
__device__ __forceinline__ u32x4v lds_ld16(const lds_byte* p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4v*>(p);
}
// whether one of the eight 16-bit values is infinite or NaN
template <bool BF>
__device__ __forceinline__ bool not_finite8(u32x4v u) {
  constexpr uint32_t M = BF ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad |= (u[i] & M) == M || (u[i] >> 16 & M) == M;
  return bad;
}

template <int D, bool BF, bool KCOL, int RT, int WR>
__global__ __launch_bounds__(256, 2) void tree_attn_kernel(const TreeAttnArgs a) {
  constexpr int WK = 4 / WR;         // waves that share the rows and differ in keys
  constexpr int RB = 16 * RT * WR;   // rows of the workgroup
  constexpr int NKT = 4 / WK;        // 16-key blocks of a wave in a tile
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int ROW = 2 * D;         // bytes of an LDS row
  constexpr int NCH = D / 32;        // 16-byte chunks of a tile per thread
  constexpr int CPR = D / 8;         // chunks of a row
  constexpr int KPI = 256 / CPR;     // rows per pass of the workgroup
  __shared__ __align__(16) unsigned char smem[2 * kTile * ROW];
  __shared__ float mx[4][16 * RT], lx[4][16 * RT];
  lds_byte* const kt_lds = (lds_byte*)smem;
  lds_byte* const vt_lds = kt_lds + kTile * ROW;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / WK, wk = wave % WK;
  const int li = lane & 15, lg = lane >> 4;

  // this workgroup's unit; the row blocks of a unit sit 8 apart, on one XCD
  const int span = 8 * a.blocks;
  const int rem = (int)blockIdx.x % span;
  const int unit = (int)blockIdx.x / span * 8 + rem % 8;
  const int rblk = rem / 8;
  const int part = tree_part_tiles(a, lane);
  int first = 0, b = -1, tiles = 0, parts = 1;  // units before b
  for (int b0 = 0; b0 < a.batch && b < 0; b0 += 64) {
    const int t = tree_tiles(a, b0 + lane);
    const int p = tree_parts(t, part);
    const int u = b0 + lane < a.batch ? p * a.kv_heads : 0;
    int scan = u;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(scan, off, 64);
      if (lane >= off) scan += o;
    }
    const uint64_t hit = __ballot(unit < first + scan);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = b0 + l;
      first += __builtin_amdgcn_readlane(scan - u, l);
      tiles = __builtin_amdgcn_readlane(t, l);
      parts = __builtin_amdgcn_readlane(p, l);
    } else {
      first += __builtin_amdgcn_readlane(scan, 63);
    }
  }
  if (b < 0) return;
  const int kvh = (unit - first) % a.kv_heads, piece = (unit - first) / a.kv_heads;
  const int per = (tiles + parts - 1) / parts;
  const int t0 = piece * per, t1 = min(tiles, t0 + per);

  const int64_t len = tiles ? a.lengths[b] : 0, end = len + a.n;
  const uint16_t* kb = a.k + (int64_t)b * a.ks_b + kvh * a.ks_h;
  const uint16_t* vb = a.v + (int64_t)b * a.vs_b + kvh * a.vs_h;

  // staging: chunk c = tid + 256 i; by position: row c / CPR, chunk c % CPR; keys by
  // dimension: dimension c / 8, eight positions c % 8
  const int srow = tid / CPR, sch = tid % CPR;
  const uint16_t* vp = vb + srow * a.vs_l + sch * 8;
  const uint16_t* kp = KCOL ? kb + (tid >> 3) * a.ks_d + (tid & 7) * 8 : kb + srow * a.ks_l + sch * 8;
  u32x4v kr[NCH], vr[NCH];
  auto load_tile = [&](int t) {
    const int64_t p0 = (int64_t)t * kTile;
    if (p0 + kTile <= end) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if constexpr (KCOL)
          __builtin_memcpy(&kr[i], kp + i * 32 * a.ks_d + p0, 16);
        else
          kr[i] = *reinterpret_cast<const u32x4v*>(kp + (p0 + i * KPI) * a.ks_l);
        vr[i] = *reinterpret_cast<const u32x4v*>(vp + (p0 + i * KPI) * a.vs_l);
      }
      return;
    }
    // the last tile: rows from `end` on are not read; values there are zeros
    const int left = (int)(end - p0);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int row = srow + i * KPI;
      vr[i] = u32x4v{0, 0, 0, 0};
      if (row < left) vr[i] = *reinterpret_cast<const u32x4v*>(vp + (p0 + i * KPI) * a.vs_l);
      if constexpr (KCOL) {
        const uint16_t* s = kp + i * 32 * a.ks_d + p0;
        const int here = left - (tid & 7) * 8;  // positions of this chunk before `end`
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < here) w[e / 2] |= (uint32_t)s[e] << (16 * (e & 1));
        kr[i] = u32x4v{w[0], w[1], w[2], w[3]};
      } else {
        kr[i] = u32x4v{0, 0, 0, 0};
        if (row < left) kr[i] = *reinterpret_cast<const u32x4v*>(kp + (p0 + i * KPI) * a.ks_l);
      }
    }
  };
  // LDS places: chunks are permuted within rows so that the reads below, 16 bytes of
  // 16 rows or 32 bytes of 8 rows at a time, touch every bank once
  auto k_swz = [](int key) { return D == 64 ? key >> 1 & 7 : key & 15; };
  auto v_swz = [](int key) { return D == 64 ? key >> 1 & 3 : key & 7; };
  auto kc_swz = [](int d) { return (d >> 1 & 1) | (d >> 3 & 1) << 1; };
  auto store_tile = [&]() {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int row = srow + i * KPI;
      lds_byte* vd = vt_lds + row * ROW + ((sch >> 1 ^ v_swz(row)) << 5) + (sch & 1) * 16;
      *reinterpret_cast<__attribute__((address_space(3))) u32x4v*>(vd) = vr[i];
      lds_byte* kd;
      if constexpr (KCOL) {
        const int d = (tid >> 3) + 32 * i, c = tid & 7;
        kd = kt_lds + d * 128 + ((c >> 1 ^ kc_swz(d)) << 5) + (c & 1) * 16;
      } else {
        kd = kt_lds + row * ROW + ((sch ^ k_swz(row)) << 4);
      }
      *reinterpret_cast<__attribute__((address_space(3))) u32x4v*>(kd) = kr[i];
    }
  };

  // Q fragments (B operand: lane = row li, dimensions 32 ks + 8 lg ..) and the
  // masks of the lane's rows
  u32x4v qf[RT][KS];
  uint64_t mask[RT];
  const uint64_t all = a.n == 64 ? ~0ull : (1ull << a.n) - 1;
  if (t0 < t1) load_tile(t0);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rblk * RB + (wr * RT + rt) * 16 + li;
    const bool there = r < a.rows;
    const int node = there ? r / a.group : 0, g = there ? r - node * a.group : 0;
    mask[rt] = there ? (uint64_t)a.masks[b * a.m_b + node] & all : 0;
    const uint16_t* q = a.q + b * a.q_b + node * a.q_n + ((int64_t)kvh * a.group + g) * D + 8 * lg;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[rt][ks] = u32x4v{0, 0, 0, 0};
      if (there) qf[rt][ks] = *reinterpret_cast<const u32x4v*>(q + 32 * ks);
    }
  }
  float4v o[RT][DT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff();
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  const float c = a.scale * kTreeLog2e;
  // the lane's bases in the tiles
  const int kfirst = wk * (kTile / WK);  // the wave's first key
  const lds_byte* kl = KCOL ? kt_lds + (8 * lg + (li >> 2)) * 128 + (li & 3) * 8
                            : kt_lds + (kfirst + li) * ROW;
  const int kx = KCOL ? kc_swz(8 * lg + (li >> 2)) : k_swz(li);
  const int vrow = 4 * lg + (li >> 2);
  const lds_byte* vl = vt_lds + (kfirst + vrow) * ROW + (li & 3) * 8;
  const int vx = v_swz(vrow);

  for (int t = t0; t < t1; ++t) {
    const int64_t p0 = (int64_t)t * kTile;
    const bool tail = p0 + kTile > len;
    __syncthreads();  // the tile before is done with
    store_tile();
    bool slow = false;
    if (!tail) {
      __syncthreads();
    } else {
      // a drafted token's value that is infinite or NaN must not reach, as 0 x inf,
      // the rows that do not see it
      bool bad = false;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        bad |= p0 + srow + i * KPI >= len && not_finite8<BF>(vr[i]);
      slow = __syncthreads_or(bad);
    }
    if (t + 1 < t1) load_tile(t + 1);

    float4v s[NKT][RT];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[kt][rt] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4v kf;
        if constexpr (KCOL) {
          const lds_byte* p = kl + ks * 32 * 128 + ((wk * NKT + kt ^ kx) << 5);
          const u32x2v lo = lds_tr(p), hi = lds_tr(p + 4 * 128);
          kf = u32x4v{lo[0], lo[1], hi[0], hi[1]};
        } else {
          kf = lds_ld16(kl + kt * 16 * ROW + ((4 * ks + lg ^ kx) << 4));
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[kt][rt] = mfma32<BF>(kf, qf[rt][ks], s[kt][rt]);
      }
    }
    // softmax of the tile; a lane holds keys 16 kt + 4 lg + e of row li
    u32x2v pf[NKT][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = -__builtin_inff();
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[kt][rt][e] * c;
          if (tail) {
            const int64_t rel = p0 - len + kfirst + 16 * kt + 4 * lg + e;
            if (rel >= 0 && (rel >= 64 || !(mask[rt] >> rel & 1))) x = -__builtin_inff();
          }
          s[kt][rt][e] = x;
          top = fmaxf(top, x);
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m[rt], top);
      const float base = mn == -__builtin_inff() ? 0.f : mn;
      if (__any(mn > m[rt])) {
        const float al = __builtin_amdgcn_exp2f(m[rt] - base);
        l[rt] *= al;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= al;
        m[rt] = mn;
      }
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = __builtin_amdgcn_exp2f(s[kt][rt][e] - base);
          l[rt] += p[e];
        }
        pf[kt][rt] = u32x2v{pack16x2(p[0], p[1], BF), pack16x2(p[2], p[3], BF)};
      }
    }
    if (__builtin_expect(!slow, 1)) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const lds_byte* p = vl + ((dt ^ vx) << 5);
        if constexpr (NKT == 1) {
          const u32x2v vf = lds_tr(p);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16<BF>(vf, pf[0][rt], o[rt][dt]);
        } else {
#pragma unroll
          for (int kt = 0; kt < NKT; kt += 2) {
            const u32x2v lo = lds_tr(p + kt * 16 * ROW), hi = lds_tr(p + (kt + 1) * 16 * ROW);
            const u32x4v vf{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              o[rt][dt] = mfma32<BF>(vf, u32x4v{pf[kt][rt][0], pf[kt][rt][1], pf[kt + 1][rt][0],
                                                pf[kt + 1][rt][1]}, o[rt][dt]);
          }
        }
      }
    } else {
      // key by key, skipping what a row does not see
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
        for (int key = 0; key < 16; ++key) {
          const int at = kfirst + 16 * kt + key;
          const int64_t rel = p0 - len + at;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const uint32_t two = (key & 2) ? pf[kt][rt][1] : pf[kt][rt][0];
            const uint32_t got = __shfl(two, li | (key >> 2) << 4, 64);
            const float p = f16or_bf((uint16_t)((key & 1) ? got >> 16 : got & 0xffff), BF);
            if (rel < 0 || (rel < 64 && (mask[rt] >> rel & 1))) {
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                const u32x2v w = *reinterpret_cast<const lds_u32x2*>(
                    vt_lds + at * ROW + ((dt ^ v_swz(at)) << 5) + lg * 8);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  o[rt][dt][e] = __builtin_fmaf(
                      p, f16or_bf((uint16_t)(w[e / 2] >> (16 * (e & 1))), BF), o[rt][dt][e]);
              }
            }
          }
        }
    }
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16, 64);
    l[rt] += __shfl_xor(l[rt], 32, 64);
  }
  if constexpr (WK > 1) {  // join the waves that share rows, in their order
    if (lg == 0)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) mx[wave][rt * 16 + li] = m[rt];
    __syncthreads();
    float4v* buf = reinterpret_cast<float4v*>(smem);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = mx[wr * WK][rt * 16 + li];
#pragma unroll
      for (int k = 1; k < WK; ++k) top = fmaxf(top, mx[wr * WK + k][rt * 16 + li]);
      const float al = __builtin_amdgcn_exp2f(m[rt] - (top == -__builtin_inff() ? 0.f : top));
      m[rt] = top;
      l[rt] *= al;
      if (lg == 0) lx[wave][rt * 16 + li] = l[rt];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        o[rt][dt] *= al;
        if (wk > 0) buf[(((wr * (WK - 1) + wk - 1) * RT + rt) * DT + dt) * 64 + lane] = o[rt][dt];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        l[rt] += lx[wr * WK + k][rt * 16 + li];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          o[rt][dt] += buf[(((wr * (WK - 1) + k - 1) * RT + rt) * DT + dt) * 64 + lane];
      }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int local = (wr * RT + rt) * 16 + li;
    const int r = rblk * RB + local;
    if (parts == 1) {
      if (r >= a.rows) continue;
      const int node = r / a.group, g = r - node * a.group;
      uint16_t* dst = a.out + (((int64_t)b * a.n + node) * a.kv_heads * a.group +
                               (int64_t)kvh * a.group + g) * D + 4 * lg;
      const float inv = l[rt] > 0.f || l[rt] != l[rt] ? 1.f / l[rt] : 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<uint2*>(dst + 16 * dt) =
            make_uint2(pack16x2(o[rt][dt][0] * inv, o[rt][dt][1] * inv, BF),
                       pack16x2(o[rt][dt][2] * inv, o[rt][dt][3] * inv, BF));
    } else {
      float* dst = a.parts + ((int64_t)unit * a.blocks + rblk) * part_words(RB, D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4v*>(dst + local * D + 16 * dt + 4 * lg) = o[rt][dt];
      if (lg == 0) {
        dst[RB * D + local] = m[rt];
        dst[RB * D + RB + local] = l[rt];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// out = sum of the parts of a row, each weighted exp2(m_part - m) / l: one wave
// per row of a KV head, lane = dimensions, parts in order
// ---------------------------------------------------------------------------
template <int D, bool BF>
__global__ __launch_bounds__(256) void tree_join_kernel(const TreeAttnArgs a, int rb) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int r = (int)blockIdx.x * 4 + (threadIdx.x >> 6), kvh = blockIdx.y, b = blockIdx.z;
  const int part = tree_part_tiles(a, lane);
  int first = 0;
  for (int b0 = 0; b0 < b; b0 += 64)
    first += b0 + lane < b ? tree_parts(tree_tiles(a, b0 + lane), part) : 0;
  first = wave_sum_i32(first) * a.kv_heads;
  const int parts = tree_parts(tree_tiles(a, b), part);
  if (parts == 1 || r >= a.rows) return;
  const int64_t words = part_words(rb, D);
  const int local = r % rb;
  const float* base = a.parts + ((int64_t)(first + kvh) * a.blocks + r / rb) * words;
  const int64_t step = (int64_t)a.kv_heads * a.blocks * words;  // to the next part
  float m = -__builtin_inff();
  for (int s = lane; s < parts; s += 64) m = fmaxf(m, base[s * step + rb * D + local]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if (m == -__builtin_inff()) m = 0.f;
  float l = 0.f, o[E] = {};
  for (int s0 = 0; s0 < parts; s0 += 64) {
    float w = 0.f;
    if (s0 + lane < parts) {
      const float* p = base + (s0 + lane) * step + rb * D + local;
      w = __builtin_amdgcn_exp2f(p[0] - m);
      l += w * p[rb];
    }
    const int here = min(64, parts - s0);
    for (int s = 0; s < here; ++s) {
      const float ws = __shfl(w, s, 64);
      const float* p = base + (s0 + s) * step + local * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(ws, p[e], o[e]);
    }
  }
  l = wave_sum(l);
  const int node = r / a.group, g = r - node * a.group;
  uint16_t* dst = a.out + (((int64_t)b * a.n + node) * a.kv_heads * a.group +
                           (int64_t)kvh * a.group + g) * D + lane * E;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = to16(o[e] * inv, BF);
}

// rows of a workgroup: as many as the rows of a KV head fill
static int tree_rows(int rows) { return rows <= 16 ? 16 : rows <= 64 ? 64 : 128; }

struct TreePlanHost {
  int rb, blocks;
  int64_t units;  // at most
  bool split;     // a sequence may be divided
};
static TreePlanHost tree_host(int64_t batch, int n, int heads, int kv_heads, int64_t cap) {
  TreePlanHost p;
  const int rows = n * (heads / kv_heads);
  p.rb = tree_rows(rows);
  p.blocks = (rows + p.rb - 1) / p.rb;
  const int64_t tiles = (cap + kTile - 1) / kTile;
  const int64_t most = (tiles + kTreeMinTiles - 1) / kTreeMinTiles;  // parts of a sequence
  p.split = most > 1;
  // sum over b of ceil(t_b / C) parts, C >= total tiles / (target / (KV heads, blocks))
  p.units = (batch + kTreeTarget / p.blocks / kv_heads + 1) * kv_heads;
  if (p.units > batch * most * kv_heads) p.units = batch * most * kv_heads;
  return p;
}

static bool tree_attn_shape_ok(int64_t batch, int n, int heads, int kv_heads, int dim, int64_t cap) {
  if (batch < 1 || batch > 65535 || n < 1 || n > kTreeMax || kv_heads < 1 || kv_heads > 65535 ||
      heads < 1 || heads > 65536 || heads % kv_heads || (dim != 64 && dim != 128 && dim != 256) ||
      cap < 1 || cap > INT32_MAX)
    return false;
  const TreePlanHost p = tree_host(batch, n, heads, kv_heads, cap);
  return (double)batch * kv_heads * p.blocks * ((cap + kTile - 1) / kTile) <= 2e9 &&
         (double)(p.units + 8) * p.blocks <= 2e9;
}

template <int D, bool BF, bool KCOL>
static void launch_main(const TreePlanHost& p, const TreeAttnArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)((p.units + 7) / 8 * 8 * p.blocks);
  switch (p.rb) {
    case 16: tree_attn_kernel<D, BF, KCOL, 1, 1><<<grid, 256, 0, st>>>(a); break;
    case 64: tree_attn_kernel<D, BF, KCOL, 2, 2><<<grid, 256, 0, st>>>(a); break;
    default: tree_attn_kernel<D, BF, KCOL, 2, 4><<<grid, 256, 0, st>>>(a); break;
  }
}

template <int D, bool BF>
static int launch_tree_attn(const TreePlanHost& p, const TreeAttnArgs& a, hipStream_t st) {
  if (a.ks_d == 1) launch_main<D, BF, false>(p, a, st);
  else launch_main<D, BF, true>(p, a, st);
  const int rc = launch_status();
  if (rc != PE_OK || !p.split) return rc;
  const dim3 grid((unsigned)((a.rows + 3) / 4), (unsigned)a.kv_heads, (unsigned)a.batch);
  tree_join_kernel<D, BF><<<grid, 256, 0, st>>>(a, p.rb);
  return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_tree_attention_workspace_size(int64_t batch, int n, int heads, int kv_heads,
                                                   int head_dim, int64_t cap) {
  if (!tree_attn_shape_ok(batch, n, heads, kv_heads, head_dim, cap)) return 0;
  const TreePlanHost p = tree_host(batch, n, heads, kv_heads, cap);
  return p.split ? (size_t)p.units * p.blocks * part_words(p.rb, head_dim) * 4 : 0;
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
  const size_t need = pe_tree_attention_workspace_size(batch, n, heads, kv_heads, head_dim, cap);
  if (need && (!workspace || workspace_bytes < need)) return PE_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return PE_ERR_ALIGN;
  const TreePlanHost p = tree_host(batch, n, heads, kv_heads, cap);
  TreeAttnArgs a{reinterpret_cast<const uint16_t*>(q), q_b, q_n,
                 reinterpret_cast<const uint16_t*>(k_cache),
                 reinterpret_cast<const uint16_t*>(v_cache), ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l,
                 lengths, masks, m_b, reinterpret_cast<uint16_t*>(out), (int)batch, n,
                 heads / kv_heads, kv_heads, n * (heads / kv_heads), p.blocks, cap, scale,
                 reinterpret_cast<float*>(workspace)};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim) {
    case 64: return bf ? launch_tree_attn<64, true>(p, a, st) : launch_tree_attn<64, false>(p, a, st);
    case 128: return bf ? launch_tree_attn<128, true>(p, a, st) : launch_tree_attn<128, false>(p, a, st);
    default: return bf ? launch_tree_attn<256, true>(p, a, st) : launch_tree_attn<256, false>(p, a, st);
  }
}
