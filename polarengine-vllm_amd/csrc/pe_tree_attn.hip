// Attention of the drafted tokens of a step over a cache: every token of a
// sequence sees the sequence's cached positions and, of the drafted ones behind
// them, those that its mask names (itself and its ancestors).
//
// The rows of one KV head (n nodes x group query heads) go through the matrix
// cores together, so a key or value is read from memory once for all of them.
// A workgroup of four waves takes RB = 16 RT WR rows and a run of tiles of 64
// positions:
//  * tiles of keys and values go straight to LDS, two buffers, the next tile under
//    way while one is worked on, one barrier a tile;
//  * scores S^T = K Q^T (v_mfma_f32_16x16x32, keys as A, so a lane holds four
//    keys of one row and the row's maximum needs two exchanges), Q in registers;
//  * one pass with running maximum and sum in fp32; the probabilities, rounded to
//    the cache's 16-bit type, are the B operand of O^T = V^T P^T just as S^T left
//    them (the order of a product's keys is free as long as V^T has the same). The
//    matrix cores take 16 bits. Each probability is off by half a step, in the sum that
//    divides alike: at most one step of sum p |v| / sum p in all, on random scores 1.4
//    times the error of the result's own rounding. A second product with what the
//    rounding leaves brings it to that (512 rows over 32,700 positions 93 -> 118 us, up
//    to 64 rows 0 to 6%), but makes NaN of an infinite value that a row sees;
//  * V^T, and K where it is stored by dimension, come out of LDS through
//    ds_read_b64_tr_b16: within 16 lanes, lane i gives the address of 8 bytes of
//    row i / 4 and gets column i of the 4 x 16 block.
// WR waves share a tile's keys and differ in their rows, 4 / WR differ in their
// keys (few rows): those join their sums in LDS at the end.
// The tiles of all sequences and KV heads form one line, cut into equal runs, one a
// workgroup, by the lengths read on the device; a second launch joins the parts of a
// sequence that a cut divides.
//
// Bound by HBM where a KV head has few rows: 32 sequences x 8 nodes, 32 rows, up to
// 16,000 positions 262 us for both launches, 5.4 TB/s (tiles through registers 493, equal
// parts of each sequence instead of the line 315). With 512 rows over 32,700 positions 94
// us, 0.73 PFLOP/s: the softmax between the products keeps the matrix cores busy 29% of
// the time. One sequence of 777 and 16 rows: 11.5 us, latency.

#include <type_traits>

#include "pe_tree.h"

namespace pe {

constexpr int kTile = 64;          // positions of a tile
constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;      // powers of two that an exponent may exceed its base by
// fp16 probabilities are 2^7 times as large: the largest lies in 2^7 .. 2^15, what is below
// 2^-21 of it (2^-29 where the base is behind) loses bits and what is below 2^-32 (2^-40)
// vanishes. Without it, beside a key 18 above 32,000 others, results were off by 4.2e-4
// of 5.8e-4. The row's sum has the factor too; no time is lost. bf16 has fp32's exponents.
constexpr float kLiftF16 = 7.f;

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
  int runs;      // workgroups of one row block
  float* parts;  // [runs][blocks][2]: a run divides at most its first and its last sequence
};

// fp32 words of one part: RB x D sums, RB maxima, RB sums
__host__ __device__ inline int64_t part_words(int rb, int dim) { return (int64_t)rb * (dim + 2); }

// ---------------------------------------------------------------------------
// The line of tiles: sequence after sequence, within one KV head after KV head.
// An empty slot of the batch has one tile, without positions, for its zeros. Both
// launches find their way from the lengths alone, in a workgroup that works together
// one wave for all.
// ---------------------------------------------------------------------------
// running sum over the 64 lanes: DPP row_shr within 16 lanes, then the rows
__device__ __forceinline__ int wave_scan_i32(int v, int lane) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = r0 + __builtin_amdgcn_readlane(v, 31);
  const int r2 = r1 + __builtin_amdgcn_readlane(v, 47);
  return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}
__device__ __forceinline__ bool tree_active(const TreeAttnArgs& a, int64_t len) {
  return len >= 0 && len <= a.cap - a.n;
}
// 64 sequences of the batch, one a lane
struct TreeChunk {
  int64_t len;
  int tiles, scan;  // and their running sum
};
__device__ __forceinline__ TreeChunk tree_chunk(const TreeAttnArgs& a, int b0, int lane) {
  TreeChunk c{-1, 0, 0};
  if (b0 + lane < a.batch) {
    c.len = a.lengths[b0 + lane];
    if (!tree_active(a, c.len)) c.len = -1;
    c.tiles = c.len >= 0 ? (int)((c.len + a.n + kTile - 1) / kTile) : 1;
  }
  c.scan = wave_scan_i32(c.tiles, lane);
  return c;
}
// tiles of all sequences, one KV head of each; c: the first chunk
__device__ __forceinline__ int tree_total(const TreeAttnArgs& a, const TreeChunk& c, int lane) {
  int total = __builtin_amdgcn_readlane(c.scan, 63);
  for (int b0 = 64; b0 < a.batch; b0 += 64)
    total += __builtin_amdgcn_readlane(tree_chunk(a, b0, lane).scan, 63);
  return total;
}
// a sequence: its number, tiles, the tiles before it, and its length (-1: empty slot)
struct TreePlace {
  int b, tiles, before;
  int64_t len;
};
__device__ __forceinline__ TreePlace tree_lane(const TreeChunk& c, int b0, int before, int l) {
  const int t = __builtin_amdgcn_readlane(c.tiles, l);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)c.len, l);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)c.len >> 32), l);
  return TreePlace{b0 + l, t, before + __builtin_amdgcn_readlane(c.scan, l) - t,
                   (int64_t)((uint64_t)hi << 32 | lo)};
}
// the sequence that holds place `at` of the line
__device__ __forceinline__ TreePlace tree_find(const TreeAttnArgs& a, TreeChunk c, int at, int lane) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const uint64_t hit = __ballot((before + c.scan) * a.kv_heads > at);
    if (hit) return tree_lane(c, b0, before, __builtin_ctzll(hit));
    before += __builtin_amdgcn_readlane(c.scan, 63);
    c = tree_chunk(a, b0 + 64, lane);
  }
  // only if the lengths change under the kernel: an empty slot
  return TreePlace{a.batch - 1, 1, at / a.kv_heads, -1};
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
// two values rounded to the 16-bit type, in one instruction
typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const float2v v{lo, hi};
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2v));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
}
typedef __attribute__((address_space(3))) s16x4v lds_s16x4;
typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(1))) const unsigned char glb_byte;
__device__ __forceinline__ u32x2v lds_tr(const lds_byte* p) {
  return __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
__device__ __forceinline__ u32x4v lds_ld16(const lds_byte* p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4v*>(p);
}
__device__ __forceinline__ void lds_st16v(lds_byte* p, u32x4v v) {
  *reinterpret_cast<__attribute__((address_space(3))) u32x4v*>(p) = v;
}
// maximum over the four lanes li, li + 16, li + 32, li + 48, in each of them
__device__ __forceinline__ float rows_max(float v) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  u = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
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
__global__ __launch_bounds__(256, D == 256 ? 1 : RT == 2 || D == 128 ? 2 : 3) void tree_attn_kernel(
    const TreeAttnArgs a) {
  constexpr int WK = 4 / WR;         // waves that share the rows and differ in keys
  constexpr int RB = 16 * RT * WR;   // rows of the workgroup
  constexpr int NKT = 4 / WK;        // 16-key blocks of a wave in a tile
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int ROW = 2 * D;         // bytes of an LDS row
  constexpr int NCH = D / 32;        // 16-byte chunks of a tile per thread
  constexpr int CPR = D / 8;         // chunks of a row
  constexpr int KPI = 256 / CPR;     // rows per pass of the workgroup
  constexpr int VT = kTile * ROW;    // a buffer: keys, then values
  // two objects, so that the compiler knows that a tile on its way into one is not
  // what is read from the other
  __shared__ __align__(16) unsigned char buf0[2 * VT];
  __shared__ __align__(16) unsigned char buf1[2 * VT];
  __shared__ float mx[4][16 * RT], lx[4][16 * RT];
  __shared__ TreePlace line_place;
  __shared__ int line_total;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / WK, wk = wave % WK;

  // this workgroup's run; the row blocks of a run sit 8 apart, on one XCD
  const int span = 8 * a.blocks;
  const int rem = (int)blockIdx.x % span;
  const int run = (int)blockIdx.x / span * 8 + rem % 8;
  const int rblk = rem / 8;
  TreeChunk chunk{};
  if (wave == 0) {
    chunk = tree_chunk(a, 0, threadIdx.x & 63);
    const int total = tree_total(a, chunk, threadIdx.x & 63);
    if (threadIdx.x == 0) line_total = total * a.kv_heads;
  }
  __syncthreads();
  const int total = __builtin_amdgcn_readfirstlane(line_total);
  const int size = (total + a.runs - 1) / a.runs;
  if ((int64_t)run * size >= total) return;
  const int line_end = (int)min((int64_t)total, (int64_t)(run + 1) * size);
  for (int at = run * size; at < line_end;) {
  int tid = threadIdx.x;
  // what follows from the lane is worked out anew for each sequence: kept across
  // them it would not leave registers enough for the tiles
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, li = lane & 15, lg = lane >> 4;
  if (wave == 0) {
    const TreePlace p = tree_find(a, chunk, at, lane);
    if (lane == 0) line_place = p;
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(line_place.b);
  const int tiles = __builtin_amdgcn_readfirstlane(line_place.tiles);
  const int before = __builtin_amdgcn_readfirstlane(line_place.before);
  const int kvh = (at - before * a.kv_heads) / tiles;
  const int t0 = at - before * a.kv_heads - kvh * tiles;
  const int t1 = min(tiles, t0 + line_end - at);
  at += t1 - t0;
  const int64_t found = (int64_t)(
      (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)line_place.len >> 32)) << 32 |
      (uint32_t)__builtin_amdgcn_readfirstlane((int)line_place.len));
  const bool live = found >= 0;
  const int64_t len = live ? found : 0, end = len + a.n;
  const uint16_t* kb = a.k + (int64_t)b * a.ks_b + kvh * a.ks_h;
  const uint16_t* vb = a.v + (int64_t)b * a.vs_b + kvh * a.vs_h;

  // Staging, straight into LDS: pass i of thread tid fills chunk tid + 256 i of a
  // tile, row c / CPR. Chunks are permuted within rows (by the source address) so
  // that the reads below, 16 bytes of 16 rows or 32 bytes of 8 rows at a time, touch
  // every bank once; the permutations are linear in the bits of the row, so pass i
  // adds a constant. Addresses are a uniform 64-bit base and the thread's 32-bit
  // offset (strides below 2^26). Rows past the cache repeat the last one. Keys by
  // dimension have any alignment and go through registers: chunk c is dimension
  // c / 8, eight positions c % 8.
  auto k_swz = [](int key) { return D == 64 ? key >> 1 & 7 : key & 15; };
  auto v_swz = [](int key) { return D == 64 ? key >> 1 & 3 : key & 7; };
  auto kc_swz = [](int d) { return (d >> 1 & 1) | (d >> 3 & 1) << 1; };
  const int srow = tid / CPR, sch = tid % CPR;
  const int vch = ((sch >> 1 ^ v_swz(srow)) << 1 | (sch & 1)) * 16, kch = (sch ^ k_swz(srow)) * 16;
  const int kst = (tid >> 3) * 128 + ((((tid & 7) >> 1) ^ kc_swz(tid >> 3)) << 5) + (tid & 1) * 16;
  const uint32_t voff = (uint32_t)srow * (uint32_t)a.vs_l * 2u + vch;
  const uint32_t koff = KCOL ? (uint32_t)(tid >> 3) * (uint32_t)a.ks_d * 2u + (tid & 7) * 16
                             : (uint32_t)srow * (uint32_t)a.ks_l * 2u + kch;
  const uint32_t koff1 = koff - kch + (kch ^ k_swz(KPI) << 4);  // of odd passes
  u32x4v kr[KCOL ? NCH : 1];
  auto issue = [&](lds_byte* to, int t) {
    const int64_t p0 = (int64_t)t * kTile;
    auto v_base = [&](int i) { return reinterpret_cast<const char*>(vb + (p0 + i * KPI) * a.vs_l); };
    auto k_base = [&](int i) {
      return reinterpret_cast<const char*>(kb + (KCOL ? i * 32 * a.ks_d + p0 : (p0 + i * KPI) * a.ks_l));
    };
    auto dma = [&](const char* from, int i, int plane) {
      __builtin_amdgcn_global_load_lds((const glb_byte*)from, to + plane + (i * 4 + wave) * 1024, 16,
                                       0, 0);
    };
    if (p0 + kTile <= a.cap) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if constexpr (KCOL) __builtin_memcpy(&kr[i], k_base(i) + koff, 16);
        else dma(k_base(i) + (i & 1 ? koff1 : koff), i, 0);
        dma(v_base(i) + voff, i, VT);
      }
      return;
    }
    const int last = (int)(end - p0) - 1;  // the cache ends within the tile
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int row = min(srow + i * KPI, last) - i * KPI;  // may lie before the pass
      dma(v_base(i) + ((int64_t)row * (int)a.vs_l * 2 + vch), i, VT);
      if constexpr (KCOL) {
        const int first = (tid & 7) * 8;
        const uint16_t* s = reinterpret_cast<const uint16_t*>(k_base(i) + koff);
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = s[min(first + e, last) - first];
        kr[i] = u32x4v{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
      } else {
        dma(k_base(i) + ((int64_t)row * (int)a.ks_l * 2 + (kch ^ k_swz(i * KPI) << 4)), i, 0);
      }
    }
  };
  auto store_k = [&](lds_byte* to) {
    if constexpr (KCOL)
#pragma unroll
      for (int i = 0; i < NCH; ++i) lds_st16v(to + kst + i * 32 * 128, kr[i]);
  };

  // Q fragments (B operand: lane = row li, dimensions 32 ks + 8 lg ..) and the
  // masks of the lane's rows
  u32x4v qf[RT][KS];
  uint64_t mask[RT];
  const uint64_t all = a.n == 64 ? ~0ull : (1ull << a.n) - 1;
  if (live) issue((lds_byte*)buf0, t0);
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
  // l: the sums of the rounded probabilities, as a product with ones (every register of
  // it holds the row's sum): what a row's weights are divided by is then their own sum
  float m[RT];
  float4v l4[RT];
  constexpr uint32_t kOnes = BF ? 0x3F803F80u : 0x3C003C00u;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff();
    l4[rt] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  const float c = fmaxf(a.scale * kTreeLog2e, 1e-30f);  // above 0: a masked -inf stays one
  // the lane's places in a buffer
  const int kfirst = wk * (kTile / WK);  // the wave's first key
  const int kat = KCOL ? (8 * lg + (li >> 2)) * 128 + (li & 3) * 8 : (kfirst + li) * ROW;
  const int kx = KCOL ? kc_swz(8 * lg + (li >> 2)) : k_swz(li);
  const int vrow = 4 * lg + (li >> 2);
  const int vat = VT + (kfirst + vrow) * ROW + (li & 3) * 8;
  const int vx = v_swz(vrow);

  // one tile from `cur`, the next on its way to `nxt`
  auto step = [&](lds_byte* __restrict__ cur, lds_byte* __restrict__ nxt, int t, auto tail_) {
    constexpr bool kTail = decltype(tail_)::value;  // holds drafted tokens, or the end
    const int64_t p0 = (int64_t)t * kTile;
    __builtin_amdgcn_s_waitcnt(0);  // this wave's share of the tile is in LDS
    __syncthreads();                // everybody's is, and `nxt` is done with
    bool slow = false;
    if constexpr (kTail) {
      // Rows from `end` on become zeros. A drafted token's value that is infinite or
      // NaN must not reach, as 0 x inf, the rows that do not see it.
      bool bad = false;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        lds_byte* at = cur + VT + (i * 256 + tid) * 16;
        const int64_t pos = p0 + srow + i * KPI;
        if (pos >= end) lds_st16v(at, u32x4v{0, 0, 0, 0});
        else if (pos >= len) bad |= not_finite8<BF>(lds_ld16(at));
      }
      slow = __syncthreads_or(bad);
    }
    if (t + 1 < t1) issue(nxt, t + 1);

    float4v s[NKT][RT];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[kt][rt] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4v kf;
        if constexpr (KCOL) {
          const lds_byte* p = cur + kat + ks * 32 * 128 + ((wk * NKT + kt ^ kx) << 5);
          const u32x2v lo = lds_tr(p), hi = lds_tr(p + 4 * 128);
          kf = u32x4v{lo[0], lo[1], hi[0], hi[1]};
        } else {
          kf = lds_ld16(cur + kat + kt * 16 * ROW + ((4 * (ks & 3) + lg ^ kx) << 4) + (ks >> 2) * 256);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[kt][rt] = mfma32<BF>(kf, qf[rt][ks], s[kt][rt]);
      }
    }
    // softmax of the tile; a lane holds keys 16 kt + 4 lg + e of row li
    u32x2v pf[NKT][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if constexpr (kTail) {
        const int r0 = (int)(p0 - len) + kfirst + 4 * lg;  // above -64
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int rel = r0 + 16 * kt + e;
            if (rel >= 0 && (rel >= 64 || !(mask[rt] >> rel & 1))) s[kt][rt][e] = -__builtin_inff();
          }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = fmaxf(top, s[kt][rt][e]);
      top = rows_max(top) * c;
      // m is what the exponents are relative to: it moves only where they would pass
      // kSlack (a factor that neither sums nor 16-bit values mind), so that most tiles
      // leave the sums alone
      if (__any(top > m[rt] + kSlack)) {
        const float mn = fmaxf(m[rt], top);
        const float al = __builtin_amdgcn_exp2f(m[rt] - (mn == -__builtin_inff() ? 0.f : mn));
        l4[rt] *= al;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= al;
        m[rt] = mn;
      }
      const float base = (m[rt] == -__builtin_inff() ? 0.f : m[rt]) - (BF ? 0.f : kLiftF16);
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][rt][e], c, -base));
        pf[kt][rt] = u32x2v{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3])};
      }
      if constexpr (NKT == 1) {
        l4[rt] = mfma16<BF>(u32x2v{kOnes, kOnes}, pf[0][rt], l4[rt]);
      } else {
#pragma unroll
        for (int kt = 0; kt < NKT; kt += 2)
          l4[rt] = mfma32<BF>(u32x4v{kOnes, kOnes, kOnes, kOnes},
                              u32x4v{pf[kt][rt][0], pf[kt][rt][1], pf[kt + 1][rt][0],
                                     pf[kt + 1][rt][1]}, l4[rt]);
      }
    }
    if (!kTail || !slow) {
#pragma unroll
      for (int kt = 0; kt < NKT; kt += 2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const lds_byte* p = cur + vat + kt * 16 * ROW + (((dt & 7) ^ vx) << 5) + (dt >> 3) * 256;
          if constexpr (NKT == 1) {
            const u32x2v vf = lds_tr(p);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16<BF>(vf, pf[0][rt], o[rt][dt]);
          } else {
            const u32x2v lo = lds_tr(p), hi = lds_tr(p + 16 * ROW);
            const u32x4v vf{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              o[rt][dt] = mfma32<BF>(vf, u32x4v{pf[kt][rt][0], pf[kt][rt][1], pf[kt + 1][rt][0],
                                                pf[kt + 1][rt][1]}, o[rt][dt]);
          }
        }
    } else {
      // key by key, skipping what a row does not see; the probabilities take the
      // place of the keys, 64-lane words of one 16-key block after the other
      __syncthreads();
      lds_byte* const pw = cur + wave * (NKT * 512);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt)
          *reinterpret_cast<lds_u32x2*>(pw + (kt * 64 + lane) * 8) = pf[kt][rt];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int key = 0; key < 16 * NKT; ++key) {
          const int at = kfirst + key;
          const int64_t rel = p0 - len + at;
          const float p = f16or_bf(*reinterpret_cast<const lds_u16*>(
              pw + ((key >> 4) * 64 + (key >> 2 & 3) * 16 + li) * 8 + (key & 3) * 2), BF);
          if (rel < 0 || (rel < 64 && (mask[rt] >> rel & 1))) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const u32x2v w = *reinterpret_cast<const lds_u32x2*>(
                  cur + VT + at * ROW + ((dt ^ v_swz(at)) << 5) + lg * 8);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[rt][dt][e] = __builtin_fmaf(
                    p, f16or_bf((uint16_t)(w[e / 2] >> (16 * (e & 1))), BF), o[rt][dt][e]);
            }
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    if (t + 1 < t1) store_k(nxt);
  };
  if (live) store_k((lds_byte*)buf0);
  const int full = min(t1, (int)(len / kTile));  // tiles before it hold cached positions alone
  int t = live ? t0 : t1;
  for (; t + 1 < full; t += 2) {
    step((lds_byte*)buf0, (lds_byte*)buf1, t, std::false_type{});
    step((lds_byte*)buf1, (lds_byte*)buf0, t + 1, std::false_type{});
  }
  for (bool odd = false; t < t1; ++t, odd = !odd)  // an odd full tile too
    step((lds_byte*)(odd ? buf1 : buf0), (lds_byte*)(odd ? buf0 : buf1), t, std::true_type{});

  float l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) l[rt] = l4[rt][0];
  if constexpr (WK > 1) {  // join the waves that share rows, in their order
    if (lg == 0)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) mx[wave][rt * 16 + li] = m[rt];
    __syncthreads();
    float4v* buf = reinterpret_cast<float4v*>(buf0);
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
    if (wk == 0)
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
  if (wk == 0)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int local = (wr * RT + rt) * 16 + li;
    const int r = rblk * RB + local;
    if (t0 == 0 && t1 == tiles) {
      if (r >= a.rows) continue;
      const int node = r / a.group, g = r - node * a.group;
      uint16_t* dst = a.out + (((int64_t)b * a.n + node) * a.kv_heads * a.group +
                               (int64_t)kvh * a.group + g) * D + 4 * lg;
      const float inv = l[rt] > 0.f || l[rt] != l[rt] ? 1.f / l[rt] : 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<uint2*>(dst + 16 * dt) =
            make_uint2(pack2<BF>(o[rt][dt][0] * inv, o[rt][dt][1] * inv),
                       pack2<BF>(o[rt][dt][2] * inv, o[rt][dt][3] * inv));
    } else {
      // the run's first sequence, begun before it, or its last, which goes on behind it
      float* dst = a.parts + (((int64_t)run * a.blocks + rblk) * 2 + (t0 == 0)) * part_words(RB, D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4v*>(dst + local * D + 16 * dt + 4 * lg) = o[rt][dt];
      if (lg == 0) {
        dst[RB * D + local] = m[rt];
        dst[RB * D + RB + local] = l[rt];
      }
    }
  }
  __syncthreads();  // the buffers are free
  }
}

// ---------------------------------------------------------------------------
// out = sum of the parts of a row, each weighted exp2(m_part - m) / l: one wave
// per row of a KV head, lane = dimensions, parts in order
// ---------------------------------------------------------------------------
template <int D, bool BF>
__global__ __launch_bounds__(256) void tree_join_kernel(const TreeAttnArgs a, int rb) {
  constexpr int E = D / 64;
  constexpr int U = 8;  // parts on their way
  typedef float floatE __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  const int r = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.y, b = blockIdx.z;
  TreeChunk c = tree_chunk(a, 0, lane);
  const int total = tree_total(a, c, lane) * a.kv_heads;
  const int size = (total + a.runs - 1) / a.runs;
  int before = 0;
  for (int b0 = 0; b0 + 64 <= b; b0 += 64) {
    before += __builtin_amdgcn_readlane(c.scan, 63);
    c = tree_chunk(a, b0 + 64, lane);
  }
  const TreePlace place = tree_lane(c, b & ~63, before, b & 63);
  const int start = place.before * a.kv_heads + kvh * place.tiles;
  const int run0 = min(start / size, a.runs - 1);
  const int parts = min((start + place.tiles - 1) / size, a.runs - 1) - run0 + 1;
  if (parts == 1 || r >= a.rows) return;
  const int64_t words = part_words(rb, D), step = 2 * a.blocks * words;  // to the next run
  const int local = r % rb;
  // the first part is its run's last, the others are their runs' first
  const float* base = a.parts + ((int64_t)run0 * a.blocks + r / rb) * 2 * words;
  auto part = [&](int s) { return base + s * step + (s == 0 ? words : 0); };
  floatE t[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      t[u] = reinterpret_cast<const floatE*>(part(min(s0 + u, parts - 1)) + local * D)[lane];
  };
  load(0);
  float m = -__builtin_inff(), l = 0.f;
  floatE o = 0.f;
  for (int s0 = 0; s0 < parts; s0 += 64) {
    const int here = min(64, parts - s0);
    const float* p = part(s0 + min(lane, here - 1)) + rb * D + local;
    const float pm = lane < here ? p[0] : -__builtin_inff(), pl = p[rb];
    float mn = pm;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
    mn = fmaxf(mn, m);
    const float shift = mn == -__builtin_inff() ? 0.f : mn;
    const float w = __builtin_amdgcn_exp2f(pm - shift), al = __builtin_amdgcn_exp2f(m - shift);
    m = mn;
    o *= al;
    l = l * al + wave_sum_dpp(lane < here ? w * pl : 0.f);
    for (int s = 0; s < here; s += U) {
      if (s0 + s > 0) load(s0 + s);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s + u < here)
          o += t[u] * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w),
                                                                          s + u));
    }
  }
  const int node = r / a.group, g = r - node * a.group;
  uint16_t* dst = a.out + (((int64_t)b * a.n + node) * a.kv_heads * a.group +
                           (int64_t)kvh * a.group + g) * D + lane * E;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t h[E];
#pragma unroll
  for (int e = 0; e < E; ++e) h[e] = to16(o[e] * inv, BF);
  __builtin_memcpy(__builtin_assume_aligned(dst, 2 * E), h, 2 * E);
}

// Rows of a workgroup: as many as the rows of a KV head fill, 64 up to 192 of them, 128
// beyond. Up to 192 the second half of the last block, the larger parts and (heads of 256)
// the 54 to 119 registers that the 128-row form spills cost more than keys and values read
// from L2 by a block more. Beyond, 128 rows win by their fewer reads where sequences are
// long, and lose up to a sixth where they are short. Heads of 128 with keys by dimension
// stay at 64: their 128-row form does not fit the registers (80 rows, 8 sequences of up to
// 8000: 111 us, by 64 rows 65). Microseconds by 64 and by 128 rows, caches from HBM, one
// sequence of 8 KV heads (128 rows: four of 4):
//   head, keys by   66, 8000   128, 6000  192, 8000  192, 30000  256, 8000  512, 30000
//   64, position    18.1 22.5  23.4 27.8  19.6 24.8  37.2 42.6   21.8 25.5  64.9 60.5
//   64, dimension   19.2 22.7  25.4 29.7  20.8 26.1  41.9 45.3   23.7 26.9  77.5 64.9
//   128, position   26.4 27.6  33.4 38.6  26.7 36.0  59.9 65.8   34.1 37.5   112 95.7
//   256, position   49.5 56.3  65.3 73.2  63.4 69.0   158  152   72.3 71.0   357  261
//   256, dimension  52.3 62.7  78.2 90.1  69.3 85.0   184  208   79.1 88.3   413  351
static int tree_rows(int rows, int dim, bool kcol) {
  if (rows <= 64) return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  return rows <= 192 || (dim == 128 && kcol) ? 64 : 128;
}

struct TreePlanHost {
  int rb, blocks;
  int runs;
  bool split;  // a sequence may be divided
};
static TreePlanHost tree_host(int64_t batch, int n, int heads, int kv_heads, int dim, int64_t cap,
                              bool kcol) {
  TreePlanHost p;
  const int rows = n * (heads / kv_heads);
  p.rb = tree_rows(rows, dim, kcol);
  p.blocks = (rows + p.rb - 1) / p.rb;
  const int64_t tiles = (cap + kTile - 1) / kTile;
  // As many workgroups as the CUs hold at a time, each an equal run. Heads of 64 would
  // fit three or four times; two are faster (32 rows, 16 sequences of up to 8000: 40.5
  // us, three 41.7, four 43.6; 128 rows: 65, 75 and 78), their parts being fewer.
  // A run's row blocks share an XCD, so what fits is counted for each of the eight: one
  // workgroup more than its CUs hold waits for a whole run (heads of 256, 320 rows over
  // 8000 positions, three blocks: 11 runs an XCD 119 us, 10 runs 89; 768 rows 121 and 86).
  const int per_cu = dim == 256 ? 1 : 2;
  const int64_t slots = (int64_t)num_cus() * per_cu;
  const int64_t per_xcd = slots / 8 / p.blocks;
  const int64_t wanted = per_xcd ? per_xcd * 8 : slots / p.blocks;
  const int64_t most = batch * kv_heads * tiles;
  p.runs = (int)(wanted < 1 ? 1 : wanted < most ? wanted : most);
  p.split = tiles > 1 && p.runs > 1;
  return p;
}

static bool tree_attn_shape_ok(int64_t batch, int n, int heads, int kv_heads, int dim, int64_t cap) {
  if (batch < 1 || batch > 65535 || n < 1 || n > kTreeMax || kv_heads < 1 || kv_heads > 65535 ||
      heads < 1 || heads > 65536 || heads % kv_heads || (dim != 64 && dim != 128 && dim != 256) ||
      cap < 1 || cap > INT32_MAX)
    return false;
  return (double)batch * kv_heads * ((cap + kTile - 1) / kTile) <= 1e9;
}

template <int D, bool BF, bool KCOL>
static void launch_main(const TreePlanHost& p, const TreeAttnArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)((p.runs + 7) / 8 * 8 * p.blocks);
  switch (p.rb) {
    case 16: tree_attn_kernel<D, BF, KCOL, 1, 1><<<grid, 256, 0, st>>>(a); break;
    case 32: tree_attn_kernel<D, BF, KCOL, 1, 2><<<grid, 256, 0, st>>>(a); break;
    case 64: tree_attn_kernel<D, BF, KCOL, 1, 4><<<grid, 256, 0, st>>>(a); break;
    default:
      if constexpr (D != 128 || !KCOL) tree_attn_kernel<D, BF, KCOL, 2, 4><<<grid, 256, 0, st>>>(a);
      break;
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
  size_t most = 0;  // of the two layouts of the keys
  for (int kcol = 0; kcol < 2; ++kcol) {
    const TreePlanHost p = tree_host(batch, n, heads, kv_heads, head_dim, cap, kcol);
    const size_t need = p.split ? (size_t)p.runs * p.blocks * 2 * part_words(p.rb, head_dim) * 4 : 0;
    most = need > most ? need : most;
  }
  return most;
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
  if (!tree_attn_shape_ok(batch, n, heads, kv_heads, head_dim, cap) || q_b < 0 || q_n < 0 || m_b < 0 ||
      !(scale >= 0.f && scale <= 3e38f))
    return PE_ERR_DIMS;
  if (!aligned16(q) || (q_b | q_n) % 8 || !aligned16(out)) return PE_ERR_ALIGN;
  const int ok = cache_strides(k_cache, ks_b, ks_h, ks_l, ks_d, v_cache, vs_b, vs_h, vs_l);
  if (ok != PE_OK) return ok;
  const size_t need = pe_tree_attention_workspace_size(batch, n, heads, kv_heads, head_dim, cap);
  if (need && (!workspace || workspace_bytes < need)) return PE_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return PE_ERR_ALIGN;
  const TreePlanHost p = tree_host(batch, n, heads, kv_heads, head_dim, cap, ks_d != 1);
  TreeAttnArgs a{reinterpret_cast<const uint16_t*>(q), q_b, q_n,
                 reinterpret_cast<const uint16_t*>(k_cache),
                 reinterpret_cast<const uint16_t*>(v_cache), ks_b, ks_h, ks_l, ks_d, vs_b, vs_h, vs_l,
                 lengths, masks, m_b, reinterpret_cast<uint16_t*>(out), (int)batch, n,
                 heads / kv_heads, kv_heads, n * (heads / kv_heads), p.blocks, cap, scale, p.runs,
                 reinterpret_cast<float*>(workspace)};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim) {
    case 64: return bf ? launch_tree_attn<64, true>(p, a, st) : launch_tree_attn<64, false>(p, a, st);
    case 128: return bf ? launch_tree_attn<128, true>(p, a, st) : launch_tree_attn<128, false>(p, a, st);
    default: return bf ? launch_tree_attn<256, true>(p, a, st) : launch_tree_attn<256, false>(p, a, st);
  }
}
