// Attention over the paged 8-bit cache: packed rows of sequences of different lengths,
// each row over the positions up to its own, or over a window of them and the first
// few.
//
// The rows of one KV head (new tokens x group query heads) go through the matrix cores
// together, 16 RT of them. A wave takes 64 positions a step, straight from memory to
// registers:
//  * scores S^T = K Q^T (v_mfma_f32_16x16x32, keys as A). Which key is which row of A
//    is free, so row 4 g + e of product t is position 16 g + 4 t + e: a lane then
//    holds the scores of 16 neighbouring positions of one row of queries, which lie in
//    one block, so one scale serves all of them;
//  * the probabilities, in fp16, are the B operand of O^T = V^T P^T just as the scores'
//    products left them, and the lane's part of V^T is 16 neighbouring bytes of the
//    block's values, which are stored by dimension. Nothing goes through LDS;
//  * e4m3 codes are exact in fp16 and bf16 (v_cvt_scalef32_pk, two a instruction).
//    The keys' scale multiplies the fp32 scores, the values' the probabilities: what
//    goes through the second product with the codes is probability times scale;
//  * one pass with running maxima and sums in fp32, both by row: of the scores, for the
//    sum that divides, and of probability times scale. So a row's result depends on
//    what that row sees alone, whatever scales others' positions, positions behind the
//    sequence's end or hidden by a window have. A product is 2^7 times as large and
//    relative to a base that moves only when it would pass 2^15, so that fp16 keeps
//    what is 2^-20 of the row's largest whole and what is above 2^-31 of it in part.
//    Rounding them costs half an fp16 step of each: less than the rounding of a bf16
//    result, about that of an fp16 one. The sum that divides is that of the rounded
//    ones where they keep what counts in it, which does not go by the scale;
//  * NaN codes are zeros for the products, in steps that some row does not see whole; a
//    map of where they are says which sums become NaN.
// The tiles of all sequences, KV heads and row blocks form one line, cut into equal
// runs, one a workgroup, by the lengths read on the device; a second launch joins the
// parts of a row block that a cut divides.
//
// Bound by HBM where a KV head has few rows: 32 sequences of up to 16,000 positions, 4
// rows, 135 + 5 us, 5.2 TB/s in the first launch; 16 windows of 4000 with heads of 256,
// one wave a SIMD, 111 + 5 us, 4.7 TB/s. 1024 tokens behind 30,000 (4096 rows): 657 us
// for both launches, 0.78 PFLOP/s, the matrix cores busy about a third of the time; heads
// of 64 426 us (operations: 213), 512 tokens with heads of 256 930 us (423). One sequence
// of 778, one row: 15 us in one launch, a chain of loads (lengths, tables, keys and values
// of four tiles).

#include "pe_paged.h"

namespace pe {

constexpr float kPaLog2e = 1.4426950408889634f;
constexpr float kPaSlack = 8.f;    // powers of two that an exponent may exceed its base by
constexpr float kPaLift = 7.f;     // and by which products of probability and scale are larger
// A value's scale is taken for at least 2^-60 of what the row's largest product implies:
// what is smaller vanishes in fp16 either way, and the probability can be had back from
// the product in fp32.
constexpr float kPaLeast = -60.f;
// Below 2^-4 of it the sum that divides is that of the unrounded products, else that of the
// rounded ones (of which fp16 drops at most what is below 2^-27 of the largest
// probability): errors that numerator and denominator have in common cancel (relative error
// of fp16 results with a window of 4000, heads of 256, 2.4e-4, of unrounded sums 2.9e-4).
constexpr float kPaNear = -4.f;
constexpr int kPaUnit = 4;         // a row's mean is in units of 2^4 until it is rounded to the result

struct PagedAttnArgs {
  const uint16_t* q;
  int64_t q_r;
  PagedCache c;
  const int32_t* tables;
  int64_t t_b;
  int width;
  const int64_t *starts, *lengths;
  uint16_t* out;
  int rows, batch, group;
  int window;  // 0: none
  int sinks;
  float scale;
  int whole;     // row blocks are not divided: each counts as one tile of the line
  int runs;
  float* parts;  // [runs][2]: a run divides at most its first and its last row block
  struct PaCut* cuts;  // [runs], behind the parts
};

// fp32 words of one part: RB x D means, RB maxima, RB sums
__host__ __device__ inline int64_t pa_part_words(int rb, int dim) { return (int64_t)rb * (dim + 2); }

// ---------------------------------------------------------------------------
// The line of tiles: sequence after sequence, within one KV head after KV head, within
// one row block after the other. Rows of an empty sequence and behind the last have a
// tile without positions, for their zeros.
// ---------------------------------------------------------------------------
struct PaSeq {
  int first, n;    // rows
  int lead;        // rows before starts[b] (of sequence 0, where starts[0] > 0)
  int64_t p0;      // position of row `first`; -1 - n and below: none
  int blocks;      // row blocks of a KV head
};
template <int RB>
__device__ __forceinline__ PaSeq pa_seq(const PagedAttnArgs& a, int b) {
  PaSeq s{0, 0, 0, 0, 0};
  if (b > a.batch) return s;
  const int64_t rows = a.rows;
  const int64_t s0 = b == 0 ? 0 : max((int64_t)0, min(a.starts[b], rows));
  const int64_t end = b == a.batch ? rows : a.starts[b + 1];
  const int64_t s1 = max(s0, min(end, rows));
  const int64_t len = b == a.batch ? -1 : a.lengths[b];
  s.first = (int)s0;
  s.n = (int)(s1 - s0);
  s.lead = b == 0 ? (int)max((int64_t)0, min(a.starts[0], rows)) : 0;
  s.p0 = len >= 0 ? len - (end - s0) : INT64_MIN / 2;
  s.blocks = (s.n * a.group + RB - 1) / RB;
  return s;
}
// the positions of row block qb: [0, sink) and [lo, hi), in tiles
struct PaSpan {
  int lo, hi, sink;
  int sink_tiles, first_tile, tiles;
};
template <int RB, int TILE>
__device__ __forceinline__ PaSpan pa_span(const PagedAttnArgs& a, const PaSeq& s, int qb) {
  PaSpan r;
  const int cap = a.width << a.c.log_t;
  const int t0 = qb * RB / a.group;
  const int t1 = min(s.n - 1, (qb * RB + RB - 1) / a.group);
  r.hi = (int)max((int64_t)0, min(s.p0 + t1 + 1, (int64_t)cap));
  r.lo = 0;
  if (a.window) r.lo = (int)max((int64_t)0, min(s.p0 + t0 - a.window + 1, (int64_t)cap));
  r.sink = min(a.sinks, r.lo);
  r.sink_tiles = (r.sink + TILE - 1) / TILE;
  r.first_tile = max(r.lo / TILE, r.sink_tiles);
  r.tiles = max(1, r.sink_tiles + max(0, (r.hi + TILE - 1) / TILE - r.first_tile));
  return r;
}
// tiles of all row blocks of a sequence, one KV head
template <int RB, int TILE>
__device__ __forceinline__ int pa_tiles(const PagedAttnArgs& a, const PaSeq& s) {
  if (a.whole) return s.blocks;
  int sum = 0;
  for (int qb = 0; qb < s.blocks; ++qb) sum += pa_span<RB, TILE>(a, s, qb).tiles;
  return sum;
}
// a row block's place in the line
struct PaPlace {
  int b, kvh, qb, t0;  // and the tile of the row block
  int tiles;
  PaSeq seq;
};
// 64 sequences, one a lane: tiles of a KV head
template <int RB>
struct PaChunk {
  PaSeq seq;
  int tiles, scan;  // and their running sum
};
template <int RB, int TILE>
__device__ __forceinline__ PaChunk<RB> pa_chunk(const PagedAttnArgs& a, int b0, int lane) {
  PaChunk<RB> c;
  c.seq = pa_seq<RB>(a, b0 + lane);
  c.tiles = pa_tiles<RB, TILE>(a, c.seq);
  c.scan = wave_scan_i32(c.tiles, lane);
  return c;
}
__device__ __forceinline__ int pa_from(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// one wave: the length of the line; c: the first chunk
template <int RB, int TILE>
__device__ __forceinline__ int64_t pa_total(const PagedAttnArgs& a, const PaChunk<RB>& c, int lane) {
  int sum = pa_from(c.scan, 63);
  for (int b0 = 64; b0 <= a.batch; b0 += 64) sum += pa_from(pa_chunk<RB, TILE>(a, b0, lane).scan, 63);
  return (int64_t)sum * a.c.kv_heads;
}
// one wave: what holds place `at` of the line (all lanes; at below the total)
template <int RB, int TILE>
__device__ __forceinline__ PaPlace pa_find(const PagedAttnArgs& a, PaChunk<RB> c, int64_t at, int lane) {
  PaPlace r{-1, 0, 0, 0, 0, {}};
  int before = 0;
  for (int b0 = 0; b0 <= a.batch; b0 += 64) {
    if (b0) c = pa_chunk<RB, TILE>(a, b0, lane);
    const uint64_t hit = __ballot((int64_t)(before + c.scan) * a.c.kv_heads > at);
    if (!hit) {
      before += pa_from(c.scan, 63);
      continue;
    }
    const int l = __builtin_ctzll(hit);
    const int tiles = pa_from(c.tiles, l);
    const int64_t in_seq = at - (int64_t)(before + pa_from(c.scan, l) - tiles) * a.c.kv_heads;
    // below tiles kv_heads; KV heads are at most 4096, so that 64 bits are seldom needed
    r.kvh = in_seq <= UINT32_MAX ? (int)((uint32_t)in_seq / (uint32_t)tiles) : (int)(in_seq / tiles);
    int left = (int)(in_seq - (int64_t)r.kvh * tiles);
    PaSeq& s = r.seq;
    s.first = pa_from(c.seq.first, l);
    s.n = pa_from(c.seq.n, l);
    s.lead = pa_from(c.seq.lead, l);
    const uint32_t lo = pa_from((int)(uint32_t)c.seq.p0, l);
    const uint32_t hi = pa_from((int)(uint32_t)((uint64_t)c.seq.p0 >> 32), l);
    s.p0 = (int64_t)((uint64_t)hi << 32 | lo);
    s.blocks = pa_from(c.seq.blocks, l);
    if (a.whole) {
      r.b = b0 + l;
      r.qb = left;
      r.tiles = pa_span<RB, TILE>(a, s, left).tiles;
      return r;
    }
    for (int q0 = 0; q0 < s.blocks; q0 += 64) {
      const int t = q0 + lane < s.blocks ? pa_span<RB, TILE>(a, s, q0 + lane).tiles : 0;
      const int sc = wave_scan_i32(t, lane);
      const uint64_t in = __ballot(sc > left);
      if (in) {
        const int k = __builtin_ctzll(in);
        r.b = b0 + l;
        r.qb = q0 + k;
        r.tiles = pa_from(t, k);
        r.t0 = left - (pa_from(sc, k) - r.tiles);
        return r;
      }
      left -= pa_from(sc, 63);
    }
    return r;
  }
  return r;  // only if the lengths change under the kernel
}
// a place that one wave found, in every thread
__device__ __forceinline__ int pa_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ PaPlace pa_place(const PaPlace& p) {
  const uint32_t lo = pa_uniform((int)(uint32_t)p.seq.p0), hi = pa_uniform((int)(uint32_t)((uint64_t)p.seq.p0 >> 32));
  return PaPlace{pa_uniform(p.b), pa_uniform(p.kvh), pa_uniform(p.qb), pa_uniform(p.t0), pa_uniform(p.tiles),
                 PaSeq{pa_uniform(p.seq.first), pa_uniform(p.seq.n), pa_uniform(p.seq.lead),
                       (int64_t)((uint64_t)hi << 32 | lo), pa_uniform(p.seq.blocks)}};
}

// ---------------------------------------------------------------------------
// MFMA operands
// ---------------------------------------------------------------------------
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
template <bool BF>
__device__ __forceinline__ float4v pa_mfma(u32x4v a, u32x4v b, float4v c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a),
                                                   __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a),
                                                  __builtin_bit_cast(half8v, b), c, 0, 0, 0);
}
// eight e4m3 codes as bf16 or fp16
template <bool BF>
__device__ __forceinline__ u32x4v pa_unpack(uint32_t lo, uint32_t hi) {
  constexpr float s = 1.f;
  if constexpr (BF)
    return u32x4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true))};
  else
    return u32x4v{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true))};
}
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{lo, hi}), half2v));
}
template <bool BF>
__device__ __forceinline__ uint32_t pa_pack16(float lo, float hi) {
  const float2v v{lo, hi};
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2v));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
}
// maximum over the four lanes li, li + 16, li + 32, li + 48, in each of them
__device__ __forceinline__ float pa_rows_max(float v) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t x0 = x[0], x1 = x[1];
  u = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, x0), __builtin_bit_cast(float, x1)));
  auto y = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t y0 = y[0], y1 = y[1];
  return fmaxf(__builtin_bit_cast(float, y0), __builtin_bit_cast(float, y1));
}
// bit 7 of each byte that is a NaN code
__device__ __forceinline__ uint32_t pa_nan(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t pa_nan(u32x4v w) { return pa_nan(w[0]) | pa_nan(w[1]) | pa_nan(w[2]) | pa_nan(w[3]); }
// NaN among 16 codes made zeros; a bit for each
__device__ __forceinline__ uint32_t pa_clean(u32x4v& w) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t n = pa_nan(w[i]) >> 7;  // bits 0, 8, 16 and 24
    bits |= ((n * 0x10204080u) >> 28) << (4 * i);
    w[i] = w[i] & ~(n * 0xFFu);
  }
  return bits;
}

// the bits of positions below n, of 16
__device__ __forceinline__ uint32_t pa_below(int n) { return (1u << min(max(n, 0), 16)) - 1; }

// What the second launch has to know of a run: the row block that begins in it and goes
// on behind it.
struct PaCut {
  int parts;  // runs that it lies in; 0: there is none
  int first, n;  // rows of its sequence
  int kvh, qb;
};
// The runs of a launch: this workgroup's, in tiles of the line. The runs of an XCD are
// neighbours, which share keys and values.
struct PaRun {
  int64_t run, at, end, size;  // at >= end: none
};
__device__ __forceinline__ PaRun pa_run(const PagedAttnArgs& a, int64_t total) {
  total = max(total, (int64_t)1);  // less only for starts that do not rise
  const int64_t size = (total + a.runs - 1) / a.runs;
  const int64_t active = (total + size - 1) / size, per = (active + 7) / 8;
  const int64_t x = blockIdx.x & 7, y = blockIdx.x >> 3;
  // workgroups that are not needed get the numbers behind
  const int64_t run = y < per ? x * per + y : 8 * per + (y - per) * 8 + x;
  if (run < a.runs && threadIdx.x == 0 && a.cuts) a.cuts[run].parts = 0;
  if (run >= active) return PaRun{run, 0, 0, size};
  return PaRun{run, run * size, min(total, (run + 1) * size), size};
}
// where the row block at tiles t0 .. t1 of `tiles` puts its means: null if it is whole.
// A part: the run's first row block, begun before it, or its last, which goes on.
__device__ __forceinline__ float* pa_part(const PagedAttnArgs& a, const PaRun& run, const PaPlace& p, int t1,
                                          int64_t words) {
  if (p.t0 == 0 && t1 == p.tiles) return nullptr;
  if (p.t0 == 0 && threadIdx.x == 0) {
    const int64_t start = run.end - t1;
    a.cuts[run.run] = PaCut{(int)((start + p.tiles - 1) / run.size - run.run) + 1, p.seq.first, p.seq.n,
                            p.kvh, p.qb};
  }
  return a.parts + (run.run * 2 + (p.t0 == 0)) * words;
}

// 1 / l, and 0 for a row that has seen nothing
__device__ __forceinline__ float pa_inverse(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }

// What a wave keeps of RT products of 16 rows.
template <int D, int RT>
struct PaRows {
  static constexpr int KS = D / 32, DT = D / 16;
  u32x4v q[RT][KS];  // B operand: lane = row li, dimensions 64 j + 16 lg + 8 h of product 2 j + h
  int pos[RT];       // of the lane's rows, below 0: sees nothing
  float4v o[RT][DT];
  // bases, whole numbers, so that their powers of two are exact: scores are relative to
  // m (-inf: none seen yet), scores plus the values' exponent bytes, and o, to m + d
  float m[RT], d[RT];
  float l[RT];

  // rows first .. first + 16 RT - 1 of the row block
  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const PaSeq& seq, int kvh, int first, int li,
                                        int lg) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = first + rt * 16 + li;
      const int token = r / a.group, g = r - token * a.group;
      const bool there = token < seq.n;
      pos[rt] = there && token >= seq.lead
                    ? (int)max((int64_t)-1, min(seq.p0 + token, (int64_t)INT32_MAX / 2)) : -1;
      const uint16_t* src = a.q + (int64_t)(seq.first + token) * a.q_r +
                            (int64_t)(kvh * a.group + g) * D + 16 * lg;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4v{0, 0, 0, 0};
        if (there) q[rt][ks] = *reinterpret_cast<const u32x4v*>(src + 64 * (ks >> 1) + 8 * (ks & 1));
      }
      m[rt] = -__builtin_inff();
      d[rt] = 0.f;
      l[rt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = float4v{0.f, 0.f, 0.f, 0.f};
    }
  }
  // scores of positions that a row does not see; bit j of seen: the lane's position
  // x + j of 16
  __device__ __forceinline__ void mask(const PagedAttnArgs& a, float4v (&s)[RT][4], uint32_t (&seen)[RT],
                                       int x, uint32_t there) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      uint32_t hidden = 0;
      if (a.window) hidden = pa_below(pos[rt] - a.window + 1 - x) & ~pa_below(a.sinks - x);
      seen[rt] = pa_below(pos[rt] + 1 - x) & ~hidden & there;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[rt][t][e] = seen[rt] & (1u << (4 * t + e)) ? s[rt][t][e] : -__builtin_inff();
    }
  }
  // p: B operands of two products, 8 neighbouring positions each. kc: what the scores
  // of the lane are multiplied by; vb: exponent byte of its values
  __device__ __forceinline__ void softmax(float4v (&s)[RT][4], float kc, float vb, u32x4v (&p)[RT][2]) {
    // the base is a rounded product, and what is compared with it has to be
#pragma clang fp contract(off)
    float mul[RT], add[RT], lift[RT];
    bool small = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[rt][t][e]);
      top *= kc;
      // the larger of the score's and the product's exponent (NaN where nothing is seen)
      if (__any(top - m[rt] + fmaxf(vb - d[rt], 0.f) > kPaSlack)) {
        const float mn = fmaxf(m[rt], ceilf(pa_rows_max(top)));
        const float to = mn == -__builtin_inff() ? 0.f : mn;
        const float dm = m[rt] - to;
        const float dn = fmaxf(d[rt] + dm, ceilf(pa_rows_max(top - to + vb)));
        const float dz = dn == -__builtin_inff() ? 0.f : dn;
        const float al = __builtin_amdgcn_exp2f(d[rt] + dm - dz);
        l[rt] *= __builtin_amdgcn_exp2f(dm);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= al;
        m[rt] = mn;
        d[rt] = dz;
      }
      const float base = m[rt] == -__builtin_inff() ? 0.f : m[rt];
      lift[rt] = fmaxf(vb - d[rt], kPaLeast) + kPaLift;
      mul[rt] = kc;
      add[rt] = lift[rt] - base;
      small |= top > -__builtin_inff() && vb - d[rt] < kPaNear;
      // beside a base of that size the lift would be rounded, and an exponent that is
      // rounded once could pass the base, which is a rounded product, by its rounding
      if (__builtin_expect(__any(fabsf(base) > 0x1p22f), 0)) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[rt][t][e] = s[rt][t][e] * kc - base;
        mul[rt] = 1.f;
        add[rt] = lift[rt];
      }
    }
    if (__builtin_expect(__any(small), 0)) products<true>(s, mul, add, lift, p);
    else products<false>(s, mul, add, lift, p);
  }
  // SMALL: the sums are those of the unrounded products
  template <bool SMALL>
  __device__ __forceinline__ void products(const float4v (&s)[RT][4], const float (&mul)[RT], const float (&add)[RT],
                                           const float (&lift)[RT], u32x4v (&p)[RT][2]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][e], mul[rt], add[rt]));
        const uint32_t w0 = pa_pack(w[0], w[1]), w1 = pa_pack(w[2], w[3]);
        const half2v ones{(_Float16)1.f, (_Float16)1.f};
        if constexpr (SMALL) {
          sum += (w[0] + w[1]) + (w[2] + w[3]);
        } else {
          sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w0), ones, sum, false);
          sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w1), ones, sum, false);
        }
        p[rt][t >> 1][2 * (t & 1)] = w0;
        p[rt][t >> 1][2 * (t & 1) + 1] = w1;
      }
      l[rt] = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-lift[rt]), l[rt]);
    }
  }
  // A NaN among the values must not reach, as 0 x NaN, the rows that do not see it: for
  // the products it is a zero (pa_clean), and the sums of rows that see it are made NaN
  // here. map: the step's 64 positions, a bit each, of every dimension; FROM, TO: 16
  // dimensions each; seen: as mask() has it.
  template <int FROM, int TO>
  __device__ __forceinline__ void nan_values(const uint64_t* map, const uint32_t (&seen)[RT], int lg) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      unsigned long long all = (unsigned long long)seen[rt] << (16 * lg);
      all |= __shfl_xor(all, 16, 64);
      all |= __shfl_xor(all, 32, 64);
#pragma unroll
      for (int dt = FROM; dt < TO; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (map[16 * dt + 4 * lg + e] & all) o[rt][dt][e] = __builtin_nanf("");
    }
  }
  __device__ __forceinline__ void values(u32x4v v, int dt, int h, const u32x4v (&p)[RT][2]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) o[rt][dt] = pa_mfma<false>(v, p[rt][h], o[rt][dt]);
  }
  // the row's whole sum in all of its lanes, and the mean of its values, in units of
  // 2^kPaUnit: finite also where values are near the largest that bf16 has, or rounded past
  // it to a code (256 * 2^120), which their sums are not
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int unit = (int)d[rt] - 127 - (int)kPaLift - kPaUnit;
      l[rt] += __shfl_xor(l[rt], 16, 64);
      l[rt] += __shfl_xor(l[rt], 32, 64);
      const float inv = pa_inverse(l[rt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[rt][dt][e] = __builtin_ldexpf(o[rt][dt][e] * inv, unit);
    }
  }
  // result or part (of RB rows) of rows first .. of the row block
  template <bool BF, int RB>
  __device__ __forceinline__ void store(const PagedAttnArgs& a, const PaSeq& seq, int kvh, int qb,
                                        int first, float* part, int li, int lg) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int local = first + rt * 16 + li;
      if (!part) {
        const int r = qb * RB + local;
        const int token = r / a.group, g = r - token * a.group;
        if (token >= seq.n) continue;
        uint16_t* dst = a.out + ((int64_t)(seq.first + token) * (a.c.kv_heads * a.group) + kvh * a.group + g) * D +
                        4 * lg;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const float4v v = o[rt][dt] * (float)(1 << kPaUnit);
          *reinterpret_cast<uint2*>(dst + 16 * dt) = make_uint2(pa_pack16<BF>(v[0], v[1]), pa_pack16<BF>(v[2], v[3]));
        }
      } else {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<float4v*>(part + local * D + 16 * dt + 4 * lg) = o[rt][dt];
        if (lg == 0) {
          part[RB * D + local] = m[rt];
          part[RB * D + RB + local] = l[rt];
        }
      }
    }
  }
};

// blocks of positions p + 16 (li / 4) (the lane's keys) and p + 16 lg (its values and
// scales), -1 where there is none
struct PaBlocks {
  int k, v;
};
__device__ __forceinline__ PaBlocks pa_blocks(const PagedAttnArgs& a, const int32_t* table, int p, int li,
                                              int lg) {
  PaBlocks r;
  const int ik = (p + 16 * (li >> 2)) >> a.c.log_t, iv = (p + 16 * lg) >> a.c.log_t;
  r.k = table[min(ik, a.width - 1)];
  r.v = table[min(iv, a.width - 1)];
  if (ik >= a.width || r.k >= a.c.blocks) r.k = -1;
  if (iv >= a.width || r.v >= a.c.blocks) r.v = -1;
  return r;
}
// The lane's part of the keys (rows 4 t and 16-byte chunks 4 j behind it) and values
// (16 dimensions behind it) of 64 positions from p on: what does not change within a KV
// head once, then a multiply-add a step (strides of blocks are below 2^31 bytes).
template <int D>
struct PaLanes {
  const uint8_t *k, *v, *ks, *vs;
  uint32_t k_b, v_b, s_b;
  int t_mask, k_off, v_off;  // the lane's 16 positions among the 64
  __device__ __forceinline__ PaLanes(const PagedAttnArgs& a, int kvh, int li, int lg) {
    k = a.c.k + (((int64_t)kvh << a.c.log_t) + (li & 3)) * D + 16 * lg;
    v = a.c.v + (((int64_t)kvh * D + li) << a.c.log_t);
    ks = a.c.ks + kvh;
    vs = a.c.vs + kvh;
    k_b = (uint32_t)a.c.k_b;
    v_b = (uint32_t)a.c.v_b;
    s_b = (uint32_t)a.c.s_b;
    t_mask = (1 << a.c.log_t) - 1;
    k_off = 16 * (li >> 2);
    v_off = 16 * lg;
  }
  __device__ __forceinline__ const uint8_t* keys(int p, int block) const {
    return k + ((uint64_t)(uint32_t)max(block, 0) * k_b + (uint32_t)(((p + k_off) & t_mask) * D));
  }
  __device__ __forceinline__ const uint8_t* values(int p, int block) const {
    return v + ((uint64_t)(uint32_t)max(block, 0) * v_b + (uint32_t)((p + v_off) & t_mask));
  }
  __device__ __forceinline__ uint64_t scale(int block) const {
    return (uint64_t)(uint32_t)max(block, 0) * s_b;
  }
};
// ---------------------------------------------------------------------------
// Few rows: the four waves of a workgroup take 64 positions each of a tile of 256,
// straight from memory to registers, and join their sums in LDS at the end of a row
// block. The loads of the next 64 keys go out when the scores are done with these, those
// of the values after the second product (both at once, with registers for two steps of
// values, made heads of 256 slower by spills: 112 -> 133 us).
// ---------------------------------------------------------------------------
template <int D, bool BF, int RT>
__global__ __launch_bounds__(256, RT == 1 && D != 256 ? 2 : 1) void paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int RB = 16 * RT, TILE = 256;
  constexpr int KS = D / 32, KL = D / 64, DT = D / 16;
  __shared__ __align__(16) float4v join[2][RT * DT * 64];  // and, until then, each wave's map of NaN
  __shared__ float join_m[4][RB], join_l[4][RB];
  __shared__ PaPlace place;
  __shared__ int64_t line;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  PaChunk<RB> chunk{};
  if (wave == 0) {
    chunk = pa_chunk<RB, TILE>(a, 0, lane);
    const int64_t total = pa_total<RB, TILE>(a, chunk, lane);
    if (lane == 0) line = total;
  }
  __syncthreads();
  const PaRun run = pa_run(a, line);

  for (int64_t at = run.at; at < run.end;) {
    if (wave == 0) {
      const PaPlace p = pa_find<RB, TILE>(a, chunk, at, lane);
      if (lane == 0) place = p;
    }
    __syncthreads();
    const PaPlace here = pa_place(place);
    const int b = here.b, kvh = here.kvh, qb = here.qb, t0 = here.t0;
    if (b < 0) return;
    const int t1 = a.whole ? here.tiles : (int)min((int64_t)here.tiles, t0 + (run.end - at));
    at += a.whole ? 1 : t1 - t0;
    const PaSeq seq = here.seq;
    const PaSpan span = pa_span<RB, TILE>(a, seq, qb);
    const int32_t* table = a.tables + (int64_t)min(b, a.batch - 1) * a.t_b;
    // positions of the block's first and last row (of fewer rows, if some are absent)
    const int64_t p_low = seq.lead ? -1 : seq.p0 + qb * RB / a.group;
    const int64_t p_high = seq.p0 + (qb * RB + RB - 1) / a.group;
    PaRows<D, RT> w;
    w.begin(a, seq, kvh, qb * RB, li, lg);
    const float c = a.scale * kPaLog2e;

    const PaLanes<D> at_lane(a, kvh, li, lg);
    // the wave's 64 positions of tile i of the row block, and whether any row sees one
    auto first_pos = [&](int i) {
      return (i < span.sink_tiles ? i : span.first_tile + i - span.sink_tiles) * TILE + wave * 64;
    };
    auto next_tile = [&](int i) {  // the first from i on of which the wave sees something
      for (; i < t1; ++i) {
        const int p = first_pos(i);
        if (p < span.hi && (p + 63 >= span.lo || p < span.sink)) break;
      }
      return i;
    };
    u32x4v kr[4][KL], vr[DT];
    uint32_t ksb, vsb;
    uint16_t* const nan_map = reinterpret_cast<uint16_t*>(&join[0][0]) + wave * D * 4;
    auto load_k = [&](int p, PaBlocks bl) {
      const uint8_t* k = at_lane.keys(p, bl.k);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < KL; ++j)
          kr[t][j] = *reinterpret_cast<const u32x4v*>(k + 4 * t * D + 64 * j);
      ksb = at_lane.ks[at_lane.scale(bl.v)];
    };
    auto load_v = [&](int p, PaBlocks bl) {
      const uint8_t* v = at_lane.values(p, bl.v);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vr[dt] = *reinterpret_cast<const u32x4v*>(v + ((16 * dt) << a.c.log_t));
      vsb = at_lane.vs[at_lane.scale(bl.v)];
    };

    int i = next_tile(t0);
    PaBlocks cur{-1, -1}, nxt{-1, -1};
    if (i < t1) {
      cur = pa_blocks(a, table, first_pos(i), li, lg);
      load_k(first_pos(i), cur);
      load_v(first_pos(i), cur);
    }
    while (i < t1) {
      const int p = first_pos(i);
      const int in = next_tile(i + 1);
      if (in < t1) nxt = pa_blocks(a, table, first_pos(in), li, lg);
      // whether all rows see all of it
      const bool full = p + 63 <= p_low && !__any(cur.v < 0) &&
                        (!a.window || p > p_high - a.window || p + 64 <= a.sinks);
      float4v s[RT][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][t] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4v kf = pa_unpack<BF>(kr[t][ks >> 1][2 * (ks & 1)], kr[t][ks >> 1][2 * (ks & 1) + 1]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][t] = pa_mfma<BF>(kf, w.q[rt][ks], s[rt][t]);
        }
      }
      // above 0: a masked -inf stays one
      const float kc = fmaxf(e8m0(ksb) * c, 1e-37f);
      if (in < t1) load_k(first_pos(in), nxt);
      uint32_t seen[RT];
      bool some_nan = false;
      if (!full) {
        w.mask(a, s, seen, p + 16 * lg, cur.v >= 0 ? 0xFFFFu : 0u);
        uint32_t bad = 0;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) bad |= pa_nan(vr[dt]);
        some_nan = __any(bad != 0);
        if (__builtin_expect(some_nan, 0))
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) nan_map[(16 * dt + li) * 4 + lg] = (uint16_t)pa_clean(vr[dt]);
      }
      u32x4v pf[RT][2];
      w.softmax(s, kc, (float)vsb, pf);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w.values(pa_unpack<false>(vr[dt][2 * h], vr[dt][2 * h + 1]), dt, h, pf);
      if (__builtin_expect(some_nan, 0)) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // other lanes' bits
        w.template nan_values<0, DT>(reinterpret_cast<const uint64_t*>(nan_map), seen, lg);
      }
      if (in < t1) load_v(first_pos(in), nxt);
      cur = nxt;
      i = in;
    }

    // the four waves' means, each by its share of the sum, in the order (0 + 2) + (1 + 3)
    w.finish();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      if (lg == 0) {
        join_m[wave][rt * 16 + li] = w.m[rt];
        join_l[wave][rt * 16 + li] = w.l[rt];
      }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + li;
      const float top = fmaxf(fmaxf(join_m[0][r], join_m[1][r]), fmaxf(join_m[2][r], join_m[3][r]));
      const float base = top == -__builtin_inff() ? 0.f : top;
      float sum[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] = join_l[k][r] * __builtin_amdgcn_exp2f(join_m[k][r] - base);
      const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
      const float al = w.l[rt] * __builtin_amdgcn_exp2f(w.m[rt] - base) * pa_inverse(all);
      w.m[rt] = top;
      w.l[rt] = all;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        w.o[rt][dt] *= al;
        if (wave >= 2) join[wave - 2][(rt * DT + dt) * 64 + lane] = w.o[rt][dt];
      }
    }
    __syncthreads();
    if (wave < 2)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) w.o[rt][dt] += join[wave][(rt * DT + dt) * 64 + lane];
    __syncthreads();
    if (wave == 1)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) join[0][(rt * DT + dt) * 64 + lane] = w.o[rt][dt];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) w.o[rt][dt] += join[0][(rt * DT + dt) * 64 + lane];
      }
      float* part = pa_part(a, run, here, t1, pa_part_words(RB, D));
      w.template store<BF, RB>(a, seq, kvh, qb, 0, part, li, lg);
    }
    __syncthreads();  // the buffers are free
  }
}

// ---------------------------------------------------------------------------
// Many rows (chunks of prompts): the four waves of a workgroup take 16 RT rows each and
// share 64 positions a step. Two waves bring the keys and two the values, convert them
// and put them to LDS in the order in which lanes read them (64 lanes x 16 bytes an
// operand, from the addresses that the other form loads), so that a code is converted
// once for all rows: the conversions, one instruction for two codes, would otherwise be
// a third of the vector instructions beside the products (1024 tokens behind 30,000 were
// 749 us that way and 676 this way, before later changes). Two buffers: while a step is
// worked on, the next one's operands are written and the loads of the one behind it are
// under way; one barrier a step. The waves that bring values look for NaN in them, in
// steps that some row of the block does not see whole, for all waves: looked for behind
// the barrier by every wave, with the products of the rare path in its code, the steps
// had no registers left (1024 tokens behind 30,000: 992 us, with spills).
// ---------------------------------------------------------------------------
// workgroups a CU: as many as the registers hold (heads of 64, microseconds by two and
// three: 1024 tokens behind 30,000 507 426, 16 x 64 behind 4000 91 85, 2048 tokens of a
// prompt 87 78)
constexpr int pa_chunk_wgs(int dim) { return dim == 256 ? 1 : dim == 64 ? 3 : 2; }
template <int D, bool BF, int RT>
__global__ __launch_bounds__(256, pa_chunk_wgs(D)) void paged_chunk_kernel(const PagedAttnArgs a) {
  constexpr int RB = 64 * RT, TILE = 64;
  constexpr int KL = D / 64, DT = D / 16;
  constexpr int PER = DT / 2;          // 16-byte loads of a wave; 4 KL = DT of keys and of values
  constexpr int KF = 2 * DT;           // operands of keys, 1 KB each, then as many of values
  __shared__ __align__(16) u32x4v buf0[2 * KF * 64];
  __shared__ __align__(16) u32x4v buf1[2 * KF * 64];
  // positions of NaN by dimension, and whether a wave that brings values had any
  __shared__ uint64_t nan0[D], nan1[D];
  __shared__ uint32_t some0[2], some1[2];
  __shared__ PaPlace place;
  __shared__ int64_t line;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  PaChunk<RB> chunk{};
  if (wave == 0) {
    chunk = pa_chunk<RB, TILE>(a, 0, lane);
    const int64_t total = pa_total<RB, TILE>(a, chunk, lane);
    if (lane == 0) line = total;
  }
  __syncthreads();
  const PaRun run = pa_run(a, line);

  for (int64_t at = run.at; at < run.end;) {
    if (wave == 0) {
      const PaPlace p = pa_find<RB, TILE>(a, chunk, at, lane);
      if (lane == 0) place = p;
    }
    __syncthreads();
    const PaPlace here = pa_place(place);
    const int b = here.b, kvh = here.kvh, qb = here.qb, t0 = here.t0;
    if (b < 0) return;
    const int t1 = a.whole ? here.tiles : (int)min((int64_t)here.tiles, t0 + (run.end - at));
    at += a.whole ? 1 : t1 - t0;
    const PaSeq seq = here.seq;
    const PaSpan span = pa_span<RB, TILE>(a, seq, qb);
    const int32_t* table = a.tables + (int64_t)min(b, a.batch - 1) * a.t_b;
    // the wave's rows, and positions of the first and the last of them
    const int first = qb * RB + wave * 16 * RT;
    const int token0 = first / a.group, token1 = (first + 16 * RT - 1) / a.group;
    const int64_t p_low = seq.lead ? -1 : seq.p0 + token0;
    const int64_t p_high = seq.p0 + min(token1, seq.n - 1);
    const bool idle = token0 >= seq.n;
    // and of the row block's
    const int64_t block_low = seq.lead ? -1 : seq.p0 + qb * RB / a.group;
    const int64_t block_high = seq.p0 + min((qb * RB + RB - 1) / a.group, seq.n - 1);
    PaRows<D, RT> w;
    w.begin(a, seq, kvh, first, li, lg);
    const float c = a.scale * kPaLog2e;

    auto first_pos = [&](int i) {
      return (i < span.sink_tiles ? i : span.first_tile + i - span.sink_tiles) * TILE;
    };
    auto in_sight = [&](int i) {  // of the row block
      const int p = first_pos(i);
      return p < span.hi && (p + 63 >= span.lo || p < span.sink);
    };
    auto next_tile = [&](int i) {
      while (i < t1 && !in_sight(i)) ++i;
      return i;
    };
    const PaLanes<D> at_lane(a, kvh, li, lg);
    // a step on its way: the wave's part of it, the scales of the lane's 16 positions
    u32x4v raw[PER];
    uint32_t rk, rv;
    int rblock;
    PaBlocks nb;
    auto load = [&](int p, PaBlocks bl) {
      if (wave < 2) {
        const uint8_t* k = at_lane.keys(p, bl.k);
#pragma unroll
        for (int n = 0; n < PER; ++n) {
          const int f = wave * PER + n;
          raw[n] = *reinterpret_cast<const u32x4v*>(k + 4 * (f / KL) * D + 64 * (f % KL));
        }
      } else {
        const uint8_t* v = at_lane.values(p, bl.v) + (((wave - 2) * PER * 16) << a.c.log_t);
#pragma unroll
        for (int n = 0; n < PER; ++n) raw[n] = *reinterpret_cast<const u32x4v*>(v + ((16 * n) << a.c.log_t));
      }
      const uint64_t sc = at_lane.scale(bl.v);
      rk = at_lane.ks[sc];
      rv = at_lane.vs[sc];
      rblock = bl.v;
    };
    // of the step that is worked on, and of the one whose operands are in LDS next
    uint32_t sc = 0, nsc = 0;
    auto convert = [&](u32x4v* to, uint64_t* nan_map, uint32_t* some_nan, int p) {
      nsc = rk | rv << 8 | (rblock >= 0 ? 1u << 16 : 0u);
      if (wave >= 2) {
        // a NaN that all rows see makes them all NaN as it is
        uint32_t bad = 0;
        if (p + 63 > block_low || __any(rblock < 0) ||
            (a.window && p <= block_high - a.window && p + 64 > a.sinks)) {
#pragma unroll
          for (int n = 0; n < PER; ++n) bad |= pa_nan(raw[n]);
        }
        const bool some = __any(bad != 0);
        if (__builtin_expect(some, 0))
#pragma unroll
          for (int n = 0; n < PER; ++n)
            reinterpret_cast<uint16_t*>(nan_map)[(((wave - 2) * PER + n) * 16 + li) * 4 + lg] =
                (uint16_t)pa_clean(raw[n]);
        if (lane == 0) some_nan[wave - 2] = some;
      }
      u32x4v* dst = to + (wave * PER * 2) * 64 + lane;
#pragma unroll
      for (int n = 0; n < PER; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          dst[(2 * n + h) * 64] = BF && wave < 2 ? pa_unpack<true>(raw[n][2 * h], raw[n][2 * h + 1])
                                                 : pa_unpack<false>(raw[n][2 * h], raw[n][2 * h + 1]);
    };
    int i = next_tile(t0), in = next_tile(i + 1), after = next_tile(in + 1);
    if (i < t1) {
      load(first_pos(i), pa_blocks(a, table, first_pos(i), li, lg));
      convert(buf0, nan0, some0, first_pos(i));
      if (in < t1) load(first_pos(in), pa_blocks(a, table, first_pos(in), li, lg));
      if (after < t1) nb = pa_blocks(a, table, first_pos(after), li, lg);
    }
    auto step = [&](const u32x4v* from, const uint64_t* nan_map, const uint32_t* some_nan, u32x4v* to,
                    uint64_t* nan_to, uint32_t* some_to) {
      const int p = first_pos(i);
      sc = nsc;
      __syncthreads();  // the operands are there, and `to` is done with
      if (in < t1) {
        convert(to, nan_to, some_to, first_pos(in));
        if (after < t1) {
          load(first_pos(after), nb);
          const int behind = next_tile(after + 1);
          if (behind < t1) nb = pa_blocks(a, table, first_pos(behind), li, lg);
          i = in;
          in = after;
          after = behind;
        } else {
          i = in;
          in = after;
        }
      } else {
        i = in;
      }
      // a wave whose rows see nothing of the step leaves it
      const bool none = idle || p > p_high ||
                        (a.window && p + 63 <= max(p_low, (int64_t)-1) - a.window && p >= a.sinks);
      if (none) return;
      const bool full = p + 63 <= p_low && !__any(!(sc >> 16)) &&
                        (!a.window || p > p_high - a.window || p + 64 <= a.sinks);
      const uint32_t nan_low = some_nan[0], nan_high = some_nan[1];  // under way until they are needed
      const u32x4v* kf = from + lane;
      const u32x4v* vf = kf + KF * 64;
      // operands A ahead of their products; the fences keep the compiler from bringing
      // them all at once, for which there are no registers
      constexpr int A = 4;
      float4v s[RT][4];
      __builtin_amdgcn_s_setprio(1);  // the other workgroup's wave has vector work meanwhile
      {
        u32x4v g[A];
#pragma unroll
        for (int f = 0; f < A; ++f) g[f] = kf[f * 64];
#pragma unroll
        for (int f = 0; f < KF; ++f) {
          const int t = f / (2 * KL), j = f % (2 * KL);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            s[rt][t] = pa_mfma<BF>(g[f % A], w.q[rt][j], j ? s[rt][t] : float4v{0.f, 0.f, 0.f, 0.f});
          if (f + A < KF) g[f % A] = kf[(f + A) * 64];
          if (f & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      // above 0: a masked -inf stays one
      const float kc = fmaxf(e8m0(sc & 0xFFu) * c, 1e-37f);
      const uint32_t there = sc >> 16 ? 0xFFFFu : 0u;
      uint32_t seen[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) seen[rt] = 0xFFFFu;
      if (!full) w.mask(a, s, seen, p + 16 * lg, there);
      u32x4v pf[RT][2];
      w.softmax(s, kc, (float)(sc >> 8 & 0xFFu), pf);
      {
        u32x4v v[A];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < A; ++f) v[f] = vf[f * 64];
#pragma unroll
        for (int f = 0; f < KF; f += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) w.values(v[(f + h) % A], f >> 1, h, pf);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (f + h + A < KF) v[(f + h) % A] = vf[(f + h + A) * 64];
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
      }
      if (__builtin_expect(pa_uniform(nan_low | nan_high), 0)) {
        if (pa_uniform(nan_low)) w.template nan_values<0, DT / 2>(nan_map, seen, lg);
        if (pa_uniform(nan_high)) w.template nan_values<DT / 2, DT>(nan_map, seen, lg);
      }
    };
    while (i < t1) {
      step(buf0, nan0, some0, buf1, nan1, some1);
      if (i < t1) step(buf1, nan1, some1, buf0, nan0, some0);
    }
    w.finish();
    float* part = pa_part(a, run, here, t1, pa_part_words(RB, D));
    w.template store<BF, RB>(a, seq, kvh, qb, wave * 16 * RT, part, li, lg);
    __syncthreads();  // the buffers are free
  }
}

// ---------------------------------------------------------------------------
// The row block that begins in a run and goes on behind it: out = sum of its parts'
// means, each weighted l_part exp2(m_part - m) / l, in order. A wave a row, lane =
// dimensions.
// ---------------------------------------------------------------------------
template <int D, bool BF, int RB>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
  // rows of a wave: of 128 its workgroups would be many, most of them with nothing to do
  // (1024 tokens behind 30,000: 27 us by one row)
  constexpr int ROWS = RB == 128 ? 4 : 1;
  constexpr int E = D / 64, U = ROWS == 1 ? 8 : 4;
  typedef float floatE __attribute__((ext_vector_type(E)));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t run = blockIdx.x;
  const PaCut cut = a.cuts[run];
  const int parts = cut.parts;
  if (!parts) return;
  const int64_t words = pa_part_words(RB, D);
  const float* base = a.parts + run * 2 * words;
  // the first part is its run's last, the others are their runs' first
  auto part = [&](int s) { return base + s * 2 * words + (s == 0 ? words : 0); };
  const int first = (blockIdx.y * 4 + wave) * ROWS;
  if ((cut.qb * RB + first) / a.group >= cut.n) return;
  float m[ROWS], l[ROWS];
  floatE o[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    m[i] = -__builtin_inff();
    l[i] = 0.f;
    o[i] = 0.f;
  }
  for (int s0 = 0; s0 < parts; s0 += 64) {
    const int here = min(64, parts - s0);
    float w[ROWS];
    const float* p = part(s0 + min(lane, here - 1)) + RB * D + first;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float pm = lane < here ? p[i] : -__builtin_inff(), pl = p[RB + i];
      float mn = pm;
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
      mn = fmaxf(mn, m[i]);
      const float shift = mn == -__builtin_inff() ? 0.f : mn;
      w[i] = lane < here ? pl * __builtin_amdgcn_exp2f(pm - shift) : 0.f;
      const float before = l[i] * __builtin_amdgcn_exp2f(m[i] - shift);
      m[i] = mn;
      l[i] = before + wave_sum_dpp(w[i]);
      const float inv = pa_inverse(l[i]);
      o[i] *= before * inv;
      w[i] *= inv;
    }
    for (int s = 0; s < here; s += U) {
      floatE t[U][ROWS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* q = part(s0 + min(s + u, here - 1)) + first * D;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) t[u][i] = reinterpret_cast<const floatE*>(q + i * D)[lane];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s + u < here)
#pragma unroll
          for (int i = 0; i < ROWS; ++i)
            o[i] += t[u][i] *
                    __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[i]), s + u));
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = cut.qb * RB + first + i;
    const int token = r / a.group, g = r - token * a.group;
    if (token >= cut.n) return;
    uint16_t h[E];
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = to16(o[i][e] * (float)(1 << kPaUnit), BF);
    uint16_t* dst = a.out + ((int64_t)(cut.first + token) * a.c.kv_heads * a.group + cut.kvh * a.group + g) * D +
                    lane * E;
    __builtin_memcpy(__builtin_assume_aligned(dst, 2 * E), h, 2 * E);
  }
}

// The form, by the rows of a KV head that a sequence has in the mean: 16 rows a workgroup
// up to 32 (two row blocks cost no more than one of 32), 32 rows up to 64 (not for heads
// of 256, where they do not fit the registers), 128 beyond. That form's steps are dearer
// where there are few of them: up to 128 rows it needs 64 (sequence, KV head) pairs. The
// mean is over what the call has on the host, empty slots and padding among it; a step of
// long chunks beside single tokens has one form for both.
// Microseconds by 16, 32 and 128 rows, from a graph, one sequence of 8000 and of 30,000
// and 16 of 4000 positions, 8 KV heads, equal counts:
//   head    rows      1 x 8000      1 x 30,000       16 x 4000
//    64       32    23  24  29      24   32   46      28   32   42
//             64    21  22  34      29   35   50      42   41   47
//            128    22  24  45      41   49   67      72   78   56
//            256    28  29  43      62   74   63     118  135   85
//   128       32    25  27  49      33   41   66      43   42   68
//             64    26  27  60      44   46   74      69   54   77
//            128    32  31  75      73   64   91     135  106   85
//            256    43  38  58     120   98   92     236  182  122
//   256       32    27   -  52      59    -   97      76    -  160
//             64    35   -  64      87    -  107     153    -  165
//            128    48   -  75     154    -  121     276    -  175
//            256    73   -  77     224    -  166     501    -  302
// Not the fewest by this rule: 256 rows behind 8000 (heads of 64 43 for 28, of 128 58 for
// 38) and 128 rows of heads of 256 behind 30,000 (154 for 121).
// Workgroups a CU: two of 16 rows (one with heads of 256: 16 rows, 16 x 4000, 58 us, two
// 70), one of 32 (64 rows, 16 x 4000, 56 us, two 72); of 128 as above.
//
// Row blocks of up to four tiles (1024 positions that the tables have room for) are not
// divided: no second launch. Microseconds divided and whole, heads of 128, one row block
// a sequence, graph and eager: one sequence of 700 14.1 13.7 and 17.6 13.7, of 1400 13.7
// 18.8 and 17.4 17.5; 16 of 959 17.3 16.7 and 17.4 15.8; 64 of 959 29.6 27.1 and 28.0
// 25.7. Heads of 256 lose more by a whole block's steps (one sequence of 700: 18.0 20.5
// eager), 128 rows by their fewer workgroups (256 rows of 64 tokens behind 700: 30.1 36.3).
constexpr int kPaWhole = 4;
struct PaPlan {
  int rb;      // rows of a row block
  int runs;
  bool whole;  // row blocks of so few tiles that they are not divided
  bool split;  // a row block may be divided
  bool fits;   // the tiles of a KV head can be counted in 32 bits
};
static PaPlan pa_plan(int64_t rows, int64_t batch, int heads, int kv_heads, int dim, int64_t positions) {
  PaPlan p;
  const int group = heads / kv_heads;
  const int64_t mean = (rows + batch - 1) / batch * group;
  if (mean > 128 || (mean > 64 && batch * kv_heads >= 64)) p.rb = 128;
  else p.rb = mean > 32 && dim != 256 ? 32 : 16;
  const int tile = p.rb == 128 ? 64 : 256;
  const int64_t tiles = (positions + tile - 1) / tile;
  const int64_t blocks = rows * group / p.rb + batch + 1;  // row blocks of a KV head, at most
  p.fits = (double)blocks * (double)tiles < 1e9;
  p.whole = tiles <= (p.rb != 128 && dim != 256 ? kPaWhole : 1);
  const double most = p.fits ? (double)blocks * (p.whole ? 1 : tiles) * kv_heads : 1e9;
  const int64_t wanted = (int64_t)num_cus() * (p.rb == 128 ? pa_chunk_wgs(dim) : p.rb == 16 && dim != 256 ? 2 : 1);
  p.runs = (int)((double)wanted < most ? (double)wanted : most);
  p.split = !p.whole && p.runs > 1;
  return p;
}

static bool pa_shape_ok(int64_t rows, int64_t batch, int heads, int kv_heads, int dim) {
  return rows >= 0 && rows <= kPagedMaxRows && batch >= 0 && batch <= kPagedMaxBatch &&
         kv_heads >= 1 && heads >= 1 && heads <= 65535 && heads % kv_heads == 0 &&
         (rows + 1) * (heads / kv_heads) <= INT32_MAX - 256 &&  // rows of a KV head
         (dim == 64 || dim == 128 || dim == 256);
}

template <int D, bool BF>
static int launch_pa(const PaPlan& p, const PagedAttnArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)((p.runs + 7) / 8 * 8);
  const dim3 join((unsigned)p.runs, (unsigned)(p.rb == 128 ? p.rb / 16 : p.rb / 4));
  switch (p.rb) {
    case 16: paged_attn_kernel<D, BF, 1><<<grid, 256, 0, st>>>(a); break;
    case 32:
      if constexpr (D != 256) paged_attn_kernel<D, BF, 2><<<grid, 256, 0, st>>>(a);
      break;
    default: paged_chunk_kernel<D, BF, 2><<<grid, 256, 0, st>>>(a); break;
  }
  const int rc = launch_status();
  if (rc != PE_OK || !p.split) return rc;
  switch (p.rb) {
    case 16: paged_join_kernel<D, BF, 16><<<join, 256, 0, st>>>(a); break;
    case 32:
      if constexpr (D != 256) paged_join_kernel<D, BF, 32><<<join, 256, 0, st>>>(a);
      break;
    default: paged_join_kernel<D, BF, 128><<<join, 256, 0, st>>>(a); break;
  }
  return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_paged_attention_workspace_size(int64_t rows, int64_t batch, int heads,
                                                    int kv_heads, int head_dim, int64_t positions) {
  if (!pa_shape_ok(rows, batch, heads, kv_heads, head_dim) || rows < 1 || batch < 1 || positions < 1)
    return 0;
  const PaPlan p = pa_plan(rows, batch, heads, kv_heads, head_dim, positions);
  return p.split ? (size_t)p.runs * (2 * pa_part_words(p.rb, head_dim) * 4 + sizeof(PaCut)) : 0;
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
  if (!pa_shape_ok(rows, batch, heads, kv_heads, head_dim) || width < 1 || width > kPagedMaxWidth ||
      t_b < width || q_r < 0 || window < 0 || sinks < 0 || !(scale >= 0.f && scale <= 3e38f))
    return PE_ERR_DIMS;
  if (!aligned16(q) || q_r % 8 || !aligned16(out)) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  if (batch == 0) return PE_ERR_DIMS;
  const PaPlan p = pa_plan(rows, batch, heads, kv_heads, head_dim, width * block_size);
  if (!p.fits) return PE_ERR_DIMS;
  const size_t need = pe_paged_attention_workspace_size(rows, batch, heads, kv_heads, head_dim,
                                                        width * block_size);
  if (need && (!workspace || workspace_bytes < need)) return PE_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return PE_ERR_ALIGN;
  a.q = reinterpret_cast<const uint16_t*>(q);
  a.q_r = q_r;
  a.tables = tables;
  a.t_b = t_b;
  a.width = (int)width;
  a.starts = starts;
  a.lengths = lengths;
  a.out = reinterpret_cast<uint16_t*>(out);
  a.rows = (int)rows;
  a.batch = (int)batch;
  a.group = heads / kv_heads;
  // past every position there is no difference
  a.window = (int)(window < kPagedMaxPositions ? window : 0);
  a.sinks = a.window ? (int)(sinks < kPagedMaxPositions ? sinks : kPagedMaxPositions) : 0;
  a.scale = scale;
  a.whole = p.whole;
  a.runs = p.runs;
  a.parts = reinterpret_cast<float*>(workspace);
  a.cuts = p.split ? reinterpret_cast<PaCut*>(a.parts + (int64_t)p.runs * 2 * pa_part_words(p.rb, head_dim))
                   : nullptr;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (head_dim * 2 + bf) {
    case 128: return launch_pa<64, false>(p, a, st);
    case 129: return launch_pa<64, true>(p, a, st);
    case 256: return launch_pa<128, false>(p, a, st);
    case 257: return launch_pa<128, true>(p, a, st);
    case 512: return launch_pa<256, false>(p, a, st);
    default: return launch_pa<256, true>(p, a, st);
  }
}
