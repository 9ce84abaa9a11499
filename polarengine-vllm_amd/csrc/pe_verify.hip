// Verification of drafted tokens: which nodes of a chain or tree of drafts stand
// against the target's distribution, from given uniform numbers, and the token
// that follows them. Rejection sampling: with every number uniform the tokens
// are distributed as the target's own.
//
// Everything that decides is in 64 bits: the answers are whole numbers, and over
// a vocabulary of 150,000 an error of 1e-7 in a cumulative sum moves about one
// sampled token in a hundred.
//
// Three launches. The first reads every logit once, 8192 of a row per workgroup, and
// leaves each piece's maximum, its place and its sum of exp((x - max) / T). The
// second joins the pieces of every row and walks the trees, one workgroup a sequence
// (64 nodes: one wave, lane = node). In the third the workgroups of a sequence sum
// the weights of 2048 tokens each at the node that the walk ends in; the last one to
// finish finds the piece and the token in it. The counters of that hand-over are
// cleared by the second launch, so the workspace needs no state between calls.
//
// Measured: 8 x 64 nodes over 151,936 32-bit logits 74.7 + 13.9 + 15.6 us (the read
// 4.2 TB/s beside 64-bit exponentials; greedy, without them, 55.4 + 13.0 + 4.5); 32 x 8
// nodes over 100,003 16-bit ones 20.8 + 6.2 + 19.1 (greedy 13.0 + 4.8 + 1.8); one
// sequence of five nodes 7.5 + 4.9 + 11.1, each launch a chain of loads and sums. With
// the walk in every workgroup of the draw, two launches: 115, 52 and 23 us in all.

#include "pe_tree.h"

namespace pe {

constexpr int kStatChunk = 8192;
constexpr int kPickChunk = 2048;

struct RowStat {
  float max;
  int first;  // lowest place of the maximum
  double sum;
};

// where a sequence's walk ends
struct WalkEnd {
  int node, count;
  float max;         // of the node's logits
  int done;          // the next token is known (or the slot empty): nothing to draw
  double sum;        // of exp((x - max) / T)
  uint64_t children; // of the node: all rejected
};

struct VerifyArgs {
  const void* logits;
  int64_t l_b, l_n;  // strides, elements
  const int64_t* tokens;
  const int64_t* parents;  // null: a chain
  int64_t p_b;
  const float* uniforms;
  const float* temps;  // null: `temp` for every sequence
  float temp;
  const float* probs;  // null: drafts without probabilities
  int64_t q_b, q_n;
  int64_t *out, *path, *count;
  int n, V, nc, np;
  RowStat* stats;   // [batch * n][nc]
  double* sums;     // [batch][np][2]
  WalkEnd* ends;    // [batch]
  uint32_t* done;   // [batch]
};

// NaN counts as -inf (fmax takes the other operand)
template <int DT>
__device__ __forceinline__ float logit(const void* p, int64_t i) {
  float x;
  if constexpr (DT == PE_DTYPE_F32) x = reinterpret_cast<const float*>(p)[i];
  else x = f16or_bf(reinterpret_cast<const uint16_t*>(p)[i], DT == PE_DTYPE_BF16);
  return fmaxf(x, -__builtin_inff());
}

// 2^z for z <= 0, relative error 2e-14: z = k + f with |f| <= 1/2, 2^f by its
// interpolation of degree 9 at the Chebyshev nodes of [-1/2, 1/2]. ZERO: 0 where it is
// below the normal range, for -inf and for NaN; else about 1e-307 there, in one
// instruction less of the slower kind.
template <bool ZERO>
__device__ __forceinline__ double exp2_f64(double z) {
  z = fmax(z, ZERO ? -1100.0 : -1020.0);
  constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are rint(z)
  const double t = z + kRound;
  const double f = z - (t - kRound);
  double p = 1.0205905413765595e-07;
  p = __builtin_fma(p, f, 1.325964524488711e-06);
  p = __builtin_fma(p, f, 1.5252672924850737e-05);
  p = __builtin_fma(p, f, 0.0001540343375125101);
  p = __builtin_fma(p, f, 0.0013333558200794592);
  p = __builtin_fma(p, f, 0.009618129193934313);
  p = __builtin_fma(p, f, 0.05550410866465167);
  p = __builtin_fma(p, f, 0.2402265069564034);
  p = __builtin_fma(p, f, 0.6931471805599462);
  p = __builtin_fma(p, f, 1.0000000000000135);
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, t);
  if constexpr (ZERO) return __builtin_ldexp(p, (int)k);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  return __builtin_bit_cast(double, (uint64_t)((uint32_t)(bits >> 32) + (k << 20)) << 32 |
                                        (uint32_t)bits);
}
// exp((x - m) / T) with the scale log2(e) / T, 1 at the maximum itself (also where
// that is infinite)
__device__ __forceinline__ double weight(float x, float m, double scale) {
  const double e = exp2_f64<true>(((double)x - (double)m) * scale);
  return x == m ? 1.0 : e;
}
// log2(e) / T, above 0 also for an infinite T (a product with -inf stays -inf)
__device__ __forceinline__ double weight_scale(float t) {
  return fmax(1.4426950408889634 / (double)t, 1e-300);
}

// G groups of VE = 4 or 8 logits (16 bytes each), group i from place v + i step on,
// -inf from V on; `whole`, for the workgroup: none reaches V. All loads go out
// before the first is waited for. Rows have any alignment.
template <int DT, int G, int VE>
__device__ __forceinline__ void logits16(const void* row, int v, int step, int V, bool whole,
                                         float (&x)[G][VE]) {
  static_assert(VE == (DT == PE_DTYPE_F32 ? 4 : 8), "16 bytes");
  if (whole) {
    u32x4v u[G];
#pragma unroll
    for (int i = 0; i < G; ++i)
      __builtin_memcpy(&u[i], reinterpret_cast<const char*>(row) + (int64_t)(v + i * step) * (16 / VE), 16);
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const uint32_t w = u[i][VE == 4 ? j : j / 2];
        if constexpr (DT == PE_DTYPE_F32) x[i][j] = __builtin_bit_cast(float, w);
        else x[i][j] = f16or_bf((uint16_t)(w >> (16 * (j & 1))), DT == PE_DTYPE_BF16);
        x[i][j] = fmaxf(x[i][j], -__builtin_inff());
      }
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const int at = v + i * step + j;
        x[i][j] = logit<DT>(row, min(at, V - 1));
        if (at >= V) x[i][j] = -__builtin_inff();
      }
  }
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// lane moves of 64-bit values as two of 32 (DPP control word CTRL; lanes without a
// source get 0)
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// running sum over the 64 lanes: row_shr 1, 2, 4, 8 within 16 lanes, then the rows
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {
  v += dpp_f64<0x111>(v);
  v += dpp_f64<0x112>(v);
  v += dpp_f64<0x114>(v);
  v += dpp_f64<0x118>(v);
  const double r0 = lane_f64(v, 15), r1 = r0 + lane_f64(v, 31), r2 = r1 + lane_f64(v, 47);
  const int row = lane >> 4;
  return v + (row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}
// sum over the 64 lanes, in every lane
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<0x111>(v);
  v += dpp_f64<0x112>(v);
  v += dpp_f64<0x114>(v);
  v += dpp_f64<0x118>(v);
  return (lane_f64(v, 15) + lane_f64(v, 31)) + (lane_f64(v, 47) + lane_f64(v, 63));
}

// sums of two pieces of a row: (max, first, sum) each, sums relative to their maxima
__device__ __forceinline__ void join_stats(float& m, int& first, double& s, float om, int of,
                                           double os, double scale) {
  const float mn = fmaxf(m, om);
  first = om > m ? of : om == m ? min(first, of) : first;
  s = (s > 0.0 ? s * weight(m, mn, scale) : 0.0) + (os > 0.0 ? os * weight(om, mn, scale) : 0.0);
  m = mn;
}

template <int DT>
__global__ __launch_bounds__(256) void verify_stats_kernel(const VerifyArgs a) {
  __shared__ RowStat ws[4];
  const int64_t row = blockIdx.x / a.nc;
  const int piece = (int)(blockIdx.x - row * a.nc);
  const int64_t b = row / a.n;
  const int node = (int)(row - b * a.n);
  const int64_t* tok = a.tokens + b * a.n;
  // rows of absent drafts and of empty sequences are not looked at
  if (tok[node] < 0 || tok[node] >= a.V || tok[0] < 0 || tok[0] >= a.V) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* base = reinterpret_cast<const char*>(a.logits) +
                     (b * a.l_b + node * a.l_n) * (DT == PE_DTYPE_F32 ? 4 : 2);
  const int v0 = piece * kStatChunk;
  const float t = a.temps ? a.temps[b] : a.temp;
  constexpr int VE = DT == PE_DTYPE_F32 ? 4 : 8;
  constexpr int G = kStatChunk / 256 / VE;  // loads of 16 bytes
  float x[G][VE];
  logits16<DT>(base, v0 + tid * VE, 256 * VE, a.V, v0 + kStatChunk <= a.V, x);
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) m = fmaxf(m, x[i][j]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  // sums relative to the wave's own maximum, so that no wave waits for another
  double s = 0.0, scale = 0.0;
  int first = a.V;
  if (t > 0.f) {
    scale = weight_scale(t);
    if (__builtin_expect(m == __builtin_inff(), 0)) {  // those share the distribution
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j) s += x[i][j] == m ? 1.0 : 0.0;
    } else if (m != -__builtin_inff()) {
      // The difference before the scale, as weight() has it: x scale - m scale would keep
      // an error of 2^-53 m scale, which at a temperature of 1e-16 is several powers of two
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j)
          s += exp2_f64<false>(((double)x[i][j] - (double)m) * scale);
    }
    s = wave_sum_f64(s);
  } else {
#pragma unroll
    for (int i = G - 1; i >= 0; --i)
#pragma unroll
      for (int j = VE - 1; j >= 0; --j) {
        const int v = v0 + (i * 256 + tid) * VE + j;
        if (x[i][j] == m && v < a.V) first = v;
      }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) first = min(first, __shfl_xor(first, off, 64));
  }
  if (lane == 0) ws[wave] = RowStat{m, first, s};
  __syncthreads();
  if (wave > 0) return;
  RowStat r = ws[lane & 3];
#pragma unroll
  for (int off = 1; off < 4; off <<= 1)
    join_stats(r.max, r.first, r.sum, __shfl_xor(r.max, off, 64), __shfl_xor(r.first, off, 64),
               __shfl_xor(r.sum, off, 64), scale);
  if (lane == 0) a.stats[blockIdx.x] = r;
}

__device__ __forceinline__ void st_dev64(double* p, double v) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double ld_dev64(const double* p) {
  return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p),
                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <int DT>
__global__ __launch_bounds__(256) void verify_walk_kernel(const VerifyArgs a) {
  __shared__ float rmax[kTreeMax];
  __shared__ int rfirst[kTreeMax];
  __shared__ double rsum[kTreeMax];
  __shared__ int order[kTreeMax];
  const int tid = threadIdx.x;
  const int n = a.n, V = a.V;
  const int64_t b = blockIdx.x;
  const int64_t* tok = a.tokens + b * n;
  int64_t *out = a.out + b * n, *path = a.path + b * n;
  if (tid == 0) a.done[b] = 0;
  const int64_t root = tok[0];
  if (root < 0 || root >= V) {  // an empty slot of the batch
    if (tid < n) out[tid] = path[tid] = -1;
    if (tid == 0) {
      a.count[b] = 0;
      a.ends[b].done = 1;
    }
    return;
  }
  const float t = a.temps ? a.temps[b] : a.temp;
  const bool greedy = !(t > 0.f);
  const double scale = greedy ? 0.0 : weight_scale(t);

  // the rows' maxima and sums, from their pieces: a few lanes a row
  const int tpr = n > 32 ? 4 : n > 16 ? 8 : 16;
  {
    const int r = tid / tpr, c0 = tid & (tpr - 1);
    const bool there = r < n && tok[r] >= 0 && tok[r] < V;
    float m = -__builtin_inff();
    int first = V;
    double s = 0.0;
    if (there) {
      const RowStat* st = a.stats + (b * n + r) * a.nc;
      constexpr int kBatch = 8;  // pieces on their way at once
      for (int c = c0; c < a.nc; c += kBatch * tpr) {
        RowStat p[kBatch];
        float mn = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          p[k] = RowStat{-__builtin_inff(), V, 0.0};
          if (c + k * tpr < a.nc) p[k] = st[c + k * tpr];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (p[k].max > mn || (p[k].max == mn && p[k].first < first)) first = p[k].first;
          mn = fmaxf(mn, p[k].max);
        }
        if (!greedy && mn != -__builtin_inff()) {
          s = s > 0.0 ? s * weight(m, mn, scale) : 0.0;
#pragma unroll
          for (int k = 0; k < kBatch; ++k)
            if (p[k].sum > 0.0) s += p[k].sum * weight(p[k].max, mn, scale);
        }
        m = mn;
      }
    }
    for (int off = 1; off < tpr; off <<= 1)
      join_stats(m, first, s, __shfl_xor(m, off, 64), __shfl_xor(first, off, 64),
                 __shfl_xor(s, off, 64), scale);
    if (r < n && c0 == 0) {
      rmax[r] = m;
      rfirst[r] = first;
      rsum[r] = s;
    }
  }
  __syncthreads();
  if (tid >= 64) return;

  // the walk: lane = node
  const int i = tid;
  const int64_t x = i < n ? tok[i] : -1;
  int64_t par = -1;
  if (i > 0 && i < n && x >= 0 && x < V) par = a.parents ? a.parents[b * a.p_b + i] : i - 1;
  const uint64_t mask = tree_mask(par, i, n);
  const bool there = i > 0 && mask != 0;
  const int p = there ? (int)par : 0;
  const char* lrow = reinterpret_cast<const char*>(a.logits) +
                     (b * a.l_b + p * a.l_n) * (DT == PE_DTYPE_F32 ? 4 : 2);
  double px = 0.0, qx = 1.0, u = 0.0;
  if (there) {
    const float m = rmax[p];
    const float lx = logit<DT>(lrow, x);
    u = a.uniforms[b * n + i];
    if (a.probs) {
      const float q = a.probs[b * a.q_b + p * a.q_n + x];
      qx = q > 0.f && q < __builtin_inff() ? q : 0.0;
    }
    if (greedy) px = x == rfirst[p] && m != -__builtin_inff() ? 1.0 : 0.0;
    else if (m != -__builtin_inff()) px = weight(lx, m, scale) / rsum[p];
  }
  bool blocked = false, ok = there && u * qx < px;
  double rem = 1.0;
  if (a.parents) {  // in order of the nodes: what a rejection leaves to later siblings
    for (uint64_t todo = __ballot(there); todo; todo &= todo - 1) {
      const int j = __builtin_ctzll(todo);
      const bool after = there && i > j && p == __builtin_amdgcn_readlane(p, j);
      if (!__ballot(after)) continue;
      const int jx = __builtin_amdgcn_readlane((int)x, j);
      const double jq = lane_f64(px, j);
      const bool jok = __builtin_amdgcn_readlane((int)ok, j);
      if (after) {
        blocked |= jok;
        rem -= jq;
        if ((int)x == jx) px = 0.0;  // rejected once: nothing is left of it
        ok = u * rem < px;
      }
    }
  }
  const uint64_t taken = __ballot(i == 0 || (ok && !blocked));
  const uint64_t on = __ballot(i < n && mask != 0 && !(mask & ~taken));
  const int last = 63 - __builtin_clzll(on);
  const uint64_t children = __ballot(there && p == last);
  const int count = __popcll(on);
  const float m = rmax[last];
  const bool none = m == -__builtin_inff();

  // lane = place on the path
  if (on >> i & 1) order[__popcll(on & ((1ull << i) - 1))] = i;
  __builtin_amdgcn_wave_barrier();
  const int at = i < count ? order[i] : 0;
  const int64_t said = __shfl((long long)x, __shfl(at, (i + 1) & 63, 64), 64);
  if (i < n) {
    path[i] = i < count ? at : -1;
    out[i] = i < count - 1 ? said : i == count - 1 && !none && greedy ? rfirst[last] : -1;
  }
  if (i == 0) {
    a.count[b] = count;
    a.ends[b] = WalkEnd{last, count, m, greedy || none, rsum[last], children};
  }
}

// The next token. A workgroup sums the weights that are left of a piece, and the row's own
// (for where nothing is left), E consecutive tokens a thread; the last one to finish finds
// the piece that holds the token and goes through it once more.
template <int DT>
__global__ __launch_bounds__(256) void verify_pick_kernel(const VerifyArgs a) {
  __shared__ uint32_t gone[kPickChunk / 32];  // the piece's tokens that were rejected
  __shared__ double part[2][4];
  __shared__ int s_piece, s_found;
  __shared__ double s_target;
  __shared__ bool s_last, s_own;
  constexpr int E = kPickChunk / 256;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int V = a.V;
  const int64_t b = blockIdx.y;
  const WalkEnd end = a.ends[b];
  if (end.done) return;
  const double scale = weight_scale(a.temps ? a.temps[b] : a.temp);
  const char* row = reinterpret_cast<const char*>(a.logits) +
                    (b * a.l_b + end.node * a.l_n) * (DT == PE_DTYPE_F32 ? 4 : 2);
  const bool residual = a.probs && end.children;
  const float* q = residual ? a.probs + b * a.q_b + end.node * a.q_n : nullptr;
  double* sums = a.sums + b * a.np * 2;

  int piece = blockIdx.x;
  for (bool find = false;; find = true) {
    const int v0 = piece * kPickChunk + tid * E;
    constexpr int VE = DT == PE_DTYPE_F32 ? 4 : 8;
    const bool whole = (piece + 1) * kPickChunk <= V;
    float x[E / VE][VE], qv[E / 4][4] = {};
    if (residual) logits16<PE_DTYPE_F32>(q, v0, 4, V, whole, qv);
    logits16<DT>(row, v0, VE, V, whole, x);
    if (!residual) {
      for (int i = tid; i < kPickChunk / 32; i += 256) gone[i] = 0;
      __syncthreads();
      if (tid < a.n && (end.children >> tid & 1)) {
        const int64_t t = a.tokens[b * a.n + tid];
        if (t / kPickChunk == piece) atomicOr(&gone[t % kPickChunk / 32], 1u << (t & 31));
      }
      __syncthreads();
    }
    double w[E], own[E], s0 = 0.0, s1 = 0.0;
    const uint32_t lost = residual ? 0 : gone[tid * E / 32] >> (tid * E & 31);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      own[k] = v0 + k < V ? weight(x[k / VE][k % VE], end.max, scale) : 0.0;
      w[k] = own[k];
      if (residual) {
        const float qk = qv[k / 4][k % 4];
        const double qd = qk > 0.f && qk < __builtin_inff() ? (double)qk : 0.0;
        w[k] = fmax(__builtin_fma(-qd, end.sum, own[k]), 0.0);
      } else if (lost >> k & 1) {
        w[k] = 0.0;
      }
      s0 += w[k];
      s1 += own[k];
    }
    if (find) {
      // running sums over the workgroup: the first token that passes the target
      const bool use_own = s_own;
      const double mine = use_own ? s1 : s0;
      const double scan = wave_scan_f64(mine, lane);
      if (lane == 63) part[0][wave] = scan;
      __syncthreads();
      double run = 0.0;
      for (int k = 0; k < wave; ++k) run += part[0][k];
      run += scan - mine;
      int hit = V, any = -1;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const double wk = use_own ? own[k] : w[k];
        if (wk > 0.0) {
          any = v0 + k;
          run += wk;
          if (hit == V && run > s_target) hit = any;
        }
      }
      if (hit < V) atomicMin(&s_found, hit);
      __syncthreads();
      int found = s_found;
      if (found == V) {  // rounding left the target behind the last weight
        __syncthreads();
        if (tid == 0) s_found = -1;
        __syncthreads();
        if (any >= 0) atomicMax(&s_found, any);
        __syncthreads();
        found = s_found;
      }
      if (tid == 0) a.out[b * a.n + end.count - 1] = found;
      return;
    }
    s0 = wave_sum_f64(s0);
    s1 = wave_sum_f64(s1);
    if (lane == 0) {
      part[0][wave] = s0;
      part[1][wave] = s1;
    }
    __syncthreads();
    if (tid == 0) {
      st_dev64(sums + 2 * piece, (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]));
      st_dev64(sums + 2 * piece + 1, (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]));
      __builtin_amdgcn_s_waitcnt(0);
      s_last = atomicAdd(&a.done[b], 1u) + 1 == (uint32_t)a.np;
    }
    __syncthreads();
    if (!s_last) return;

    // the piece: the first whose running sum passes u_0 of the total
    if (wave == 0) {
      double total = 0.0;
      int use = 0;
      for (;; use = 1) {
        total = 0.0;
        for (int c = lane; c < a.np; c += 64) total += ld_dev64(sums + 2 * c + use);
        total = wave_sum_f64(total);
        if (use == 1 || total > 0.0) break;  // nothing is left: the target's own distribution
      }
      const double target = fmin(fmax((double)a.uniforms[b * a.n], 0.0), 1.0) * total;
      double run = 0.0, before = 0.0;
      int found = 0;  // without a hit the last piece that has weight
      for (int c0 = 0; c0 < a.np; c0 += 64) {
        const double s = c0 + lane < a.np ? ld_dev64(sums + 2 * (c0 + lane) + use) : 0.0;
        const double scan = wave_scan_f64(s, lane);
        const double excl = run + (scan - s);
        const uint64_t hit = __ballot(s > 0.0 && run + scan > target);
        const uint64_t some = hit ? hit : __ballot(s > 0.0);
        if (some) {
          const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
          found = c0 + l;
          before = lane_f64(excl, l);
        }
        if (hit) break;
        run += lane_f64(scan, 63);
      }
      if (lane == 0) {
        s_piece = found;
        s_target = target - before;
        s_own = use == 1;
        s_found = V;
      }
    }
    __syncthreads();
    piece = s_piece;
  }
}

static int pieces(int64_t V, int chunk) { return (int)((V + chunk - 1) / chunk); }

static bool verify_shape_ok(int64_t batch, int n, int64_t vocab) {
  return batch >= 1 && batch <= 65535 && n >= 1 && n <= kTreeMax && vocab >= 1 &&
         vocab <= (int64_t)1 << 24 &&
         batch * n * pieces(vocab, kStatChunk) <= kTreeMaxGrid;
}

static size_t stats_bytes(int64_t batch, int n, int64_t vocab) {
  return (size_t)batch * n * pieces(vocab, kStatChunk) * sizeof(RowStat);
}
static size_t sums_bytes(int64_t batch, int64_t vocab) {
  return (size_t)batch * pieces(vocab, kPickChunk) * 16;
}
static size_t ends_bytes(int64_t batch) { return round_up((size_t)batch * sizeof(WalkEnd), 16); }

template <int DT>
static int launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t st) {
  verify_stats_kernel<DT><<<(unsigned)(batch * a.n * a.nc), 256, 0, st>>>(a);
  int rc = launch_status();
  if (rc != PE_OK) return rc;
  verify_walk_kernel<DT><<<(unsigned)batch, 256, 0, st>>>(a);
  rc = launch_status();
  if (rc != PE_OK) return rc;
  verify_pick_kernel<DT><<<dim3((unsigned)a.np, (unsigned)batch), 256, 0, st>>>(a);
  return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_verify_drafts_workspace_size(int64_t batch, int n, int64_t vocab) {
  if (!verify_shape_ok(batch, n, vocab)) return 0;
  return stats_bytes(batch, n, vocab) + sums_bytes(batch, vocab) + ends_bytes(batch) +
         round_up((size_t)batch * 4, 16);
}

extern "C" int pe_verify_drafts(const void* logits, int dtype, int64_t l_b, int64_t l_n,
                                int64_t batch, int n, int64_t vocab, const int64_t* tokens,
                                const int64_t* parents, int64_t p_b, const float* uniforms,
                                const float* temps, float temp, const float* probs, int64_t q_b,
                                int64_t q_n, int64_t* out, int64_t* path, int64_t* count,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !tokens || !uniforms || !out || !path || !count) return PE_ERR_NULL;
  if (dtype != PE_DTYPE_F32 && bf16_flag(dtype) < 0) return PE_ERR_DTYPE;
  if (batch == 0) return PE_OK;
  if (!verify_shape_ok(batch, n, vocab) || l_b < 0 || l_n < 0 || p_b < 0 || q_b < 0 || q_n < 0 ||
      (parents && probs))
    return PE_ERR_DIMS;
  if (!workspace || workspace_bytes < pe_verify_drafts_workspace_size(batch, n, vocab))
    return PE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return PE_ERR_ALIGN;
  char* ws = reinterpret_cast<char*>(workspace);
  char* sums = ws + stats_bytes(batch, n, vocab);
  char* ends = sums + sums_bytes(batch, vocab);
  VerifyArgs a{logits, l_b, l_n, tokens, parents, p_b, uniforms, temps, temp, probs, q_b, q_n,
               out, path, count, n, (int)vocab, pieces(vocab, kStatChunk),
               pieces(vocab, kPickChunk), reinterpret_cast<RowStat*>(ws),
               reinterpret_cast<double*>(sums), reinterpret_cast<WalkEnd*>(ends),
               reinterpret_cast<uint32_t*>(ends + ends_bytes(batch))};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PE_DTYPE_F32) return launch_verify<PE_DTYPE_F32>(a, batch, st);
  if (dtype == PE_DTYPE_BF16) return launch_verify<PE_DTYPE_BF16>(a, batch, st);
  return launch_verify<PE_DTYPE_F16>(a, batch, st);
}
