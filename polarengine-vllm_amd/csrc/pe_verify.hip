// Verification of drafted tokens: which nodes of a chain or tree of drafts stand
// against the target's distribution, from given uniform numbers, and the token
// that follows them. Rejection sampling: with every number uniform the tokens
// are distributed as the target's own.
//
// Everything that decides is in 64 bits: the answers are whole numbers, and over
// a vocabulary of 150,000 an error of 1e-7 in a cumulative sum moves about one
// sampled token in a hundred.
//
// Two launches. The first reads every logit once, 8192 of a row per workgroup, and
// leaves each piece's maximum, its place and its sum of exp((x - max) / T). In the
// second every workgroup of a sequence walks the tree for itself (64 nodes: one
// wave, lane = node; 19 KB of sums from L2), then sums the weights of 2048 tokens
// of the node that the walk ends in; the last one to finish finds the piece and
// the token in it. The counters of that hand-over are cleared by the first
// launch, so the workspace needs no state between calls.

#include "pe_tree.h"

namespace pe {

constexpr int kStatChunk = 8192;
constexpr int kPickChunk = 2048;

struct RowStat {
  float max;
  int first;  // lowest place of the maximum
  double sum;
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
// interpolation of degree 9 at the Chebyshev nodes of [-1/2, 1/2]. About 18 64-bit
// instructions; at the rate of 64-bit fma a card passes 2.1e12 values a second, what
// it reads of 32-bit logits in the same time.
__device__ __forceinline__ double exp2_f64(double z) {
  z = fmax(z, -1100.0);  // 0, also for -inf and NaN
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
  return __builtin_ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, t));
}
// exp((x - m) / T) with the scale log2(e) / T, 1 at the maximum itself (also where
// that is infinite)
__device__ __forceinline__ double weight(float x, float m, double scale) {
  const double e = exp2_f64(((double)x - (double)m) * scale);
  return x == m ? 1.0 : e;
}
// log2(e) / T, above 0 also for an infinite T (a product with -inf stays -inf)
__device__ __forceinline__ double weight_scale(float t) {
  return fmax(1.4426950408889634 / (double)t, 1e-300);
}

// VE consecutive logits (16 bytes) from place v on, -inf from V on
template <int DT>
__device__ __forceinline__ void logits16(const void* row, int v, int V,
                                         float (&x)[DT == PE_DTYPE_F32 ? 4 : 8]) {
  constexpr int VE = DT == PE_DTYPE_F32 ? 4 : 8;
  if (v + VE <= V) {  // rows have any alignment
    u32x4v u;
    __builtin_memcpy(&u, reinterpret_cast<const char*>(row) + (int64_t)v * (16 / VE), 16);
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const uint32_t w = u[VE == 4 ? j : j / 2];
      if constexpr (DT == PE_DTYPE_F32) x[j] = __builtin_bit_cast(float, w);
      else x[j] = f16or_bf((uint16_t)(w >> (16 * (j & 1))), DT == PE_DTYPE_BF16);
      x[j] = fmaxf(x[j], -__builtin_inff());
    }
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      x[j] = v + j < V ? logit<DT>(row, v + j) : -__builtin_inff();
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
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
  if (piece == 0 && node == 0 && threadIdx.x == 0) a.done[b] = 0;
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
#pragma unroll
  for (int i = 0; i < G; ++i) logits16<DT>(base, v0 + (i * 256 + tid) * VE, a.V, x[i]);
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
    if (m != -__builtin_inff()) {
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j) s += weight(x[i][j], m, scale);
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
__global__ __launch_bounds__(256) void verify_pick_kernel(const VerifyArgs a) {
  __shared__ float rmax[kTreeMax];
  __shared__ int rfirst[kTreeMax];
  __shared__ double rsum[kTreeMax];
  __shared__ uint32_t gone[kPickChunk / 32];  // this piece's tokens that were rejected
  __shared__ double part[2][4];
  __shared__ int s_piece, s_found;
  __shared__ double s_before;
  __shared__ bool s_last, s_alt;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.n, V = a.V;
  const int64_t b = blockIdx.y;
  const int64_t* tok = a.tokens + b * n;
  int64_t *out = a.out + b * n, *path = a.path + b * n;
  const int64_t root = tok[0];
  if (root < 0 || root >= V) {  // an empty slot of the batch
    if (blockIdx.x == 0) {
      if (tid < n) out[tid] = path[tid] = -1;
      if (tid == 0) a.count[b] = 0;
    }
    return;
  }
  const float t = a.temps ? a.temps[b] : a.temp;
  const bool greedy = !(t > 0.f);
  if (greedy && blockIdx.x > 0) return;
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
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (c + k * tpr < a.nc) p[k] = st[c + k * tpr];
          else p[k] = RowStat{-__builtin_inff(), V, 0.0};
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (c + k * tpr < a.nc) join_stats(m, first, s, p[k].max, p[k].first, p[k].sum, scale);
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
  for (int i = tid; i < kPickChunk / 32; i += 256) gone[i] = 0;
  __syncthreads();

  // the walk: lane = node
  const int i = lane;
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
    if (greedy) px = x == rfirst[p] && m != -__builtin_inff() ? 1.0 : 0.0;
    else if (m != -__builtin_inff()) px = weight(logit<DT>(lrow, x), m, scale) / rsum[p];
    u = a.uniforms[b * n + i];
    if (a.probs) {
      const float q = a.probs[b * a.q_b + p * a.q_n + x];
      qx = q > 0.f && q < __builtin_inff() ? q : 0.0;
    }
  }
  bool blocked = false, ok = false;
  double rem = 1.0;
  for (int j = 1; j < n; ++j) {
    if (i == j) ok = there && (a.probs ? u * qx : u * rem) < px;
    const bool jt = __builtin_amdgcn_readlane((int)there, j);
    if (!jt) continue;
    const int jp = __builtin_amdgcn_readlane(p, j);
    const int jx = __builtin_amdgcn_readlane((int)x, j);
    const double jq = lane_f64(px, j);
    const bool jok = __builtin_amdgcn_readlane((int)ok, j);
    if (there && i > j && p == jp) {
      blocked |= jok;
      if (!a.probs) {
        rem -= jq;
        if ((int)x == jx) px = 0.0;  // rejected once: nothing is left of it
      }
    }
  }
  const uint64_t taken = __ballot(i == 0 || (ok && !blocked));
  const uint64_t on = __ballot(i < n && mask != 0 && !(mask & ~taken));
  const int last = 63 - __builtin_clzll(on);
  const bool child = there && p == last;
  const bool any_child = __ballot(child) != 0;
  const int count = __popcll(on);

  auto finish = [&](int64_t token) {  // wave 0 of one workgroup; lane = place on the path
    int at = 0;
    for (int j = 0; j < n; ++j)
      if ((on >> j & 1) && __popcll(on & ((1ull << j) - 1)) == i) at = j;
    const int64_t said = __shfl((long long)x, __shfl(at, (i + 1) & 63, 64), 64);
    if (i < n) {
      path[i] = i < count ? at : -1;
      out[i] = i < count - 1 ? said : i == count - 1 ? token : -1;
    }
    if (i == 0) a.count[b] = count;
  };
  const float m = rmax[last];
  if (greedy || m == -__builtin_inff()) {
    if (blockIdx.x == 0 && wave == 0) finish(m == -__builtin_inff() ? -1 : rfirst[last]);
    return;
  }
  const double total_e = rsum[last];

  // weights of this workgroup's piece
  const char* row = reinterpret_cast<const char*>(a.logits) +
                    (b * a.l_b + last * a.l_n) * (DT == PE_DTYPE_F32 ? 4 : 2);
  const bool residual = a.probs && any_child;
  const float* q = a.probs + (a.probs ? b * a.q_b + last * a.q_n : 0);
  constexpr int E = kPickChunk / 256;
  auto mark = [&](int piece) {  // rejected tokens of the piece (drafts without probabilities)
    if (!a.probs && wave == 0 && child && x / kPickChunk == piece)
      atomicOr(&gone[(x % kPickChunk) / 32], 1u << (x & 31));
  };
  // what is left of tokens v .. v + 7, times the row's sum, and the row's own weights
  auto weights = [&](int v, double (&w)[E], double (&own)[E]) {
    float x[E], qv[E];
    constexpr int VE = DT == PE_DTYPE_F32 ? 4 : 8;
#pragma unroll
    for (int g = 0; g < E; g += VE) {
      float y[VE];
      logits16<DT>(row, v + g, V, y);
#pragma unroll
      for (int j = 0; j < VE; ++j) x[g + j] = y[j];
    }
    if (residual) {
#pragma unroll
      for (int g = 0; g < E; g += 4) {
        float y[4];
        logits16<PE_DTYPE_F32>(q, v + g, V, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) qv[g + j] = y[j];
      }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      own[j] = v + j < V ? weight(x[j], m, scale) : 0.0;
      w[j] = own[j];
      if (residual)
        w[j] = fmax(__builtin_fma(-(qv[j] > 0.f && qv[j] < __builtin_inff() ? (double)qv[j] : 0.0),
                                  total_e, own[j]), 0.0);
      else if (gone[((v + j) % kPickChunk) / 32] >> ((v + j) & 31) & 1)
        w[j] = 0.0;
    }
  };
  mark(blockIdx.x);
  __syncthreads();
  double s0 = 0.0, s1 = 0.0;
  {
    double w[E], own[E];
    weights((int)blockIdx.x * kPickChunk + tid * E, w, own);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      s0 += w[k];
      s1 += own[k];
    }
  }
  s0 = wave_sum_f64(s0);
  s1 = wave_sum_f64(s1);
  if (lane == 0) {
    part[0][wave] = s0;
    part[1][wave] = s1;
  }
  __syncthreads();
  if (tid == 0) {
    double* sum = a.sums + (b * a.np + blockIdx.x) * 2;
    st_dev64(sum, (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]));
    st_dev64(sum + 1, (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]));
    __builtin_amdgcn_s_waitcnt(0);
    s_last = atomicAdd(&a.done[b], 1u) + 1 == (uint32_t)a.np;
  }
  __syncthreads();
  if (!s_last) return;

  // the piece: the first whose running sum passes u_0 of the total
  const double* sums = a.sums + b * a.np * 2;
  if (wave == 0) {
    double total[2] = {0.0, 0.0};
    for (int c = lane; c < a.np; c += 64) {
      total[0] += ld_dev64(sums + 2 * c);
      total[1] += ld_dev64(sums + 2 * c + 1);
    }
    total[0] = wave_sum_f64(total[0]);
    total[1] = wave_sum_f64(total[1]);
    const int alt = total[0] > 0.0 ? 0 : 1;  // nothing is left: the target's own distribution
    const double target = fmin(fmax((double)a.uniforms[b * n], 0.0), 1.0) * total[alt];
    double run = 0.0, before = 0.0;
    int found = 0;  // without a hit the last piece that has weight
    for (int c0 = 0; c0 < a.np; c0 += 64) {
      const double s = c0 + lane < a.np ? ld_dev64(sums + 2 * (c0 + lane) + alt) : 0.0;
      double scan = s;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(scan, off, 64);
        if (lane >= off) scan += o;
      }
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
      s_before = target - before;
      s_alt = alt != 0;
      s_found = V;
    }
  }
  for (int k = tid; k < kPickChunk / 32; k += 256) gone[k] = 0;
  __syncthreads();
  const int piece = s_piece;
  mark(piece);
  __syncthreads();
  // each thread takes consecutive tokens; running sums over the workgroup
  double w[E], own[E], mine = 0.0;
  weights(piece * kPickChunk + tid * E, w, own);
#pragma unroll
  for (int k = 0; k < E; ++k) {
    if (s_alt) w[k] = own[k];
    mine += w[k];
  }
  double scan = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o = __shfl_up(scan, off, 64);
    if (lane >= off) scan += o;
  }
  if (lane == 63) part[0][wave] = scan;
  __syncthreads();
  double run = 0.0;
  for (int k = 0; k < wave; ++k) run += part[0][k];
  run += scan - mine;
  int hit = V, any = -1;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    if (w[k] > 0.0) {
      any = piece * kPickChunk + tid * E + k;
      run += w[k];
      if (hit == V && run > s_before) hit = any;
    }
  }
  if (hit < V) atomicMin(&s_found, hit);
  __syncthreads();
  if (s_found == V) {  // rounding left the target behind the last weight
    __syncthreads();
    if (tid == 0) s_found = -1;
    __syncthreads();
    if (any >= 0) atomicMax(&s_found, any);
    __syncthreads();
  }
  if (wave == 0) finish(s_found);
}

static int pieces(int64_t V, int chunk) { return (int)((V + chunk - 1) / chunk); }

static bool verify_shape_ok(int64_t batch, int n, int64_t vocab) {
  return batch >= 1 && batch <= 65535 && n >= 1 && n <= kTreeMax && vocab >= 1 &&
         vocab <= (int64_t)1 << 24 &&
         batch * n * pieces(vocab, kStatChunk) <= INT32_MAX;
}

static size_t stats_bytes(int64_t batch, int n, int64_t vocab) {
  return (size_t)batch * n * pieces(vocab, kStatChunk) * sizeof(RowStat);
}
static size_t sums_bytes(int64_t batch, int64_t vocab) {
  return (size_t)batch * pieces(vocab, kPickChunk) * 16;
}

template <int DT>
static int launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t st) {
  verify_stats_kernel<DT><<<(unsigned)(batch * a.n * a.nc), 256, 0, st>>>(a);
  const int rc = launch_status();
  if (rc != PE_OK) return rc;
  verify_pick_kernel<DT><<<dim3((unsigned)a.np, (unsigned)batch), 256, 0, st>>>(a);
  return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_verify_drafts_workspace_size(int64_t batch, int n, int64_t vocab) {
  if (!verify_shape_ok(batch, n, vocab)) return 0;
  return stats_bytes(batch, n, vocab) + sums_bytes(batch, vocab) + round_up((size_t)batch * 4, 16);
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
  VerifyArgs a{logits, l_b, l_n, tokens, parents, p_b, uniforms, temps, temp, probs, q_b, q_n,
               out, path, count, n, (int)vocab, pieces(vocab, kStatChunk),
               pieces(vocab, kPickChunk), reinterpret_cast<RowStat*>(ws),
               reinterpret_cast<double*>(ws + stats_bytes(batch, n, vocab)),
               reinterpret_cast<uint32_t*>(ws + stats_bytes(batch, n, vocab) +
                                           sums_bytes(batch, vocab))};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PE_DTYPE_F32) return launch_verify<PE_DTYPE_F32>(a, batch, st);
  if (dtype == PE_DTYPE_BF16) return launch_verify<PE_DTYPE_BF16>(a, batch, st);
  return launch_verify<PE_DTYPE_F16>(a, batch, st);
}
