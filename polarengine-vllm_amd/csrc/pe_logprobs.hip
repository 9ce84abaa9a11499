// Log probabilities of given tokens, their ranks, the entropy and the likeliest
// alternatives, in one pass over the logits:
//
//   lse = m + log z, z = sum e^(x - m), entropy = log z - (sum (x - m) e^(x - m)) / z
//
// Bound by reading the logits; a row is cut into pieces, a workgroup each, where there
// are few rows, and a second launch joins them. A wave reads chunks of eight values a
// lane, the next one's loads under way. A lane's sums are relative to its own maximum,
// eight values at a time in fp32 and those in 64 bits, so that a row of 200,000 tokens
// is no less exact than one of a thousand. Ranks are counted by ballots. The wave's
// likeliest tokens so far lie sorted across its lanes; a chunk is looked through only
// if one of its values passes the last of them, which is rare behind the first chunks.
//
// 2048 rows of 151,936 fp32: 227 us, 5.5 TB/s (bf16: 151 us, 4.1 TB/s, about twelve
// vector instructions a value, one of them for signalling NaN, 2% of either); one row
// with 20 alternatives 8 us and 6 us for the join, 7.4 us without alternatives; 48 rows of
// 100,003 bf16 with 5: 15 + 5 us, of which the read would be 2.

#include "pe_internal.h"

namespace pe {

constexpr int kTopMax = 64;        // a lane each
constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr float kLpLog2e = 1.4426950408889634f;

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  int rows, vocab, top;
  float* logprob;
  int64_t* rank;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  int pieces;    // of a row
  int granules;  // of 16 bytes of a piece, a multiple of a chunk's
  char* parts;   // [rows][pieces]: LpSums, then [rows][pieces][top]: LpKey
};
struct LpSums {
  double z, e;
  float m;
  int rank;
};

template <int DT>
__device__ __forceinline__ float lp_logit(const void* p, int64_t i) {
  if constexpr (DT == PE_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  else return f16or_bf(reinterpret_cast<const uint16_t*>(p)[i], DT == PE_DTYPE_BF16);
}

// A NaN logit is one of -inf: the token is ruled out.
__device__ __forceinline__ float lp_ruled(float x) { return x != x ? -__builtin_inff() : x; }

// A token as one number: the larger the logit the larger, of equal logits the lower
// token; 0: none.
typedef uint64_t LpKey;
__device__ __forceinline__ LpKey lp_key(float x, int i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 is 0
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)o << 32 | ~(uint32_t)i;
}
__device__ __forceinline__ float lp_value(LpKey k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return k ? __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o) : -__builtin_inff();
}
__device__ __forceinline__ int lp_token(LpKey k) { return k ? (int)~(uint32_t)k : -1; }

template <int M>
__device__ __forceinline__ uint32_t lp_xor32(uint32_t v, int lane) {
  if constexpr (M <= 8) {
    return __builtin_bit_cast(uint32_t, lane_xor<M>(__builtin_bit_cast(float, v)));
  } else if constexpr (M == 16) {
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return lane & 16 ? r0 : r1;
  } else {
    auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return lane & 32 ? r0 : r1;
  }
}
template <int M>
__device__ __forceinline__ LpKey lp_xor(LpKey k, int lane) {
  return (uint64_t)lp_xor32<M>((uint32_t)(k >> 32), lane) << 32 | lp_xor32<M>((uint32_t)k, lane);
}
// one step of a bitonic network: the larger of lanes l and l ^ M in the one where
// lane & M is not set, unless `up`
template <int M>
__device__ __forceinline__ LpKey lp_step(LpKey k, bool up, int lane) {
  const LpKey o = lp_xor<M>(k, lane);
  const bool low = ((lane & M) == 0) != up;
  return (o > k) == low ? o : k;
}
// a bitonic sequence in order, falling unless `up`
template <int M>
__device__ __forceinline__ LpKey lp_merge(LpKey k, bool up, int lane) {
  k = lp_step<M>(k, up, lane);
  if constexpr (M > 1) k = lp_merge<M / 2>(k, up, lane);
  return k;
}
// rising over the 64 lanes
__device__ __forceinline__ LpKey lp_sort(LpKey k, int lane) {
  k = lp_merge<1>(k, (lane & 2) == 0, lane);
  k = lp_merge<2>(k, (lane & 4) == 0, lane);
  k = lp_merge<4>(k, (lane & 8) == 0, lane);
  k = lp_merge<8>(k, (lane & 16) == 0, lane);
  k = lp_merge<16>(k, (lane & 32) == 0, lane);
  return lp_merge<32>(k, true, lane);
}

// The wave's 64 likeliest tokens, falling over the lanes; `last`, uniform, is the
// top-th of them, which a candidate has to pass.
struct LpList {
  LpKey k, last;
  float last_x;
  __device__ __forceinline__ void begin() {
    k = last = 0;
    last_x = -__builtin_inff();
  }
  __device__ __forceinline__ void set_last(int top) {
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), top - 1);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)k, top - 1);
    last = (uint64_t)hi << 32 | lo;
    last_x = lp_value(last);
  }
  // 64 more, rising over the lanes: the larger of each pair are the 64 likeliest of both
  __device__ __forceinline__ void join(LpKey rising, int lane, int top) {
    k = lp_merge<32>(rising > k ? rising : k, false, lane);
    set_last(top);
  }
  // eight candidates a lane: the best of each lane at a time, as long as some pass
  __device__ __forceinline__ void offer(LpKey (&c)[8], int lane, int top) {
    for (int round = 0; round < 8; ++round) {
      LpKey best = c[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) best = c[j] > best ? c[j] : best;
      uint64_t pass = __ballot(best > last);
      if (!pass) return;
      if (__builtin_popcountll(pass) > 3) {
        join(lp_sort(best > last ? best : 0, lane), lane, top);
      } else {
        while (pass) {  // one by one: the lanes behind its place move by one
          const int l = __builtin_ctzll(pass);
          const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(best >> 32), l);
          const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)best, l);
          const LpKey n = (uint64_t)hi << 32 | lo;
          const LpKey up = __shfl_up((unsigned long long)k, 1, 64);
          k = k > n ? k : lane == 0 || up > n ? n : up;
          pass &= pass - 1;
        }
        set_last(top);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = c[j] == best ? 0 : c[j];
    }
  }
};

// The lists of a workgroup's waves, in the first wave's.
__device__ __forceinline__ void lp_join_lists(LpList& list, LpKey (*shared)[64], int lane, int wave, int top) {
  shared[wave][lane] = list.k;
  __syncthreads();
  if (wave == 0)
    for (int w = 1; w < kLpWaves; ++w) list.join(shared[w][63 - lane], lane, top);
}

// A workgroup's sums, in every thread.
__device__ __forceinline__ LpSums lp_join(LpSums s, LpSums* shared, int lane, int wave) {
  float m = s.m;
#pragma unroll
  for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  auto onto = [](LpSums v, float to) {  // relative to `to`
    const float d = v.m - to;
    const double f = v.z > 0 ? (double)__builtin_amdgcn_exp2f(d * kLpLog2e) : 0.0;
    v.e = f > 0 ? f * (v.e + d * v.z) : 0.0;  // d may be -inf, also of finite logits
    v.z *= f;
    v.m = to;
    return v;
  };
  s = onto(s, m);
#pragma unroll
  for (int k = 32; k; k >>= 1) {
    s.z += __shfl_xor(s.z, k, 64);
    s.e += __shfl_xor(s.e, k, 64);
    s.rank += __shfl_xor(s.rank, k, 64);
  }
  if (lane == 0) shared[wave] = s;
  __syncthreads();
  for (int w = 0; w < kLpWaves; ++w) m = fmaxf(m, shared[w].m);
  LpSums t{0, 0, m, 0};
  for (int w = 0; w < kLpWaves; ++w) {
    const LpSums o = onto(shared[w], m);
    t.z += o.z;
    t.e += o.e;
    t.rank += o.rank;
  }
  return t;
}

// The row's answers, by one wave that holds its list. xt: the token's logit.
template <int DT>
__device__ __forceinline__ void lp_answer(const LogprobArgs& a, int row, const LpSums& s, const LpList& list,
                                          int lane) {
  const double lz = log(s.z);
  if (lane < a.top) {
    a.top_logprobs[(int64_t)row * a.top + lane] = (float)((double)(lp_value(list.k) - s.m) - lz);
    a.top_tokens[(int64_t)row * a.top + lane] = lp_token(list.k);
  }
  if (lane == 0) {
    const int64_t tok = a.tokens[row];
    float lp = 0.f;
    int64_t rank = -1;
    if (tok >= 0 && tok < a.vocab) {
      const float xt = lp_ruled(lp_logit<DT>(a.logits, row * a.ld + tok));
      lp = (float)((double)(xt - s.m) - lz);
      rank = s.rank;
    }
    a.logprob[row] = lp;
    a.rank[row] = rank;
    a.entropy[row] = (float)(lz - s.e / s.z);
  }
}

template <int DT, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(const LogprobArgs a) {
  constexpr int SZ = DT == PE_DTYPE_F32 ? 4 : 2, PER = 16 / SZ;  // values of a granule
  constexpr int U = 8 / PER;                                    // granules of a lane and chunk
  __shared__ LpSums sums[kLpWaves];
  __shared__ LpKey tops[kLpWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x, piece = blockIdx.y;
  // 16-byte granules from the one that holds the row's first value; value j of granule g
  // is token g PER + j - off
  const char* start = reinterpret_cast<const char*>(a.logits) + row * a.ld * SZ;
  const int off = (int)(reinterpret_cast<uintptr_t>(start) & 15) / SZ;
  const u32x4v* base = reinterpret_cast<const u32x4v*>(start - off * SZ);
  const int all = (a.vocab + off + PER - 1) / PER;
  const int g0 = piece * a.granules, g1 = min(all, g0 + a.granules);
  const int64_t tok64 = a.tokens[row];
  const bool there = tok64 >= 0 && tok64 < a.vocab;
  const int tok = there ? (int)tok64 : 0;
  const float xt = there ? lp_ruled(lp_logit<DT>(a.logits, row * a.ld + tok)) : __builtin_nanf("");
  // Among ruled-out tokens NaN and -inf tie: such a token's rank is counted apart, so that
  // a comparison for which NaN does not hold serves all others.
  const bool ruled = xt == -__builtin_inff();

  LpList list;
  list.begin();
  float m = -__builtin_inff();
  double z = 0, e = 0;
  int rank = 0;
  constexpr int STEP = kLpWaves * 64 * U;  // granules of the workgroup's chunks
  u32x4v nxt[U];
  auto load = [&](int c) {
#pragma unroll
    for (int u = 0; u < U; ++u) nxt[u] = base[min(c + u * 64 + lane, all - 1)];
  };
  int c = g0 + wave * 64 * U;
  if (c < g1) load(c);
  for (; c < g1; c += STEP) {
    u32x4v cur[U];
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = nxt[u];
    if (c + STEP < g1) load(c + STEP);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = cur[j / PER][j % PER * SZ / 4];
      if constexpr (DT == PE_DTYPE_F32) x[j] = __builtin_bit_cast(float, w);
      else if constexpr (DT == PE_DTYPE_BF16)
        x[j] = __builtin_bit_cast(float, j & 1 ? w & 0xFFFF0000u : w << 16);
      else x[j] = h2f((uint16_t)(w >> (16 * (j & 1))));
    }
    // a signalling NaN would take the maximum's other operand with it (fp16's are quiet
    // after their conversion)
    if constexpr (DT != PE_DTYPE_F16)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_canonicalizef(x[j]);
    auto index = [&](int j) { return (c + (j / PER) * 64 + lane) * PER + j % PER - off; };
    // outside the row and past the piece: NaN, which no comparison holds for
    auto outside = [&](int j) {
      return ((uint32_t)index(j) >= (uint32_t)a.vocab) | (c + (j / PER) * 64 + lane >= g1);
    };
    const bool edge = c == 0 || c + 64 * U > g1 || c + 64 * U >= all;
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = outside(j) ? __builtin_nanf("") : x[j];
    }
    float cm = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(cm > m)) {
      const float mn = fmaxf(m, cm);
      if (mn > m) {
        const float d = m - mn;
        const double f = __builtin_amdgcn_exp2f(d * kLpLog2e);
        e = f > 0 ? f * (e + d * z) : 0.0;  // d may be -inf, also of finite logits
        z *= f;
        m = mn;
      }
    }
    const float sub = m == -__builtin_inff() ? 0.f : m;
    float zs = 0.f, es = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = fmaxf(x[j] - sub, -1e4f);  // -inf and NaN: a weight of 0
      const float w = __builtin_amdgcn_exp2f(d * kLpLog2e);
      zs += w;
      es = __builtin_fmaf(w, d, es);
    }
    z += zs;
    e += es;
    // ties count where they come before the token; its own granule is looked at below
    if (__builtin_expect(ruled, 0)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        rank += __builtin_popcountll(__ballot(x[j] > xt || (!outside(j) && index(j) < tok)));
    } else
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t before = __ballot((c + u * 64 + lane) * PER + PER - 1 - off < tok);
#pragma unroll
      for (int j = u * PER; j < u * PER + PER; ++j)
        rank += __builtin_popcountll(__ballot(x[j] > xt) | (__ballot(x[j] == xt) & before));
    }
    if constexpr (TOP)
      if (__any(cm > list.last_x) || list.last == 0) {
        LpKey k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = lp_key(lp_ruled(x[j]), index(j));
        if (edge)
#pragma unroll
          for (int j = 0; j < 8; ++j) k[j] = outside(j) ? 0 : k[j];
        list.offer(k, lane, a.top);
      }
  }
  rank = lane == 0 ? rank : 0;
  if (there && !ruled && piece == 0 && wave == 0 && lane < PER) {
    // ties before the token in its granule
    const int i = (tok + off) / PER * PER - off + lane;
    rank += i >= 0 && i < tok && lp_logit<DT>(a.logits, row * a.ld + i) == xt;
  }
  const LpSums s = lp_join(LpSums{z, e, m, rank}, sums, lane, wave);
  if constexpr (TOP) lp_join_lists(list, tops, lane, wave, a.top);
  if (wave) return;
  if (a.pieces == 1) {
    lp_answer<DT>(a, row, s, list, lane);
    return;
  }
  const int64_t part = (int64_t)row * a.pieces + piece;
  if (lane == 0) reinterpret_cast<LpSums*>(a.parts)[part] = s;
  if (TOP && lane < a.top)
    reinterpret_cast<LpKey*>(reinterpret_cast<LpSums*>(a.parts) + (int64_t)a.rows * a.pieces)
        [part * a.top + lane] = list.k;
}

// a workgroup a row: its pieces' sums and lists
template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(const LogprobArgs a) {
  __shared__ LpSums sums[kLpWaves];
  __shared__ LpKey tops[kLpWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x;
  const LpSums* parts = reinterpret_cast<const LpSums*>(a.parts) + (int64_t)row * a.pieces;
  const int count = a.pieces * a.top;
  const LpKey* cand = reinterpret_cast<const LpKey*>(reinterpret_cast<const LpSums*>(a.parts) +
                                                     (int64_t)a.rows * a.pieces) + (int64_t)row * count;
  LpSums s{0, 0, -__builtin_inff(), 0};
  if ((int)threadIdx.x < a.pieces) s = parts[threadIdx.x];
  LpList list;
  list.begin();
  for (int c = wave * 512; c < count; c += kLpWaves * 512) {
    LpKey k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = c + j * 64 + lane;
      k[j] = cand[min(i, count - 1)];
      k[j] = i < count ? k[j] : 0;
    }
    list.offer(k, lane, a.top);
  }
  s = lp_join(s, sums, lane, wave);
  if (a.top) lp_join_lists(list, tops, lane, wave, a.top);
  if (wave == 0) lp_answer<DT>(a, row, s, list, lane);
}

// Pieces of a row: one where the rows alone fill the card, else as many as make about
// kLpTarget workgroups, of at least a chunk of the workgroup's. Microseconds by 300, 512,
// 1024, 2048 and 4096: 16 rows of 151,936 fp32 with 5 alternatives 18.8 17.1 16.2 15.7
// 15.8, 64 rows bf16 with 20 38.5 33.3 29.8 31.4 31.8, 300 rows fp32 with 5 67.8 58.5 53.1
// 55.6 60.6.
constexpr int kLpTarget = 1024;
constexpr int kLpMaxPieces = kLpThreads;  // a thread each in the join
struct LpPlan {
  int pieces, granules;
};
static LpPlan lp_plan(int64_t rows, int64_t vocab, int dtype) {
  const int per = dtype == PE_DTYPE_F32 ? 4 : 8, step = kLpWaves * 64 * (8 / per);
  const int64_t all = (vocab + 2 * per - 2) / per;  // at most, wherever the row begins
  int64_t n = (kLpTarget + rows - 1) / rows;
  n = n < kLpMaxPieces ? n : kLpMaxPieces;
  int64_t granules = ((all + n - 1) / n + step - 1) / step * step;
  return LpPlan{(int)((all + granules - 1) / granules), (int)granules};
}
static size_t lp_bytes(const LpPlan& p, int64_t rows, int top) {
  return p.pieces == 1 ? 0 : (size_t)rows * p.pieces * (sizeof(LpSums) + (size_t)top * sizeof(LpKey));
}
static bool lp_shape_ok(int64_t rows, int64_t vocab, int top) {
  return rows >= 0 && rows < (1 << 24) && vocab >= 1 && vocab <= (1 << 24) && top >= 0 && top <= kTopMax &&
         top <= vocab;
}

template <int DT>
static int launch_lp(const LogprobArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.rows, (unsigned)a.pieces);
  if (a.top) logprob_kernel<DT, true><<<grid, kLpThreads, 0, st>>>(a);
  else logprob_kernel<DT, false><<<grid, kLpThreads, 0, st>>>(a);
  const int rc = launch_status();
  if (rc != PE_OK || a.pieces == 1) return rc;
  logprob_join_kernel<DT><<<(unsigned)a.rows, kLpThreads, 0, st>>>(a);
  return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int top) {
  if (!lp_shape_ok(rows, vocab, top) || rows == 0) return 0;
  // of the types, the one with more pieces
  const size_t a = lp_bytes(lp_plan(rows, vocab, PE_DTYPE_F32), rows, top);
  const size_t b = lp_bytes(lp_plan(rows, vocab, PE_DTYPE_F16), rows, top);
  return a > b ? a : b;
}

extern "C" int pe_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t ld,
                                 int64_t vocab, const int64_t* tokens, int top, float* logprob,
                                 int64_t* rank, float* entropy, float* top_logprobs,
                                 int64_t* top_tokens, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!logits || !tokens || !logprob || !rank || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
    return PE_ERR_NULL;
  if (dtype != PE_DTYPE_F32 && bf16_flag(dtype) < 0) return PE_ERR_DTYPE;
  if (!lp_shape_ok(rows, vocab, top) || ld < vocab) return PE_ERR_DIMS;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == PE_DTYPE_F32 ? 4 : 2)) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  const LpPlan p = lp_plan(rows, vocab, dtype);
  const size_t need = lp_bytes(p, rows, top);
  if (need && (!workspace || workspace_bytes < need)) return PE_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return PE_ERR_ALIGN;
  const LogprobArgs a{logits, ld, tokens, (int)rows, (int)vocab, top, logprob, rank, entropy,
                      top_logprobs, top_tokens, p.pieces, p.granules, reinterpret_cast<char*>(workspace)};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PE_DTYPE_F32) return launch_lp<PE_DTYPE_F32>(a, st);
  if (dtype == PE_DTYPE_BF16) return launch_lp<PE_DTYPE_BF16>(a, st);
  return launch_lp<PE_DTYPE_F16>(a, st);
}
