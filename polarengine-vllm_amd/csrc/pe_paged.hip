// The paged 8-bit cache: block tables and slot maps of a step, blocks back to the
// pool, and the quantizing write of keys and values.

#include <type_traits>

#include "pe_paged.h"

namespace pe {

constexpr int kPlanThreads = 1024;

// Running sums over a workgroup in order of thread; `total` in every thread.
// Values and sums stop at kPlanCap, which is past any number of rows or blocks.
constexpr uint32_t kPlanCap = 1u << 30;
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t* waves, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(v, off, 64);
    if (lane >= off) v = min(v + u, kPlanCap);
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) {
    if (w < wave) before = min(before + waves[w], kPlanCap);
    total = min(total + waves[w], kPlanCap);
  }
  return min(before + v, kPlanCap);
}

// ---------------------------------------------------------------------------
// The plan, one workgroup: a thread a sequence, then a thread a row. What bounds it is
// the chain of loads: lengths, table entries, free blocks, the rows' entries. A
// sequence's first kPlanShort entries are its thread's, at once; of longer ones a wave
// takes 64 at a time (a thread alone: 27.6 us for 496 users beside four chunks of up to
// 2800 rows, this way 13.4; their release 17.2 -> 5.9). 64 users' step: 4.7 us, 3.4 for
// its release.
// ---------------------------------------------------------------------------
constexpr int kPlanShort = 4;

// sequences of a pass that have more than kPlanShort entries to look at
struct PlanLong {
  uint32_t count;
  uint16_t of[kPlanThreads];
};
__device__ __forceinline__ bool plan_long(PlanLong& l, bool mine) {
  if (!__syncthreads_or(mine)) return false;
  if (threadIdx.x == 0) l.count = 0;
  __syncthreads();
  if (mine) l.of[atomicAdd(&l.count, 1u)] = (uint16_t)threadIdx.x;  // in any order
  __syncthreads();
  return true;
}

__global__ __launch_bounds__(kPlanThreads) void plan_step_kernel(
    const int64_t* __restrict__ lengths, const int64_t* __restrict__ counts, int32_t* tables,
    int64_t t_b, int batch, int64_t width, const int32_t* __restrict__ free_blocks, int64_t free_cap,
    int64_t* free_count, int rows, int log_t, int64_t* __restrict__ starts,
    int64_t* __restrict__ positions, int64_t* __restrict__ slots, int64_t* __restrict__ out_lengths) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  __shared__ uint32_t used;
  __shared__ PlanLong longs;
  __shared__ uint32_t needs[kPlanThreads];
  __shared__ int64_t firsts[kPlanThreads], lasts[kPlanThreads];
  // of the step: each sequence's end among the rows, and position minus row (kNone: it
  // got nothing)
  constexpr int kNone = INT32_MIN;
  __shared__ int ends[kPagedMaxBatch], offsets[kPagedMaxBatch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int threads = blockDim.x, n_waves = threads / 64;
  const uint32_t have = (uint32_t)max((int64_t)0, min(*free_count, free_cap));
  if (tid == 0) {
    starts[0] = 0;
    used = 0;
  }
  uint32_t row0 = 0, need0 = 0;  // of the sequences before these
  for (int b0 = 0; b0 < batch; b0 += threads) {
    const int b = b0 + tid;
    const int64_t len = b < batch ? lengths[b] : -1;
    // a count past the rows is as good as one row more
    const uint32_t n = len >= 0 ? (uint32_t)max((int64_t)0, min(counts[b], (int64_t)rows + 1)) : 0;
    uint32_t total;
    const uint32_t end = min(row0 + plan_scan(n, waves, total), (uint32_t)rows + 1);
    row0 = min(row0 + total, (uint32_t)rows + 1);
    const bool fits = len >= 0 && len <= (width << log_t) - (int64_t)n && end <= (uint32_t)rows;
    const int64_t j0 = len >> log_t, j1 = fits && n ? (len + n - 1) >> log_t : j0 - 1;
    int32_t* row = tables + (int64_t)b * t_b;
    uint32_t need = 0;
    int32_t entry[kPlanShort];
#pragma unroll
    for (int i = 0; i < kPlanShort; ++i) entry[i] = j0 + i <= j1 ? row[j0 + i] : 0;
#pragma unroll
    for (int i = 0; i < kPlanShort; ++i) need += entry[i] < 0;
    const bool is_long = j1 - j0 >= kPlanShort;
    firsts[tid] = j0;
    lasts[tid] = j1;
    const bool any_long = plan_long(longs, is_long);
    for (uint32_t k = wave; any_long && k < longs.count; k += n_waves) {
      const int t = longs.of[k];
      const int32_t* r = tables + (int64_t)(b0 + t) * t_b;
      uint32_t lacks = 0;
      for (int64_t j = firsts[t] + lane; j - lane <= lasts[t]; j += 64)
        lacks += __builtin_popcountll(__ballot(j <= lasts[t] && r[min(j, lasts[t])] < 0));
      if (lane == 0) needs[t] = lacks;
    }
    if (any_long) __syncthreads();
    if (is_long) need = needs[tid];
    const uint32_t cum = need0 + plan_scan(need, waves, total);
    need0 = min(need0 + total, kPlanCap);
    const bool taken = fits && (need == 0 || cum <= have);
    if (b < batch) {
      starts[b + 1] = min(end, (uint32_t)rows);
      out_lengths[b] = taken ? len + n : -1;
      ends[b] = (int)min(end, (uint32_t)rows);
      offsets[b] = taken ? (int)len - (int)(end - n) : kNone;
    }
    if (taken && need && !is_long) {
      uint32_t at = cum - need;
#pragma unroll
      for (int i = 0; i < kPlanShort; ++i)
        if (entry[i] < 0) row[j0 + i] = free_blocks[have - 1 - at++];
    }
    needs[tid] = taken && need ? cum - need : UINT32_MAX;  // rank of the first block
    if (taken && need) atomicMax(&used, cum);
    __syncthreads();
    for (uint32_t k = wave; any_long && k < longs.count; k += n_waves) {
      const int t = longs.of[k];
      if (needs[t] == UINT32_MAX) continue;
      int32_t* r = tables + (int64_t)(b0 + t) * t_b;
      uint32_t at = needs[t];
      for (int64_t j = firsts[t] + lane; j - lane <= lasts[t]; j += 64) {
        const bool lacks = j <= lasts[t] && r[min(j, lasts[t])] < 0;
        const uint64_t all = __ballot(lacks);
        if (lacks) r[j] = free_blocks[have - 1 - (at + __builtin_popcountll(all & ((1ull << lane) - 1)))];
        at += __builtin_popcountll(all);
      }
    }
    if (any_long) __syncthreads();
  }
  if (tid == 0) *free_count = (int64_t)have - used;
  // R rows a thread at a time, so that their entries' loads go out together
  auto place = [&](auto R_) {
    constexpr int R = decltype(R_)::value;
    for (int r0 = tid; r0 < rows; r0 += R * threads) {
      int64_t pos[R];
      int32_t block[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = min(r0 + i * threads, rows - 1);
        int lo = 0, hi = batch;  // the first sequence that ends behind row r
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (ends[mid] > r) hi = mid;
          else lo = mid + 1;
        }
        const int off = lo < batch ? offsets[lo] : kNone;
        pos[i] = off != kNone ? off + r : -1;
        block[i] = off != kNone ? tables[lo * t_b + (pos[i] >> log_t)] : 0;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = r0 + i * threads;
        if (r < rows) {
          positions[r] = pos[i];
          slots[r] = pos[i] >= 0 ? ((int64_t)block[i] << log_t) + (pos[i] & ((1 << log_t) - 1)) : -1;
        }
      }
    }
  };
  if (rows <= threads) place(std::integral_constant<int, 1>{});
  else place(std::integral_constant<int, 8>{});
}

__global__ __launch_bounds__(kPlanThreads) void release_kernel(
    int32_t* tables, int64_t t_b, int batch, int64_t width, const int64_t* __restrict__ keep,
    int32_t* __restrict__ free_blocks, int64_t free_cap, int64_t* free_count, int log_t) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  __shared__ PlanLong longs;
  __shared__ uint32_t ns[kPlanThreads], ats[kPlanThreads];
  __shared__ int64_t firsts[kPlanThreads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int threads = blockDim.x, n_waves = threads / 64;
  const int64_t have = max((int64_t)0, min(*free_count, free_cap));
  int64_t first;
  int32_t entry[kPlanShort];
  bool is_long, any_long = false;
  // how many blocks of sequence b0 + tid go back; `longs` has those of more than kPlanShort
  auto count = [&](int b0) {
    const int b = b0 + tid;
    const int64_t k = b < batch ? keep[b] : -1;
    first = k < 0 ? width : min(width, (k >> log_t) + ((k & ((1 << log_t) - 1)) != 0));
#pragma unroll
    for (int i = 0; i < kPlanShort; ++i)
      entry[i] = first + i < width ? tables[b * t_b + first + i] : -1;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < kPlanShort; ++i) n += n == (uint32_t)i && entry[i] >= 0;
    is_long = n == kPlanShort;
    firsts[tid] = first;
    any_long = plan_long(longs, is_long);
    for (uint32_t l = wave; any_long && l < longs.count; l += n_waves) {
      const int t = longs.of[l];
      const int32_t* r = tables + (int64_t)(b0 + t) * t_b;
      uint32_t m = 0;
      for (int64_t j = firsts[t] + lane;; j += 64) {
        const uint64_t there = __ballot(j < width && r[min(j, width - 1)] >= 0);
        m += ~there ? __builtin_ctzll(~there) : 64;
        if (~there) break;
      }
      if (lane == 0) ns[t] = m;
    }
    if (any_long) __syncthreads();
    if (is_long) n = ns[tid];
    return n;
  };
  uint32_t all = 0, total, n = 0;
  for (int b0 = 0; b0 < batch; b0 += threads) {
    n = count(b0);
    plan_scan(n, waves, total);
    all += total;
  }
  if (have + all > free_cap) return;
  uint32_t before = 0;
  for (int b0 = 0; b0 < batch; b0 += threads) {
    if (batch > threads) n = count(b0);
    const uint32_t at = before + plan_scan(n, waves, total) - n;
    before += total;
    int32_t* row = tables + (int64_t)(b0 + tid) * t_b + first;
    // from the stack's new end on, downwards
    int32_t* top = free_blocks + have + all - 1;
    if (!is_long) {
#pragma unroll
      for (int i = 0; i < kPlanShort; ++i)
        if ((uint32_t)i < n) {
          top[-(int64_t)(at + i)] = entry[i];
          row[i] = -1;
        }
    }
    if (!any_long) continue;
    ats[tid] = at;
    ns[tid] = n;
    __syncthreads();
    for (uint32_t l = wave; l < longs.count; l += n_waves) {
      const int t = longs.of[l];
      int32_t* r = tables + (int64_t)(b0 + t) * t_b + firsts[t];
      for (uint32_t i = lane; i < ns[t]; i += 64) {
        top[-(int64_t)(ats[t] + i)] = r[i];
        r[i] = -1;
      }
    }
    __syncthreads();
  }
  if (tid == 0) *free_count = have + all;
}

// ---------------------------------------------------------------------------
// The write. A workgroup looks for runs that begin among its `per` rows (one in a
// decode step, so that every token has a workgroup; up to 32 in a prompt) and takes
// those of one KV head, keys or values, one after the other. A thread holds 4 slots x 8
// dimensions: the run is read once, its largest |x| gives the scale, then codes go out.
// Threads of a wave run over dimensions first for keys (rows of the block) and over
// slots first for values (which the block stores by dimension), so that either writes
// neighbouring bytes. What bounds it is the chain of slots, rows, largest value and codes
// of a run: 32 rows of 8 heads of 128 6.4 us, 4 x 2048 rows 17 us (50 MB, 2.9 TB/s; with
// a workgroup for every row 628).
// ---------------------------------------------------------------------------
// four codes; NaN where a value is not finite (the conversion itself would saturate)
__device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  uint32_t u = (uint32_t)r;
  u = fabsf(a) <= 3.4e38f ? u : u | 0x7Fu;
  u = fabsf(b) <= 3.4e38f ? u : u | 0x7F00u;
  u = fabsf(c) <= 3.4e38f ? u : u | 0x7F0000u;
  u = fabsf(d) <= 3.4e38f ? u : u | 0x7F000000u;
  return u;
}
// the smallest e with amax <= 448 2^e
__device__ __forceinline__ int f8_exp(float amax) {
  if (amax == 0.f) return kMinExp;
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  // amax = 1.m 2^x: x - 8, one more where 1.m passes 1.75
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
  return max(e, kMinExp);
}

struct WriteArgs {
  const uint16_t *k, *v;
  int64_t k_r, k_h, v_r, v_h;
  const int64_t* slots;
  PagedCache c;
  int rows, per, log_d;
};

template <bool BF, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS <= 256 ? 6 : 4) void write_blocks_kernel(const WriteArgs a) {
  __shared__ float red[THREADS / 64];
  const int h = blockIdx.y;
  const bool val = blockIdx.z;
  const int log_t = a.c.log_t, T = 1 << log_t, log_d = a.log_d, D = 1 << log_d;
  const int tid = threadIdx.x, lane = tid & 63;
  const int row0 = blockIdx.x * a.per;
  const int64_t n_slots = a.c.blocks << log_t;
  // the thread's part of a block: slots 4 sg .. + 3 and dimensions 8 ch .. + 7
  const int sg = val ? tid & ((T >> 2) - 1) : tid >> (log_d - 3);
  const int ch = val ? tid >> (log_t - 2) : tid & ((D >> 3) - 1);
  const bool in = tid < T * D / 32;
  // 64 rows' slots, a lane each: which of the first `per` rows begin a run
  const int64_t mine = a.slots[min(row0 + lane, a.rows - 1)];
  int64_t prev = __shfl_up((long long)mine, 1, 64);
  if (lane == 0) prev = row0 ? a.slots[row0 - 1] : -1;
  const bool within = row0 + lane > 0 && prev == mine - 1 && (mine & (T - 1));
  const bool valid = row0 + lane < a.rows && mine >= 0 && mine < n_slots;
  uint64_t begins = __ballot(lane < a.per && valid && !within);
  const uint64_t on = __ballot(valid && within);  // goes on what the row before it does
  for (; begins; begins &= begins - 1) {
    const int l = __builtin_ctzll(begins), row = row0 + l;
    const int64_t slot = __shfl((long long)mine, l, 64);
    const int off = (int)(slot & (T - 1));
    const uint64_t rest = l < 63 ? ~(on >> (l + 1)) : ~0ull;
    int n = 1 + (rest ? __builtin_ctzll(rest) : 64);  // rows of the run
    n = min(n, 64 - l);
    // on behind the 64
    for (int i0 = 64 - l; n == i0 && off + n < T; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t more = __ballot(off + i < T && row + i < a.rows &&
                                     a.slots[min(row + i, a.rows - 1)] == slot + i);
      n += ~more ? __builtin_ctzll(~more) : 64;
    }
    const int64_t block = slot >> log_t;
    const uint16_t* src = val ? a.v + row * a.v_r + h * a.v_h : a.k + row * a.k_r + h * a.k_h;
    const int64_t s_r = val ? a.v_r : a.k_r;
    uint8_t* dst = (val ? a.c.v + block * a.c.v_b : a.c.k + block * a.c.k_b) + ((int64_t)h << (log_t + log_d));
    uint8_t* scale = (val ? a.c.vs : a.c.ks) + block * a.c.s_b + h;
    const int old = (int)*scale - 127;
    const int s0 = 4 * sg - off;  // of the run's rows
    const bool act = in && s0 + 3 >= 0 && s0 < n;
    u32x4v x[4];
    float amax = 0.f;
    if (act) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[t] = u32x4v{0, 0, 0, 0};
        if (s0 + t >= 0 && s0 + t < n) x[t] = *reinterpret_cast<const u32x4v*>(src + (s0 + t) * s_r + 8 * ch);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t u = x[t][w];
          const float lo = fabsf(f16or_bf((uint16_t)u, BF)), hi = fabsf(f16or_bf((uint16_t)(u >> 16), BF));
          amax = fmaxf(amax, lo <= 3.4e38f ? lo : 0.f);
          amax = fmaxf(amax, hi <= 3.4e38f ? hi : 0.f);
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
    __syncthreads();  // the last run's sums and stores are done with
    if (lane == 0) red[tid >> 6] = amax;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 64; ++w) amax = fmaxf(amax, red[w]);
    const int e = off ? max(old, f8_exp(amax)) : f8_exp(amax);
    if (off && e > old) {
      uint32_t* codes = reinterpret_cast<uint32_t*>(dst);
      for (int i = tid; i < T * D / 4; i += blockDim.x) {
        const uint32_t u = codes[i];
        float f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t one = u >> (8 * k);
          f[k] = __builtin_ldexpf(__builtin_amdgcn_cvt_f32_fp8(one, 0), old - e);
        }
        codes[i] = f8_codes(f[0], f[1], f[2], f[3]);
      }
      __syncthreads();
    }
    if (tid == 0) *scale = (uint8_t)(e + 127);
    if (!act) continue;
    uint32_t code[4][2];  // of each slot, eight dimensions
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t u = x[t][2 * w], v = x[t][2 * w + 1];
        code[t][w] = f8_codes(__builtin_ldexpf(f16or_bf((uint16_t)u, BF), -e),
                              __builtin_ldexpf(f16or_bf((uint16_t)(u >> 16), BF), -e),
                              __builtin_ldexpf(f16or_bf((uint16_t)v, BF), -e),
                              __builtin_ldexpf(f16or_bf((uint16_t)(v >> 16), BF), -e));
      }
    if (!val) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (s0 + t >= 0 && s0 + t < n)
          *reinterpret_cast<uint2*>(dst + ((4 * sg + t) << log_d) + 8 * ch) = make_uint2(code[t][0], code[t][1]);
    } else {
      const bool whole = s0 >= 0 && s0 + 3 < n;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        uint32_t u = 0;  // four slots of a dimension
#pragma unroll
        for (int t = 0; t < 4; ++t) u |= (code[t][d >> 2] >> (8 * (d & 3)) & 0xFFu) << (8 * t);
        uint8_t* to = dst + ((8 * ch + d) << log_t) + 4 * sg;
        if (whole) {
          *reinterpret_cast<uint32_t*>(to) = u;
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (s0 + t >= 0 && s0 + t < n) to[t] = (uint8_t)(u >> (8 * t));
        }
      }
    }
  }
}

// workgroups that a write is cut into, by giving each of them up to 32 rows
constexpr int64_t kWriteWgs = 4096;

static bool plan_shape_ok(int64_t batch, int64_t width, int64_t t_b, int64_t free_cap,
                          int block_size) {
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return false;
  return batch >= 0 && batch <= kPagedMaxBatch && width >= 1 && width <= kPagedMaxWidth &&
         t_b >= width && free_cap >= 1 && free_cap <= INT32_MAX;
}
// a small plan's barriers are cheaper among four waves
static unsigned plan_threads(int64_t items) { return items <= 256 ? 256 : kPlanThreads; }
static int log2_of(int block_size) {
  return block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
}

}  // namespace pe

using namespace pe;

extern "C" int pe_plan_step(const int64_t* lengths, const int64_t* counts, int32_t* tables,
                            int64_t t_b, int64_t batch, int64_t width, const int32_t* free_blocks,
                            int64_t free_cap, int64_t* free_count, int64_t rows, int block_size,
                            int64_t* starts, int64_t* positions, int64_t* slots,
                            int64_t* out_lengths, void* stream) {
  if (!lengths || !counts || !tables || !free_blocks || !free_count || !starts || !out_lengths ||
      (rows > 0 && (!positions || !slots)))
    return PE_ERR_NULL;
  if (!plan_shape_ok(batch, width, t_b, free_cap, block_size) || rows < 0 || rows > kPagedMaxRows)
    return PE_ERR_DIMS;
  if (batch == 0) return PE_OK;
  plan_step_kernel<<<1, plan_threads(batch > rows ? batch : rows), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      lengths, counts, tables, t_b, (int)batch, width, free_blocks, free_cap, free_count, (int)rows,
      log2_of(block_size), starts, positions, slots, out_lengths);
  return launch_status();
}

extern "C" int pe_release_blocks(int32_t* tables, int64_t t_b, int64_t batch, int64_t width,
                                 const int64_t* keep, int32_t* free_blocks, int64_t free_cap,
                                 int64_t* free_count, int block_size, void* stream) {
  if (!tables || !keep || !free_blocks || !free_count) return PE_ERR_NULL;
  if (!plan_shape_ok(batch, width, t_b, free_cap, block_size)) return PE_ERR_DIMS;
  if (batch == 0) return PE_OK;
  release_kernel<<<1, plan_threads(batch), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      tables, t_b, (int)batch, width, keep, free_blocks, free_cap, free_count, log2_of(block_size));
  return launch_status();
}

extern "C" int pe_write_blocks(const void* k, const void* v, int dtype, int64_t rows, int64_t k_r,
                               int64_t k_h, int64_t v_r, int64_t v_h, const int64_t* slots,
                               void* k_codes, int64_t k_b, void* v_codes, int64_t v_b, void* k_scale,
                               void* v_scale, int64_t s_b, int64_t blocks, int kv_heads,
                               int block_size, int head_dim, void* stream) {
  if (!k || !v || !slots) return PE_ERR_NULL;
  const int bf = bf16_flag(dtype);
  if (bf < 0) return PE_ERR_DTYPE;
  WriteArgs a;
  const int ok = paged_cache(a.c, k_codes, k_b, v_codes, v_b, k_scale, v_scale, s_b, blocks, kv_heads,
                             block_size, head_dim);
  if (ok != PE_OK) return ok;
  if (rows < 0 || rows > kPagedMaxRows || k_r < 0 || k_h < 0 || v_r < 0 || v_h < 0) return PE_ERR_DIMS;
  if (!aligned16(k) || !aligned16(v) || (k_r | k_h | v_r | v_h) % 8) return PE_ERR_ALIGN;
  if (rows == 0) return PE_OK;
  a.k = reinterpret_cast<const uint16_t*>(k);
  a.v = reinterpret_cast<const uint16_t*>(v);
  a.k_r = k_r;
  a.k_h = k_h;
  a.v_r = v_r;
  a.v_h = v_h;
  a.slots = slots;
  a.rows = (int)rows;
  a.log_d = head_dim == 64 ? 6 : head_dim == 128 ? 7 : 8;
  const int64_t per = (rows * kv_heads * 2 + kWriteWgs - 1) / kWriteWgs;
  a.per = (int)(per < 32 ? per : 32);
  const dim3 grid((unsigned)((rows + a.per - 1) / a.per), (unsigned)kv_heads, 2);
  const int parts = block_size * head_dim / 32;  // of 4 slots x 8 dimensions: a thread each
  const unsigned threads = parts < 64 ? 64 : parts;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (threads <= 256) {
    if (bf) write_blocks_kernel<true, 256><<<grid, threads, 0, st>>>(a);
    else write_blocks_kernel<false, 256><<<grid, threads, 0, st>>>(a);
  } else {
    if (bf) write_blocks_kernel<true, 1024><<<grid, threads, 0, st>>>(a);
    else write_blocks_kernel<false, 1024><<<grid, threads, 0, st>>>(a);
  }
  return launch_status();
}
