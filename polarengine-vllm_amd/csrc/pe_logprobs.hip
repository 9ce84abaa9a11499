// Log probabilities of given tokens, their ranks, the entropy and the likeliest
// alternatives: a workgroup a row.

#include "pe_internal.h"

namespace pe {

constexpr int kTopMax = 64;

template <int DT>
__device__ __forceinline__ float logit(const void* p, int64_t i) {
  if constexpr (DT == PE_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  else return f16or_bf(reinterpret_cast<const uint16_t*>(p)[i], DT == PE_DTYPE_BF16);
}

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
};

template <int DT>
__global__ __launch_bounds__(1024) void logprob_kernel(const LogprobArgs a) {
  __shared__ double rd[16];
  __shared__ float rf[16];
  __shared__ int ri[16];
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const int64_t base = row * a.ld;
  auto best = [&](float v, int i) {  // the largest, the first of equals
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      const float ov = __shfl_xor(v, m, 64);
      const int oi = __shfl_xor(i, m, 64);
      if (ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
      }
    }
    __syncthreads();
    if ((tid & 63) == 0) {
      rf[wave] = v;
      ri[wave] = i;
    }
    __syncthreads();
    v = rf[0];
    i = ri[0];
    for (int w = 1; w < 16; ++w)
      if (rf[w] > v || (rf[w] == v && ri[w] < i)) {
        v = rf[w];
        i = ri[w];
      }
  return make_float2(v, __builtin_bit_cast(float, i));
  };
  auto sum = [&](double v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, 64);
    __syncthreads();
    if ((tid & 63) == 0) rd[wave] = v;
    __syncthreads();
    double t = 0;
    for (int w = 0; w < 16; ++w) t += rd[w];
    return t;
  };
  const int64_t tok = a.tokens[row];
  const bool there = tok >= 0 && tok < a.vocab;
  const float xt = there ? logit<DT>(a.logits, base + tok) : 0.f;
  float mx = -__builtin_inff();
  int mi = a.vocab;
  for (int i = tid; i < a.vocab; i += 1024) {
    const float x = logit<DT>(a.logits, base + i);
    if (x > mx || (x == mx && i < mi)) {
      mx = x;
      mi = i;
    }
  }
  float2 w = best(mx, mi);
  const float top = w.x;
  double z = 0, e = 0, r = 0;
  for (int i = tid; i < a.vocab; i += 1024) {
    const float x = logit<DT>(a.logits, base + i), d = x - top;
    const float p = expf(d);
    z += p;
    if (p > 0.f || p != p) e += (double)p * d;
    r += x > xt || (x == xt && i < tok);
  }
  z = sum(z);
  e = sum(e);
  r = sum(r);
  const double lz = log(z);
  if (tid == 0) {
    a.logprob[row] = there ? (float)((double)(xt - top) - lz) : 0.f;
    a.rank[row] = there ? (int64_t)r : -1;
    a.entropy[row] = (float)(lz - e / z);
  }
  int last = -1;  // the one taken before
  float lv = 0.f;
  for (int k = 0; k < a.top; ++k) {
    if (k) {
      mx = -__builtin_inff();
      mi = a.vocab;
      for (int i = tid; i < a.vocab; i += 1024) {
        const float x = logit<DT>(a.logits, base + i);
        if (!(x < lv || (x == lv && i > last))) continue;
        if (x > mx || (x == mx && i < mi)) {
          mx = x;
          mi = i;
        }
      }
      w = best(mx, mi);
    }
    lv = w.x;
    last = __builtin_bit_cast(int, w.y);
    if (tid == 0) {
      a.top_logprobs[(int64_t)row * a.top + k] = (float)((double)(lv - top) - lz);
      a.top_tokens[(int64_t)row * a.top + k] = last < a.vocab ? last : -1;
    }
  }
}

}  // namespace pe

using namespace pe;

extern "C" size_t pe_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int top) { return 0; }

extern "C" int pe_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t ld,
                                 int64_t vocab, const int64_t* tokens, int top, float* logprob,
                                 int64_t* rank, float* entropy, float* top_logprobs,
                                 int64_t* top_tokens, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!logits || !tokens || !logprob || !rank || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
    return PE_ERR_NULL;
  if (dtype != PE_DTYPE_F32 && bf16_flag(dtype) < 0) return PE_ERR_DTYPE;
  if (rows < 0 || rows > kTopMax * (int64_t)(1 << 18) || vocab < 1 || vocab > (1 << 24) || ld < vocab ||
      top < 0 || top > kTopMax || top > vocab)
    return PE_ERR_DIMS;
  if (rows == 0) return PE_OK;
  const LogprobArgs a{logits, ld, tokens, (int)rows, (int)vocab, top, logprob, rank, entropy,
                      top_logprobs, top_tokens};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PE_DTYPE_F32) logprob_kernel<PE_DTYPE_F32><<<(unsigned)rows, 1024, 0, st>>>(a);
  else if (dtype == PE_DTYPE_BF16) logprob_kernel<PE_DTYPE_BF16><<<(unsigned)rows, 1024, 0, st>>>(a);
  else logprob_kernel<PE_DTYPE_F16><<<(unsigned)rows, 1024, 0, st>>>(a);
  return launch_status();
}
