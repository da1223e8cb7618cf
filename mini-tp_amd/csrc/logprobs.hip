// Log-probabilities of given tokens. For a row x of V logits and its token t,
// with m = max x and Z = sum_v exp(x_v - m):
//     log p_t = (x_t - m) - log Z
//     entropy = log Z - sum_v exp(x_v - m) (x_v - m) / Z
// the number of tokens in front of t, and the first k tokens of the order:
// larger logits first, equal ones by the lower token, NaN before every number.
#include <cmath>

#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  int V, top;
  const int64_t* tokens;
  float *logprobs, *entropy;
  int64_t *ranks, *top_tokens;
  float* top_logprobs;
};

// Logits as whole numbers in their order (-0 is 0, NaN above all), and with
// their token, the lower token ahead.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
  return (uint64_t)order_of(x) << 32 | ~token;
}

template <typename F>
__device__ __forceinline__ double block_sum(double v, double* scratch, F join) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = join(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return join(join(scratch[0], scratch[1]), join(scratch[2], scratch[3]));
}

template <typename T>
__global__ __launch_bounds__(256) void logprob_rows_kernel(LogprobArgs a) {
  __shared__ double scratch[4];
  __shared__ uint64_t best[4];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x;
  const T* x = (const T*)a.logits + b * a.ld;
  const int64_t t = a.tokens[b];
  const bool given = t >= 0 && t < a.V;
  const float xt = given ? load_f32<T>(x, t) : 0.f;
  const uint64_t kt = order_key(xt, (uint32_t)t);
  auto max2 = [](double p, double q) { return p > q ? p : q; };
  auto add2 = [](double p, double q) { return p + q; };
  double top = -__builtin_inf(), ahead = 0.0, nan = 0.0;
  for (int i = tid; i < a.V; i += 256) {
    const float v = load_f32<T>(x, i);
    nan += v != v;
    top = max2(top, (double)v);
    ahead += order_key(v, i) > kt;
  }
  top = block_sum(top, scratch, max2);
  ahead = block_sum(ahead, scratch, add2);
  nan = block_sum(nan, scratch, add2);
  double z = 0.0, s = 0.0;
  const float m = (float)top;
  for (int i = tid; i < a.V; i += 256) {
    const float d = load_f32<T>(x, i) - m, e = expf(d);
    z += e;
    s += e == 0.f ? 0.f : e * d;
  }
  z = block_sum(z, scratch, add2);
  s = block_sum(s, scratch, add2);
  const bool none = nan > 0.0 || fabs(top) == __builtin_inf();
  const double lse = none ? __builtin_nan("") : log(z);
  if (tid == 0) {
    a.logprobs[b] = given ? (float)((double)xt - top - lse) : __builtin_nanf("");
    a.entropy[b] = (float)(lse - s / z);
    a.ranks[b] = given ? (int64_t)ahead : -1;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t mine = 0;
    for (int i = tid; i < a.V; i += 256) {
      const uint64_t key = order_key(load_f32<T>(x, i), i);
      if (key < last || (k == 0 && key == last)) mine = std::max(mine, key);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mine = std::max<uint64_t>(mine, __shfl_xor(mine, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) best[tid >> 6] = mine;
    __syncthreads();
    last = std::max(std::max(best[0], best[1]), std::max(best[2], best[3]));
    if (tid == 0) {
      const uint32_t token = ~(uint32_t)last;
      a.top_tokens[b * a.top + k] = token;
      a.top_logprobs[b * a.top + k] = (float)((double)load_f32<T>(x, token) - top - lse);
    }
  }
}

}  // namespace

int64_t token_logprobs_workspace_bytes(int, int64_t B, int64_t, int64_t) { return B >= (1LL << 24) ? -1 : 0; }

int launch_token_logprobs(hipStream_t st, int dtype, const TokenLogprobs& t, void*, int64_t) {
  if (t.B >= (1LL << 24)) {
    set_error("token_logprobs: %lld rows of %lld logits are too many for one call", (long long)t.B, (long long)t.V);
    return MINITP_ERR_UNSUPPORTED;
  }
  const LogprobArgs a{t.logits,   t.ld,      (int)t.V, (int)t.top,   t.tokens,
                      t.logprobs, t.entropy, t.ranks,  t.top_tokens, t.top_logprobs};
  if (dtype == MINITP_F32)
    logprob_rows_kernel<float><<<(unsigned)t.B, 256, 0, st>>>(a);
  else
    logprob_rows_kernel<bf16><<<(unsigned)t.B, 256, 0, st>>>(a);
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

}  // namespace minitp
