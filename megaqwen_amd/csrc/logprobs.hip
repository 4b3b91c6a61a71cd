// logprobs.hip — log probability of a given token in every row of logits, the row's entropy and its
// most likely tokens.  With m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//   log p(token) = x[token] - m - log s,   entropy = log s - t / s.
// One workgroup per row: one pass for m, s and t, then one pass per alternative.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_device.h"
#include "mq_logprobs.h"

namespace {

#define LP_THREADS 512
#define LP_LOG2E 1.44269504088896340736f
#define LP_LN2 0.69314718055994530942f

template <int TYPE> MQ_DEV float lp_load(const void* p, long long i) {
  if constexpr (TYPE == 2) return ((const float*)p)[i];
  else if constexpr (TYPE == 1) return (float)((const _Float16*)p)[i];
  else return bf16_to_f32(((const uint16_t*)p)[i]);
}

// Sums of a running softmax: m = max, s = sum e^(x - m), t = sum e^(x - m) (x - m).  No element yet
// (or only -inf): m = -inf, s = t = 0.  A NaN element makes m NaN.
struct LpSum {
  float m, s, t;
};
MQ_DEV LpSum lp_join(LpSum a, LpSum b) {
  LpSum r;
  r.m = __builtin_elementwise_maximum(a.m, b.m);
  // (-inf) - (-inf) is NaN, which fmaxf drops; e^-150 has no weight next to 1
  const float da = fmaxf(a.m - r.m, -150.f), db = fmaxf(b.m - r.m, -150.f);
  const float fa = __builtin_amdgcn_exp2f(da * LP_LOG2E), fb = __builtin_amdgcn_exp2f(db * LP_LOG2E);
  r.s = fa * a.s + fb * b.s;
  r.t = fa * fmaf(a.s, da, a.t) + fb * fmaf(b.s, db, b.t);
  return r;
}

template <int TYPE>
__global__ void __launch_bounds__(LP_THREADS) lp_row_kernel(MqLogprobArgs a) {
  __shared__ LpSum sums[LP_THREADS / 64];
  __shared__ uint64_t keys[LP_THREADS / 64];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const void* x = (const char*)a.logits + (size_t)((long long)row * a.stride) * (TYPE == 2 ? 4 : 2);
  LpSum r = {-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
    const float v = lp_load<TYPE>(x, i);
    r = lp_join(r, LpSum{v, v == -INFINITY ? 0.f : 1.f, 0.f});
  }
  for (int d = 1; d < 64; d <<= 1)
    r = lp_join(r, LpSum{xor_lane(r.m, d), xor_lane(r.s, d), xor_lane(r.t, d)});
  if (lane == 0) sums[wave] = r;
  __syncthreads();
  r = sums[0];
  for (int w = 1; w < LP_THREADS / 64; ++w) r = lp_join(r, sums[w]);
  const bool bad = !(r.m < INFINITY), empty = r.m == -INFINITY;
  const float ls = empty ? 0.f : __builtin_amdgcn_logf(r.s) * LP_LN2;
  if (threadIdx.x == 0) {
    const long long tok = a.tok64 ? ((const long long*)a.tokens)[row] : ((const int*)a.tokens)[row];
    float lp = -INFINITY;
    if (tok >= 0 && tok < a.vocab && !empty) lp = lp_load<TYPE>(x, tok) - r.m - ls;
    a.logprob[row] = bad ? NAN : lp;
    a.entropy[row] = bad ? NAN : empty ? 0.f : ls - r.t / r.s;
  }
  uint64_t prev = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
      // -0 counts as +0; in a row with a NaN the order is by index alone
      const float v = r.m != r.m ? 0.f : lp_load<TYPE>(x, i) + 0.f;
      const uint64_t key = argmax_key(v, (uint32_t)i);
      if (key < prev && key > best) best = key;
    }
    best = wave_max_u64(best);
    __syncthreads();
    if (lane == 0) keys[wave] = best;
    __syncthreads();
    for (int w = 0; w < LP_THREADS / 64; ++w) best = u64_max(best, keys[w]);
    prev = best;
    if (threadIdx.x == 0) {
      const int i = (int)argmax_key_index(best);
      a.top_tok[(size_t)row * a.top_k + k] = i;
      a.top_lp[(size_t)row * a.top_k + k] = bad ? NAN : empty ? -INFINITY : lp_load<TYPE>(x, i) - r.m - ls;
    }
  }
}

}  // namespace

size_t mq_logprobs_workspace(int, int, int) { return 0; }

int mq_launch_token_logprobs(const MqLogprobArgs& a, void*, hipStream_t stream) {
  auto kernel = a.type == 2 ? lp_row_kernel<2> : a.type == 1 ? lp_row_kernel<1> : lp_row_kernel<0>;
  hipLaunchKernelGGL(kernel, dim3(a.rows), dim3(LP_THREADS), 0, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
