// w4.hip — products with 4-bit weights and group scales:
//   out[m][n] = sum_g s[n][g] sum_{k in g} (u[n][k] - z[n][g]) x[m][k]  (+ residual[m][n])
// One wave per output: lanes take 8 consecutive weights (4 bytes) each, fp32 sums.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_device.h"
#include "mq_q4.h"

namespace {

MQ_DEV float from16(uint32_t bits, bool f16) {
  return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : bf16_to_f32((bf16_t)bits);
}

MQ_DEV void store_out(void* out, size_t i, float v, int type) {
  if (type == MQ_T_F32) ((float*)out)[i] = v;
  else if (type == MQ_T_F16) ((uint16_t*)out)[i] = __builtin_bit_cast(uint16_t, (_Float16)v);
  else ((uint16_t*)out)[i] = f32_to_bf16(v);
}
MQ_DEV float load_out(const void* out, size_t i, int type) {
  return type == MQ_T_F32 ? ((const float*)out)[i] : from16(((const uint16_t*)out)[i], type == MQ_T_F16);
}

__global__ void __launch_bounds__(256) w4_kernel(MqW4Args a) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y;
  if (n >= a.N) return;
  const int groups = a.K / a.G;
  const uint8_t* qr = a.qw + (size_t)n * (a.K / 2);
  const uint16_t* xr = a.x + (size_t)m * a.K;
  float acc = 0.f;
  for (int k = 8 * lane; k < a.K; k += 512) {
    const int g = k / a.G;
    const uint32_t w = *(const uint32_t*)(qr + k / 2);
    const float z = a.zeros != nullptr ? (float)a.zeros[(size_t)n * groups + g] : 8.0f;
    float part = 0.f;
    for (int i = 0; i < 8; ++i)
      part = fmaf((float)((w >> (4 * i)) & 15u) - z, from16(xr[k + i], a.x_type == MQ_T_F16), part);
    acc = fmaf(from16(a.scales[(size_t)n * groups + g], a.s_type == MQ_T_F16), part, acc);
  }
  acc = wave_sum(acc);
  if (lane == 0) {
    const size_t i = (size_t)m * a.N + n;
    if (a.residual != nullptr) acc += load_out(a.residual, i, a.o_type);
    store_out(a.out, i, acc, a.o_type);
  }
}

}  // namespace

int mq_launch_w4_linear(const MqW4Args& a, hipStream_t stream) {
  for (int m0 = 0; m0 < a.M; m0 += 65535) {
    MqW4Args b = a;
    b.x = a.x + (size_t)m0 * a.K;
    b.M = a.M - m0 < 65535 ? a.M - m0 : 65535;
    const size_t skip = (size_t)m0 * a.N * (a.o_type == MQ_T_F32 ? 4 : 2);
    b.out = (char*)a.out + skip;
    if (a.residual != nullptr) b.residual = (const char*)a.residual + skip;
    hipLaunchKernelGGL(w4_kernel, dim3((a.N + 3) / 4, b.M), dim3(256), 0, stream, b);
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
