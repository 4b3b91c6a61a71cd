// kv4.hip — a key/value cache held in 4 bits: rows are quantised into it (append), read back as
// the values they stand for (read), and attended over (attend).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_device.h"
#include "mq_q4.h"

namespace {

MQ_DEV float from16(uint32_t bits, bool f16) {
  return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : bf16_to_f32((bf16_t)bits);
}
MQ_DEV uint16_t to16(float v, bool f16) {
  return f16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : f32_to_bf16(v);
}

// One thread per group of G values of a key (i = 0) or value (i = 1) row.
//   s = bf16(max|x| / 7), u = clamp(rint(x / s), -7, 7) + 8; s = 0: u = 8; a group that holds an
//   infinity or a NaN gets s = NaN, so that all of its values read as NaN.
__global__ void __launch_bounds__(256)
kv4_append_kernel(MqKv4 c, const uint16_t* k, MqStrides ks, const uint16_t* v, MqStrides vs, bool f16) {
  const int ng = c.D / c.G;
  long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long long)c.B * c.T * c.Hkv * 2 * ng) return;
  const int g = (int)(id % ng); id /= ng;
  const int which = (int)(id & 1); id >>= 1;
  const int h = (int)(id % c.Hkv); id /= c.Hkv;
  const int t = (int)(id % c.T), b = (int)(id / c.T);
  const long long pos = (long long)c.lengths[b] - c.T + t;
  if (pos < 0 || pos >= c.S) return;
  const MqStrides st = which ? vs : ks;
  const uint16_t* x = (which ? v : k) + b * st.b + t * st.t + h * st.h + g * c.G;
  float amax = 0.f;
  bool bad = false;
  for (int i = 0; i < c.G; ++i) {
    const float f = fabsf(from16(x[i], f16));
    bad |= !(f < INFINITY);
    amax = fmaxf(amax, f);
  }
  const uint16_t sb = bad ? 0x7fc0 : f32_to_bf16(amax / 7.0f);
  const float s = bf16_to_f32(sb);
  const size_t row = ((size_t)b * c.Hkv + h) * c.S + pos;
  c.scales[(row * 2 + which) * ng + g] = sb;
  uint8_t* dst = (which ? c.vq : c.kq) + row * (c.D / 2) + g * (c.G / 2);
  for (int i = 0; i < c.G; i += 2) {
    uint32_t u[2];
    for (int e = 0; e < 2; ++e) {
      const float r = s > 0.f ? rintf(from16(x[i + e], f16) / s) : 0.f;
      u[e] = (uint32_t)(int)(fminf(fmaxf(r, -7.f), 7.f) + 8.f);
    }
    dst[i / 2] = (uint8_t)(u[0] | (u[1] << 4));
  }
}

// One thread per byte (two values) of a row; rows outside [0, S) read as 0.
__global__ void __launch_bounds__(256) kv4_read_kernel(MqKv4 c, void* k, void* v, int o_type) {
  const int half = c.D / 2, ng = c.D / c.G;
  long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long long)c.B * c.T * c.Hkv * 2 * half) return;
  const int d = (int)(id % half); id /= half;
  const int which = (int)(id & 1); id >>= 1;
  const size_t o = (size_t)id * c.D + 2 * d;
  const int h = (int)(id % c.Hkv); id /= c.Hkv;
  const int t = (int)(id % c.T), b = (int)(id / c.T);
  const long long pos = (long long)c.lengths[b] - c.T + t;
  float lo = 0.f, hi = 0.f;
  if (pos >= 0 && pos < c.S) {
    const size_t row = ((size_t)b * c.Hkv + h) * c.S + pos;
    const float s = bf16_to_f32(c.scales[(row * 2 + which) * ng + 2 * d / c.G]);
    const uint32_t u = (which ? c.vq : c.kq)[row * half + d];
    lo = s * (float)((int)(u & 15) - 8);
    hi = s * (float)((int)(u >> 4) - 8);
  }
  void* out = which ? v : k;
  if (o_type == MQ_T_F32) {
    ((float*)out)[o] = lo;
    ((float*)out)[o + 1] = hi;
  } else {
    ((uint16_t*)out)[o] = to16(lo, o_type == MQ_T_F16);
    ((uint16_t*)out)[o + 1] = to16(hi, o_type == MQ_T_F16);
  }
}

// One wave per (sequence, query row, query head): lanes hold 2 (D = 128) or 1 values of the head.
__global__ void __launch_bounds__(64)
kv4_attend_kernel(MqKv4 c, const uint16_t* q, MqStrides qs, uint16_t* out, int Hq, int max_len,
                  bool f16, float scale_log2) {
  const int lane = threadIdx.x, h = blockIdx.x % Hq, t = blockIdx.x / Hq, b = blockIdx.y;
  const int hk = h / (Hq / c.Hkv), ng = c.D / c.G, per = c.D / 64;
  const long long end = min((long long)c.lengths[b] - c.T + t + 1, (long long)min(c.S, max_len));
  float qv[2] = {0.f, 0.f}, o[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < per; ++e) qv[e] = from16(q[b * qs.b + t * qs.t + h * qs.h + per * lane + e], f16);
  for (long long p = 0; p < end; ++p) {
    const size_t row = ((size_t)b * c.Hkv + hk) * c.S + p;
    const int g = per * lane / c.G;
    float s = 0.f, vv[2];
    for (int e = 0; e < per; ++e) {
      const int d = per * lane + e;
      const int ku = (c.kq[row * (c.D / 2) + d / 2] >> (4 * (d & 1))) & 15;
      const int vu = (c.vq[row * (c.D / 2) + d / 2] >> (4 * (d & 1))) & 15;
      s = fmaf(qv[e], bf16_to_f32(c.scales[(row * 2) * ng + g]) * (float)(ku - 8), s);
      vv[e] = bf16_to_f32(c.scales[(row * 2 + 1) * ng + g]) * (float)(vu - 8);
    }
    s = wave_sum(s) * scale_log2;
    const float mn = fmaxf(m, s), alpha = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = fmaf(l, alpha, w);
    for (int e = 0; e < per; ++e) o[e] = fmaf(o[e], alpha, w * vv[e]);
  }
  uint16_t* dst = out + (((size_t)b * c.T + t) * Hq + h) * c.D + per * lane;
  for (int e = 0; e < per; ++e) dst[e] = to16(end > 0 ? o[e] / l : 0.f, f16);
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : -1; }

}  // namespace

int mq_launch_kv4_append(const MqKv4& c, const uint16_t* k, MqStrides ks, const uint16_t* v,
                         MqStrides vs, bool f16, hipStream_t stream) {
  const long long n = (long long)c.B * c.T * c.Hkv * 2 * (c.D / c.G);
  hipLaunchKernelGGL(kv4_append_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, c, k,
                     ks, v, vs, f16);
  return launched();
}

int mq_launch_kv4_read(const MqKv4& c, void* k, void* v, int o_type, hipStream_t stream) {
  const long long n = (long long)c.B * c.T * c.Hkv * c.D;
  hipLaunchKernelGGL(kv4_read_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, c, k, v,
                     o_type);
  return launched();
}

size_t mq_kv4_attend_workspace(int, int, int, int, int, int, int) { return 0; }

int mq_launch_kv4_attend(const MqKv4& c, const uint16_t* q, MqStrides qs, uint16_t* out, int Hq,
                         int max_len, bool f16, float scale_log2, void*, hipStream_t stream) {
  hipLaunchKernelGGL(kv4_attend_kernel, dim3((unsigned)(c.T * Hq), c.B), dim3(64), 0, stream, c, q, qs,
                     out, Hq, max_len, f16, scale_log2);
  return launched();
}
