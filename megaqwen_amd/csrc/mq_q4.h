// 4-bit weights and the 4-bit key/value cache (w4.hip, kv4.hip): host launchers.
//
// A code u (0..15) stands for s (u - z): s is the scale of its group of consecutive values, z = 8
// where there are no zero points.  A byte holds two codes, the even value in its low half.
// Every launcher returns 0, or -1 if the launch failed.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

// Storage types, numbered as MQ_DTYPE_* of the C interface.
enum { MQ_T_BF16 = 0, MQ_T_F16 = 1, MQ_T_F32 = 2 };

// out[m][n] = sum_k x[m][k] w[n][k] (+ residual[m][n]) for rows m < M.  x: contiguous [M, K] of
// x_type (bf16 or fp16), 16-byte aligned; qw: bytes [N, K / 2], 16-byte aligned; scales [N, K / G]
// of s_type (bf16 or fp16); zeros: bytes [N, K / G] or null; residual (or null) and out:
// contiguous [M, N] of o_type.  G is 32, 64 or 128 and divides K; M, N, K >= 1.
struct MqW4Args {
  const uint16_t* x;
  const uint8_t* qw;
  const uint16_t* scales;
  const uint8_t* zeros;
  const void* residual;
  void* out;
  int M, N, K, G, x_type, s_type, o_type;
};
int mq_launch_w4_linear(const MqW4Args& a, hipStream_t stream);

// The cache: codes [B, Hkv, S, D / 2] for keys and for values, scales (bf16) [B, Hkv, S, 2, D / G],
// the key's scales before the value's.  lengths (device, int32 [B]) counts a sequence's rows with
// the T rows of the call: row t of sequence b is at position lengths[b] - T + t.
struct MqKv4 {
  uint8_t* kq;
  uint8_t* vq;
  uint16_t* scales;
  const int* lengths;
  int B, T, Hkv, D, S, G;
};
// Element strides of a [B, T, H, D] tensor whose last dimension is contiguous.
struct MqStrides {
  long long b, t, h;
};
// Quantises rows k, v [B, T, Hkv, D] (bf16, or fp16 if f16) into the cache.
int mq_launch_kv4_append(const MqKv4& c, const uint16_t* k, MqStrides ks, const uint16_t* v,
                         MqStrides vs, bool f16, hipStream_t stream);
// The values of the T rows of every sequence, contiguous [B, T, Hkv, D] of o_type.
int mq_launch_kv4_read(const MqKv4& c, void* k, void* v, int o_type, hipStream_t stream);
// Attention of queries [B, T, Hq, D] over the cache, out contiguous [B, T, Hq, D] of the same type.
// max_len bounds the positions looked at.  ws: mq_kv4_attend_workspace() bytes.
size_t mq_kv4_attend_workspace(int B, int T, int Hq, int Hkv, int D, int G, int max_len);
int mq_launch_kv4_attend(const MqKv4& c, const uint16_t* q, MqStrides qs, uint16_t* out, int Hq,
                         int max_len, bool f16, float scale_log2, void* ws, hipStream_t stream);
