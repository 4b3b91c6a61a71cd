// w4.hip — products with 4-bit weights and group scales:
//   out[m][n] = sum_g s[n][g] sum_{k in g} (u[n][k] - z[n][g]) x[m][k]  (+ residual[m][n])
//
// A wave takes 16 outputs n and up to 64 rows m, 128 inputs k at a time: lane (n = l % 16, j = l / 16)
// loads the 16 bytes of codes 32 j .. 32 j + 31 of its output's row (64 bytes of 16 rows per load), which
// become operands of 16 x 16 x 32 matrix products with a shift and an and-or per two codes
// (mq_nibble.h); the matrix cores do the multiplying, so that one row costs what 16 do.  The rows of x
// wait in LDS in operand order, with their sum over every group:
//   sum_{k in g} (u - z) x = sum (16 + u) x - (16 + z) sum x,
// the second term being where the products' sum starts.  It is scaled and added in fp32 per group.
// All four lanes of an output must work on the same group in one product.  With groups of 128 they do;
// for 64 and 32 the words are first exchanged between the lanes of an output (permlane swaps, one
// instruction per word or half of one), which keeps the 16-byte loads.
// 8 waves share the rows of x: KW of them split the inputs of the same outputs and join at the end.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mq_device.h"
#include "mq_nibble.h"
#include "mq_q4.h"

namespace {

#define W4_WAVES 8
#define W4_THREADS (64 * W4_WAVES)
#define W4_FAR 0x40000000               // a buffer offset behind every buffer: its load returns 0
// blocks of 128 inputs that a wave has in flight, for mt tiles of 16 rows
constexpr int w4_unroll(int mt) { return mt <= 2 ? 4 : 2; }
#define W4_LDS 61440                    // bytes of x (and its sums) staged at a time

MQ_DEV float w4_from16(uint32_t bits, bool f16) {
  return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __uint_as_float(bits << 16);
}
MQ_DEV void w4_store(void* out, size_t i, float v, int type) {
  if (type == MQ_T_F32) ((float*)out)[i] = v;
  else if (type == MQ_T_F16) ((uint16_t*)out)[i] = __builtin_bit_cast(uint16_t, (_Float16)v);
  else ((uint16_t*)out)[i] = f32_to_bf16(v);
}
MQ_DEV float w4_residual(const void* r, size_t i, int type) {
  return type == MQ_T_F32 ? ((const float*)r)[i] : w4_from16(((const uint16_t*)r)[i], type == MQ_T_F16);
}

// Words d[s] of lane j as step s of the products: afterwards step s's four lanes hold words of one group.
template <int G> MQ_DEV void w4_exchange(uint32_t (&d)[4]) {
  if constexpr (G <= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    d[0] = p[0]; d[1] = q[0]; d[2] = p[1]; d[3] = q[1];
  }
  if constexpr (G == 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(d[0], d[1], false, false);
    const auto q = __builtin_amdgcn_permlane16_swap(d[2], d[3], false, false);
    d[0] = p[0]; d[1] = p[1]; d[2] = q[0]; d[3] = q[1];
  }
}
// Where the 8 inputs 8 piece .. of a block of 128 are then: 4 * step + lane j
template <int G> MQ_DEV int w4_slot(int piece) {
  const int p = piece >> 2, d = piece & 3;         // loaded by lane p as word d
  if constexpr (G == 128) return 4 * d + p;
  else if constexpr (G == 64) return 4 * (2 * (p >> 1) + (d & 1)) + 2 * (d >> 1) + (p & 1);
  else return 4 * p + d;
}

struct W4Plan {
  int blocks;         // of 128 inputs, the last one possibly cut
  int kw;             // waves that split the inputs; W4_WAVES / kw tiles of 16 outputs per workgroup
  int steps;          // times w4_unroll() blocks per wave for all of K
  int chunk;          // such steps per staging of x
  int lds;            // bytes
  bool wide_scales;   // a block's scales (and zeros) are one aligned load
};

template <bool F16, int G, int MT, bool ONE>
__global__ void __launch_bounds__(W4_THREADS, MT <= 2 ? 4 : 2) w4_kernel(MqW4Args a, W4Plan pl) {
  constexpr int PER = 128 / G, U = w4_unroll(MT);      // groups of a block; blocks of a step
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = wave / pl.kw, kw = wave - nw * pl.kw;
  const int n0 = (blockIdx.x * (W4_WAVES / pl.kw) + nw) * 16;
  const int m0 = blockIdx.y * (16 * MT), rows = min(16 * MT, a.M - m0);
  const int groups = a.K / G, tile_rows = max(0, min(16, a.N - n0));
  const int cblocks = pl.chunk * U * pl.kw;                  // blocks staged at a time
  const int xstride = cblocks * 128 + 8;                             // (8: rows start in different banks)
  uint16_t* xs = (uint16_t*)lds;                                     // [rows][block][step][j][8]
  float* xsum = (float*)(lds + (((size_t)rows * xstride * 2 + 15) & ~(size_t)15));   // [group][16 MT]

  // Rows of this wave's outputs: loads of rows >= N, and of inputs >= K, return 0 without an access.
  auto rsrc = [&](const void* p, int row_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)p + (size_t)n0 * row_bytes), (short)0, tile_rows * row_bytes, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t wr = rsrc(a.qw, a.K / 2), sr = rsrc(a.scales, groups * 2), zr = rsrc(a.zeros, groups);
  struct Block {
    uint32_t w[4], s[PER > 1 ? PER / 2 : 1], z;
  };
  auto load = [&](Block& x, int b) {
    const int k = 128 * b + 32 * j;
    const auto w = __builtin_amdgcn_raw_buffer_load_b128(wr, k < a.K ? col * (a.K / 2) + k / 2 : W4_FAR, 0, 0);
    for (int i = 0; i < 4; ++i) x.w[i] = w[i];
    const int g = col * groups + PER * b;
    x.z = 0x08080808u;
    if (PER == 1 || pl.wide_scales) {
      const int so = b < pl.blocks ? 2 * g : W4_FAR;
      if constexpr (PER == 4) {
        const auto s = __builtin_amdgcn_raw_buffer_load_b64(sr, so, 0, 0);
        x.s[0] = s[0];
        x.s[1] = s[1];
      } else if constexpr (PER == 2) x.s[0] = __builtin_amdgcn_raw_buffer_load_b32(sr, so, 0, 0);
      else x.s[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, so, 0, 0);
      if (a.zeros != nullptr) {
        const int zo = b < pl.blocks ? g : W4_FAR;
        if constexpr (PER == 4) x.z = __builtin_amdgcn_raw_buffer_load_b32(zr, zo, 0, 0);
        else if constexpr (PER == 2) x.z = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(zr, zo, 0, 0);
        else x.z = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, zo, 0, 0);
      }
    } else if constexpr (PER > 1) {
      uint32_t z = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const bool in = PER * b + i < groups;
        const uint32_t s = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, in ? 2 * (g + i) : W4_FAR, 0, 0);
        x.s[i / 2] = i & 1 ? x.s[i / 2] | (s << 16) : s;
        if (a.zeros != nullptr) z |= (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, in ? g + i : W4_FAR, 0, 0) << (8 * i);
      }
      if (a.zeros != nullptr) x.z = z;
    }
  };
  auto load_step = [&](Block (&x)[U], int step) {
#pragma unroll
    for (int u = 0; u < U; ++u) load(x[u], (step * U + u) * pl.kw + kw);
  };

  // Rows m0 .. m0 + rows of inputs from 128 c0 on, in operand order, and the sums of their groups.
  auto stage = [&](int c0) {
    const int blocks = min(cblocks, pl.blocks - c0), pieces = blocks * 16;
    for (int id = tid; id < rows * pieces; id += W4_THREADS) {
      const int m = id / pieces, q = id - m * pieces, b = q >> 4, k = (c0 + b) * 128 + 8 * (q & 15);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (k < a.K) v = ld16(a.x + (size_t)(m0 + m) * a.K + k);
      *(uint4*)(xs + (size_t)m * xstride + b * 128 + 8 * w4_slot<G>(q & 15)) = nb_order8(v);
      float s = nb_sum8<F16>(v);
      s += dpp_f<MQ_DPP_QUAD_XOR1>(s);
      s += dpp_f<MQ_DPP_QUAD_XOR2>(s);
      if constexpr (G >= 64) s += dpp_f<MQ_DPP_ROW_HALF_MIRROR>(s);
      if constexpr (G >= 128) s += dpp_f<MQ_DPP_ROW_MIRROR>(s);
      if ((q & (G / 8 - 1)) == 0) xsum[(size_t)(q / (G / 8)) * (16 * MT) + m] = s;
    }
  };

  nb_f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
  int xrow[MT];                          // (rows past the last read it again; their results are not stored)
#pragma unroll
  for (int t = 0; t < MT; ++t) xrow[t] = (ONE ? 0 : min(16 * t + col, rows - 1)) * xstride + 8 * j;
  const bool s16 = a.s_type == MQ_T_F16;

  auto compute = [&](const Block& x, int b) {        // b: block of the staged ones
    uint32_t d[4] = {x.w[0], x.w[1], x.w[2], x.w[3]};
    w4_exchange<G>(d);
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      const float z = -NB_OFFSET - (float)((x.z >> (8 * g)) & 255u);
      const float* sums = xsum + (size_t)(b * PER + g) * (16 * MT) + (ONE ? 0 : 4 * j);
      nb_f32x4 c[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (ONE) c[t] = nb_f32x4{z * sums[0], 0.f, 0.f, 0.f};
        else c[t] = *(const nb_f32x4*)(sums + 16 * t) * z;
      }
#pragma unroll
      for (int s = 4 / PER * g; s < 4 / PER * (g + 1); ++s) {
        const uint4 w = nb_expand8<F16>(d[s]);
#pragma unroll
        for (int t = 0; t < MT; ++t) c[t] = nb_mfma<F16>(*(const uint4*)(xs + xrow[t] + b * 128 + 32 * s), w, c[t]);
      }
      const float sc = w4_from16((x.s[g / 2] >> (16 * (g & 1))) & 0xffffu, s16);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (ONE) acc[t][0] = fmaf(sc, c[t][0], acc[t][0]);
        else
          for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(sc, c[t][i], acc[t][i]);
      }
    }
  };

  Block cur[U];
  load_step(cur, 0);
  for (int step = 0; step < pl.steps; ++step) {
    Block nxt[U];
    const int c0 = step / pl.chunk * pl.chunk * U * pl.kw;
    if (step % pl.chunk == 0) {
      if (step > 0) __syncthreads();
      stage(c0);
      __syncthreads();
    }
    if (step + 1 < pl.steps) load_step(nxt, step + 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = (step * U + u) * pl.kw + kw;
      if (b < pl.blocks) compute(cur[u], b - c0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = nxt[u];
  }

  // Results: column col is output n0 + col, register i of tile t row 16 t + 4 j + i
  auto write = [&](int m, int n, float v) {
    if (m >= rows || n >= a.N) return;
    const size_t at = (size_t)(m0 + m) * a.N + n;
    if (a.residual != nullptr) v += w4_residual(a.residual, at, a.o_type);
    w4_store(a.out, at, v, a.o_type);
  };
  if (pl.kw == 1) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < (ONE ? 1 : 4); ++i) write(16 * t + 4 * j + i, n0 + col, acc[t][i]);
    return;
  }
  __syncthreads();
  constexpr int R = ONE ? 1 : 4;
  float* red = (float*)lds;              // [wave][MT][R][64]
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < R; ++i) red[((wave * MT + t) * R + i) * 64 + lane] = acc[t][i];
  __syncthreads();
  for (int id = tid; id < W4_WAVES / pl.kw * MT * R * 64; id += W4_THREADS) {
    const int ln = id & 63, v = id >> 6, t = v / R % MT, i = v % R, w = v / (R * MT);
    float sum = 0.f;
    for (int q = 0; q < pl.kw; ++q) sum += red[(((w * pl.kw + q) * MT + t) * R + i) * 64 + ln];
    write(16 * t + 4 * (ln >> 4) + i, (blockIdx.x * (W4_WAVES / pl.kw) + w) * 16 + (ln & 15), sum);
  }
}

}  // namespace

int mq_launch_w4_linear(const MqW4Args& a, hipStream_t stream) {
  const int mt = a.M > 48 ? 4 : (a.M + 15) / 16, rows = a.M < 16 * mt ? a.M : 16 * mt;
  const long long tiles = (a.N + 15) / 16;
  const int unroll = w4_unroll(mt);
  W4Plan p;
  p.blocks = (a.K + 127) / 128;
  p.kw = W4_WAVES;
  while (p.kw > 1 && (tiles * p.kw > 4096 || p.kw > p.blocks)) p.kw /= 2;
  p.steps = (p.blocks + unroll * p.kw - 1) / (unroll * p.kw);
  // x and its sums of some steps: rows * (256 blocks + 16 of padding) + 4 * 16 mt * (128 / G) blocks
  auto bytes = [&](int chunk) {
    const size_t blocks = (size_t)chunk * unroll * p.kw;
    return ((size_t)rows * (blocks * 256 + 16) + 15) / 16 * 16 + blocks * (128 / a.G) * 64 * mt;
  };
  while (p.kw > 1 && bytes(1) > W4_LDS) {
    p.kw /= 2;
    p.steps = (p.blocks + unroll * p.kw - 1) / (unroll * p.kw);
  }
  p.chunk = 1;
  while (p.chunk < p.steps && bytes(p.chunk + 1) <= W4_LDS) ++p.chunk;
  const size_t red = p.kw > 1 ? (size_t)W4_WAVES * mt * 1024 : 0;
  p.lds = (int)(bytes(p.chunk) > red ? bytes(p.chunk) : red);
  p.wide_scales = a.K % 128 == 0 && ((uintptr_t)a.scales & 7) == 0 && ((uintptr_t)a.zeros & 3) == 0;
  const int per = W4_WAVES / p.kw;
  const unsigned gx = (unsigned)((tiles + per - 1) / per);
  auto go = [&](auto f16, auto g) {
    constexpr bool F = decltype(f16)::value;
    constexpr int G = decltype(g)::value;
    for (int m0 = 0; m0 < a.M; m0 += 65535 * 64) {          // the grid's second dimension
      MqW4Args b = a;
      const size_t out = a.o_type == MQ_T_F32 ? 4 : 2;
      b.x = a.x + (size_t)m0 * a.K;
      b.out = (char*)a.out + (size_t)m0 * a.N * out;
      if (a.residual != nullptr) b.residual = (const char*)a.residual + (size_t)m0 * a.N * out;
      b.M = a.M - m0 < 65535 * 64 ? a.M - m0 : 65535 * 64;
      const dim3 grid(gx, (unsigned)((b.M + 16 * mt - 1) / (16 * mt)));
      if (b.M == 1 && mt == 1) hipLaunchKernelGGL((w4_kernel<F, G, 1, true>), grid, dim3(W4_THREADS), p.lds, stream, b, p);
      else if (mt == 1) hipLaunchKernelGGL((w4_kernel<F, G, 1, false>), grid, dim3(W4_THREADS), p.lds, stream, b, p);
      else if (mt == 2) hipLaunchKernelGGL((w4_kernel<F, G, 2, false>), grid, dim3(W4_THREADS), p.lds, stream, b, p);
      else if (mt == 3) hipLaunchKernelGGL((w4_kernel<F, G, 3, false>), grid, dim3(W4_THREADS), p.lds, stream, b, p);
      else hipLaunchKernelGGL((w4_kernel<F, G, 4, false>), grid, dim3(W4_THREADS), p.lds, stream, b, p);
    }
  };
  auto pick = [&](auto f16) {
    using std::integral_constant;
    if (a.G == 128) go(f16, integral_constant<int, 128>());
    else if (a.G == 64) go(f16, integral_constant<int, 64>());
    else go(f16, integral_constant<int, 32>());
  };
  if (a.x_type == MQ_T_F16) pick(std::true_type());
  else pick(std::false_type());
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
