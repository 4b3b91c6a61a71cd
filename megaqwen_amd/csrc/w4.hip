// w4.hip — products with 4-bit weights and group scales:
//   out[m][n] = sum_g s[n][g] sum_{k in g} (u[n][k] - z[n][g]) x[m][k]  (+ residual[m][n])
//
// A wave takes 16 outputs n and up to 64 rows m, 128 inputs k at a time: lane (n = l % 16, j = l / 16)
// loads the 16 bytes of codes 32 j .. 32 j + 31 of its output's row, which become operands of 16 x 16 x 32
// matrix products with a shift and an and-or per two codes (mq_nibble.h): the matrix cores do the
// multiplying, so that one row costs what 16 do.  A second product with the constant -(16 + z) takes the
// offset and the zero point off,
//   sum_{k in g} (u - z) x = sum (16 + u) x + sum -(16 + z) x,
// both exact in fp32 but for the sums' roundings; matrix cycles are there to spare, vector instructions
// are not.  A group's sum is scaled and added in fp32.
// All four lanes of an output must work on the same group in one product.  With groups of 128 they do;
// for 64 and 32 the words are first exchanged between the lanes of an output (permlane swaps, one
// instruction per word or half of one), which keeps the 16-byte loads.
//
// Three kernels, by the sizes (w4_plan()):
//   w4_direct_kernel   few outputs: the 8 waves of a workgroup split the inputs of 16 outputs and 16 rows
//                      and load their own pieces of x; nothing waits before the first product
//   w4_whole_kernel    several tiles of 16 outputs per workgroup share the rows of x, which wait in LDS in
//                      operand order; kw waves split a tile's inputs
//   w4_stretch_kernel  the same where the rows do not fit: 512 inputs after the other, two such in LDS
//
// Measured, weights from memory: one row of 1024 to 151936 outputs in fp32 16.4 us, 4.95 TB/s, the rate of a
// large copy; to 4096 outputs 3.0 us of kernel, 7 rows of 3072 to 1024 outputs 4.9, both the latency of
// codes, products and join one after the other; 33 rows of 4096 to 16001 outputs in groups of 32 20 us,
// where vector instructions (47 per 32 inputs of a tile, 6 of them products) are issued in half of the
// cycles, LDS reads take a little less and 16 waves meet at a barrier every 512 inputs.  (Its rows in an order
// that no LDS read conflicts in: no faster, the writes or the loads of x take as much more.)
// x through LDS also keeps the loads of weights ahead of their use: loads return in order, so one of x
// behind them would wait for memory.
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
MQ_DEV void w4_write(const MqW4Args& a, int m, int n, float v) {
  const size_t at = (size_t)m * a.N + n;
  if (a.residual != nullptr) v += w4_residual(a.residual, at, a.o_type);
  w4_store(a.out, at, v, a.o_type);
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
// Step s of lane j is then on the 8 inputs 8 piece .. of the block,
template <int G> MQ_DEV int w4_piece(int step, int j) {
  if constexpr (G == 128) return 4 * j + step;
  else if constexpr (G == 64) return 4 * ((j & 1) + 2 * (step >> 1)) + (step & 1) + 2 * (j >> 1);
  else return 4 * step + j;
}
// and those inputs are at 4 * step + j.
template <int G> MQ_DEV int w4_slot(int piece) {
  const int p = piece >> 2, d = piece & 3;         // loaded by lane p as word d
  if constexpr (G == 128) return 4 * d + p;
  else if constexpr (G == 64) return 4 * (2 * (p >> 1) + (d & 1)) + 2 * (d >> 1) + (p & 1);
  else return 4 * p + d;
}

// Rows n0 .. n0 + rows of a tensor (in scalar registers)
MQ_DEV int w4_outputs(const MqW4Args& a, int n0, int most = 16) { return __builtin_amdgcn_readfirstlane(max(0, min(most, a.N - n0))); }
MQ_DEV __amdgpu_buffer_rsrc_t w4_rsrc(const void* p, int row_bytes, int n0, int rows) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)p + (size_t)n0 * row_bytes), (short)0, rows * row_bytes, 0x00020000);
}
MQ_DEV void w4_codes(uint32_t (&w)[4], __amdgpu_buffer_rsrc_t wr, int K, int col, int j, int b) {
  const int k = 128 * b + 32 * j;
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(wr, k < K ? col * (K / 2) + k / 2 : W4_FAR, 0, 0);
  for (int i = 0; i < 4; ++i) w[i] = v[i];
}

// Scales and zero points of the NS groups of U blocks of 128 inputs of one output.
template <int NS> struct W4Scales {
  uint32_t s[(NS + 1) / 2], z[(NS + 3) / 4];
  MQ_DEV uint32_t scale(int g) const { return g & 1 ? s[g / 2] >> 16 : s[g / 2]; }     // in the low 16 bits
  MQ_DEV uint32_t zero(int g) const { return (z[g / 4] >> (8 * (g & 3))) & 255u; }
};
// Loads the weights of the 16 outputs from n0 on, U blocks at a time: those of outputs >= N and inputs >= K
// return 0 without an access.
template <int G, int U> struct W4Weights {
  static constexpr int NS = U * 128 / G;
  __amdgpu_buffer_rsrc_t wr, sr, zr;
  int K, groups, col, j;
  bool wide, zeros;
  MQ_DEV W4Weights(const MqW4Args& a, int n0, bool wide_scales, int lane, int outputs = 16) {     // (a power of two)
    K = a.K;
    groups = K / G;
    col = lane & (outputs - 1);
    j = lane >> 4;
    wide = wide_scales;
    zeros = a.zeros != nullptr;
    const int rows = w4_outputs(a, n0, outputs);
    wr = w4_rsrc(a.qw, K / 2, n0, rows);
    sr = w4_rsrc(a.scales, groups * 2, n0, rows);
    zr = w4_rsrc(a.zeros, groups, n0, rows);
  }
  // words of block b
  MQ_DEV void codes(uint32_t (&w)[4], int b) const { w4_codes(w, wr, K, col, j, b); }
  // groups of blocks U unit .. U unit + U; those >= groups have scale 0 (and not the next output's first,
  // which may be infinite)
  MQ_DEV void scales(W4Scales<NS>& x, int unit) const {
    int g = NS * unit < groups ? col * groups + NS * unit : W4_FAR / 2;
    asm volatile("" : "+v"(g));          // (opaque: or every group's offset below has a register of its own)
    for (int i = 0; i < (NS + 3) / 4; ++i) x.z[i] = 0x08080808u;
    if (wide) {                          // NS groups are there, and aligned
      if constexpr (NS == 1) x.s[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, 2 * g, 0, 0);
      else if constexpr (NS == 2) x.s[0] = __builtin_amdgcn_raw_buffer_load_b32(sr, 2 * g, 0, 0);
      else if constexpr (NS == 4) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(sr, 2 * g, 0, 0);
        x.s[0] = v[0];
        x.s[1] = v[1];
      } else {
#pragma unroll
        for (int q = 0; q < NS / 8; ++q) {
          const auto v = __builtin_amdgcn_raw_buffer_load_b128(sr, 2 * g + 16 * q, 0, 0);
          for (int i = 0; i < 4; ++i) x.s[4 * q + i] = v[i];
        }
      }
      if (zeros) {
        if constexpr (NS == 1) x.z[0] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, g, 0, 0);
        else if constexpr (NS == 2) x.z[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(zr, g, 0, 0);
        else {
#pragma unroll
          for (int q = 0; q < NS / 4; ++q) x.z[q] = __builtin_amdgcn_raw_buffer_load_b32(zr, g + 4 * q, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const bool in = NS * unit + i < groups;
        const uint32_t s = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, in ? 2 * (g + i) : W4_FAR, 0, 0);
        x.s[i / 2] = i & 1 ? x.s[i / 2] | (s << 16) : s;
        if (zeros) {
          const uint32_t z = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, in ? g + i : W4_FAR, 0, 0);
          x.z[i / 4] = i & 3 ? x.z[i / 4] | (z << (8 * (i & 3))) : z;
        }
      }
    }
  }
};

// acc[t] += the products of a block whose first group is the first-th of sc (fp16: its type; else bf16); x_of(t, step) is the operand of row tile t.  AHEAD: a step's operands are read one step
// ahead, and no further: steps mixed by the scheduler take more registers than there are.
template <bool F16, int G, int MT, bool ONE, bool AHEAD = true, class S, class X>
MQ_DEV void w4_block(nb_f32x4 (&acc)[MT], uint32_t (&d)[4], const S& sc, int first, bool fp16, X x_of) {
  constexpr int SPG = G / 32;            // steps of a group
  w4_exchange<G>(d);
  // (a branch for all scales of the block at once; one per group moves all groups' sums behind the last)
  float f[4 / SPG];
  if (fp16) {
#pragma unroll
    for (int i = 0; i < 4 / SPG; ++i) f[i] = w4_from16(sc.scale(first + i) & 0xffffu, true);
  } else {
#pragma unroll
    for (int i = 0; i < 4 / SPG; ++i) f[i] = __uint_as_float(sc.scale(first + i) << 16);
  }
  uint4 x[MT], zero;
  nb_f32x4 c[MT];
  if constexpr (AHEAD)
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = x_of(t, 0);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    uint4 xn[MT];
    if constexpr (!AHEAD) {
#pragma unroll
      for (int t = 0; t < MT; ++t) x[t] = x_of(t, s);
    } else if (s < 3) {
#pragma unroll
      for (int t = 0; t < MT; ++t) xn[t] = x_of(t, s + 1);
    }
    const int g = first + s / SPG;
    if (s % SPG == 0) {
      const uint32_t z = sc.zero(g), zc = F16 ? 0xcc00u + (z << 6) : 0xc180u + (z << 3);
      const uint32_t zz = zc | (zc << 16);                    // -(16 + z), twice
      zero = make_uint4(zz, zz, zz, zz);
#pragma unroll
      for (int t = 0; t < MT; ++t) c[t] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const uint4 w = nb_expand8<F16>(d[s]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      c[t] = nb_mfma<F16>(x[t], zero, c[t]);
      c[t] = nb_mfma<F16>(x[t], w, c[t]);
    }
    if (s % SPG == SPG - 1) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < (ONE ? 1 : 4); ++i) acc[t][i] = fmaf(f[s / SPG], c[t][i], acc[t][i]);
#pragma unroll
      for (int t = 0; t < MT; ++t) asm volatile("" : "+v"(acc[t]));      // (here, and not behind the next loads)
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (AHEAD)
#pragma unroll
      for (int t = 0; t < MT; ++t) x[t] = xn[t];
  }
}

// Joins the kw waves of every tile of outputs and writes: column col is output n0 + col, register i of
// row tile t row 16 t + 4 j + i.
template <int MT, bool ONE>
MQ_DEV void w4_finish(const MqW4Args& a, const nb_f32x4 (&acc)[MT], int m0, int rows, int wave, int kw, float* red) {
  constexpr int R = ONE ? 1 : 4;
  const int tid = threadIdx.x, lane = tid & 63, tiles = (blockDim.x >> 6) / kw, first = blockIdx.x * tiles * 16;
  if (kw == 1) {
    const int n = first + 16 * wave + (lane & 15);
    if (n >= a.N) return;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int m = 16 * t + 4 * (lane >> 4) + i;
        if (m < rows) w4_write(a, m0 + m, n, acc[t][i]);
      }
    return;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < R; ++i) red[((wave * MT + t) * R + i) * 64 + lane] = acc[t][i];
  __syncthreads();
  for (int id = tid; id < tiles * MT * R * 64; id += blockDim.x) {
    const int ln = id & 63, v = id >> 6, i = v % R, t = v / R % MT, w = v / (R * MT);
    const int m = 16 * t + 4 * (ln >> 4) + i, n = first + 16 * w + (ln & 15);
    if (m >= rows || n >= a.N) continue;
    float sum = 0.f;
    for (int q = 0; q < kw; ++q) sum += red[(((w * kw + q) * MT + t) * R + i) * 64 + ln];
    w4_write(a, m0 + m, n, sum);
  }
}

// 16 rows of the products, 2^slices slices of the inputs: row r is row r % R of x in slice r / R, R = 16 >>
// slices, column c output c % R of the workgroup's R in slice c / R, and what counts of the result is where
// the slices agree.  With few rows of x and few outputs that puts more compute units to work, each of which
// has only so many loads in flight.  Wave w takes blocks w, w + 8, .. of every slice.
template <bool F16, int G, bool ONE>
__global__ void __launch_bounds__(W4_THREADS, 4) w4_direct_kernel(MqW4Args a, bool wide_scales, int slices) {
  constexpr int U = 3;                  // blocks in flight, with their pieces of x
  typedef W4Weights<G, 1> Weights;
  __shared__ float red[W4_WAVES * (ONE ? 1 : 4) * 64];
  const int lane = threadIdx.x & 63, col = lane & 15, j = lane >> 4;
  const int shift = 4 - slices, R = 1 << shift, blocks = (((a.K + 127) / 128) + (1 << slices) - 1) >> slices;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = (col >> shift) * blocks;
  const Weights wt(a, blockIdx.x * R, wide_scales, lane, R);
  const int m0 = 16 * blockIdx.y, rows = min(R, a.M - m0);
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (size_t)m0 * a.K), (short)0, rows * a.K * 2, 0x00020000);
  const int xrow = (ONE ? 0 : min(col & (R - 1), rows - 1)) * a.K;     // (rows past the last read it again)
  struct Stretch {
    uint32_t w[4];
    W4Scales<Weights::NS> sc;
    uint4 x[4];
  };
  auto load = [&](Stretch& y, int b) {
    wt.codes(y.w, first + b);
    wt.scales(y.sc, first + b);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = 128 * (first + b) + 8 * w4_piece<G>(s, j);
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, k < a.K ? 2 * (xrow + k) : W4_FAR, 0, 0);
      y.x[s] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  };
  const bool s16 = a.s_type == MQ_T_F16;
  nb_f32x4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
  Stretch y[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (wave + W4_WAVES * u < blocks) load(y[u], wave + W4_WAVES * u);
  // One output per thread at the end; its residual is on the way from here.
  const int ol = threadIdx.x & (R - 1), om = threadIdx.x >> shift, on = R * blockIdx.x + ol;
  const bool mine = om < rows && on < a.N;
  const size_t out_at = (size_t)(m0 + om) * a.N + on;
  const float residual = mine && a.residual != nullptr ? w4_residual(a.residual, out_at, a.o_type) : 0.f;
  for (int b = wave; b < blocks; b += W4_WAVES * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + W4_WAVES * u < blocks)
        w4_block<F16, G, 1, ONE>(acc, y[u].w, y[u].sc, 0, s16, [&](int, int s) { return nb_order8(y[u].x[s]); });
      if (b + W4_WAVES * (u + U) < blocks) load(y[u], b + W4_WAVES * (u + U));
    }
  }
  constexpr int REGS = ONE ? 1 : 4;     // (one row is in register 0: R is 4 at least)
#pragma unroll
  for (int i = 0; i < REGS; ++i) red[(wave * REGS + i) * 64 + lane] = acc[0][i];
  __syncthreads();
  if (!mine) return;
  float sum = 0.f;
  for (int p = 0; p < 1 << slices; ++p) {
    const int r = R * p + om, at = (r & 3) * 64 + (r >> 2) * 16 + R * p + ol;
#pragma unroll
    for (int q = 0; q < W4_WAVES; ++q) sum += red[q * REGS * 64 + at];
  }
  w4_store(a.out, out_at, sum + residual, a.o_type);
}

struct W4Plan {
  enum { DIRECT, WHOLE, STRETCH } kind;
  int mt;             // tiles of 16 rows
  int kw, waves;      // waves that split the inputs, waves of a workgroup
  int units;          // per wave: w4_unit() blocks each
  int slices;         // w4_direct_kernel
  int lds;            // bytes
  bool wide_scales;   // the scales (and zeros) of a unit (or block, DIRECT) are whole, aligned loads
};

// Rows of x in LDS, in operand order: [rows][block][step][j][8], rows 16 bytes further apart than their
// length, so that they start in different banks.
template <int G> struct W4Rows {
  const uint16_t* x;
  int K, rows, per_row, stride;          // 16-byte pieces of a row; elements
  MQ_DEV W4Rows(const MqW4Args& a, int m0, int rows_, int blocks) {
    x = a.x + (size_t)m0 * a.K;
    K = a.K;
    rows = rows_;
    per_row = 16 * blocks;
    stride = 128 * blocks + 8;
  }
  // piece `id`, zeros from K on
  MQ_DEV uint4 fetch(int id) const {
    const int m = id / per_row, k = 8 * (id - m * per_row);
    return k < K ? ld16(x + (size_t)m * K + k) : make_uint4(0u, 0u, 0u, 0u);
  }
  MQ_DEV void put(uint16_t* dst, int id, uint4 v) const {
    const int m = id / per_row, q = id - m * per_row;
    *(uint4*)(dst + (size_t)m * stride + (q >> 4) * 128 + 8 * w4_slot<G>(q & 15)) = nb_order8(v);
  }
  MQ_DEV void all(uint16_t* dst) const {
    const int total = rows * per_row, threads = blockDim.x;
    for (int id = threadIdx.x; id < total; id += 4 * threads) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (id + i * threads < total) v[i] = fetch(id + i * threads);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (id + i * threads < total) put(dst, id + i * threads, v[i]);
    }
  }
};

#define W4_WHOLE_UNIT 4      // blocks of 128 inputs that a wave has in flight
#define W4_STRETCH_KW 4      // waves that split the inputs, and blocks of a stretch
#define W4_STRETCH_TILES 4   // tiles of 16 outputs
#define W4_STRETCH_WAVES (W4_STRETCH_KW * W4_STRETCH_TILES)
#define W4_STRETCH_ROW (128 * W4_STRETCH_KW + 8)

template <bool F16, int G, int MT, bool ONE>
__global__ void __launch_bounds__(W4_THREADS, MT == 2 ? 2 : G == 32 && !ONE ? 3 : 4) w4_whole_kernel(MqW4Args a, W4Plan pl) {
  constexpr int U = W4_WHOLE_UNIT;
  typedef W4Weights<G, U> Weights;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, col = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = wave / pl.kw, kw = wave - nw * pl.kw;
  const int m0 = blockIdx.y * (16 * MT), rows = min(16 * MT, a.M - m0);
  uint16_t* xs = (uint16_t*)lds;
  const Weights wt(a, (blockIdx.x * (pl.waves / pl.kw) + nw) * 16, pl.wide_scales, lane);
  const bool s16 = a.s_type == MQ_T_F16;
  uint32_t w[U][4];
  W4Scales<Weights::NS> sc;
#pragma unroll
  for (int u = 0; u < U; ++u) wt.codes(w[u], kw * U + u);
  wt.scales(sc, kw);
  const W4Rows<G> rx(a, m0, rows, pl.units * U * pl.kw);
  rx.all(xs);
  nb_f32x4 acc[MT];
  int xrow[MT];                          // (rows past the last read it again; their results are not stored)
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    acc[t] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
    xrow[t] = (ONE ? 0 : min(16 * t + col, rows - 1)) * rx.stride + 8 * j;
  }
  __syncthreads();
  for (int i = 0; i < pl.units; ++i) {
    const bool more = i + 1 < pl.units;
    const int unit = i * pl.kw + kw, next = unit + pl.kw;
    W4Scales<Weights::NS> nsc;
    if (more) wt.scales(nsc, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t d[4] = {w[u][0], w[u][1], w[u][2], w[u][3]};
      if (more) wt.codes(w[u], next * U + u);
      const uint16_t* at = xs + (unit * U + u) * 128;
      w4_block<F16, G, MT, ONE>(acc, d, sc, u * (128 / G), s16, [&](int t, int s) { return *(const uint4*)(at + xrow[t] + 32 * s); });
    }
    sc = nsc;
  }
  if (pl.kw > 1) __syncthreads();
  w4_finish<MT, ONE>(a, acc, m0, rows, wave, pl.kw, (float*)lds);
}

// Scales and zero points of the groups of a block of 128 inputs of one output, packed (WIDE) or one to a
// register.
template <int G, bool WIDE> struct W4BlockScales {
  static constexpr int NS = 128 / G;
  uint32_t s[WIDE ? (NS + 1) / 2 : NS], z[WIDE ? 1 : NS], flip;
  MQ_DEV uint32_t scale(int g) const { return WIDE ? (g & 1 ? s[g / 2] >> 16 : s[g / 2]) : s[g]; }     // in the low 16 bits
  MQ_DEV uint32_t zero(int g) const { return ((WIDE ? z[0] ^ flip : z[g] ^ flip) >> (WIDE ? 8 * g : 0)) & 255u; }
};
// W4Weights a block at a time and without a branch: the compiler's wait for a load that may or may not have
// been followed by others is a wait for all of them, which costs the stretches 10%.  (In the other kernels
// the loads that a branch saves are worth more, about 20 cycles of a compute unit each: the vocabulary's
// product of one row took 20.4 us for 16.4, the q|k|v product of one row 3.7 for 2.6.)
// WIDE: a block's scales are one aligned load, and its zero points.
template <int G, bool WIDE> struct W4Block {
  typedef W4BlockScales<G, WIDE> Scales;
  static constexpr int NS = Scales::NS;
  __amdgpu_buffer_rsrc_t wr, sr, zr;
  int K, groups, col, j;
  uint32_t no_zeros;                     // no zero points: they read as 0, and these bits make them 8
  MQ_DEV W4Block(const MqW4Args& a, int n0, int lane) {
    K = a.K;
    groups = K / G;
    col = lane & 15;
    j = lane >> 4;
    no_zeros = a.zeros == nullptr ? 0x08080808u : 0u;
    const int rows = w4_outputs(a, n0);
    wr = w4_rsrc(a.qw, K / 2, n0, rows);
    sr = w4_rsrc(a.scales, groups * 2, n0, rows);
    zr = w4_rsrc(a.zeros, groups, n0, a.zeros == nullptr ? 0 : rows);
  }
  // words of block b
  MQ_DEV void codes(uint32_t (&w)[4], int b) const { w4_codes(w, wr, K, col, j, b); }
  // its groups; those behind the last have scale 0 (and not the next output's first, which may be infinite)
  MQ_DEV void scales(Scales& x, int b) const {
    x.flip = no_zeros;
    if constexpr (WIDE) {
      int g = NS * b < groups ? col * groups + NS * b : W4_FAR / 2;
      if constexpr (NS == 1) {
        x.s[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, 2 * g, 0, 0);
        x.z[0] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, g, 0, 0);
      } else if constexpr (NS == 2) {
        x.s[0] = __builtin_amdgcn_raw_buffer_load_b32(sr, 2 * g, 0, 0);
        x.z[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(zr, g, 0, 0);
      } else {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(sr, 2 * g, 0, 0);
        x.s[0] = v[0];
        x.s[1] = v[1];
        x.z[0] = __builtin_amdgcn_raw_buffer_load_b32(zr, g, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int g = NS * b + i < groups ? col * groups + NS * b + i : W4_FAR / 2;
        x.s[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, 2 * g, 0, 0);
        x.z[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, g, 0, 0);
      }
    }
  }
};

template <bool F16, int G, bool WIDE, int MT>
__global__ void __launch_bounds__(64 * W4_STRETCH_WAVES, 4) w4_stretch_kernel(MqW4Args a) {
  typedef W4Block<G, WIDE> Weights;
  constexpr int HALF = 16 * MT * W4_STRETCH_ROW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* xs = (uint16_t*)lds;                       // [2] stretches of [16 MT] rows
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = wave / W4_STRETCH_KW, kw = wave % W4_STRETCH_KW;
  const int m0 = blockIdx.y * (16 * MT), rows = min(16 * MT, a.M - m0);
  const Weights wt(a, (blockIdx.x * W4_STRETCH_TILES + nw) * 16, lane);
  const bool s16 = a.s_type == MQ_T_F16;
  // A wave carries 64 pieces of rows wave, wave + 16, ..; rows that are not there are zeros.
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (size_t)m0 * a.K), (short)0, rows * a.K * 2, 0x00020000);
  uint16_t* const put = xs + wave * W4_STRETCH_ROW + (lane >> 4) * 128 + 8 * w4_slot<G>(lane & 15);
  auto fetch = [&](uint4 (&v)[MT], int step) {
    const int k = 128 * W4_STRETCH_KW * step + 8 * lane, at = k < a.K ? 2 * (wave * a.K + k) : W4_FAR;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b128(xr, at + 32 * t * a.K, 0, 0);
      v[t] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  };
  auto store = [&](const uint4 (&v)[MT], int half) {
#pragma unroll
    for (int t = 0; t < MT; ++t) *(uint4*)(put + half * HALF + 16 * t * W4_STRETCH_ROW) = nb_order8(v[t]);
  };
  const int steps = (a.K + 128 * W4_STRETCH_KW - 1) / (128 * W4_STRETCH_KW);
  uint32_t w[2][4];                      // this stretch's and the next's weights
  typename Weights::Scales sc[2];
  uint4 v[2][MT];                        // rows of the next stretch and the one after it
  fetch(v[0], 0);
#pragma unroll
  for (int p = 0; p < 2; ++p) {          // (behind the last block: zeros)
    wt.codes(w[p], W4_STRETCH_KW * p + kw);
    wt.scales(sc[p], W4_STRETCH_KW * p + kw);
  }
  fetch(v[1], 1);
  store(v[0], 0);
  nb_f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
  const uint16_t* const get = xs + col * W4_STRETCH_ROW + 8 * j + 128 * kw;
  auto stretch = [&](auto p_tag, int step) {
    constexpr int P = decltype(p_tag)::value;
    __syncthreads();
    fetch(v[P], step + 2);
    w4_block<F16, G, MT, false, MT < 4>(acc, w[P], sc[P], 0, s16, [&](int t, int s) {
      return *(const uint4*)(get + P * HALF + 16 * t * W4_STRETCH_ROW + 32 * s);
    });
    wt.codes(w[P], W4_STRETCH_KW * (step + 2) + kw);
    wt.scales(sc[P], W4_STRETCH_KW * (step + 2) + kw);
    store(v[1 - P], 1 - P);              // (its readers passed the barrier above)
  };
  for (int step = 0; step < steps; step += 2) {
    stretch(std::integral_constant<int, 0>(), step);
    if (step + 1 < steps) stretch(std::integral_constant<int, 1>(), step + 1);
  }
  __syncthreads();
  w4_finish<MT, false>(a, acc, m0, rows, wave, W4_STRETCH_KW, (float*)lds);
}

// Which kernel, measured in us with weights from memory, groups of 64, bf16 (outputs x inputs):
//  - DIRECT while its workgroups of 16 outputs by 16 rows are few.  They read x for themselves, and further
//    tiles of rows the weights again:
//      rows  outputs x inputs        DIRECT     other    |  outputs x inputs        DIRECT     other
//        1    4096 x 4096               5.2       5.3    |   6144 x 4096               9.5       7.3
//       16    8192 x 1024, 8192    5.3 25.1   6.2 23.3   |  12288 x 1024, 8192    7.3 35.6   6.3 32.1
//       33    4096 x 1024, 8192    6.4 30.5   8.5 33.7   |   8192 x 1024, 8192   10.4 57.2   8.6 33.7
//       64    2048 x 1024, 8192    5.1 23.6   9.6 35.0   |   4096 x 1024, 8192    8.6 45.1   9.8 38.2
//    Its slices, 1, 2 and 4: as many as the rows leave room for while all workgroups are on the chip at once
//    and a slice has 4 blocks, one row of 1024 outputs: 512 inputs 2.5 2.6 2.8, 1024 2.8 2.7 2.9, 3072 5.0 3.6
//    3.3, 8192 8.9 6.0 4.4; 7 rows, 3072: 5.8 4.5.  (16 waves in place of 8, without slices: 5.7.)
//  - WHOLE if two workgroups with all rows of x fit a compute unit: 60000 x 1024, groups of 32: 4 rows 12.2
//    (STRETCH 13.5), 16 rows 14.1 (14.4), 32 rows 18.6 (23.3); 20000 x 2048: 4 rows 12.1 (14.2), 16 rows
//    15.5 (14.9).
//  - Waves that split the inputs leave fewer outputs to share x: as many as fill the chip one and a half
//    times (one row, 40000 x 2048: 15.2, once 16.3; 16 rows, 30000 x 2048: 16.4, twice 21.2).
W4Plan w4_plan(const MqW4Args& a) {
  W4Plan p;
  const int tiles = (a.N + 15) / 16, blocks = (a.K + 127) / 128, rows = a.M < 64 ? a.M : 64;
  p.mt = (rows + 15) / 16;
  p.waves = p.kw = a.M == 1 ? 4 : W4_WAVES;
  p.kind = (long long)tiles * ((a.M + 15) / 16) <= (a.M == 1 ? 256 : a.M <= 16 ? 512 : 768) ? W4Plan::DIRECT
           : p.mt <= 2 && (long long)rows * a.K * 2 <= 65536 ? W4Plan::WHOLE : W4Plan::STRETCH;
  const int unit = p.kind == W4Plan::WHOLE ? W4_WHOLE_UNIT : 1;
  const int ns = unit * 128 / a.G;       // groups loaded at a time
  p.wide_scales = a.K % (ns * a.G) == 0 && ((uintptr_t)a.scales & 15) == 0 && ((uintptr_t)a.zeros & 15) == 0;
  if (p.kind == W4Plan::DIRECT) {
    p.slices = 0;
    while (p.slices < 2 && a.M <= (8 >> p.slices) && (tiles << (p.slices + 1)) <= 256 && (blocks >> (p.slices + 1)) >= 4) ++p.slices;
    return p;
  }
  if (p.kind == W4Plan::STRETCH) {
    p.waves = W4_STRETCH_WAVES;
    p.kw = W4_STRETCH_KW;
    p.lds = 2 * 16 * p.mt * W4_STRETCH_ROW * 2;        // (more than the 16 x 64 x 4 mt sums of the join)
    return p;
  }
  while (p.kw > 1 && (tiles * p.kw > 6144 || unit * (p.kw / 2) >= blocks)) p.kw /= 2;
  p.units = (blocks + unit * p.kw - 1) / (unit * p.kw);
  const int x = rows * (p.units * unit * p.kw * 256 + 16), red = p.kw > 1 ? p.waves * p.mt * 1024 : 0;
  p.lds = x > red ? x : red;
  return p;
}

}  // namespace

int mq_launch_w4_linear(const MqW4Args& a, hipStream_t stream) {
  const W4Plan p = w4_plan(a);
  const int per = 16 * (p.waves / p.kw);                         // outputs of a workgroup
  const unsigned gx = (unsigned)(((long long)a.N + per - 1) / per);
  auto go = [&](auto f16, auto g) {
    constexpr bool F = decltype(f16)::value;
    constexpr int G = decltype(g)::value;
    if (p.kind == W4Plan::DIRECT) {
      const int outputs = 16 >> p.slices;
      const dim3 grid((a.N + outputs - 1) / outputs, (a.M + 15) / 16);
      if (a.M == 1) hipLaunchKernelGGL((w4_direct_kernel<F, G, true>), grid, dim3(W4_THREADS), 0, stream, a, p.wide_scales, p.slices);
      else hipLaunchKernelGGL((w4_direct_kernel<F, G, false>), grid, dim3(W4_THREADS), 0, stream, a, p.wide_scales, p.slices);
      return;
    }
    for (int m0 = 0; m0 < a.M; m0 += 65535 * 64) {               // the grid's second dimension
      MqW4Args b = a;
      const size_t out = a.o_type == MQ_T_F32 ? 4 : 2;
      b.x = a.x + (size_t)m0 * a.K;
      b.out = (char*)a.out + (size_t)m0 * a.N * out;
      if (a.residual != nullptr) b.residual = (const char*)a.residual + (size_t)m0 * a.N * out;
      b.M = a.M - m0 < 65535 * 64 ? a.M - m0 : 65535 * 64;
      const dim3 grid(gx, (unsigned)((b.M + 16 * p.mt - 1) / (16 * p.mt)));
      if (p.kind == W4Plan::WHOLE) {
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * p.waves), p.lds, stream, b, p); };
        launch(a.M == 1 ? w4_whole_kernel<F, G, 1, true> : p.mt == 1 ? w4_whole_kernel<F, G, 1, false> : w4_whole_kernel<F, G, 2, false>);
      } else {
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * p.waves), p.lds, stream, b); };
        auto tiles = [&](auto wide) {
          constexpr bool W = decltype(wide)::value;
          launch(p.mt == 1 ? w4_stretch_kernel<F, G, W, 1> : p.mt == 2 ? w4_stretch_kernel<F, G, W, 2> : p.mt == 3 ? w4_stretch_kernel<F, G, W, 3> : w4_stretch_kernel<F, G, W, 4>);
        };
        if constexpr (G == 128) tiles(std::true_type());             // (always one load)
        else if (p.wide_scales) tiles(std::true_type());
        else tiles(std::false_type());
      }
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
  return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}
