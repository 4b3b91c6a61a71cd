// kv4.hip — a key/value cache held in 4 bits: rows are quantised into it (append), read back as
// the values they stand for (read), and attended over (attend).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mq_device.h"
#include "mq_nibble.h"
#include "mq_q4.h"

namespace {

MQ_DEV uint16_t to16(float v, bool f16) {
  return f16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : f32_to_bf16(v);
}

// Rows of 8-value pieces: a thread takes one of (t, piece), the grid's second dimension is (key or
// value, kv head) and its third the sequence.  A head's rows are neighbours in the cache, so that a
// wave writes (append) or reads 256 bytes of codes in a row; on the other side every row of a head
// is D 2 bytes in a row.  3 x 2731 tokens of 8 heads of 128, keys and values: append 9.8 us, read 10.9, of 42 MB
// each (4.3 and 3.9 TB/s; memory bounds both, a large copy reaches 5.1).  Append took 17 us with divisions,
// for quotients and for the thread's place.
struct KvPiece {
  int t, piece, h;
  bool which, in;                  // value rows; a row of the call
  long long pos;                   // the cache row, or < 0 or >= S
};
MQ_DEV KvPiece kv_piece(const MqKv4& c, int b) {
  const int shift = c.D == 128 ? 4 : 3, id = blockIdx.x * 256 + threadIdx.x;
  KvPiece p;
  p.t = id >> shift;
  p.piece = id & ((1 << shift) - 1);
  p.which = blockIdx.y >= (unsigned)c.Hkv;
  p.h = p.which ? blockIdx.y - c.Hkv : blockIdx.y;
  p.in = p.t < c.T;
  p.pos = (long long)c.lengths[b] - c.T + p.t;
  return p;
}

//   s = bf16(max|x| / 7) over the group's G / 8 threads, u = clamp(rint(x / s), -7, 7) + 8; s = 0:
//   u = 8; a group that holds an infinity or a NaN gets s = NaN, so that all of its values read as NaN.
// Quotients are reciprocals with one correction, q' = q + (x - q s) r: off by an ulp or two of fp32 at
// most, and exact where x / s has few bits.  x has up to 11 bits and s 8, so x / s is either exactly
// half a step, and then so is q', or at least 2^-12 of it away: no code differs from the exact
// quotient's.  The same holds for max / 7 and the midpoints of bf16.  Below 2^-60 the products could
// underflow, and the quotients are divisions.
template <bool F16, int G>
__global__ void __launch_bounds__(256) kv4_append_kernel(MqKv4 c, const uint16_t* k, MqStrides ks, const uint16_t* v, MqStrides vs) {
  const int b = blockIdx.z;
  const KvPiece p = kv_piece(c, b);
  if (!p.in) return;               // (whole groups)
  const MqStrides st = p.which ? vs : ks;
  const uint4 x = nb_load16((p.which ? v : k) + b * st.b + p.t * st.t + p.h * st.h + 8 * p.piece);
  const float f[8] = {nb_lo<F16>(x.x), nb_hi<F16>(x.x), nb_lo<F16>(x.y), nb_hi<F16>(x.y),
                      nb_lo<F16>(x.z), nb_hi<F16>(x.z), nb_lo<F16>(x.w), nb_hi<F16>(x.w)};
  // (maximum keeps a NaN; the lanes of a group are in the same row of 16)
  float m = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __builtin_elementwise_maximum(m, fabsf(f[i]));
  m = __builtin_elementwise_maximum(m, dpp_f<MQ_DPP_QUAD_XOR1>(m));
  m = __builtin_elementwise_maximum(m, dpp_f<MQ_DPP_QUAD_XOR2>(m));
  if constexpr (G >= 64) m = __builtin_elementwise_maximum(m, dpp_f<MQ_DPP_ROW_HALF_MIRROR>(m));
  if constexpr (G >= 128) m = __builtin_elementwise_maximum(m, dpp_f<MQ_DPP_ROW_MIRROR>(m));
  auto quotient = [](float a, float d, float r) {
    const float q = a * r;
    return fmaf(fmaf(-q, d, a), r, q);
  };
  uint32_t w = 0;
  uint16_t sb;
  if (m >= 0x1p-60f && m < INFINITY) {
    sb = f32_to_bf16(quotient(m, 7.0f, 1.0f / 7.0f));
    const float s = bf16_to_f32(sb), r = __builtin_amdgcn_rcpf(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the sum's last bits: its rounding is rint's, 8 is added, and the constant ends in four zeros
      const float u = __builtin_amdgcn_fmed3f(quotient(f[i], s, r), -7.f, 7.f) + (0x1.8p23f + 8.f);
      w |= (__float_as_uint(u) & 15u) << (4 * i);
    }
  } else {
    sb = m < INFINITY ? f32_to_bf16(m / 7.0f) : 0x7fc0;
    const float s = bf16_to_f32(sb);
    for (int i = 0; i < 8; ++i) {
      const float r = s > 0.f ? rintf(f[i] / s) : 0.f;
      w |= (uint32_t)(int)(fminf(fmaxf(r, -7.f), 7.f) + 8.f) << (4 * i);
    }
  }
  if (p.pos < 0 || p.pos >= c.S) return;
  const size_t row = ((size_t)b * c.Hkv + p.h) * c.S + p.pos;
  ((uint32_t*)(p.which ? c.vq : c.kq))[row * (c.D / 8) + p.piece] = w;
  if (p.piece % (G / 8) == 0) c.scales[(row * 2 + p.which) * (c.D / G) + p.piece / (G / 8)] = sb;
}

// Rows outside [0, S) read as 0.
__global__ void __launch_bounds__(256) kv4_read_kernel(MqKv4 c, void* k, void* v, int o_type) {
  const int b = blockIdx.z, per = c.D / 8, gshift = c.G == 32 ? 2 : c.G == 64 ? 3 : 4;
  const KvPiece p = kv_piece(c, b);
  if (!p.in) return;
  float s = 0.f;
  uint32_t u = 0;
  if (p.pos >= 0 && p.pos < c.S) {
    const size_t row = ((size_t)b * c.Hkv + p.h) * c.S + p.pos;
    s = bf16_to_f32(c.scales[(row * 2 + p.which) * (per >> gshift) + (p.piece >> gshift)]);
    u = ((const uint32_t*)(p.which ? c.vq : c.kq))[row * per + p.piece];
  }
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = s * (float)((int)((u >> (4 * i)) & 15u) - 8);
  const size_t o = ((((size_t)b * c.T + p.t) * c.Hkv + p.h) * per + p.piece) * 8;
  void* out = p.which ? v : k;
  if (o_type == MQ_T_F32) {
    float4* dst = (float4*)((float*)out + o);
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    const bool f16 = o_type == MQ_T_F16;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)to16(f[2 * i], f16) | ((uint32_t)to16(f[2 * i + 1], f16) << 16);
    *(uint4*)((uint16_t*)out + o) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- attention
//
// A workgroup is (sequence, kv head, a tile of its query rows, a share of the positions); its waves take
// 32 positions at a time and join their (max, sum, O) at the end.  Query rows of a kv head are
// r = t (Hq / Hkv) + head, so that a cached row is read once for all of them.
//   * S = K Q^T by 16 x 16 x 32 products of the codes (mq_nibble.h) and the unrounded queries.  A
//     key row has a scale per group of its dims, which no product can sum over: the 16 columns are
//     (query row, group) pairs, column c holding row c / NG with all dims outside group c % NG
//     zero.  Each score is the sum of its NG columns, times their scales, over neighbouring lanes.
//   * the result's layout, a lane with 2 x 4 positions of one column, is the operand layout of
//     O^T += V^T P^T: the weights go from registers into the next product.  Column (row, g) carries
//     the weights times the value scales of group g, and only the dims of group g are kept of it.
//   * weights enter as a truncated bf16 and the bf16 of the remainder (16 bits of each), so that their
//     rounding stays far below the output's; one bf16 would add an error of the output's own size.
// Softmax statistics and sums are fp32.  Codes are 4 bytes (8 dims) per lane for values, so that a
// lane sees 8 positions of the same dims without a transpose through LDS.  (16 bytes of a position per
// lane, exchanged among 4 lanes, are 2 loads for 8 but more instructions: 5 to 10% slower.)
//
// Measured, bf16 and fp16 with the join: one sequence of 32768 rows, 8 kv heads of 2 query heads, groups of
// 32, 15.4 us (37.8 MB, 2.45 TB/s: 9.5 us of kernel and 3.9 of join); 24 sequences up to 8191 rows, 4 query
// heads per kv head, 34 us (112 MB, 3.3 TB/s); 509 queries over 6007 rows 45 us (540 TFLOP/s).  Vector
// instructions bound it: about 260 per 32 positions and column tile (310 for two tiles), issued in 70% of the
// cycles, beside 26 products (52).
#define AT_TILE 32                 // positions per wave and step
#define AT_RAISE 8.0f              // a column's reference point moves when a score exceeds it by 2^8
#define AT_BIAS (NB_OFFSET + 8.0f)

struct AtArgs {
  MqKv4 c;
  const uint16_t* q;
  MqStrides qs;
  uint16_t* out;
  float2* ml;                      // [rows][nsplit] (max, sum) and
  float* part;                     // [rows][nsplit][D] unnormalised sums, if nsplit > 1
  int Hq, ratio, max_len, nsplit;
  uint32_t by_ratio, by_hkv;       // at_magic()
  float scale_log2;
};
// n / d as the upper half of n ceil(2^32 / d): exact for n (d - 1) < 2^32 (d <= 256 and n <= 2^24 here)
uint32_t at_magic(int d) { return d == 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d); }
MQ_DEV int at_div(int n, uint32_t magic) { return magic == 0 ? n : (int)__umulhi((uint32_t)n, magic); }

// 16 bits of a word as the upper half of an fp32 (a bf16 scale), chosen by a byte selector
MQ_DEV float at_pick(uint32_t hi, uint32_t lo, uint32_t sel) { return __uint_as_float(__builtin_amdgcn_perm(hi, lo, sel)); }
MQ_DEV float at_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }    // (fmaxf canonicalises its operands first)
// a + a's value in the lane that DPP control CTRL names
template <int CTRL> MQ_DEV float at_add_dpp(float a) {
#pragma clang fp contract(off)
  return a + dpp_f<CTRL>(a);
}
// a b, and 0 where a or b is 0 whatever the other: a masked position's weight is 0, its scale may be NaN.
// (The instruction by its intrinsic: between transcendentals and matrix products the compiler has to place
// wait states, which it does not for instructions written as inline assembly.)
extern "C" __device__ float at_mul0(float a, float b) __asm("llvm.amdgcn.fmul.legacy");
// Two weights as the truncated bf16 and the bf16 of the remainder
MQ_DEV void at_split2(float w0, float w1, uint32_t& hi, uint32_t& lo) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  hi = __builtin_amdgcn_perm(__float_as_uint(w1), __float_as_uint(w0), 0x07060302u);
  // w - hi as a two-element product with (-1, 0) and (0, -1), in registers that the compiler cannot see
  // through: as a constant it would encode (-1, 0) as -1.0, which the hardware reads as (0, -1)
  uint32_t c0 = 0x0000bf80u, c1 = 0xbf800000u;
  asm("" : "+s"(c0), "+s"(c1));
  const v2 h = __builtin_bit_cast(v2, hi);
  const f2 r = {__builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(v2, c0), w0, false),
                __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(v2, c1), w1, false)};
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2));
}

// Scales of positions 16 t + 4 j + i of a tile, as a lane holds them
template <int NG> struct AtScales {
  uint32_t s[NG == 1 ? 8 : 16];
};

template <bool F16, int D, int NG, int CT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, CT == 1 ? 4 : 2) kv4_attend_kernel(AtArgs a) {
  constexpr int KW = D / 32;       // words of a key row per lane
  constexpr int DPL = D / 16;      // dims of a value row per lane
  constexpr int RQ = 16 / NG;      // query rows per column tile
  constexpr int G = D / NG;
  typedef AtScales<NG> Scales;
  __shared__ float red[WAVES][4 * DPL][64];
  __shared__ float4 red_ml[WAVES][CT][16];       // m, l, and the sum that the offset is taken off by
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, j = lane >> 4, g = col % NG;
  // the kv head is the fastest index: workgroups go round the 8 XCDs, so that those that read the
  // same rows share an L2
  const int rt = at_div(blockIdx.x, a.by_hkv), hk = blockIdx.x - rt * a.c.Hkv, split = blockIdx.y, b = blockIdx.z;
  const int rows = a.c.T * a.ratio, r0 = rt * (CT * RQ);
  const int cap = min(a.c.S, a.max_len);
  // rows of this (sequence, kv head): loads beyond its last row return 0 without an access
  const size_t row = ((size_t)b * a.c.Hkv + hk) * a.c.S;
  auto rsrc = [&](const void* base, int row_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + row * row_bytes), (short)0, cap * row_bytes, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t kr = rsrc(a.c.kq, D / 2), vr = rsrc(a.c.vq, D / 2), sr = rsrc(a.c.scales, 4 * NG);
  // A tile: K words of position 16 t + col, dims (D / 4) j + ..; value dims DPL col + .. of positions
  // 16 t + 4 j + i.  The next tile's words are loaded over a tile's as soon as those are used.
  uint32_t kw[2][KW], vw[8];
  auto load_keys = [&](int p) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int ko = (p + 16 * t + col) * (D / 2) + j * (4 * KW);
      if constexpr (KW == 4) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b128(kr, ko, 0, 0);
        for (int s = 0; s < 4; ++s) kw[t][s] = w[s];
      } else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(kr, ko, 0, 0);
        for (int s = 0; s < 2; ++s) kw[t][s] = w[s];
      }
    }
  };
  auto load_values = [&](int p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pos = p + 16 * (e >> 2) + 4 * j + (e & 3);
      if constexpr (DPL == 8) vw[e] = __builtin_amdgcn_raw_buffer_load_b32(vr, pos * (D / 2) + 4 * col, 0, 0);
      else vw[e] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vr, pos * (D / 2) + 2 * col, 0, 0);
    }
  };
  auto load_scales = [&](Scales& x, int p) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (NG == 1) {           // (key, value) scale pairs of 4 positions
        const auto w = __builtin_amdgcn_raw_buffer_load_b128(sr, (p + 16 * t + 4 * j) * 4, 0, 0);
        for (int i = 0; i < 4; ++i) x.s[4 * t + i] = w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = p + 16 * t + 4 * j + i, e = 4 * t + i;
        if constexpr (NG == 2) {         // both groups of key and value, two positions at a time
          if (i & 1) continue;
          const auto w = __builtin_amdgcn_raw_buffer_load_b128(sr, pos * 8, 0, 0);
          for (int q = 0; q < 4; ++q) x.s[2 * e + q] = w[q];
        } else if constexpr (NG == 4) {
          x.s[2 * e] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, pos * 16 + 2 * g, 0, 0);
          x.s[2 * e + 1] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, pos * 16 + 8 + 2 * g, 0, 0);
        }
      }
    }
  };
  // positions that query t looks at: first + t, in [0, cap]
  const int first = min(max(a.c.lengths[b], 0), 1 << 28) - a.c.T + 1;
  auto limit = [&](int r) { return max(0, min(cap, first + at_div(r, a.by_ratio))); };
  const int end = limit(min(r0 + CT * RQ, rows) - 1), sure = limit(r0);
  // A range is contiguous (ranges dealt out tile by tile read 15% slower); without ranges a wave's first
  // tile does not depend on the length.
  constexpr int STRIDE = AT_TILE * WAVES;
  int p = AT_TILE * wave, p1 = end;
  if (a.nsplit > 1) {
    const int chunk = ((end + a.nsplit - 1) / a.nsplit + STRIDE - 1) / STRIDE * STRIDE;
    p += split * chunk;
    p1 = min(end, (split + 1) * chunk);
  }
  Scales sx, sy;
  load_keys(p);
  load_scales(sx, p);
  load_values(p);
  // scores are taken with the scale's sign in the queries, so that the largest stays the largest; a scale
  // of 0 is one next to it, so that a masked score, -inf, stays -inf
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);

  uint4 qf[CT][KW];
  // m: a column's reference point (lowest: none yet), l: its sum of weights in this lane's positions
  float m[CT], l[CT];
  int lim[CT];
  nb_f32x4 acc[CT][DPL], sv[CT];   // sv: the sums of the weights times the value scales, in every row
  nb_f32x4 cinit[CT];              // -24 times the sum of the column's queries: the codes' offset
  constexpr uint32_t BIAS2 = F16 ? 0xce00ce00u : 0xc1c0c1c0u;         // (-24, -24)
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int r = r0 + ct * RQ + col / NG;
    const bool there = r < rows;
    const int t = there ? at_div(r, a.by_ratio) : 0, h = there ? hk * a.ratio + r - t * a.ratio : 0;
    const uint16_t* qr = a.q + b * a.qs.b + t * a.qs.t + h * a.qs.h;
    cinit[ct] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      const int d = (D / 4) * j + 8 * s;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (there && d / G == g) {
        x = nb_order8(nb_load16(qr + d));
        x = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
      }
      qf[ct][s] = x;
      cinit[ct] = nb_mfma<F16>(make_uint4(BIAS2, BIAS2, BIAS2, BIAS2), x, cinit[ct]);
    }
    lim[ct] = there ? limit(r) : 0;
    m[ct] = -3.402823466e38f;
    l[ct] = 0.f;
    sv[ct] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[ct][i] = nb_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint32_t half = NG == 2 && g == 1 ? 0x03020c0cu : 0x01000c0cu;      // (0x0c: a zero byte)
  auto key_scale = [&](const Scales& x, int e) {
    if constexpr (NG == 1) return __uint_as_float(x.s[e] << 16);
    else if constexpr (NG == 2) return at_pick(x.s[2 * e], x.s[2 * e], half);
    else return __uint_as_float(x.s[2 * e] << 16);
  };
  auto value_scale = [&](const Scales& x, int e) {
    if constexpr (NG == 1) return __uint_as_float(x.s[e] & 0xffff0000u);
    else if constexpr (NG == 2) return at_pick(x.s[2 * e + 1], x.s[2 * e + 1], half);
    else return __uint_as_float(x.s[2 * e + 1] << 16);
  };

  auto step = [&](const Scales& x, Scales& next, int p) {
    // scores z[ct][e], not yet scaled, of positions p + 16 (e / 4) + 4 j + e % 4
    float z[CT][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      nb_f32x4 s[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct] = cinit[ct];
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint4 kx = nb_expand8<F16>(kw[t][w]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[ct] = nb_mfma<F16>(kx, qf[ct][w], s[ct]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ks = key_scale(x, 4 * t + i);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          float v = s[ct][i] * ks;
          if constexpr (NG >= 2) v = at_add_dpp<MQ_DPP_QUAD_XOR1>(v);
          if constexpr (NG >= 4) v = at_add_dpp<MQ_DPP_QUAD_XOR2>(v);
          z[ct][4 * t + i] = v;
        }
      }
    }
    load_keys(p + STRIDE);               // (past the end: not used)
    load_scales(next, p + STRIDE);
    if (p + AT_TILE > sure) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (p + 16 * (e >> 2) + 4 * j + (e & 3) >= lim[ct]) z[ct][e] = -INFINITY;
          asm volatile("" : "+v"(z[ct][e]));     // (keeps this a branch: few tiles need it)
        }
    }
    uint4 ph[CT], pl[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mt = at_max(at_max(at_max(z[ct][0], z[ct][1]), z[ct][2]), at_max(at_max(z[ct][3], z[ct][4]), at_max(z[ct][5], at_max(z[ct][6], z[ct][7]))));
      float2 pr = swap16(mt);
      mt = at_max(pr.x, pr.y);
      pr = swap32(mt);
      mt = at_max(pr.x, pr.y) * scale;
      if (__builtin_amdgcn_ballot_w64(mt > m[ct] + AT_RAISE) != 0) {
        const bool up = mt > m[ct] + AT_RAISE;
        const float alpha = up ? __builtin_amdgcn_exp2f(m[ct] - mt) : 1.0f;
        m[ct] = up ? mt : m[ct];
        l[ct] *= alpha;
        sv[ct] *= alpha;
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[ct][i] *= alpha;
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p_ = __builtin_amdgcn_exp2f(fmaf(z[ct][e + i], scale, -m[ct]));
          l[ct] += p_;
          w[i] = at_mul0(p_, value_scale(x, e + i));
        }
        at_split2(w[0], w[1], hi[e / 2], lo[e / 2]);
      }
      ph[ct] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      pl[ct] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) sv[ct] = nb_mfma<false>(ones, pl[ct], nb_mfma<false>(ones, ph[ct], sv[ct]));
    // value codes of position pairs in the halves of a word: words f of wl hold dims DPL col + f
    uint32_t wl[4], wh[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      wl[t] = __builtin_amdgcn_perm(vw[2 * t + 1], vw[2 * t], 0x05040100u);
      if constexpr (DPL == 8) wh[t] = __builtin_amdgcn_perm(vw[2 * t + 1], vw[2 * t], 0x07060302u);
    }
    load_values(p + STRIDE);
    auto values = [&](auto f_tag, const uint32_t (&w)[4], int i) {
      constexpr int f = decltype(f_tag)::value;
      const uint4 va = make_uint4(nb_pair<false, f>(w[0]), nb_pair<false, f>(w[1]), nb_pair<false, f>(w[2]), nb_pair<false, f>(w[3]));
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        acc[ct][i] = nb_mfma<false>(va, ph[ct], acc[ct][i]);
        acc[ct][i] = nb_mfma<false>(va, pl[ct], acc[ct][i]);
      }
    };
    values(std::integral_constant<int, 0>(), wl, 0);
    values(std::integral_constant<int, 1>(), wl, 1);
    values(std::integral_constant<int, 2>(), wl, 2);
    values(std::integral_constant<int, 3>(), wl, 3);
    if constexpr (DPL == 8) {
      values(std::integral_constant<int, 0>(), wh, 4);
      values(std::integral_constant<int, 1>(), wh, 5);
      values(std::integral_constant<int, 2>(), wh, 6);
      values(std::integral_constant<int, 3>(), wh, 7);
    }
  };
  for (; p < p1; p += 2 * STRIDE) {
    step(sx, sy, p);
    if (p + STRIDE >= p1) break;
    step(sy, sx, p + STRIDE);
  }

  // Join the waves.  A column's O, without the codes' offset, is in value order i' DPL + i, where
  // dim = DPL (4 j + i') + i.
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] = sum_xor32(sum_xor16(l[ct]));
    if (j == 0) red_ml[wave][ct][col] = make_float4(m[ct], l[ct], sv[ct][0], 0.f);
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DPL; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][e * DPL + i][lane] = acc[ct][i][e];
    __syncthreads();
    if (wave >= 4) continue;
    float mx = -INFINITY, sum = 0.f, off = 0.f, f[WAVES];
    float4 v[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v[w] = red_ml[w][ct][col];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, v[w].x);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {      // (a wave without a position: sums of 0 at the lowest m)
      f[w] = __builtin_amdgcn_exp2f(v[w].x - mx);
      sum = fmaf(v[w].y, f[w], sum);
      off = fmaf(v[w].z, f[w], off);
    }
    // wave i' of the workgroup: dims DPL (4 j + i') .. + DPL of the lane's column
    float o[DPL];
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      o[i] = -AT_BIAS * off;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) o[i] = fmaf(red[w][wave * DPL + i][lane], f[w], o[i]);
    }
    const int r = r0 + ct * RQ + col / NG, d = DPL * (4 * j + wave);
    if (r >= rows || d / G != g) continue;
    const int t = at_div(r, a.by_ratio);
    const size_t at = ((size_t)b * a.c.T + t) * a.Hq + hk * a.ratio + r - t * a.ratio;
    if (a.nsplit == 1) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      uint32_t w[DPL / 2];
#pragma unroll
      for (int i = 0; i < DPL; i += 2)
        w[i / 2] = (uint32_t)to16(o[i] * inv, F16) | ((uint32_t)to16(o[i + 1] * inv, F16) << 16);
      uint32_t* dst = (uint32_t*)(a.out + at * D + d);
#pragma unroll
      for (int i = 0; i < DPL / 2; ++i) dst[i] = w[i];
    } else {
      if (d == 0) a.ml[at * a.nsplit + split] = make_float2(mx, sum);
      if (sum != 0.f) {
        float* dst = a.part + (at * a.nsplit + split) * D + d;
#pragma unroll
        for (int i = 0; i < DPL; ++i) dst[i] = o[i];
      }
    }
  }
}

// Joins the ranges of a query row.  A row is WAVES waves (1 for few ranges, 4 for many), a thread 4
// dims of every SLOTS-th range; ranges without a position (sum 0) have nothing stored.
template <int D, int WAVES>
__global__ void __launch_bounds__(256) kv4_join_kernel(const float2* ml, const float* part, uint16_t* out, int rows, int nsplit, bool f16) {
  constexpr int DT = D / 4, SLOTS = 64 * WAVES / DT;
  __shared__ float4 red[4][DT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = lane % DT, slot = (threadIdx.x & (64 * WAVES - 1)) / DT;
  const size_t at = (size_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  if (at >= (size_t)rows) return;                       // (whole waves; with 4 waves a row there is no rest)
  const float2* mr = ml + at * nsplit;
  float mx = -INFINITY, sum = 0.f;
  for (int s = lane; s < nsplit; s += 64) mx = fmaxf(mx, mr[s].x);
  mx = wave_max(mx);
  for (int s = lane; s < nsplit; s += 64) {
    const float2 v = mr[s];
    sum = v.y == 0.f ? sum : fmaf(v.y, __builtin_amdgcn_exp2f(v.x - mx), sum);
  }
  sum = wave_sum(sum);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = slot; s < nsplit; s += SLOTS) {
    const float4 p = ((const float4*)part)[(at * nsplit + s) * DT + d];
    const float2 v = mr[s];
    const float f = __builtin_amdgcn_exp2f(v.x - mx);
    o.x = v.y == 0.f ? o.x : fmaf(p.x, f, o.x);
    o.y = v.y == 0.f ? o.y : fmaf(p.y, f, o.y);
    o.z = v.y == 0.f ? o.z : fmaf(p.z, f, o.z);
    o.w = v.y == 0.f ? o.w : fmaf(p.w, f, o.w);
  }
  auto across = [](float v) {
    v = sum_xor32(v);
    return DT == 16 ? sum_xor16(v) : v;
  };
  o = make_float4(across(o.x), across(o.y), across(o.z), across(o.w));
  if constexpr (WAVES == 4) {
    if (lane < DT) red[wave][lane] = o;
    __syncthreads();
    if (threadIdx.x >= DT) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 p = red[w][d];
      o = make_float4(o.x + p.x, o.y + p.y, o.z + p.z, o.w + p.w);
    }
  } else if (lane >= DT) {
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const uint32_t lo = (uint32_t)to16(o.x * inv, f16) | ((uint32_t)to16(o.y * inv, f16) << 16);
  const uint32_t hi = (uint32_t)to16(o.z * inv, f16) | ((uint32_t)to16(o.w * inv, f16) << 16);
  ((uint2*)out)[at * DT + d] = make_uint2(lo, hi);
}

// How a call is laid out.  Measured on 8 kv heads of 128 dims, bf16 and fp16:
//  - query rows: one column tile if they fit, else two tiles per step, so that a tile's codes are
//    read out of the registers twice (509 queries over 6007 rows: one tile 55 us, two 45 us).
//  - waves: a workgroup's waves go through its positions in turns of 32.  Two column tiles take 8
//    waves (4: 51 us for the 45 above), one tile 4 (a batch of 24 ragged sequences up to 8191 rows,
//    4 query heads per kv head: 33.8 us, 8 waves 36.6 at their best; one sequence of 32768 rows 15.4
//    and 14.8).
//  - ranges: every workgroup costs about 2 us besides its positions, so one sequence gets as many as
//    fill the 256 CUs once (32768 rows: 256 workgroups 15.4 us, 512 15.6, 1024 19.6; the 509
//    queries: 256 45 us, 512 58).  Sequences in a batch differ in length and their workgroups with
//    them; more per CU even that out: four of one tile (256 43 us, 512 40, 1024 34, 1536 36), two of
//    two tiles (24 sequences of 4 query rows of 4 heads: 256 56 us, 512 53, 1024 66; of 2 rows of 2
//    heads in groups of 32: 41, 36, 32; 5 sequences of 16 rows of 2 heads: 30, 34, 43).
//    No range is shorter than AT_RANGE positions, and up to twice that one workgroup takes them all:
//    the join is a kernel more.
constexpr int AT_RANGE = 256;
struct AtPlan {
  int ct, row_tiles, nsplit;
};
AtPlan at_plan(int B, int T, int Hq, int Hkv, int D, int G, int max_len) {
  AtPlan p;
  const int rq = 16 / (D / G), rows = T * (Hq / Hkv);
  p.ct = rows <= rq ? 1 : 2;
  p.row_tiles = (rows + p.ct * rq - 1) / (p.ct * rq);
  const long long wgs = (long long)B * Hkv * p.row_tiles, fill = B == 1 ? 256 : p.ct == 2 ? 512 : 1024;
  const int want = (int)((fill + wgs - 1) / wgs), most = max_len <= 2 * AT_RANGE ? 1 : (max_len + AT_RANGE - 1) / AT_RANGE;
  p.nsplit = want < most ? want : most;
  return p;
}

int launched() { return hipPeekAtLastError() == hipSuccess ? 0 : -1; }

}  // namespace

// (the host has checked T Hkv <= 2^26 and Hkv <= 256)
static dim3 kv4_row_grid(const MqKv4& c) { return dim3(((unsigned)c.T * (c.D / 8) + 255) / 256, 2 * c.Hkv, c.B); }

int mq_launch_kv4_append(const MqKv4& c, const uint16_t* k, MqStrides ks, const uint16_t* v,
                         MqStrides vs, bool f16, hipStream_t stream) {
  auto go = [&](auto f16_, auto g) {
    hipLaunchKernelGGL((kv4_append_kernel<decltype(f16_)::value, decltype(g)::value>), kv4_row_grid(c), dim3(256), 0, stream, c,
                       k, ks, v, vs);
  };
  auto pick = [&](auto f16_) {
    if (c.G == 32) go(f16_, std::integral_constant<int, 32>());
    else if (c.G == 64) go(f16_, std::integral_constant<int, 64>());
    else go(f16_, std::integral_constant<int, 128>());
  };
  if (f16) pick(std::true_type());
  else pick(std::false_type());
  return launched();
}

int mq_launch_kv4_read(const MqKv4& c, void* k, void* v, int o_type, hipStream_t stream) {
  hipLaunchKernelGGL(kv4_read_kernel, kv4_row_grid(c), dim3(256), 0, stream, c, k, v, o_type);
  return launched();
}

size_t mq_kv4_attend_workspace(int B, int T, int Hq, int Hkv, int D, int G, int max_len) {
  const AtPlan p = at_plan(B, T, Hq, Hkv, D, G, max_len);
  if (p.nsplit == 1) return 0;
  const size_t rows = (size_t)B * T * Hq * p.nsplit;
  return (rows * sizeof(float2) + 15) / 16 * 16 + rows * D * sizeof(float);
}

int mq_launch_kv4_attend(const MqKv4& c, const uint16_t* q, MqStrides qs, uint16_t* out, int Hq,
                         int max_len, bool f16, float scale_log2, void* ws, hipStream_t stream) {
  const AtPlan p = at_plan(c.B, c.T, Hq, c.Hkv, c.D, c.G, max_len);
  const size_t rows = (size_t)c.B * c.T * Hq;
  AtArgs a = {c, q, qs, out, (float2*)ws, (float*)((char*)ws + (rows * p.nsplit * sizeof(float2) + 15) / 16 * 16),
              Hq, Hq / c.Hkv, max_len, p.nsplit, at_magic(Hq / c.Hkv), at_magic(c.Hkv), scale_log2};
  const dim3 grid((unsigned)(c.Hkv * p.row_tiles), (unsigned)p.nsplit, (unsigned)c.B), block(p.ct == 2 ? 512 : 256);
  auto go = [&](auto f16_, auto d, auto ng) {
    constexpr bool F = decltype(f16_)::value;
    constexpr int D = decltype(d)::value, NG = decltype(ng)::value;
    if (p.ct == 2) hipLaunchKernelGGL((kv4_attend_kernel<F, D, NG, 2, 8>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv4_attend_kernel<F, D, NG, 1, 4>), grid, block, 0, stream, a);
    if (p.nsplit >= 16)
      hipLaunchKernelGGL((kv4_join_kernel<D, 4>), dim3((unsigned)rows), dim3(256), 0, stream, a.ml, a.part, out, (int)rows, p.nsplit, F);
    else if (p.nsplit > 1)
      hipLaunchKernelGGL((kv4_join_kernel<D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a.ml, a.part, out, (int)rows, p.nsplit, F);
  };
  auto pick = [&](auto f16_) {
    using std::integral_constant;
    const int ng = c.D / c.G;
    if (c.D == 128) {
      if (ng == 4) go(f16_, integral_constant<int, 128>(), integral_constant<int, 4>());
      else if (ng == 2) go(f16_, integral_constant<int, 128>(), integral_constant<int, 2>());
      else go(f16_, integral_constant<int, 128>(), integral_constant<int, 1>());
    } else {
      if (ng == 2) go(f16_, integral_constant<int, 64>(), integral_constant<int, 2>());
      else go(f16_, integral_constant<int, 64>(), integral_constant<int, 1>());
    }
  };
  if (f16) pick(std::true_type());
  else pick(std::false_type());
  return launched();
}
