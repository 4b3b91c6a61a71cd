// logprobs.hip — log probability of a given token in every row of logits, the row's entropy and its
// most likely tokens, in one pass over the logits.  With m = max x, y = (x - m) log2 e,
// s = sum 2^y and t = sum 2^y y:
//   log p(token) = x[token] - m - log s,   entropy = ln 2 (log2 s - t / s).
// A workgroup takes a slice of a row: all of it where there are rows enough to fill the chip, one of
// up to 64 otherwise, which a second kernel joins.
//
// The top_k (k <= 32) of a slice: the workgroup's threads fall into 32 groups of 16 lanes, and the
// k-th largest of the groups' maxima, B, is a lower bound of the k-th largest value.  Only threads
// whose own maximum reaches B look at their elements again, which finds somewhat more than k
// candidates (value, index), ranked by counting.
//
// Measured: 2047 rows of 151936 bf16 logits with 5 alternatives 115 us, 5.4 TB/s: memory bounds it.  One row
// in fp32 with 20 alternatives: slices 6.4 us, join 4.9, the latency of each kernel's few dependent passes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mq_device.h"
#include "mq_logprobs.h"

namespace {

#define LP_THREADS 512
#define LP_WAVES (LP_THREADS / 64)
#define LP_GROUPS (LP_THREADS / 16)   // at least MQ_TOP_MAX
#define LP_CAP 1024                   // candidates of a slice held in LDS
#define LP_SLICES 64                  // most slices of a row (one lane each in the join)
#define LP_LOG2E 1.44269504088896340736f
#define LP_LN2 0.69314718055994530942f
#define LP_FLOOR -216.f               // 2^-216 is 0: weights from there on are, and y stays finite

template <int TYPE> struct LpType {
  static constexpr int VEC = TYPE == 2 ? 4 : 8;
  typedef typename std::conditional<TYPE == 2, float, uint16_t>::type raw;
};
template <int TYPE> MQ_DEV float lp_float(typename LpType<TYPE>::raw v) {
  if constexpr (TYPE == 2) return v;
  else if constexpr (TYPE == 1) return (float)__builtin_bit_cast(_Float16, v);
  else return bf16_to_f32(v);
}
// 16 bytes at any address aligned to an element, as floats
template <int TYPE> MQ_DEV void lp_load(const typename LpType<TYPE>::raw* p, float* x) {
  struct __attribute__((packed, aligned(TYPE == 2 ? 4 : 2))) Loose { uint32_t w[4]; };
  const Loose v = *(const Loose*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TYPE == 2) x[i] = __uint_as_float(v.w[i]);
    else {
      x[2 * i] = lp_float<TYPE>((uint16_t)v.w[i]);
      x[2 * i + 1] = lp_float<TYPE>((uint16_t)(v.w[i] >> 16));
    }
  }
}

MQ_DEV float lp_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN stays

// Sums of a running softmax; m = -inf, s = t = 0: no element, or -inf alone.  NaN: m = NaN.
struct LpSum {
  float m, s, t;
};
MQ_DEV float lp_y(float x, float m) { return fmaxf((x - m) * LP_LOG2E, LP_FLOOR); }    // (-inf) - (-inf): the floor
MQ_DEV LpSum lp_join(LpSum a, LpSum b) {
  LpSum r;
  r.m = lp_max(a.m, b.m);
  const float da = lp_y(a.m, r.m), db = lp_y(b.m, r.m);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  r.s = fa * a.s + fb * b.s;
  r.t = fa * fmaf(a.s, da, a.t) + fb * fmaf(b.s, db, b.t);
  return r;
}
// Over the 64 lanes: the maximum first, then the sums at it.
MQ_DEV float lp_wave_max(float v) {
  v = lp_max(v, dpp_f<MQ_DPP_QUAD_XOR1>(v));
  v = lp_max(v, dpp_f<MQ_DPP_QUAD_XOR2>(v));
  v = lp_max(v, dpp_f<MQ_DPP_ROW_HALF_MIRROR>(v));
  v = lp_max(v, dpp_f<MQ_DPP_ROW_MIRROR>(v));
  float2 p = swap16(v);
  p = swap32(lp_max(p.x, p.y));
  return lp_max(p.x, p.y);
}
// (lane 0's in every lane: the order of a sum differs between lanes)
MQ_DEV LpSum lp_wave_join(LpSum r) {
  auto first = [](float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); };
  const float m = first(lp_wave_max(r.m)), d = lp_y(r.m, m), f = __builtin_amdgcn_exp2f(d);
  return LpSum{m, first(wave_sum(f * r.s)), first(wave_sum(f * fmaf(r.s, d, r.t)))};
}
// n more elements
template <int N> MQ_DEV void lp_add(LpSum& r, const float (&x)[N]) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = lp_max(mx, x[i]);
  const float m = lp_max(r.m, mx), d = lp_y(r.m, m), f = __builtin_amdgcn_exp2f(d);
  r.t = f * fmaf(r.s, d, r.t);
  r.s *= f;
  r.m = m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = lp_y(x[i], m), e = __builtin_amdgcn_exp2f(y);
    r.s += e;
    r.t = fmaf(e, y, r.t);
  }
}

MQ_DEV uint64_t lp_key(float v, int i) { return argmax_key(v + 0.f, (uint32_t)i); }    // -0 counts as +0
MQ_DEV float lp_key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

struct LpShared {
  LpSum sums[LP_WAVES];
  alignas(16) float group[LP_GROUPS];
  int n_gt, n_eq, n_scan;
  uint64_t best[LP_WAVES];
  uint16_t scan[LP_THREADS];
  uint64_t gt[LP_CAP], eq[LP_CAP];
};

// Where a row's results go
struct LpRow {
  float lse_m, ls;            // log p = x - lse_m - ls
  bool bad, empty;
};
MQ_DEV float lp_of(const LpRow& r, float x) { return r.bad ? NAN : r.empty ? -INFINITY : x - r.lse_m - r.ls; }
MQ_DEV LpRow lp_row(LpSum r) {
  LpRow w;
  w.bad = !(r.m < INFINITY);
  w.empty = r.m == -INFINITY;
  w.lse_m = r.m;
  w.ls = __builtin_amdgcn_logf(r.s) * LP_LN2;
  return w;
}
// The logit of a row's token, and whether it has one (loaded at a kernel's start, used at its end)
struct LpToken {
  float x;
  bool in;
};
template <int TYPE> MQ_DEV LpToken lp_token(const MqLogprobArgs& a, int row) {
  const long long tok = a.tok64 ? ((const long long*)a.tokens)[row] : ((const int*)a.tokens)[row];
  const bool in = tok >= 0 && tok < a.vocab;
  return LpToken{lp_float<TYPE>(((const typename LpType<TYPE>::raw*)a.logits)[(long long)row * a.stride + (in ? tok : 0)]), in};
}
MQ_DEV void lp_write(const MqLogprobArgs& a, int row, LpSum r, const LpRow& w, LpToken tok) {
  a.logprob[row] = tok.in ? lp_of(w, tok.x) : w.bad ? NAN : -INFINITY;
  a.entropy[row] = w.bad ? NAN : w.empty ? 0.f : (__builtin_amdgcn_logf(r.s) - r.t / r.s) * LP_LN2;
}

// Ranks the n keys of LDS and hands key i of the first k to put(i, key).
template <class Put> MQ_DEV void lp_rank(const uint64_t* keys, int n, int k, Put put) {
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const uint64_t mine = keys[c];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += keys[i] > mine;
    if (rank < k) put(rank, mine);
  }
}

template <int TYPE>
__global__ void __launch_bounds__(LP_THREADS) lp_slice_kernel(MqLogprobArgs a, int slices, int slice, LpSum* part_sum, uint64_t* part_key) {
  typedef typename LpType<TYPE>::raw raw;
  constexpr int VEC = LpType<TYPE>::VEC, UNROLL = 4;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / slices, sl = blockIdx.x - row * slices;
  const int lo = sl * slice, n = min(slice, a.vocab - lo);      // n >= 1
  const raw* x = (const raw*)a.logits + (long long)row * a.stride + lo;
  LpToken tok = {};
  if (slices == 1 && tid == 0) tok = lp_token<TYPE>(a, row);

  // Thread t has vectors t, t + 512, ..  and one of the last elements, or, in a slice too short to give
  // every thread a vector, elements t, t + 512, ..
  const bool wide = n >= LP_THREADS * VEC;
  const int nvec = wide ? n / VEC : 0, rest = wide ? n - nvec * VEC : 0;
  LpSum r = {-INFINITY, 0.f, 0.f};
  if (wide) {
    int v = tid;
    for (; v + (UNROLL - 1) * LP_THREADS < nvec; v += UNROLL * LP_THREADS) {
      float e[UNROLL * VEC];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) lp_load<TYPE>(x + (size_t)(v + u * LP_THREADS) * VEC, e + u * VEC);
      lp_add(r, e);
    }
    for (; v < nvec; v += LP_THREADS) {
      float e[VEC];
      lp_load<TYPE>(x + (size_t)v * VEC, e);
      lp_add(r, e);
    }
    if (tid < rest) {
      const float e[1] = {lp_float<TYPE>(x[nvec * VEC + tid])};
      lp_add(r, e);
    }
  } else {
    for (int i = tid; i < n; i += LP_THREADS) {
      const float e[1] = {lp_float<TYPE>(x[i])};
      lp_add(r, e);
    }
  }
  const float mine = r.m;
  r = lp_wave_join(r);
  if (lane == 0) sh.sums[wave] = r;
  // (a group's maximum: NaN counts as the largest here; such a row's order is by index, below)
  float gm = mine;
  gm = lp_max(gm, dpp_f<MQ_DPP_QUAD_XOR1>(gm));
  gm = lp_max(gm, dpp_f<MQ_DPP_QUAD_XOR2>(gm));
  gm = lp_max(gm, dpp_f<MQ_DPP_ROW_HALF_MIRROR>(gm));
  gm = lp_max(gm, dpp_f<MQ_DPP_ROW_MIRROR>(gm));
  if ((lane & 15) == 0) sh.group[tid >> 4] = gm;
  if (tid == 0) sh.n_gt = sh.n_eq = sh.n_scan = 0;
  __syncthreads();
  r = lane < LP_WAVES ? sh.sums[lane] : LpSum{-INFINITY, 0.f, 0.f};
  r = lp_wave_join(r);
  const LpRow out = lp_row(r);
  if (tid == 0) {
    if (slices == 1) lp_write(a, row, r, out, tok);
    else part_sum[blockIdx.x] = r;
  }
  const int k = a.top_k;
  if (k == 0) return;
  auto put = [&](int i, uint64_t key) {
    if (slices > 1) {
      part_key[(size_t)blockIdx.x * k + i] = key;
    } else {
      a.top_tok[(size_t)row * k + i] = (int)argmax_key_index(key);
      a.top_lp[(size_t)row * k + i] = lp_of(out, lp_key_value(key));
    }
  };
  const int kk = min(k, n);
  if (tid >= kk && tid < k) put(tid, 0);          // a slice of fewer than k elements (never a whole row)
  if (r.m != r.m) {
    // a NaN in the row: tokens in the order of their index (the join orders the slices' NaN by index too)
    if (tid < kk) put(tid, lp_key(NAN, lo + tid));
    return;
  }
  // B: the kk-th largest of the groups' maxima; lane l counts, of those larger than group l % 32's, the
  // ones in one half of the groups
  const int gi = lane & (LP_GROUPS - 1), g0 = (lane >> 5) * (LP_GROUPS / 2);
  const float g = sh.group[gi];
  int above = 0;
#pragma unroll
  for (int i = 0; i < LP_GROUPS / 2; ++i) {
    const float o = sh.group[g0 + i];
    above += o > g || (o == g && g0 + i < gi);
  }
  above += __builtin_amdgcn_ds_bpermute((lane ^ 32) << 2, above);
  const uint64_t at = __builtin_amdgcn_ballot_w64(above == kk - 1);
  const float bound = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), __builtin_ctzll(at)));
  if (mine >= bound) sh.scan[atomicAdd(&sh.n_scan, 1)] = (uint16_t)tid;
  __syncthreads();
  auto look = [&](float v, int i) {
    if (v > bound) {
      const int c = atomicAdd(&sh.n_gt, 1);
      if (c < LP_CAP) sh.gt[c] = lp_key(v, lo + i);
    } else if (v == bound) {
      const int c = atomicAdd(&sh.n_eq, 1);
      if (c < LP_CAP) sh.eq[c] = lp_key(v, lo + i);
    }
  };
  // (thread, vector) pairs over the workgroup; a thread's last element counts as a vector
  const int scans = sh.n_scan, full = wide ? (nvec + LP_THREADS - 1) / LP_THREADS : (n + LP_THREADS - 1) / LP_THREADS;
  const int per = full + (rest > 0);
  for (int id = tid; id < scans * per; id += LP_THREADS) {
    const int c = id / per, q = id - c * per, t = sh.scan[c], v = t + q * LP_THREADS;
    if (!wide) {
      if (v < n) look(lp_float<TYPE>(x[v]), v);
    } else if (q == full) {
      if (t < rest) look(lp_float<TYPE>(x[nvec * VEC + t]), nvec * VEC + t);
    } else if (v < nvec) {
      float e[VEC];
      lp_load<TYPE>(x + (size_t)v * VEC, e);
      float mx = e[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) mx = fmaxf(mx, e[i]);
      if (mx >= bound) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) look(e[i], v * VEC + i);
      }
    }
  }
  __syncthreads();
  const int n_gt = sh.n_gt, n_eq = sh.n_eq;
  if (n_gt > LP_CAP) {
    // Too many above B (values crowded into few threads): one pass per alternative.
    uint64_t prev = ~0ull;
    for (int i = 0; i < kk; ++i) {
      uint64_t best = 0;
      for (int e = tid; e < n; e += LP_THREADS) {
        const uint64_t key = lp_key(lp_float<TYPE>(x[e]), lo + e);
        if (key < prev && key > best) best = key;
      }
      best = wave_max_u64(best);
      __syncthreads();
      if (lane == 0) sh.best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < LP_WAVES; ++w) best = u64_max(best, sh.best[w]);
      prev = best;
      if (tid == 0) put(i, best);
    }
    return;
  }
  if (n_gt >= kk) {
    lp_rank(sh.gt, n_gt, kk, put);
    return;
  }
  if (n_eq > LP_CAP) {
    // Many values equal to B (-inf or the lowest value as a mask, flat rows): the lowest indices, by an
    // ordered walk of wave 0 that ends when it has enough.
    if (wave == 0) {
      int have = 0;
      for (int i0 = 0; i0 < n && have < kk - n_gt; i0 += 64) {
        const bool hit = i0 + lane < n && lp_float<TYPE>(x[min(i0 + lane, n - 1)]) == bound;
        const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
        const int c = have + __popcll(hits & ((1ull << lane) - 1));
        if (hit && c < kk - n_gt) put(n_gt + c, lp_key(bound, lo + i0 + lane));
        have += __popcll(hits);
      }
    }
  } else {
    lp_rank(sh.eq, n_eq, kk - n_gt, [&](int i, uint64_t key) { put(n_gt + i, key); });
  }
  lp_rank(sh.gt, n_gt, n_gt, put);
}

// Joins a row's slices: one workgroup of 256 threads per row.  The j-th keys of the slices,
// j = ceil(k / slices), bound the k-th largest key from below by their ceil(k / j)-th largest.
template <int TYPE>
__global__ void __launch_bounds__(256) lp_join_kernel(MqLogprobArgs a, int slices, const LpSum* part_sum, const uint64_t* part_key) {
  constexpr int HELD = LP_SLICES * MQ_TOP_MAX / 256;
  __shared__ uint64_t cand[LP_SLICES * MQ_TOP_MAX], lead[LP_SLICES];
  __shared__ int count;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, k = a.top_k;
  const uint64_t* keys = part_key + (size_t)row * slices * k;
  const int j = k > 0 ? (k + slices - 1) / slices : 1, need = (k + j - 1) / j, total = slices * k;      // need <= slices
  // everything that is read, at once
  LpToken tok = {};
  if (tid == 0) tok = lp_token<TYPE>(a, row);
  LpSum r = {-INFINITY, 0.f, 0.f};
  if (lane < slices) r = part_sum[(size_t)row * slices + lane];
  uint64_t mine = 0, held[HELD];
  if (k > 0 && lane < slices) mine = keys[(size_t)lane * k + j - 1];
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = tid + 256 * i < total ? keys[tid + 256 * i] : 0;
  r = lp_wave_join(r);
  const LpRow out = lp_row(r);
  if (tid == 0) {
    lp_write(a, row, r, out, tok);
    count = 0;
  }
  if (k == 0) return;
  if (r.m != r.m) {
    if (tid < k) {
      a.top_tok[(size_t)row * k + tid] = tid;
      a.top_lp[(size_t)row * k + tid] = NAN;
    }
    return;
  }
  if (tid < slices) lead[tid] = mine;
  __syncthreads();
  // Every wave: the rank of each slice's j-th key (keys are different, but for 0: no key), and B
  int above = 0;
  for (int i = 0; i < slices; ++i) {
    const uint64_t o = lead[i];
    above += o > mine || (o == mine && i < lane);
  }
  const uint64_t at = __builtin_amdgcn_ballot_w64(lane < slices && above == need - 1);
  const uint64_t bound = lead[__builtin_ctzll(at)];
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (held[i] >= bound && held[i] != 0) cand[atomicAdd(&count, 1)] = held[i];
  __syncthreads();
  lp_rank(cand, count, k, [&](int i, uint64_t key) {
    a.top_tok[(size_t)row * k + i] = (int)argmax_key_index(key);
    a.top_lp[(size_t)row * k + i] = lp_of(out, lp_key_value(key));
  });
}

// Slices of a row, and their length: about 512 workgroups in all while a slice keeps 2048 elements.
struct LpPlan {
  int slices, slice;
};
LpPlan lp_plan(int rows, int vocab) {
  int s = rows >= 512 ? 1 : (512 + rows - 1) / rows;
  s = s > LP_SLICES ? LP_SLICES : s;
  const int most = vocab / 2048 > 1 ? vocab / 2048 : 1;
  s = s > most ? most : s;
  LpPlan p;
  p.slice = ((vocab + s - 1) / s + 7) / 8 * 8;
  p.slices = (vocab + p.slice - 1) / p.slice;
  return p;
}
size_t lp_sums_bytes(int rows, int slices) { return ((size_t)rows * slices * sizeof(LpSum) + 15) / 16 * 16; }

}  // namespace

size_t mq_logprobs_workspace(int rows, int vocab, int top_k) {
  const LpPlan p = lp_plan(rows, vocab);
  return p.slices == 1 ? 0 : lp_sums_bytes(rows, p.slices) + (size_t)rows * p.slices * top_k * sizeof(uint64_t);
}

int mq_launch_token_logprobs(const MqLogprobArgs& a, void* ws, hipStream_t stream) {
  const LpPlan p = lp_plan(a.rows, a.vocab);
  LpSum* sums = (LpSum*)ws;
  uint64_t* keys = (uint64_t*)((char*)ws + lp_sums_bytes(a.rows, p.slices));
  auto go = [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
    hipLaunchKernelGGL((lp_slice_kernel<TYPE>), dim3((unsigned)((size_t)a.rows * p.slices)), dim3(LP_THREADS), 0, stream, a,
                       p.slices, p.slice, sums, keys);
    if (p.slices > 1)
      hipLaunchKernelGGL((lp_join_kernel<TYPE>), dim3(a.rows), dim3(256), 0, stream, a, p.slices, sums, keys);
  };
  if (a.type == 2) go(std::integral_constant<int, 2>());
  else if (a.type == 1) go(std::integral_constant<int, 1>());
  else go(std::integral_constant<int, 0>());
  return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}
