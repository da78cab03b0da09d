// Log probabilities of given tokens with the logsumexp, entropy and top tokens of
// their rows, and the gradient of the logits, on gfx950 (MI355X, CDNA4).
//
//   lse = M + log sum e^{x - M};  logp_t = x_t - lse;  H = log sum e^{x - M} - sum (x - M) e^{x - M} / sum e^{x - M}
//   grad_j = sum_l g_l [t_l = j] + sum_k h_k [i_k = j] + p_j (g_lse - sum g - sum h - g_H (x_j - lse + H))
//
// HBM-bound: the rows are read once (the backward reads them once more and writes as
// much). A row is cut into chunks of 512 vectors of 16 bytes; a wave takes one chunk, 8
// vectors a lane, all loaded before any math, and leaves the chunk's maximum, sum and
// weighted sum, so no wave waits for another and a single row still fills many CUs. A second
// launch joins a row's chunks, looks up the given tokens and finds the top ones:
// the chunk kernel also leaves the maximum of each group of 64 consecutive vectors, and the K
// largest values of a row lie in the K groups of largest maximum (of equal ones those
// of lowest index), which alone are read again.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "dan_readout.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
extern thread_local char g_err[512];
}  // namespace dan

namespace dan_logp {

#define DAN_GLOBAL __attribute__((address_space(1)))

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kVecs = 8;               // vectors a lane
constexpr int kChunk = 64 * kVecs;     // vectors a wave

// A vector of 16 bytes at an address that only the type's own alignment holds for
// (rows of an odd number of values): the hardware reads it in one piece.
template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  static constexpr int n = 8;
  typedef __bf16 type __attribute__((ext_vector_type(8)));
  typedef type loose __attribute__((aligned(2)));
  typedef float f32 __attribute__((ext_vector_type(8)));
};
template <>
struct Vec<_Float16> {
  static constexpr int n = 8;
  typedef _Float16 type __attribute__((ext_vector_type(8)));
  typedef type loose __attribute__((aligned(2)));
  typedef float f32 __attribute__((ext_vector_type(8)));
};
template <>
struct Vec<float> {
  static constexpr int n = 4;
  typedef float type __attribute__((ext_vector_type(4)));
  typedef type loose __attribute__((aligned(4)));
  typedef float f32 __attribute__((ext_vector_type(4)));
};

#define DAN_DPP(x, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), ctrl, 0xF, 0xF, false))
#define DAN_LANE(x, n) __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), n))
__device__ inline float wave_max(float v) {
  v = fmaxf(v, DAN_DPP(v, 0xB1));
  v = fmaxf(v, DAN_DPP(v, 0x4E));
  v = fmaxf(v, DAN_DPP(v, 0x141));
  v = fmaxf(v, DAN_DPP(v, 0x140));
  return fmaxf(fmaxf(DAN_LANE(v, 0), DAN_LANE(v, 16)), fmaxf(DAN_LANE(v, 32), DAN_LANE(v, 48)));
}
__device__ inline float wave_sum(float v) {
  v += DAN_DPP(v, 0xB1);
  v += DAN_DPP(v, 0x4E);
  v += DAN_DPP(v, 0x141);
  v += DAN_DPP(v, 0x140);
  return (DAN_LANE(v, 0) + DAN_LANE(v, 16)) + (DAN_LANE(v, 32) + DAN_LANE(v, 48));
}

struct Params {
  const void *x;
  const int64_t *tokens;
  float *logprobs, *lse, *entropy, *top_logprobs;
  int64_t *top_ids;
  float *part;  // [N, chunks, 4]: maximum, sum e, sum e t (t in log2 units); then [N, chunks * kVecs] group maxima
  int64_t x_st, t_st;
  int32_t N, V, L, K, chunks;
};

// The row's vector `at` (from its first value on; what lies past its end is -inf). Vectors past
// the last whole one load that instead, or the row's start where there is none.
template <typename T>
__device__ inline void load_chunk(typename Vec<T>::f32 (&x)[kVecs], const T *row, int vocab, int first, int lane) {
  constexpr int n = Vec<T>::n;
  const int whole = vocab / n;
  typename Vec<T>::type raw[kVecs];
  if (whole > 0) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      raw[k] = *(const DAN_GLOBAL typename Vec<T>::loose *)(row + (int64_t)n * min(first + 64 * k + lane, whole - 1));
  }
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int at = first + 64 * k + lane;
    if (at < whole) {
      x[k] = __builtin_convertvector(raw[k], typename Vec<T>::f32);
    } else {
#pragma unroll
      for (int e = 0; e < n; ++e) x[k][e] = n * (int64_t)at + e < vocab ? (float)row[n * at + e] : -INFINITY;
    }
  }
}

template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(256) void chunk_kernel(const Params p) {
  constexpr int n = Vec<T>::n;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = (int64_t)blockIdx.x * 4 + wave;
  if (at >= (int64_t)p.N * p.chunks) return;
  const int64_t r = at / p.chunks;
  const int c = (int)(at - r * p.chunks);
  typename Vec<T>::f32 x[kVecs];
  load_chunk<T>(x, static_cast<const T *>(p.x) + r * p.x_st, p.V, c * kChunk, lane);
  float most[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    most[k] = x[k][0];
#pragma unroll
    for (int e = 1; e < n; ++e) most[k] = fmaxf(most[k], x[k][e]);
  }
  float m;
  if constexpr (TOP) {
    m = -INFINITY;
    float mine = 0.f;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const float w = wave_max(most[k]);
      m = fmaxf(m, w);
      mine = lane == k ? w : mine;
    }
    if (lane < kVecs) p.part[(int64_t)p.N * p.chunks * 4 + at * kVecs + lane] = mine;
  } else {
#pragma unroll
    for (int k = 1; k < kVecs; ++k) most[0] = fmaxf(most[0], most[k]);
    m = wave_max(most[0]);
  }
  float l = 0.f, a = 0.f;
  // Sums of 2^t and of t 2^t, t(x) = (x - m) log2 e.
  auto sums = [&](auto exponent) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const float t = exponent(x[k][e]);
        const float w = __builtin_amdgcn_exp2f(t);
        l += w;
        if constexpr (ENTROPY) a = __builtin_fmaf(w, fmaxf(t, -1000.0f), a);  // 0 times -inf else
      }
  };
  if (fabsf(m) < 1e38f) {
    // One operation a value: t + d, d being what the product's rounding adds to all of them, taken back below.
    const float sub = -m * kLog2e, d = __builtin_fmaf(m, kLog2e, sub);
    sums([&](float v) { return __builtin_fmaf(v, kLog2e, sub); });
    const float by = __builtin_amdgcn_exp2f(-d);
    a = by * __builtin_fmaf(-d, l, a);
    l *= by;
  } else {  // m log2 e overflows (a chunk of the type's lowest value), or nothing is finite here
    const float sub = m == -INFINITY ? 0.0f : m;
    sums([&](float v) { return (v - sub) * kLog2e; });
  }
  l = wave_sum(l);
  if constexpr (ENTROPY) a = wave_sum(a);
  if (lane == 0) *(f32x4 *)(p.part + at * 4) = (f32x4){m, l, a, 0};
}

// The row's maximum, sum and weighted sum from its chunks', in every lane of a wave.
struct Row {
  float m, l, a;
};
__device__ inline Row join(const Params &p, int64_t r, int lane) {
  const f32x4 *part = (const f32x4 *)p.part + r * p.chunks;
  float m = -INFINITY;
  for (int c = lane; c < p.chunks; c += 64) m = fmaxf(m, part[c][0]);
  m = wave_max(m);
  const float sub = m == -INFINITY ? 0.0f : m;
  float l = 0.f, a = 0.f;
  for (int c = lane; c < p.chunks; c += 64) {
    const f32x4 q = part[c];
    const float t = fmaxf((q[0] - sub) * kLog2e, -1000.0f), by = __builtin_amdgcn_exp2f(t);  // 0 times -inf else
    l = __builtin_fmaf(by, q[1], l);
    a = __builtin_fmaf(by, __builtin_fmaf(t, q[1], q[2]), a);
  }
  return {m, wave_sum(l), wave_sum(a)};
}

// Writes the row's logsumexp, entropy and the given tokens' log probabilities
// (threads `tid` of `count`); returns what a logit's log probability subtracts: M, then log sum.
template <typename T>
__device__ inline void write_row(const Params &p, int64_t r, const Row &row, int tid, int count, float &m, float &logl) {
  m = row.m == -INFINITY ? 0.0f : row.m;
  logl = logf(row.l);
  if (tid == 0) {
    p.lse[r] = m + logl;
    if (p.entropy) p.entropy[r] = row.l == 0.0f ? 0.0f : logl - row.a / row.l * kLn2;
  }
  const T *x = static_cast<const T *>(p.x) + r * p.x_st;
  for (int l = tid; l < p.L; l += count) {
    const int64_t t = p.tokens[r * p.t_st + l];
    float y = 0.0f;
    if (t >= p.V) y = __builtin_nanf("");
    else if (t >= 0) {
      const float v = (float)x[t];
      y = row.l == 0.0f ? -INFINITY : (v - m) - logl;
    }
    p.logprobs[r * p.L + l] = y;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void row_kernel(const Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.N) return;
  float m, logl;
  write_row<T>(p, r, join(p, r, lane), lane, 64, m, logl);
}

// A value's place among all values as an unsigned number: rising with it, NaN above
// all, -0 as 0.
__device__ inline uint32_t order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t o) {
  return o == 0xffffffffu ? __builtin_nanf("") : __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Larger for the larger value, and for the lower index of equal ones.
__device__ inline uint64_t key_of(uint32_t o, uint32_t index) { return (uint64_t)o << 32 | (0xffffffffu - index); }

__device__ inline uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t w = (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32 | (uint32_t)__shfl_xor((int)v, o);
    v = w > v ? w : v;
  }
  return v;
}

constexpr int kGroupKeys = 32;  // group maxima a lane: 2048 groups, rows of DAN_READOUT_MAX_TOP_VOCAB fp32 values
constexpr int kCand = 256;

template <typename T>
__global__ __launch_bounds__(256) void top_kernel(const Params p) {
  constexpr int n = Vec<T>::n, kRegs = DAN_READOUT_MAX_TOP / 4;  // vectors a lane: 64 of each group, 4 waves
  __shared__ int group[DAN_READOUT_MAX_TOP];
  __shared__ uint64_t cand[kCand];
  __shared__ uint32_t quad[64];
  __shared__ uint64_t best_of[2][4];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const Row row = join(p, r, lane);
  float m, logl;
  write_row<T>(p, r, row, tid, 256, m, logl);
  const bool empty = row.l == 0.0f;  // every logit is -inf

  // The K groups of largest maximum, by one wave: each lane keeps its best.
  const int vectors = (p.V + n - 1) / n, groups = (vectors + 63) / 64, taken = min(p.K, groups);
  if (tid == 0) count = 0;
  if (wave == 0) {
    const float *gm = p.part + (int64_t)p.N * p.chunks * 4 + r * p.chunks * kVecs;
    uint32_t o[kGroupKeys];
#pragma unroll
    for (int i = 0; i < kGroupKeys; ++i) o[i] = lane + 64 * i < groups ? order(gm[lane + 64 * i]) : 0;
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kGroupKeys; ++i) {
      const uint64_t k = lane + 64 * i < groups ? key_of(o[i], lane + 64 * i) : 0;
      best = k > best ? k : best;
    }
    for (int k = 0; k < taken; ++k) {
      const uint64_t top = wave_max64(best);
      if (lane == 0) group[k] = (int)(0xffffffffu - (uint32_t)top);
      if (best == top) {  // one lane: its next
        best = 0;
#pragma unroll
        for (int i = 0; i < kGroupKeys; ++i) {
          const uint64_t q = lane + 64 * i < groups ? key_of(o[i], lane + 64 * i) : 0;
          best = q < top && q > best ? q : best;
        }
      }
    }
  }
  __syncthreads();

  // Those groups again, wave w taking groups w, w + 4, ..
  const T *x = static_cast<const T *>(p.x) + r * p.x_st;
  const int whole = p.V / n;
  typename Vec<T>::type raw[kRegs];
  int at[kRegs];
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int k = wave + 4 * i;
    at[i] = k < taken ? group[k] * 64 + lane : vectors;
    if (whole > 0) raw[i] = *(const DAN_GLOBAL typename Vec<T>::loose *)(x + (int64_t)n * min(at[i], whole - 1));
  }
  uint32_t o[kRegs][n];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const bool there = at[i] < vectors && n * at[i] + e < p.V;
      o[i][e] = !there ? 0 : order(at[i] < whole ? (float)raw[i][e] : (float)x[n * at[i] + e]);  // order() of a value is never 0
      most = max(most, o[i][e]);
    }

  // A bound that at least K values reach: the K-th largest of the 64 maxima of four lanes each.
  uint32_t q4 = max(most, (uint32_t)__shfl_xor((int)most, 1));
  q4 = max(q4, (uint32_t)__shfl_xor((int)q4, 2));
  if ((lane & 3) == 0) quad[tid >> 2] = q4;
  __syncthreads();
  const uint32_t mine = quad[lane];
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
    above += other > mine || (other == mine && i < lane);
  }
  const uint64_t kth = __ballot(above == p.K - 1);
  const uint32_t bound = max(1u, (uint32_t)__builtin_amdgcn_readlane((int)mine, __builtin_ctzll(kth)));
  int have = 0;
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) have += o[i][e] >= bound;
  int start = have ? atomicAdd(&count, have) : 0;  // where they go does not change the result: keys differ
  if (have && start + have <= kCand) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
#pragma unroll
      for (int e = 0; e < n; ++e)
        if (o[i][e] >= bound) cand[start++] = key_of(o[i][e], n * at[i] + e);
  }
  __syncthreads();
  const int total = count;
  auto write = [&](int k, uint64_t key) {
    const float v = value_of((uint32_t)(key >> 32));
    p.top_logprobs[r * p.K + k] = empty ? -INFINITY : (v - m) - logl;
    p.top_ids[r * p.K + k] = 0xffffffffu - (uint32_t)key;
  };
  if (total <= kCand) {  // each candidate's rank among them
    if (tid < total) {
      const uint64_t k = cand[tid];
      int rank = 0;
      for (int i = 0; i < total; ++i) rank += cand[i] > k;
      if (rank < p.K) write(rank, k);
    }
    return;
  }
  // Too many reach the bound (a row of equal values, or its largest side by side): K rounds of the largest left.
  uint64_t last = ~0ull, best = 0;
  for (int k = 0; k < p.K; ++k) {
    if (k == 0 || best == last) {
      best = 0;
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
#pragma unroll
        for (int e = 0; e < n; ++e) {
          const uint64_t q = o[i][e] ? key_of(o[i][e], n * at[i] + e) : 0;
          best = q < last && q > best ? q : best;
        }
    }
    const uint64_t w = wave_max64(best);
    if (lane == 0) best_of[k & 1][wave] = w;
    __syncthreads();
    last = best_of[k & 1][0];
#pragma unroll
    for (int i = 1; i < 4; ++i) last = best_of[k & 1][i] > last ? best_of[k & 1][i] : last;
    if (tid == 0) write(k, last);
  }
}

struct GradParams {
  const void *x;
  const int64_t *tokens, *top_ids;
  const float *lse, *entropy, *g_logp, *g_lse, *g_entropy, *g_top;
  void *grad;
  int64_t x_st, t_st, g_st;
  int32_t N, V, L, K, chunks;
};

template <typename T, bool ENTROPY>
__global__ __launch_bounds__(256) void grad_kernel(const GradParams p) {
  constexpr int n = Vec<T>::n;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t work = (int64_t)blockIdx.x * 4 + wave;
  if (work >= (int64_t)p.N * p.chunks) return;
  const int64_t r = work / p.chunks;
  const int first = (int)(work - r * p.chunks) * kChunk;
  typename Vec<T>::f32 x[kVecs];
  load_chunk<T>(x, static_cast<const T *>(p.x) + r * p.x_st, p.V, first, lane);
  const float lse = p.lse[r];
  const float sub = lse == -INFINITY ? 0.0f : lse;
  // The ids of the row that take a gradient of their own (the labels, then the top tokens;
  // none where every logit is -inf), and its sum.
  const int labels = p.g_logp ? p.L : 0, ids = lse == -INFINITY ? 0 : labels + (p.g_top ? p.K : 0);
  auto id_of = [&](int i, int &id, float &g) {
    id = -1;
    g = 0.f;
    if (i >= ids) return;
    const int64_t t = i < labels ? p.tokens[r * p.t_st + i] : p.top_ids[r * p.K + i - labels];
    if (t < 0) return;
    g = i < labels ? p.g_logp[r * p.L + i] : p.g_top[r * p.K + i - labels];
    id = t < p.V ? (int)t : -1;
    if (t >= p.V) g = __builtin_nanf("");  // as its log probability
  };
  float sum = 0.f, g0 = 0.f;
  int id0 = -1;
  for (int i = 0; i < ids; i += 64) {
    int id;
    float g;
    id_of(i + lane, id, g);
    if (i == 0) id0 = id, g0 = g;
    sum += g;
  }
  sum = (p.g_lse ? p.g_lse[r] : 0.0f) - wave_sum(sum);
  const float ge = ENTROPY ? p.g_entropy[r] : 0.0f, h = ENTROPY ? p.entropy[r] : 0.0f;
  T *out = static_cast<T *>(p.grad) + r * p.g_st;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int at = first + 64 * k + lane;
    typename Vec<T>::f32 y;
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float lp = x[k][e] - sub;
      const float w = __builtin_amdgcn_exp2f(lp * kLog2e);
      float f = sum;
      if constexpr (ENTROPY) f = __builtin_fmaf(-ge, fmaxf(lp, -1000.0f) + h, f);  // 0 times -inf else
      y[e] = w * f;
    }
    // What falls into these 64 vectors is added by the lane that holds it.
    const int low = (first + 64 * k) * n;
    for (int i = 0; i < ids; i += 64) {
      int id = id0;
      float g = g0;
      if (i > 0) id_of(i + lane, id, g);
      uint64_t hits = __ballot(id >= low && id < low + 64 * n);
      while (hits) {
        const int s = __builtin_ctzll(hits);
        hits &= hits - 1;
        const int to = __builtin_amdgcn_readlane(id, s) - low;
        const float add = DAN_LANE(g, s);
#pragma unroll
        for (int e = 0; e < n; ++e) y[e] += lane == to / n && e == to % n ? add : 0.0f;
      }
    }
    const typename Vec<T>::type z = __builtin_convertvector(y, typename Vec<T>::type);
    if ((int64_t)n * at + n <= p.V) {
      *(DAN_GLOBAL typename Vec<T>::loose *)(out + (int64_t)n * at) = z;
    } else {
#pragma unroll
      for (int e = 0; e < n; ++e)
        if ((int64_t)n * at + e < p.V) out[(int64_t)n * at + e] = z[e];
    }
  }
}

inline int values_of(int dtype) { return dtype == DAN_DTYPE_F32 ? 4 : 8; }
inline int chunks_of(int dtype, int vocab) {
  const int n = values_of(dtype);
  return (int)(((int64_t)vocab + (int64_t)n * kChunk - 1) / ((int64_t)n * kChunk));
}

template <typename T>
void forward(const Params &p, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)p.N * p.chunks + 3) / 4));
  if (p.entropy) {
    if (p.K > 0) hipLaunchKernelGGL((chunk_kernel<T, true, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((chunk_kernel<T, true, false>), grid, dim3(256), 0, s, p);
  } else {
    if (p.K > 0) hipLaunchKernelGGL((chunk_kernel<T, false, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((chunk_kernel<T, false, false>), grid, dim3(256), 0, s, p);
  }
  if (p.K > 0) hipLaunchKernelGGL((top_kernel<T>), dim3((unsigned)p.N), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((row_kernel<T>), dim3((unsigned)((p.N + 3) / 4)), dim3(256), 0, s, p);
}

template <typename T>
void backward(const GradParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)p.N * p.chunks + 3) / 4));
  if (p.g_entropy) hipLaunchKernelGGL((grad_kernel<T, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((grad_kernel<T, false>), grid, dim3(256), 0, s, p);
}

// What both calls check alike; 0 when all is well.
int check(int abi, int dtype, int rows, int vocab, int labels, int top, int64_t stride, int64_t tokens_stride) {
  using dan::fail;
  if (abi != DAN_READOUT_ABI_VERSION) return fail(DAN_ERR_VERSION, "abi_version %d, readout speaks %d", abi, DAN_READOUT_ABI_VERSION);
  if (dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16 && dtype != DAN_DTYPE_F32) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16, f16 or f32", dtype);
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || labels < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "need rows >= 0, vocab in [1, 2^30] and labels >= 0");
  if (top < 0 || top > DAN_READOUT_MAX_TOP || top > vocab)
    return fail(DAN_ERR_INVALID_ARGUMENT, "top %d: at most %d and the vocabulary's %d", top, DAN_READOUT_MAX_TOP, vocab);
  if (top > 0 && vocab > DAN_READOUT_MAX_TOP_VOCAB)
    return fail(DAN_ERR_UNSUPPORTED, "top tokens of %d values: rows of at most %d", vocab, DAN_READOUT_MAX_TOP_VOCAB);
  if (stride < 0 || tokens_stride < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "row strides must be >= 0");
  if (((int64_t)rows * chunks_of(dtype, vocab) + 3) / 4 >= (int64_t)1 << 31) return fail(DAN_ERR_INVALID_ARGUMENT, "too many rows");
  return 0;
}

}  // namespace dan_logp

extern "C" {

int dan_readout_abi_version(void) { return DAN_READOUT_ABI_VERSION; }

int64_t dan_logprobs_workspace_size(int32_t dtype, int32_t rows, int32_t vocab, int32_t top) {
  using namespace dan_logp;
  if ((dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16 && dtype != DAN_DTYPE_F32) || rows < 0 || vocab < 1 || vocab > (1 << 30) || top < 0)
    return 0;
  return (int64_t)rows * chunks_of(dtype, vocab) * (16 + (top > 0 ? 4 * kVecs : 0)) + 16;
}

int dan_logprobs_fwd(const DanLogprobsArgs *a, void *stream) {
  using namespace dan_logp;
  using dan::fail;
  dan::g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const int rc = check(a->abi_version, a->dtype, a->rows, a->vocab, a->labels, a->top, a->logits_stride, a->tokens_stride)) return rc;
  if (a->rows == 0) return DAN_OK;
  if (!a->logits || !a->logsumexp || (a->labels > 0 && (!a->tokens || !a->logprobs)) || (a->top > 0 && (!a->top_logprobs || !a->top_ids)))
    return fail(DAN_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
  if ((uintptr_t)a->logits & (a->dtype == DAN_DTYPE_F32 ? 3 : 1)) return fail(DAN_ERR_INVALID_ARGUMENT, "logits must be aligned to their type");
  const int64_t need = dan_logprobs_workspace_size(a->dtype, a->rows, a->vocab, a->top);
  if (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < need)
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace: %lld bytes, 16-byte aligned; got %lld", (long long)need, (long long)a->workspace_bytes);
  Params p;
  p.x = a->logits; p.tokens = a->tokens; p.logprobs = a->logprobs; p.lse = a->logsumexp; p.entropy = a->entropy;
  p.top_logprobs = a->top_logprobs; p.top_ids = a->top_ids; p.part = static_cast<float *>(a->workspace);
  p.x_st = a->logits_stride; p.t_st = a->tokens_stride;
  p.N = a->rows; p.V = a->vocab; p.L = a->labels; p.K = a->top; p.chunks = chunks_of(a->dtype, a->vocab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == DAN_DTYPE_BF16) forward<__bf16>(p, s);
  else if (a->dtype == DAN_DTYPE_F16) forward<_Float16>(p, s);
  else forward<float>(p, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "log probabilities launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

int dan_logprobs_bwd(const DanLogprobsGradArgs *a, void *stream) {
  using namespace dan_logp;
  using dan::fail;
  dan::g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (const int rc = check(a->abi_version, a->dtype, a->rows, a->vocab, a->labels, a->top, a->logits_stride, a->tokens_stride)) return rc;
  if (a->rows == 0) return DAN_OK;
  if (!a->logits || !a->logsumexp || !a->grad || (a->g_entropy && !a->entropy) || (a->g_top && !a->top_ids) ||
      (a->g_logprobs && a->labels > 0 && !a->tokens))
    return fail(DAN_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
  const uintptr_t own = a->dtype == DAN_DTYPE_F32 ? 3 : 1;
  if (((uintptr_t)a->logits | (uintptr_t)a->grad) & own) return fail(DAN_ERR_INVALID_ARGUMENT, "logits and grad must be aligned to their type");
  if (a->grad_stride < a->vocab) return fail(DAN_ERR_INVALID_ARGUMENT, "grad_stride %lld < vocab", (long long)a->grad_stride);
  GradParams p;
  p.x = a->logits; p.tokens = a->tokens; p.top_ids = a->top_ids; p.lse = a->logsumexp; p.entropy = a->entropy;
  p.g_logp = a->g_logprobs; p.g_lse = a->g_logsumexp; p.g_entropy = a->g_entropy; p.g_top = a->g_top; p.grad = a->grad;
  p.x_st = a->logits_stride; p.t_st = a->tokens_stride; p.g_st = a->grad_stride;
  p.N = a->rows; p.V = a->vocab; p.L = a->labels; p.K = a->top; p.chunks = chunks_of(a->dtype, a->vocab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == DAN_DTYPE_BF16) backward<__bf16>(p, s);
  else if (a->dtype == DAN_DTYPE_F16) backward<_Float16>(p, s);
  else backward<float>(p, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "gradient launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
