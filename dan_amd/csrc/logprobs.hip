// Log probabilities of given tokens with the logsumexp, entropy and top tokens of
// their rows, and the gradient of the logits, on gfx950 (MI355X, CDNA4).
//
//   lse = M + log sum e^{x - M};  logp_t = x_t - lse;  H = log sum e^{x - M} - sum (x - M) e^{x - M} / sum e^{x - M}
//   grad_j = sum_l g_l [t_l = j] + sum_k h_k [i_k = j] + p_j (g_lse - sum g - sum h - g_H (x_j - lse + H))
// (lse rounded to fp32, and what that took from it, which log p_j = (x_j - lse) - rest needs)
//
// HBM-bound: the rows are read once (the backward reads them once more and writes as
// much). A row is cut into chunks of 512 vectors of 16 bytes; a wave takes one chunk, 8
// vectors a lane, all loaded before any math, and leaves the chunk's maximum, sum and
// weighted sum, so no wave waits for another and a single row still fills many CUs. A second
// launch (short rows: the same, in_one) joins a row's chunks, looks up the given tokens and finds the top ones:
// the chunk kernel also leaves the maximum of each group of 64 consecutive vectors, and the K
// largest values of a row lie in the K groups of largest maximum (of equal ones those
// of lowest index), which alone are read again.
//
// Measured, us: 2039 rows x 128256 bf16 with 5 top tokens and entropy 104 (the chunk kernel 86: 523 MB at 6.1 TB/s; the
// top kernel 16), without top tokens 87; 1 row 5.0 + 7.8 with 20 top tokens, of which
// about 4 each are a launch and its first loads; 45 rows x 50257 fp32 with 5, 5.4 + 6.7. Forward with entropy and gradient of
// 4096 x 128256 bf16 (3.15 GB) 520: 6.0 TB/s, where a large copy moves 4.9.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "cus.h"
#include "dan_readout.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
extern thread_local char g_err[512];
}  // namespace dan

namespace dan_logp {

#define DAN_GLOBAL __attribute__((address_space(1)))

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kVecs = 8;               // vectors a lane
constexpr int kChunk = 64 * kVecs;     // vectors a wave
constexpr int kWhole = 8;              // chunks of a row that one work group takes whole

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

template <typename F>
__device__ inline uint32_t wave_fold(uint32_t v, F f) {
  auto dpp = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xF, 0xF, false); };
  v = f(v, dpp(v, std::integral_constant<int, 0xB1>()));
  v = f(v, dpp(v, std::integral_constant<int, 0x4E>()));
  v = f(v, dpp(v, std::integral_constant<int, 0x141>()));
  v = f(v, dpp(v, std::integral_constant<int, 0x140>()));
  auto at = [&](int n) { return (uint32_t)__builtin_amdgcn_readlane((int)v, n); };
  return f(f(at(0), at(16)), f(at(32), at(48)));
}

struct Params {
  const void *x;
  const int64_t *tokens;
  float *logprobs, *lse, *rest, *entropy, *top_logprobs;  // rest: of lse, or NULL
  int64_t *top_ids;
  float *part;  // [N, chunks, 4]: maximum, sum e, sum e t (t in log2 units); then [N, chunks * kVecs] group maxima
  int64_t x_st, t_st;
  int32_t N, V, L, K, chunks;
};

// A lane's vectors of a chunk; what lies past the row's end is -inf. (A vector past the last whole one
// loads that instead.) The loads pass the caches by, which rows of a few hundred MB only
// sweep: 2039 x 128256 bf16 91 -> 80 us, forward and backward of 4096 rows 548 -> 521.
template <typename T>
__device__ inline void load_chunk(typename Vec<T>::f32 (&x)[kVecs], const T *row, int vocab, int first, int lane) {
  constexpr int n = Vec<T>::n;
  const int whole = vocab / n;
  typename Vec<T>::type raw[kVecs];
  if (whole > 0) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      raw[k] = __builtin_nontemporal_load((const DAN_GLOBAL typename Vec<T>::loose *)(row + (int64_t)n * min(first + 64 * k + lane, whole - 1)));
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

// A chunk's maximum, sum and weighted sum (and 0), in every lane; TOP: with lane k's `mine` the maximum of group k.
template <typename T, bool ENTROPY, bool TOP>
__device__ __forceinline__ f32x4 chunk_sums(const T *row, int vocab, int first, int lane, float &mine) {
  constexpr int n = Vec<T>::n;
  typename Vec<T>::f32 x[kVecs];
  load_chunk<T>(x, row, vocab, first, lane);
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
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const float w = wave_max(most[k]);
      m = fmaxf(m, w);
      mine = lane == k ? w : mine;
    }
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
  if (fabsf(m) < 0x1p20f) {
    // One operation a value: t + d, d being what the product's rounding adds to all of them, taken back below. d is at most
    // half a unit of m log2 e: 2^-4 here, but past m = 3e9 more than the 127 that an exponent holds.
    const float sub = -m * kLog2e, d = __builtin_fmaf(m, kLog2e, sub);
    sums([&](float v) { return __builtin_fmaf(v, kLog2e, sub); });
    const float by = __builtin_amdgcn_exp2f(-d);
    a = by * __builtin_fmaf(-d, l, a);
    l *= by;
  } else {  // a chunk of large values (as a mask's), or one that nothing finite is in
    const float sub = m == -INFINITY ? 0.0f : m;
    sums([&](float v) { return (v - sub) * kLog2e; });
  }
  l = wave_sum(l);
  if constexpr (ENTROPY) a = wave_sum(a);
  return {m, l, a, 0};
}

template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(256) void chunk_kernel(const Params p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = (int64_t)blockIdx.x * 4 + wave;
  if (at >= (int64_t)p.N * p.chunks) return;
  const int64_t r = at / p.chunks;
  float mine = 0.f;
  const f32x4 sums = chunk_sums<T, ENTROPY, TOP>(static_cast<const T *>(p.x) + r * p.x_st, p.V, (int)(at - r * p.chunks) * kChunk, lane, mine);
  if (TOP && lane < kVecs) p.part[(int64_t)p.N * p.chunks * 4 + at * kVecs + lane] = mine;
  if (lane == 0) *(f32x4 *)(p.part + at * 4) = sums;
}

// The row's maximum, sum and weighted sum from its chunks', in every lane of a wave; `first` is chunk `lane`'s
// (-inf, 0, 0 behind the last), loaded ahead.
struct Row {
  float m, l, a;
};
__device__ inline f32x4 first_chunk(const f32x4 *part, int chunks, int lane) { return lane < chunks ? part[lane] : (f32x4){-INFINITY, 0, 0, 0}; }
__device__ inline Row join(const f32x4 *part, int chunks, int lane, f32x4 first) {
  float m = first[0];
  for (int c = lane + 64; c < chunks; c += 64) m = fmaxf(m, part[c][0]);
  m = wave_max(m);
  const float sub = m == -INFINITY ? 0.0f : m;
  float l = 0.f, a = 0.f;
  auto add = [&](f32x4 q) {
    const float t = fmaxf((q[0] - sub) * kLog2e, -1000.0f), by = __builtin_amdgcn_exp2f(t);  // 0 times -inf else
    l = __builtin_fmaf(by, q[1], l);
    a = __builtin_fmaf(by, __builtin_fmaf(t, q[1], q[2]), a);
  };
  add(first);
  for (int c = lane + 64; c < chunks; c += 64) add(part[c]);
  return {m, wave_sum(l), wave_sum(a)};
}

// A thread's first given token and its logit, loaded ahead of the row's sums.
struct Given {
  int64_t token;  // -1: padding, or none for this thread
  float x;
};
template <typename T>
__device__ inline Given fetch(const Params &p, int64_t r, int l) {
  Given g = {-1, 0.0f};
  if (l < p.L) {
    g.token = p.tokens[r * p.t_st + l];
    if (g.token >= 0 && g.token < p.V) g.x = (float)static_cast<const T *>(p.x)[r * p.x_st + g.token];
  }
  return g;
}

// Writes the row's logsumexp, entropy and the given tokens' log probabilities (threads `tid` of
// `count`; the first of each in `g`), x - (M, then log sum).
template <typename T>
__device__ inline void write_row(const Params &p, int64_t r, const Row &row, Given g, int tid, int count, float m, float logl) {
  if (tid == 0) {
    const float lse = m + logl;
    p.lse[r] = lse;
    if (p.rest) {  // m + logl = lse + rest exactly, whichever of the two is larger
      const float back = lse - m;
      p.rest[r] = fabsf(lse) < INFINITY ? (m - (lse - back)) + (logl - back) : 0.0f;
    }
    if (p.entropy) p.entropy[r] = row.l == 0.0f ? 0.0f : logl - row.a / row.l * kLn2;
  }
  for (int l = tid; l < p.L; l += count) {
    if (l != tid) g = fetch<T>(p, r, l);
    float y = 0.0f;
    if (g.token >= p.V) y = __builtin_nanf("");
    else if (g.token >= 0) y = row.l == 0.0f ? -INFINITY : (g.x - m) - logl;
    p.logprobs[r * p.L + l] = y;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void row_kernel(const Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.N) return;
  const f32x4 *part = (const f32x4 *)p.part + r * p.chunks;
  const f32x4 first = first_chunk(part, p.chunks, lane);
  const Given g = fetch<T>(p, r, lane);
  const Row row = join(part, p.chunks, lane, first);
  write_row<T>(p, r, row, g, lane, 64, row.m == -INFINITY ? 0.0f : row.m, logf(row.l));
}

// Short rows in one launch: ONE: a wave takes a row of one chunk; else a work group takes a row of up to kWhole, whose
// sums meet in LDS.
template <typename T, bool ENTROPY, bool ONE>
__global__ __launch_bounds__(256) void whole_kernel(const Params p) {
  __shared__ f32x4 part[kWhole];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = ONE ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (ONE && r >= p.N) return;
  const T *x = static_cast<const T *>(p.x) + r * p.x_st;
  const Given g = fetch<T>(p, r, ONE ? lane : tid);
  float none = 0.f;
  Row row;
  if constexpr (ONE) {
    const f32x4 sums = chunk_sums<T, ENTROPY, false>(x, p.V, 0, lane, none);
    row = join(part, 1, lane, lane == 0 ? sums : (f32x4){-INFINITY, 0, 0, 0});
  } else {
    for (int c = wave; c < p.chunks; c += 4) {
      const f32x4 sums = chunk_sums<T, ENTROPY, false>(x, p.V, c * kChunk, lane, none);
      if (lane == 0) part[c] = sums;
    }
    __syncthreads();
    row = join(part, p.chunks, lane, first_chunk(part, p.chunks, lane));
  }
  write_row<T>(p, r, row, g, ONE ? lane : tid, ONE ? 64 : 256, row.m == -INFINITY ? 0.0f : row.m, logf(row.l));
}

// A value's place among all values as an unsigned number in [0x7fffff, 0xfffffffe]: rising with
// it, NaN above all, -0 as 0; and the value back.
__device__ inline uint32_t order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// Larger for the larger value, and for the lower index of equal ones.
__device__ inline uint64_t key_of(uint32_t o, uint32_t index) { return (uint64_t)o << 32 | (0xffffffffu - index); }

// The bits of a wave's 64-bit lane mask below this lane.
__device__ inline int below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// What a lane wrote to LDS is there for the other lanes of its wave.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kTaken = 32;    // groups whose values a work group holds: 8 vectors a lane of 4 waves
constexpr int kCand = 64;     // values that a wave collects
constexpr uint32_t kLowest = 0x007fffffu;  // order(-inf): every value reaches it

// Raises `bound` by bisection, between what K or more of a set's keys reach and `over`, which
// fewer do, until at most `most` reach it or the two are neighbours; `have` is how many
// do, reach(x) how many reach x.
template <typename F>
__device__ inline void bisect(uint32_t &bound, uint32_t &over, int &have, int k, int most, F reach) {
  while (have > most && over - bound > 1) {
    const uint32_t mid = bound + (over - bound) / 2;
    const int c = reach(mid);
    if (c >= k) bound = mid, have = c;
    else over = mid;
  }
}

// The K largest values of a row, one work group.
//  1. Each wave finds by bisection a bound that K and not many more of the group maxima reach, or,
//     where too many are equal at it, that value itself. K values of the row reach it, so the row's K
//     largest do, and they lie in these groups (of those whose maximum is the bound itself, in
//     the first that make up K).
//  2. The work group loads these groups and each wave collects its values that reach the bound: in
//     rows of ordinary logits few more than K in all. Of values equal to a bound that too many reach (masked
//     rows: the masked value) each wave collects its first K. Where a wave has more than 64 (no more
//     groups than K; most of the largest side by side) the bound is raised by bisection over the
//     lanes' maxima, and if need be over the values.
//  3. Each collected value's rank among them is its place in the result.
// KEYS: group maxima a lane, 64 KEYS >= groups. `part` and `gm` are the row's chunks' sums and its group
// maxima, `given` the thread's first token.
template <typename T, int KEYS>
__device__ __forceinline__ void top_row(const Params &p, const int64_t r, const f32x4 *part, const float *gm, const Given given) {
  constexpr int n = Vec<T>::n, kRegs = kTaken / 4;
  __shared__ int group[4][kTaken];
  __shared__ u32x4 kept[4][kRegs][64];
  __shared__ uint64_t cand[4][kCand];
  __shared__ uint32_t lane_max[256];
  __shared__ int counts[4], sums[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int vectors = (p.V + n - 1) / n, groups = (vectors + 63) / 64;
  const f32x4 first = first_chunk(part, p.chunks, lane);
  float g[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) g[i] = lane + 64 * i < groups ? gm[lane + 64 * i] : 0.0f;
  uint32_t o[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) o[i] = lane + 64 * i < groups ? order(g[i]) : 0;

  // 1.
  auto reach = [&](uint32_t x) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) c += __builtin_popcountll(__ballot(o[i] >= x));
    return c;
  };
  const int most = min(kTaken, p.K + p.K / 2 + 4);
  uint32_t best = o[0];
#pragma unroll
  for (int i = 1; i < KEYS; ++i) best = max(best, o[i]);
  // The smallest of the lanes' largest (of lanes that have one) is reached by each of them.
  uint32_t bound = wave_fold(best ? best : 0xffffffffu, [](uint32_t x, uint32_t y) { return min(x, y); });
  uint32_t over = wave_fold(best, [](uint32_t x, uint32_t y) { return max(x, y); }) + 1;
  int have = reach(bound);
  if (have > p.K) bisect(bound, over, have, p.K, most, reach);
  if (groups <= p.K) bound = kLowest, have = groups;  // all of them
  bool equal = have > kTaken;                         // then over = bound + 1
  const int left = equal ? p.K - reach(over) : 0, taken = equal ? p.K : have;
  {
    int at = 0, before = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      bool in = o[i] >= (equal ? over : bound);
      if (equal) {
        const uint64_t same = __ballot(o[i] == bound);
        in = in || (o[i] == bound && before + below(same) < left);
        before += __builtin_popcountll(same);
      }
      in = in && lane + 64 * i < groups;
      const uint64_t mask = __ballot(in);
      if (in) group[wave][at + below(mask)] = lane + 64 * i;
      at += __builtin_popcountll(mask);
    }
  }
  wave_sync();  // a wave reads its own list

  // 2. Wave w takes groups w, w + 4, ..; rising ones, so that of equal values the first come first.
  // What lies behind the row's end is NaN, which reaches no bound.
  const T *x = static_cast<const T *>(p.x) + r * p.x_st;
  const int whole = p.V / n, mine = (taken - wave + 3) / 4;
  // They are kept in LDS (a wave's own part), where loops over them need few registers.
  u32x4 raw[kRegs];
  int at[kRegs];
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    at[i] = i < mine ? group[wave][wave + 4 * i] * 64 + lane : vectors;
    if (whole > 0 && i < mine) raw[i] = __builtin_bit_cast(u32x4, *(const DAN_GLOBAL typename Vec<T>::loose *)(x + (int64_t)n * min(at[i], whole - 1)));
  }
  u32x4 tail = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};  // NaN in every type
  if (p.V != whole * n) {                                           // the row's last values fill no vector: one by one
    const uint16_t *last = (const uint16_t *)(x + (int64_t)n * whole);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((int)sizeof(T) * (p.V - n * whole) > 2 * e) tail[e / 2] = e % 2 ? (tail[e / 2] & 0xffffu) | (uint32_t)last[e] << 16 : (tail[e / 2] & 0xffff0000u) | last[e];
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
    if (i < mine) {
#pragma unroll
      for (int c = 0; c < 4; ++c) raw[i][c] = at[i] < whole ? raw[i][c] : at[i] == whole ? tail[c] : 0x7fff7fffu;
      kept[wave][i][lane] = raw[i];
    }
  wave_sync();

  const Row row = join(part, p.chunks, lane, first);
  const float m = row.m == -INFINITY ? 0.0f : row.m, logl = logf(row.l);
  write_row<T>(p, r, row, given, tid, 256, m, logl);
  if (!(row.l >= 0.0f)) {  // NaN: the row has no order
    if (tid < p.K) {
      p.top_logprobs[r * p.K + tid] = __builtin_nanf("");
      p.top_ids[r * p.K + tid] = tid;
    }
    return;
  }

  auto values = [&](int i) { return __builtin_convertvector(__builtin_bit_cast(typename Vec<T>::type, kept[wave][i][lane]), typename Vec<T>::f32); };
  auto largest = [&](typename Vec<T>::f32 f) {
    float y = f[0];
#pragma unroll
    for (int e = 1; e < n; ++e) y = fmaxf(y, f[e]);
    return y;
  };
  for (int stage = groups > p.K ? 0 : 1;; ++stage) {
    if (stage == 1) {  // K or more of the lanes' maxima reach it, so as many values do
      uint32_t mx = 0, q[4];
      for (int i = 0; i < mine; ++i) {
        const float y = largest(values(i));
        mx = y == y ? max(mx, order(y)) : mx;
      }
      lane_max[tid] = mx;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = lane_max[lane + 64 * i];
      auto reach_lanes = [&](uint32_t y) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c += __builtin_popcountll(__ballot(q[i] >= y));
        return c;
      };
      over = wave_fold(max(max(q[0], q[1]), max(q[2], q[3])), [](uint32_t y, uint32_t z) { return max(y, z); }) + 1;
      have = reach_lanes(bound);
      if (have > p.K) bisect(bound, over, have, p.K, most, reach_lanes);
      equal = have > most;
    } else if (stage == 2) {
      int turn = 0;
      auto reach_values = [&](uint32_t y) {
        const float v = value_of(y);  // NaN above +inf's place: reached by none
        int c = 0;
        for (int i = 0; i < mine; ++i) {
          const typename Vec<T>::f32 f = values(i);
#pragma unroll
          for (int e = 0; e < n; ++e) c += __builtin_popcountll(__ballot(f[e] >= v));
        }
        if (lane == 0) sums[turn & 1][wave] = c;
        __syncthreads();
        c = sums[turn & 1][0] + sums[turn & 1][1] + sums[turn & 1][2] + sums[turn & 1][3];
        ++turn;
        return c;
      };
      int total = reach_values(bound);
      over = 0xffffffffu;
      bisect(bound, over, total, p.K, kCand, reach_values);
      equal = total > kCand;
    }
    // The wave's values that reach the bound, or the next one where `equal`.
    const float v = value_of(equal ? over : bound);
    int c = 0;
    for (int i = 0; i < mine; ++i) {
      const typename Vec<T>::f32 f = values(i);
      const uint32_t index = n * (group[wave][wave + 4 * i] * 64 + lane);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const uint64_t mask = __ballot(f[e] >= v);
        if (mask) {  // (most have none)
          const int to = c + below(mask);
          if (f[e] >= v && to < kCand) cand[wave][to] = key_of(order(f[e]), index + e);
          c += __builtin_popcountll(mask);
        }
      }
    }
    if (equal) {  // over = bound + 1: the first K of those equal to the bound
      const float w = value_of(bound);
      int room = p.K;
      for (int i = 0; i < mine && room > 0; ++i) {
        const typename Vec<T>::f32 f = values(i);
        const uint32_t index = n * (group[wave][wave + 4 * i] * 64 + lane);
        int before = 0, all = 0;
#pragma unroll
        for (int e = 0; e < n; ++e) {
          const uint64_t mask = __ballot(f[e] == w);
          before += below(mask);
          all += __builtin_popcountll(mask);
        }
#pragma unroll
        for (int e = 0; e < n; ++e)
          if (f[e] == w) {
            if (before < room && c + before < kCand) cand[wave][c + before] = key_of(bound, index + e);
            ++before;
          }
        all = min(all, room);
        c += all;
        room -= all;
      }
    }
    if (lane == 0) counts[wave] = c;
    __syncthreads();
    if (max(max(counts[0], counts[1]), max(counts[2], counts[3])) <= kCand) break;  // at stage 2 at the latest: 64 in all, or fewer than K and K
    __syncthreads();
  }

  // 3.
  uint64_t other[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) other[w] = lane < counts[w] ? cand[w][lane] : 0;
  const uint64_t k = cand[wave][lane];
  int rank = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    for (int i = 0, c = counts[w]; i < c; ++i) {
      const uint64_t q = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(other[w] >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)other[w], i);
      rank += q > k;
    }
  if (lane < counts[wave] && rank < p.K) {
    const float y = value_of((uint32_t)(k >> 32));
    p.top_logprobs[r * p.K + rank] = row.l == 0.0f ? -INFINITY : (y - m) - logl;
    p.top_ids[r * p.K + rank] = 0xffffffffu - (uint32_t)k;
  }
}

template <typename T, int KEYS>
__global__ __launch_bounds__(256, 4) void top_kernel(const Params p) {
  const int64_t r = blockIdx.x;
  const Given given = fetch<T>(p, r, threadIdx.x);
  top_row<T, KEYS>(p, r, (const f32x4 *)p.part + r * p.chunks, p.part + (int64_t)p.N * p.chunks * 4 + r * p.chunks * kVecs, given);
}

// A short row (kWhole) with its top tokens in one launch.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(256, 4) void whole_top_kernel(const Params p) {
  __shared__ f32x4 part[kWhole];
  __shared__ float gm[kWhole * kVecs];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x;
  const Given given = fetch<T>(p, r, tid);
  for (int c = wave; c < p.chunks; c += 4) {
    float mine = 0.f;
    const f32x4 sums = chunk_sums<T, ENTROPY, true>(static_cast<const T *>(p.x) + r * p.x_st, p.V, c * kChunk, lane, mine);
    if (lane == 0) part[c] = sums;
    if (lane < kVecs) gm[c * kVecs + lane] = mine;
  }
  __syncthreads();
  top_row<T, kWhole * kVecs / 64>(p, r, part, gm, given);
}

// By how many group maxima a lane keeps in registers: the fewest that hold the row's, for each
// adds an operation to every step of the search. 128256 bf16 values (251 groups), a whole call of 1 row with 20 top
// tokens / of 2039 rows with 5, us: 4 a lane 12.8 / 108.7, 8 13.6 / 111.9, 32 18.7 / 118.9. 151936 fp32 values (594 groups),
// 1 row with 20 / 500 rows with 5: 16 a lane 14.2 / 60, 32 17.9 / 65.
template <typename T>
void launch_top(const Params &p, hipStream_t s) {
  const int groups = ((p.V + Vec<T>::n - 1) / Vec<T>::n + 63) / 64;
  if (groups <= 64 * 4) hipLaunchKernelGGL((top_kernel<T, 4>), dim3((unsigned)p.N), dim3(256), 0, s, p);
  else if (groups <= 64 * 8) hipLaunchKernelGGL((top_kernel<T, 8>), dim3((unsigned)p.N), dim3(256), 0, s, p);
  else if (groups <= 64 * 16) hipLaunchKernelGGL((top_kernel<T, 16>), dim3((unsigned)p.N), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((top_kernel<T, 32>), dim3((unsigned)p.N), dim3(256), 0, s, p);  // up to DAN_READOUT_MAX_TOP_VOCAB fp32 values
}

struct GradParams {
  const void *x;
  const int64_t *tokens, *top_ids;
  const float *lse, *rest, *entropy, *g_logp, *g_lse, *g_entropy, *g_top;
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
  // The rows from the last to the first: the forward, if it has just run, has left the last ones in cache.
  const int64_t turn = work / p.chunks, r = p.N - 1 - turn;
  const int first = (int)(work - turn * p.chunks) * kChunk;
  typename Vec<T>::f32 x[kVecs];
  load_chunk<T>(x, static_cast<const T *>(p.x) + r * p.x_st, p.V, first, lane);
  const float lse = p.lse[r];
  const float sub = lse == -INFINITY ? 0.0f : lse, rest = p.rest ? p.rest[r] : 0.0f;
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
      const float lp = (x[k][e] - sub) - rest;
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
      // past the caches, which the logits still to come then keep: forward and backward of 4096 x 128256 bf16
      // 584 -> 545 us (and 537 with the rows reversed); a product that reads the gradient next is no slower
      __builtin_nontemporal_store((typename Vec<T>::loose)z, (DAN_GLOBAL typename Vec<T>::loose *)(out + (int64_t)n * at));
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

template <typename T, bool ENTROPY>
void forward_whole(const Params &p, hipStream_t s) {
  if (p.K > 0) hipLaunchKernelGGL((whole_top_kernel<T, ENTROPY>), dim3((unsigned)p.N), dim3(256), 0, s, p);
  else if (p.chunks == 1) hipLaunchKernelGGL((whole_kernel<T, ENTROPY, true>), dim3((unsigned)((p.N + 3) / 4)), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((whole_kernel<T, ENTROPY, false>), dim3((unsigned)p.N), dim3(256), 0, s, p);
}

// Whether rows go through one launch, whose work groups take a row (or four of one chunk) whole. us in two
// launches / in one, bf16 with entropy: 1 row of 4000 4.9 / 3.6, 500 rows of 16000 7.2 / 5.2, 8000 of 4000 17.4 / 15.0,
// but 2000 of 16000 16.1 / 16.6 and 8000 47 / 55, 100 of 32000 7.0 / 7.4 (work groups wait on their own join); with 5 top tokens 1 of
// 16000 8.2 / 6.3, 500 of 32000 15.4 / 13.2, 8000 of 10000 85 / 70, but 8000 of 1000 64 / 71 (three waves of four have no
// chunk); 1 of 50257 (13 chunks) 9.9 / 13.8.
bool in_one(int rows, int chunks, bool top, int cus) {
  const bool few = rows <= 4 * (cus > 0 ? cus : 256);
  return top ? chunks <= kWhole && (few || chunks > 1) : chunks == 1 || (chunks <= 4 && few);
}

template <typename T>
void forward(const Params &p, hipStream_t s) {
  if (in_one(p.N, p.chunks, p.K > 0, dan::num_cus())) return p.entropy ? forward_whole<T, true>(p, s) : forward_whole<T, false>(p, s);
  const dim3 grid((unsigned)(((int64_t)p.N * p.chunks + 3) / 4));
  if (p.entropy) {
    if (p.K > 0) hipLaunchKernelGGL((chunk_kernel<T, true, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((chunk_kernel<T, true, false>), grid, dim3(256), 0, s, p);
  } else {
    if (p.K > 0) hipLaunchKernelGGL((chunk_kernel<T, false, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((chunk_kernel<T, false, false>), grid, dim3(256), 0, s, p);
  }
  if (p.K > 0) launch_top<T>(p, s);
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
  if (abi != DAN_READOUT_ABI_VERSION && abi != 1) return fail(DAN_ERR_VERSION, "abi_version %d, readout speaks %d and 1", abi, DAN_READOUT_ABI_VERSION);
  if (dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16 && dtype != DAN_DTYPE_F32) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16, f16 or f32", dtype);
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || labels < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "need rows >= 0, vocab in [1, 2^30] and labels >= 0");
  if (top < 0 || top > DAN_READOUT_MAX_TOP || top > vocab)
    return fail(DAN_ERR_INVALID_ARGUMENT, "top %d: at most %d and the vocabulary's %d", top, DAN_READOUT_MAX_TOP, vocab);
  if (top > 0 && vocab > DAN_READOUT_MAX_TOP_VOCAB)
    return fail(DAN_ERR_UNSUPPORTED, "top tokens of %d values: rows of at most %d", vocab, DAN_READOUT_MAX_TOP_VOCAB);
  if (stride < 0 || tokens_stride < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "row strides must be >= 0");
  // A launch has fewer than 2^32 threads: 64 a chunk, and 256 a row but for rows of one chunk without top tokens.
  const int64_t chunks = chunks_of(dtype, vocab);
  if ((rows * chunks + 3) / 4 * 256 >= (int64_t)1 << 32 || ((top > 0 || chunks > 1) && rows >= 1 << 24))
    return fail(DAN_ERR_INVALID_ARGUMENT, "%d rows: too many for one launch", rows);
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
  p.rest = a->abi_version == 1 ? nullptr : a->logsumexp_rest;
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
  p.rest = a->abi_version == 1 ? nullptr : a->logsumexp_rest;
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
