// Gradient of tree-masked attention for gfx950 (include/dan_tree_grad.h).
//
// With S = scale Q K^T, P = softmax(S) over the visible keys, O = P V, and the
// output's gradient G:
//   delta_i = sum_d G_id O_id       dP = G V^T        dS = P * (dP - delta)
//   dV = P^T G                      dQ = scale dS K   dK = scale dS^T Q
// P is computed again from Q, K and the forward pass's logsumexp. Two launches, or three:
//   grad_rows_kernel     delta, and for fp16 a bound of |dS|;
//   grad_kernel          dK and dV (grad_keys): a work group holds a run of keys and
//                        walks the query rows that see them, over the heads of the kv
//                        head; and dQ (grad_queries): it holds query rows of the heads
//                        that share a kv head and walks the keys that they see;
//   grad_sum_kernel      where few keys made several work groups share them by heads,
//                        adds those parts up;
// Each result, or part of one, is summed by one work group in a fixed order, and parts are
// added up in order, so there are no atomics
// and the results do not change from run to run. The price is that S and dP are
// computed twice: 7 products where 5 would do (dQ summed by atomics, or written and
// read again in fp32 for every run of keys, would cost 8192 rows of 32 heads x 128
// that see 7700 keys 134 MB for each run of them). Parts of dK and dV cost their
// bytes twice, in fp32 (2 D numbers a row, kv head and part): 2000 rows of 2 kv heads
// x 128 in 4 parts 16 MB, written and read again.
//
// Measured: 8192 rows in one request of 32 branches, 32/8 heads x 128, bf16: rows 28 us
// (134 MB, 4.8 TB/s), keys and queries 1.7 ms (1917 GFLOP, 1130 TFLOP/s; in launches of
// their own 0.94 and 0.73), where a library's product of 16384^3 reaches 1370. The matrix unit is
// busy 57 % (keys) and 52 % (queries) of the time at about 1.95 GHz, which the power
// holds; what it waits for is the chain from S over its exponentials to dS in each wave,
// of which one fits a SIMD (its registers are full; what is needed once in front of or behind a loop,
// 18 to 54 of them, is kept in scratch memory at head_dim 128 and 256, but for bf16's larger unit of 256). With head_dim 256 every operand read
// feeds one product instead of two, and LDS is as busy as the matrix unit: 4099 rows
// behind 1024 keys, 16/2 heads x 256: 241 us. Batches of a few thousand rows have one to
// four units a compute unit, and each loads, joins and stores by itself (10 us of its 50 to 100):
// 3413 rows in four requests, 32/8 x 128, fp16: 180 us.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "dan_tree_grad.h"
#include "tiles.h"

namespace dan {

int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
extern thread_local char g_err[512];

namespace {

using namespace tiles;

constexpr int kThreads = 256;
constexpr int kMaxPartials = 1024;  // work groups of grad_rows_kernel, and partial maxima
// fp16: P goes into its product times 2^14, so that the small probabilities of long rows keep their bits.
constexpr float kPBias = 14.0f;
constexpr int64_t kAlign = 256;

// Rows (keys, queries) that a wave holds: 64, or 32 where head_dim 256 takes twice the registers. A wave
// reads each tile of the other side from LDS once for all of them: 64 B a clock of the CU's 128 with 64 rows.
template <int D>
constexpr int kWaveRows = D == 256 ? 32 : 64;

struct GradParams {
  const void *q, *k, *v, *o, *g;
  void *dq, *dk, *dv;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, g_st, g_sh, dq_st, dq_sh, dk_st, dk_sh, dv_st, dv_sh;
  const float *lse;
  float *stats;    // [2][H][N]: (bias - lse) / c, -delta
  float *partial;  // [3][partials]: max |G row|^2, max |V row|^2, max |delta|
  float *parts;    // [splits][2][Hkv][N][D]: dK, dV
  const DanGradKeyUnit *key_units;
  const DanGradQueryUnit *query_units;
  const int32_t *row_lo, *row_end;
  const DanPastDesc *pasts;
  int32_t num_tokens, num_heads, num_kv_heads, rep, hpw, groups, num_pasts, partials, key_rows, splits, key_groups;
  float scale, c;  // c = scale * log2 e
};

template <typename T>
__device__ inline T load_unit(const T *p) {
  struct Raw {
    uint32_t w[sizeof(T) / 4];
  } raw;
  const __attribute__((address_space(4))) uint32_t *src = (const __attribute__((address_space(4))) uint32_t *)p;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) raw.w[i] = __builtin_amdgcn_readfirstlane(src[i]);
  return __builtin_bit_cast(T, raw);
}

__device__ inline float block_max(float x, float *red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  x = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return x;
}

// The larger of two sizes; an infinite or NaN one has no part in fp16's power of 2, whose batch other segments share.
__device__ inline float finite_max(float top, float x) { return x < INFINITY ? fmaxf(top, x) : top; }

// Sum of squares over the L lanes of a row, 8 values each.
template <typename T, int L>
__device__ inline float row_square(u32x4 x) {
  const f32x8 v = unpack8<T>(x);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq = fmaf(v[i], v[i], sq);
#pragma unroll
  for (int m = L / 2; m; m >>= 1) sq += __shfl_xor(sq, m);
  return sq;
}

// ---------------------------------------------------------------- delta
// One pass over G and O (2 x 67 MB at 8192 rows x 32 heads x 128: 28 us, 4.8 TB/s): a row is D / 8 lanes, 16 bytes each.
// delta takes O as it was rounded: half a step of O moves dS by as much as dS's own rounding does. With O's 16-bit rest kept beside it delta
// would be exact, and the forward pass would write, and the program keep, as many bytes again.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void grad_rows_kernel(const GradParams p) {
  constexpr int L = D / 8, R = kThreads / L;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  const int sub = threadIdx.x % L, mine = threadIdx.x / L;
  const int64_t rows = (int64_t)p.num_tokens * p.num_heads;
  float gmax = 0.f, vmax = 0.f, dmax = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * R + mine; r < rows; r += (int64_t)gridDim.x * R) {
    const int64_t n = r / p.num_heads, h = r % p.num_heads;
    const f32x8 g = unpack8<T>(load16(static_cast<const T *>(p.g) + n * p.g_st + h * p.g_sh + 8 * sub));
    const f32x8 o = unpack8<T>(load16(static_cast<const T *>(p.o) + n * p.o_st + h * p.o_sh + 8 * sub));
    float dot = 0.f, sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dot = fmaf(g[i], o[i], dot);
      if (kHalf) sq = fmaf(g[i], g[i], sq);
    }
#pragma unroll
    for (int m = L / 2; m; m >>= 1) {
      dot += __shfl_xor(dot, m);
      if (kHalf) sq += __shfl_xor(sq, m);
    }
    if (sub == 0) {
      const int64_t at = h * p.num_tokens + n;
      p.stats[at] = ((kHalf ? kPBias : 0.f) - p.lse[at]) / p.c;
      p.stats[rows + at] = -dot;
    }
    if (kHalf && p.row_end[n] > 0) {  // (rows of no segment may hold anything, and their dS is never made)
      gmax = finite_max(gmax, sq);
      dmax = finite_max(dmax, fabsf(dot));
    }
  }
  if constexpr (kHalf) {
    const int64_t vrows = (int64_t)p.num_tokens * p.num_kv_heads;
    for (int64_t r = (int64_t)blockIdx.x * R + mine; r < vrows; r += (int64_t)gridDim.x * R) {
      const int64_t n = r / p.num_kv_heads, h = r % p.num_kv_heads;
      const float sq = row_square<T, L>(load16(static_cast<const T *>(p.v) + n * p.v_st + h * p.v_sh + 8 * sub));
      if (p.row_end[n] > 0) vmax = finite_max(vmax, sq);
    }
    for (int i = 0; i < p.num_pasts; ++i) {
      const DanPastDesc pd = load_unit(p.pasts + i);
      const int64_t prows = (int64_t)pd.len * p.num_kv_heads;
      for (int64_t r = (int64_t)blockIdx.x * R + mine; r < prows; r += (int64_t)gridDim.x * R) {
        const int64_t n = r / p.num_kv_heads, h = r % p.num_kv_heads;
        vmax = finite_max(vmax, row_square<T, L>(load16(static_cast<const T *>(pd.v) + n * pd.v_stride_tok + h * pd.v_stride_head + 8 * sub)));
      }
    }
    __shared__ float red[4];
    gmax = block_max(gmax, red);
    vmax = block_max(vmax, red);
    dmax = block_max(dmax, red);
    if (threadIdx.x == 0) {
      p.partial[blockIdx.x] = gmax;
      p.partial[p.partials + blockIdx.x] = vmax;
      p.partial[2 * p.partials + blockIdx.x] = dmax;
    }
  }
}

// fp16: the power of 2 that brings every |dS| under 2^15 and keeps the rest as far above fp16's smallest
// as it goes: |dP| <= |G row| |V row|.
__device__ inline float ds_factor(const GradParams &p, float *red) {
  float g = 0.f, v = 0.f, d = 0.f;
  for (int i = threadIdx.x; i < p.partials; i += kThreads) {
    g = fmaxf(g, p.partial[i]);
    v = fmaxf(v, p.partial[p.partials + i]);
    d = fmaxf(d, p.partial[2 * p.partials + i]);
  }
  g = block_max(g, red);
  v = block_max(v, red);
  d = block_max(d, red);
  const float bound = sqrtf(g) * sqrtf(v) + d;
  if (!(bound > 0.f)) return 1.f;
  const int e = min(max(14 - ilogbf(bound), -100), 100);
  return ldexpf(1.f, e);
}

// Results of a 32x32 product whose lane holds column `lane % 32`, rows 8 (i / 4) + 4 (l / 32) + i % 4, scaled and
// stored as the lane's row of memory: lanes l and l ^ 32 trade halves, so that each stores 16 bytes at a time.
template <typename T>
__device__ inline void store_column(T *row, const f32x16 &x, float f, int hl, bool valid) {
#pragma unroll
  for (int jp = 0; jp < 2; ++jp) {
    const u32x2 even = pack4<T>(f32x4{x[8 * jp], x[8 * jp + 1], x[8 * jp + 2], x[8 * jp + 3]} * f);
    const u32x2 odd = pack4<T>(f32x4{x[8 * jp + 4], x[8 * jp + 5], x[8 * jp + 6], x[8 * jp + 7]} * f);
    // lanes below 32 get (even, the partner's even), the others (the partner's odd, odd)
    const auto a = __builtin_amdgcn_permlane32_swap(even[0], odd[0], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(even[1], odd[1], false, false);
    if (valid) store16(row + 8 * (2 * jp + hl), u32x4{a[0], b[0], a[1], b[1]});
  }
}

// 8 of a lane's 16 results, rounded and packed.
template <typename T>
__device__ inline u32x4 pack_part(const f32x16 &x, int first) {
  f32x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[first + i];
  return pack8<T>(y);
}

// ---------------------------------------------------------------- dK, dV
// Four waves: KW runs of kWaveRows keys side by side, and 4 / KW of the (32 rows, head) tiles of a step. A wave
// keeps its keys' K and V (as operands) and dK and dV (as accumulators) in registers: 384 of 512 at head_dim 128
// and 64 keys. Tiles of Q and G come to LDS by direct loads, a ring of steps ahead of their use.
// (S's and dP's operands read for each block of 32 keys by itself, so that a block's softmax has the other's products to hide
// behind, were 3 % slower at head_dim 128 and 25 % in fp16 with the smaller unit: LDS is read a third more.)
template <int D, int KW>
struct KeyLds {
  static constexpr int QW = 4 / KW;
  static constexpr int stage = 2 * QW * Tile<D>::bytes;
  static constexpr int stat_step = 1024;  // [4 waves][64 floats]
  static constexpr int ring = 4 * (stage + stat_step) <= 140 * 1024 ? 4 : 3 * (stage + stat_step) <= 140 * 1024 ? 3 : 2;
  static constexpr int stats = ring * stage;
  static constexpr int red = stats + ring * stat_step;  // 16 floats
  static constexpr int wave = 2 * kWaveRows<D> * D * 4;  // a wave's dK and dV
  static constexpr int merge = QW > 1 ? QW / 2 * KW * wave : 0;
  static constexpr int total = red + 64 > merge ? red + 64 : merge;
  static_assert(total <= 160 * 1024, "LDS");
};

template <typename T, int D, int KW>
__device__ __forceinline__ void grad_keys(const GradParams &p, int block, uint8_t *smem) {
  using Tl = Tile<D>;
  using Lds = KeyLds<D, KW>;
  constexpr int NS = kWaveRows<D> / 32, QW = 4 / KW, NK = D / 16, ND = D / 32, NB = Lds::ring;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  const uint32_t lds = (uint32_t)(uintptr_t)(DAN_TILE_LDS uint8_t *)smem;
  const int lane = threadIdx.x & 63, hl = lane >> 5, wave = uni(threadIdx.x >> 6);
  const int kw = wave % KW, qw = wave / KW;
  // A work group's unit, kv head, and part of the heads that share it.
  const int kvh = block % p.num_kv_heads, part = block / p.num_kv_heads % p.splits;
  const int head0 = kvh * p.rep + p.rep * part / p.splits, rep = kvh * p.rep + p.rep * (part + 1) / p.splits - head0;
  const DanGradKeyUnit un = load_unit(p.key_units + block / (p.num_kv_heads * p.splits));
  if (un.start < 0 || un.n <= 0 || un.start + un.n > p.num_tokens || un.key0 < 0 || un.keys <= 0 || un.keys > p.key_rows ||
      un.key0 + un.keys > un.n || un.q_end <= un.key0 || un.q_end > un.n)
    return;  // no such rows
  float factor = 1.f;
  if constexpr (kHalf) factor = ds_factor(p, reinterpret_cast<float *>(smem + Lds::red));

  // The lane's keys: row 32 s + lane % 32 of the wave's. Key x is seen by the rows [x, x + see).
  const int wkey = un.key0 + kw * kWaveRows<D>, kend = un.key0 + un.keys;
  u32x4 kf[NS][NK], vf[NS][NK];
  int key[NS], see[NS];
  int low = un.n;  // the rows below it and past the last key see every key
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    key[s] = wkey + 32 * s + (lane & 31);
    const bool valid = key[s] < kend;
    const int64_t row = un.start + min(key[s], kend - 1);
    const T *kr = static_cast<const T *>(p.k) + row * p.k_st + kvh * p.k_sh + 8 * hl;
    const T *vr = static_cast<const T *>(p.v) + row * p.v_st + kvh * p.v_sh + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      kf[s][kk] = load16(kr + 16 * kk);
      vf[s][kk] = load16(vr + 16 * kk);
    }
    const int end = valid ? p.row_end[row] : 0;
    see[s] = max(end - key[s], 0);
    low = min(low, end);
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) low = min(low, __shfl_xor(low, m));
  low = uni(low);

  f32x16 dk[NS][ND], dv[NS][ND];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int db = 0; db < ND; ++db) dk[s][db] = dv[s][db] = f32x16{};

  // Tiles in order: a head after the other, then the next 32 rows. A step takes QW of them; the KW waves that share one load it.
  const int tiles = (un.q_end - un.key0 + 31) / 32 * rep, steps = (tiles + QW - 1) / QW;
  const int64_t plane = (int64_t)p.num_heads * p.num_tokens;
  const int rest = QW % rep, whole = QW / rep;  // from a wave's tile to its next: `rest` heads and 32 `whole` rows on
  int next = min(qw, tiles - 1), next_head = next % rep, next_left = un.n - 1 - un.key0 - 32 * (next / rep);  // left: rows of the segment past the tile's first
  auto tile_at = [&](const void *base, int64_t st, int64_t sh) __attribute__((always_inline)) {
    return uniform_ptr(static_cast<const char *>(base) + 2 * ((un.start + un.key0 + 32 * (int64_t)(next / rep)) * st + (head0 + next_head) * sh));
  };
  const char *q_at = tile_at(p.q, p.q_st, p.q_sh), *g_at = tile_at(p.g, p.g_st, p.g_sh);
  const float *s_at = uniform_ptr(p.stats + (int64_t)(head0 + next_head) * p.num_tokens + un.start + un.key0 + 32 * (next / rep));
  const int64_t q_on = 2 * (rest * p.q_sh + 32 * whole * p.q_st), g_on = 2 * (rest * p.g_sh + 32 * whole * p.g_st), s_on = rest * (int64_t)p.num_tokens + 32 * whole;
  const int64_t q_wrap = 2 * (32 * p.q_st - rep * p.q_sh), g_wrap = 2 * (32 * p.g_st - rep * p.g_sh), s_wrap = 32 - rep * (int64_t)p.num_tokens;
  const uint32_t q_row = (uint32_t)(2 * p.q_st), g_row = (uint32_t)(2 * p.g_st);
  // The x-th load of a step, into ring buffer b: every wave issues LOADS for every step (past its last tile, that
  // one's again), so that a count of them says which have landed. Rows past the segment are its last row's copies.
  constexpr int LB = Tl::blocks / KW, LOADS = 2 * LB + 1;
  auto issue = [&](auto index, int b) __attribute__((always_inline)) {
    constexpr int x = decltype(index)::value % LB;
    constexpr bool kQ = decltype(index)::value < LB;
    const uint32_t dst = lds + (uint32_t)(b * Lds::stage + 2 * qw * Tl::bytes + kw * 1024);
    if constexpr (decltype(index)::value < 2 * LB) {
      const uint32_t m = (uint32_t)min(Tl::block_row(kw + KW * x, lane), next_left);
      dma16(kQ ? q_at : g_at, m * (kQ ? q_row : g_row) + Tl::block_byte(kw + KW * x, lane), dst + (uint32_t)((kQ ? 0 : Tl::bytes) + x * KW * 1024));
    } else {
      // (each wave its own copy of the tile's statistics)
      dma4(s_at, (uint32_t)(min(lane & 31, next_left) * 4 + hl * (int)(plane * 4)), lds + (uint32_t)(Lds::stats + b * Lds::stat_step + wave * 256));
      // (selections, no branches: a step is one block of instructions)
      const bool more = next + QW < tiles, wrap = more && next_head + rest >= rep;
      next += more ? QW : 0;
      next_head += (more ? rest : 0) - (wrap ? rep : 0);
      next_left -= (more ? 32 * whole : 0) + (wrap ? 32 : 0);
      q_at += (more ? q_on : 0) + (wrap ? q_wrap : 0);
      g_at += (more ? g_on : 0) + (wrap ? g_wrap : 0);
      s_at += (more ? s_on : 0) + (wrap ? s_wrap : 0);
    }
  };
  const uint32_t rows_at = Tl::rows_at(lane), cols_at = Tl::cols_at(lane);
  // A tile's four products, NK operand reads each, every read two ahead of its use:
  //   S = K Q^T | dP = V G^T, and meanwhile P = exp2(c S) | dV += P^T G, and meanwhile dS = P dP | dK += dS^T Q.
  // S starts at -lse / c and dP at -delta. With a ring of three or more the step's barrier stands before the last
  // product: the step after has landed then and every wave has left the step before, whose buffer the loads that go
  // out over that product fill, and the next tile's first operands are read at its end. With two buffers the barrier
  // stands before the first product, and the next step's loads go out over it.
  constexpr bool kEarly = NB > 2;
  auto land = [&]() __attribute__((always_inline)) {  // (a tile that no other wave reads needs no barrier)
    if constexpr (KW > 1) barrier_lds();
    else barrier_wave_lds();
  };
  f32x16 start;    // -lse / c of the tile's rows (then -delta)
  u32x4 ahead[2];  // the tile's first two operands
  auto read_stats = [&](int b, int which) __attribute__((always_inline)) {
    const uint32_t at = lds + (uint32_t)(Lds::stats + b * Lds::stat_step + wave * 256 + which * 128 + 16 * hl);
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const f32x4 x = __builtin_bit_cast(f32x4, lds_read16(at + 32 * i4));
#pragma unroll
      for (int e = 0; e < 4; ++e) start[4 * i4 + e] = x[e];
    }
  };
  auto tile_of = [&](int b) __attribute__((always_inline)) { return lds + (uint32_t)(b * Lds::stage + 2 * qw * Tl::bytes); };
  auto read_first = [&](int b) __attribute__((always_inline)) {
    read_stats(b, 0);
    ahead[0] = Tl::read_rows(tile_of(b), rows_at, 0);
    ahead[1] = Tl::read_rows(tile_of(b), rows_at, 1);
  };
  auto compute = [&](auto masked, int qb, int b) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(masked)::value;
    constexpr int EC = 16 * NS / NK;  // elements a step
    const int to = b == 0 ? NB - 1 : b - 1, after = b == NB - 1 ? 0 : b + 1;
    const uint32_t qt = tile_of(b), gt = qt + Tl::bytes;
    if constexpr (!kEarly) {
      wait_vmem<0>();
      land();
      read_first(b);
    }
    f32x16 sc[NS], dp[NS];
    u32x4 op[4 * NK], pf[NS][2], df[NS][2];
    op[0] = ahead[0];
    op[1] = ahead[1];
    auto read = [&](auto index) __attribute__((always_inline)) {
      constexpr int i = decltype(index)::value;
      if constexpr (i < NK) op[i] = Tl::read_rows(qt, rows_at, i);
      else if constexpr (i < 2 * NK) op[i] = Tl::read_rows(gt, rows_at, i - NK);
      else if constexpr (i < 3 * NK) op[i] = Tl::read_cols(gt, cols_at, (i - 2 * NK) % ND, (i - 2 * NK) / ND);
      else if constexpr (i < 4 * NK) op[i] = Tl::read_cols(qt, cols_at, (i - 3 * NK) % ND, (i - 3 * NK) / ND);
    };
    static_for<4 * NK>([&](auto index) __attribute__((always_inline)) {
      constexpr int i = decltype(index)::value, kk = i % NK, db = kk % ND, ks = kk / ND;
      if constexpr (kEarly && i == 3 * NK) {
        wait_vmem<(NB - 3) * LOADS>();
        land();
      }
      if constexpr (i == NK - 1) read_stats(b, 1);
      if constexpr (kEarly && i == 4 * NK - 2) read_first(after);
      read(std::integral_constant<int, i + 2>{});
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if constexpr (i < NK) sc[s] = mfma32<T>(op[i], kf[s][kk], kk ? sc[s] : start);
        else if constexpr (i < 2 * NK) dp[s] = mfma32<T>(op[i], vf[s][kk], kk ? dp[s] : start);
        else if constexpr (i < 3 * NK) mfma32_sum<T>(dv[s][db], op[i], pf[s][ks]);
        else mfma32_sum<T>(dk[s][db], op[i], df[s][ks]);
      }
      if constexpr (kEarly ? i >= 3 * NK : i < NK) {
        static_for<LOADS>([&](auto x) __attribute__((always_inline)) {
          if constexpr (decltype(x)::value * NK / LOADS == kk) issue(x, to);
        });
      }
      if constexpr (i >= NK && i < 3 * NK) {
        static_for<EC>([&](auto x) __attribute__((always_inline)) {
          constexpr int e = kk * EC + decltype(x)::value, s = e / 16, r = e % 16;
          if constexpr (i < 2 * NK) {
            sc[s][r] = __builtin_amdgcn_exp2f(sc[s][r] * p.c);
            if (kMask) sc[s][r] = (uint32_t)(qb + 4 * hl - key[s] + 8 * (r >> 2) + (r & 3)) < (uint32_t)see[s] ? sc[s][r] : 0.f;
            if constexpr (r % 8 == 7) pf[s][r / 8] = pack_part<T>(sc[s], r - 7);
          } else {
            dp[s][r] *= kHalf ? sc[s][r] * factor : sc[s][r];
            if (kMask) dp[s][r] = sc[s][r] != 0.f ? dp[s][r] : 0.f;  // (a hidden key's dP may be anything)
            if constexpr (r % 8 == 7) df[s][r / 8] = pack_part<T>(dp[s], r - 7);
          }
        });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  if constexpr (kHalf) factor *= 1.f / 16384.f;  // P carries 2^kPBias
  for (int i = 0; i < NB - 1; ++i) static_for<LOADS>([&](auto x) __attribute__((always_inline)) { issue(x, i); });
  int b = 0, head = qw % rep, qb = un.key0 + 32 * (qw / rep), t = qw;  // of the wave's tile
  // Steps up to `end`. A step past the wave's last tile sees nothing of it.
  if constexpr (kEarly) {
    wait_vmem<(NB - 2) * LOADS>();
    land();
    read_first(0);
  }
  auto run = [&](auto masked, int &i, int end) __attribute__((always_inline)) {
    for (; i < end; ++i) {
      compute(masked, t < tiles ? qb : 0x3fffffff, b);
      b = b == NB - 1 ? 0 : b + 1;
      t += QW;
      head += QW % rep;
      qb += 32 * (QW / rep) + (head >= rep ? 32 : 0);
      head -= head >= rep ? rep : 0;
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      settle(dk[s]);
      settle(dv[s]);
    }
  };
  // The tiles that every key of the wave is seen from are a range: from the first whose rows all come after the keys.
  const int full0 = (wkey + kWaveRows<D> - 1 - un.key0 + 31) / 32 * rep, full1 = max((low - un.key0) / 32, 0) * rep;
  auto step_of = [&](int tile) __attribute__((always_inline)) { return min(max((tile - qw + QW - 1) / QW, 0), steps); };
  int i = 0;
  run(std::true_type{}, i, full0 < full1 ? step_of(full0) : steps);
  run(std::false_type{}, i, step_of(full1));
  run(std::true_type{}, i, steps);
  wait_vmem<0>();
  if constexpr (QW > 1) {  // the waves of the same keys add up, pairwise, over LDS
#pragma unroll
    for (int h = QW / 2; h; h >>= 1) {
      barrier_lds();
      const uint32_t at = lds + (uint32_t)((qw % h * KW + kw) * Lds::wave + lane * 16);
      if (qw >= h && qw < 2 * h) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int db = 0; db < ND; ++db)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t to = at + (uint32_t)(((s * ND + db) * 8 + x) * 1024);
              *(DAN_TILE_LDS f32x4 *)(uintptr_t)to = f32x4{dk[s][db][4 * x], dk[s][db][4 * x + 1], dk[s][db][4 * x + 2], dk[s][db][4 * x + 3]};
              *(DAN_TILE_LDS f32x4 *)(uintptr_t)(to + 4096) = f32x4{dv[s][db][4 * x], dv[s][db][4 * x + 1], dv[s][db][4 * x + 2], dv[s][db][4 * x + 3]};
            }
      }
      barrier_lds();
      if (qw < h) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int db = 0; db < ND; ++db)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t from = at + (uint32_t)(((s * ND + db) * 8 + x) * 1024);
              const f32x4 a = __builtin_bit_cast(f32x4, lds_read16(from)), c = __builtin_bit_cast(f32x4, lds_read16(from + 4096));
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                dk[s][db][4 * x + e] += a[e];
                dv[s][db][4 * x + e] += c[e];
              }
            }
      }
    }
    if (qw > 0) return;
  }
  // With several parts of the heads: fp32 sums, [part][dK, dV][kv head][row], for grad_sum_kernel.
  const float fv = kHalf ? 1.f / 16384.f : 1.f, fk = kHalf ? p.scale / (factor * 16384.f) : p.scale;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int64_t row = un.start + min(key[s], kend - 1);
    if (p.splits > 1) {
      float *kp = p.parts + ((2 * (int64_t)part * p.num_kv_heads + kvh) * p.num_tokens + row) * D + 4 * hl, *vp = kp + (int64_t)p.num_kv_heads * p.num_tokens * D;
      if (key[s] < kend)
#pragma unroll
        for (int db = 0; db < ND; ++db)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            *(DAN_TILE_GLOBAL f32x4 *)(kp + 32 * db + 8 * x) = f32x4{dk[s][db][4 * x], dk[s][db][4 * x + 1], dk[s][db][4 * x + 2], dk[s][db][4 * x + 3]} * fk;
            *(DAN_TILE_GLOBAL f32x4 *)(vp + 32 * db + 8 * x) = f32x4{dv[s][db][4 * x], dv[s][db][4 * x + 1], dv[s][db][4 * x + 2], dv[s][db][4 * x + 3]} * fv;
          }
      continue;
    }
    T *kr = static_cast<T *>(p.dk) + row * p.dk_st + kvh * p.dk_sh, *vr = static_cast<T *>(p.dv) + row * p.dv_st + kvh * p.dv_sh;
#pragma unroll
    for (int db = 0; db < ND; ++db) {
      store_column<T>(kr + 32 * db, dk[s][db], fk, hl, key[s] < kend);
      store_column<T>(vr + 32 * db, dv[s][db], fv, hl, key[s] < kend);
    }
  }
}

// The parts of dK and dV added up in order, rounded once: 8 values a thread of one kv head's dK or dV. Rows that no unit
// holds are left as they are.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void grad_sum_kernel(const GradParams p) {
  constexpr int L = D / 8;
  const int n = blockIdx.x * (kThreads / L) + threadIdx.x / L, kvh = blockIdx.y, which = blockIdx.z, column = threadIdx.x % L * 8;
  if (n >= p.num_tokens || p.row_end[n] <= 0) return;
  const int64_t plane = (int64_t)p.num_kv_heads * p.num_tokens * D;
  const float *from = p.parts + which * plane + ((int64_t)kvh * p.num_tokens + n) * D + column;
  f32x4 x = {}, y = {};
  for (int i = 0; i < p.splits; ++i, from += 2 * plane) {
    x += *(const DAN_TILE_GLOBAL f32x4 *)from;
    y += *(const DAN_TILE_GLOBAL f32x4 *)(from + 4);
  }
  T *to = which ? static_cast<T *>(p.dv) + n * p.dv_st + kvh * p.dv_sh : static_cast<T *>(p.dk) + n * p.dk_st + kvh * p.dk_sh;
  store16(to + column, pack8<T>(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)));
}

// ---------------------------------------------------------------- dQ
// Four waves: hpw heads of the kv head by 4 / hpw runs of kWaveRows rows. A wave keeps its rows' Q and G and their
// dQ in registers; tiles of 32 keys of K and V come to LDS by direct loads.
template <int D>
struct QueryLds {
  static constexpr int stage = 2 * Tile<D>::bytes, ring = 4;
  static constexpr int red = ring * stage;
  static constexpr int total = red + 64;
  static_assert(total <= 160 * 1024, "LDS");
};

template <typename T, int D>
__device__ __forceinline__ void grad_queries(const GradParams &p, int block, uint8_t *smem) {
  using Tl = Tile<D>;
  using Lds = QueryLds<D>;
  constexpr int NS = kWaveRows<D> / 32, NK = D / 16, ND = D / 32, NB = Lds::ring;
  constexpr int TS = Tl::blocks / 4, SL = 2 * TS;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  const uint32_t lds = (uint32_t)(uintptr_t)(DAN_TILE_LDS uint8_t *)smem;
  const int lane = threadIdx.x & 63, hl = lane >> 5, wave = uni(threadIdx.x >> 6);
  const int group = block % p.groups, kvh = group % p.num_kv_heads, chunk = group / p.num_kv_heads;
  const DanGradQueryUnit un = load_unit(p.query_units + block / p.groups);
  if (un.start < 0 || un.n <= 0 || un.start + un.n > p.num_tokens || un.t0 < 0 || un.tq <= 0 || un.t0 + un.tq > un.n ||
      un.tq > kWaveRows<D> * 4 / p.hpw || un.trunk < 0 || un.trunk > un.n || un.branch0 < 0 ||
      (un.past_len > 0 && (un.past_idx < 0 || un.past_idx >= p.num_pasts)))
    return;  // no such rows
  float factor = 1.f;
  if constexpr (kHalf) factor = ds_factor(p, reinterpret_cast<float *>(smem + Lds::red)) * (1.f / 16384.f);

  // The keys, three runs one after the other in tiles of 32: the prefix, the trunk up to the unit's last row, and
  // the branch rows from the first one's branch on.
  const int tend = un.t0 + un.tq, t_hi = min(un.trunk, tend);
  const int past_tiles = max(un.past_len + 31, 0) / 32, trunk_tiles = (t_hi + 31) / 32;
  const int steps = past_tiles + trunk_tiles + (tend > un.trunk ? max(tend - un.branch0 + 31, 0) / 32 : 0);
  const T *pk = nullptr, *pv = nullptr;
  int64_t pk_st = 0, pv_st = 0;
  if (past_tiles) {
    const DanPastDesc pd = load_unit(p.pasts + un.past_idx);
    if (pd.len < un.past_len) return;  // no such prefix
    pk = static_cast<const T *>(pd.k) + kvh * pd.k_stride_head;
    pv = static_cast<const T *>(pd.v) + kvh * pd.v_stride_head;
    pk_st = pd.k_stride_tok;
    pv_st = pd.v_stride_tok;
  }
  const T *own_k = static_cast<const T *>(p.k) + un.start * p.k_st + kvh * p.k_sh;
  const T *own_v = static_cast<const T *>(p.v) + un.start * p.v_st + kvh * p.v_sh;

  const int hig = chunk * p.hpw + wave % p.hpw, head = min(kvh * p.rep + hig, (kvh + 1) * p.rep - 1);
  const int w0 = un.t0 + wave / p.hpw * kWaveRows<D>;
  const bool work = hig < p.rep && w0 < tend && wave / p.hpw < 4 / p.hpw;
  const int64_t plane = (int64_t)p.num_heads * p.num_tokens;
  u32x4 qf[NS][NK], gf[NS][NK];
  float nl[NS], nd[NS];
  int row[NS], lo[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    row[s] = w0 + 32 * s + (lane & 31);
    const int64_t r = un.start + min(row[s], tend - 1);
    const T *qr = static_cast<const T *>(p.q) + r * p.q_st + head * p.q_sh + 8 * hl;
    const T *gr = static_cast<const T *>(p.g) + r * p.g_st + head * p.g_sh + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      qf[s][kk] = load16(qr + 16 * kk);
      gf[s][kk] = load16(gr + 16 * kk);
    }
    nl[s] = p.stats[head * (int64_t)p.num_tokens + r];
    nd[s] = p.stats[plane + head * (int64_t)p.num_tokens + r];
    lo[s] = p.row_lo[r];
  }
  f32x16 dq[NS][ND];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int db = 0; db < ND; ++db) dq[s][db] = f32x16{};

  // What the next tile is loaded from: its first row, the rows of its run past that one, and the two runs still to come.
  const int branch_left = tend > un.trunk ? tend - un.branch0 - 1 : -1;  // (-1: no such run)
  const char *k_at = (const char *)(past_tiles ? pk : own_k), *v_at = (const char *)(past_tiles ? pv : own_v);
  const char *k_branch = (const char *)(own_k + un.branch0 * p.k_st), *v_branch = (const char *)(own_v + un.branch0 * p.v_st);
  if (!past_tiles && !trunk_tiles) {
    k_at = k_branch;
    v_at = v_branch;
  }
  k_at = uniform_ptr(k_at);
  v_at = uniform_ptr(v_at);
  uint32_t k_row = (uint32_t)(2 * (past_tiles ? pk_st : p.k_st)), v_row = (uint32_t)(2 * (past_tiles ? pv_st : p.v_st));
  int at_run = past_tiles ? 0 : trunk_tiles ? 1 : 2, next_left = at_run == 0 ? un.past_len - 1 : at_run == 1 ? t_hi - 1 : branch_left;
  // The x-th load of a step, into ring buffer b (past the last step: the last tile's again).
  constexpr int LOADS = SL;
  auto issue = [&](auto index, int b) __attribute__((always_inline)) {
    constexpr int x = decltype(index)::value % TS;
    constexpr bool kK = decltype(index)::value < TS;
    const uint32_t m = (uint32_t)min(Tl::block_row(4 * x + wave, lane), next_left);
    dma16(kK ? k_at : v_at, m * (kK ? k_row : v_row) + Tl::block_byte(4 * x + wave, lane),
          lds + (uint32_t)(b * Lds::stage + wave * 1024 + (kK ? 0 : Tl::bytes) + x * 4096));
    if constexpr (decltype(index)::value == LOADS - 1) {  // (selections, no branches: a step is one block of instructions)
      const bool same = next_left >= 32, trunk = !same && at_run == 0 && trunk_tiles > 0, branch = !same && !trunk && at_run < 2 && branch_left >= 0;
      next_left = same ? next_left - 32 : trunk ? t_hi - 1 : branch ? branch_left : next_left;
      k_at = same ? k_at + 32 * (int64_t)k_row : trunk ? (const char *)own_k : branch ? k_branch : k_at;
      v_at = same ? v_at + 32 * (int64_t)v_row : trunk ? (const char *)own_v : branch ? v_branch : v_at;
      k_row = trunk || branch ? (uint32_t)(2 * p.k_st) : k_row;
      v_row = trunk || branch ? (uint32_t)(2 * p.v_st) : v_row;
      at_run = trunk ? 1 : branch ? 2 : at_run;
    }
  };
  const uint32_t rows_at = Tl::rows_at(lane), cols_at = Tl::cols_at(lane);
  // A tile's three products for the wave's NS blocks of 32 rows:
  //   S = Q K^T of each block, and over the second block's P = exp2(c S) of the first; dP = G V^T of each block, and over them P of
  //   the second and dS = P dP of the first; dQ += dS K of both, each operand read once for them.
  // S starts at -lse / c and dP at -delta. K's and V's operands stay for the second block. The step's barrier stands
  // before the last product: the step after has landed then and every wave has left the step before, whose buffer the
  // loads that go out over that product fill, and the next tile's first operands are read at its end.
  u32x4 ahead[2];  // the tile's first two operands
  auto read_first = [&](int b) __attribute__((always_inline)) {
    ahead[0] = Tl::read_rows(lds + (uint32_t)(b * Lds::stage), rows_at, 0);
    ahead[1] = Tl::read_rows(lds + (uint32_t)(b * Lds::stage), rows_at, 1);
  };
  auto land = [&]() __attribute__((always_inline)) {
    wait_vmem<(NB - 3) * LOADS>();
    barrier_lds();
  };
  auto compute = [&](auto masked, int kb, int run, int b) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(masked)::value;
    constexpr int EC = 16 / NK > 0 ? 16 / NK : 1;  // elements of a block a step
    const int to = b == 0 ? NB - 1 : b - 1, after = b == NB - 1 ? 0 : b + 1;
    const uint32_t kt = lds + (uint32_t)(b * Lds::stage), vt = kt + Tl::bytes;
    int first[NS];
    uint32_t see[NS];
    if constexpr (kMask) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {  // the row sees `see` keys of this run, of which `first` lie past the lane's first one
        const int at = run < 2 ? 0 : row[s] < un.trunk ? row[s] + 1 : lo[s], last = run == 0 ? un.past_len - 1 : run == 1 ? min(row[s], un.trunk - 1) : row[s];
        first[s] = kb + 4 * hl - at;
        see[s] = (uint32_t)max(last - at + 1, 0);
      }
    }
    f32x16 sc[NS], dp[NS];
    u32x4 op[3 * NK], df[NS][2];
    auto read = [&](auto index) __attribute__((always_inline)) {
      constexpr int i = decltype(index)::value;
      if constexpr (i < NK) op[i] = Tl::read_rows(kt, rows_at, i);
      else if constexpr (i < 2 * NK) op[i] = Tl::read_rows(vt, rows_at, i - NK);
      else if constexpr (i < 3 * NK) op[i] = Tl::read_cols(kt, cols_at, (i - 2 * NK) % ND, (i - 2 * NK) / ND);
    };
    auto exps = [&](auto block, auto step) __attribute__((always_inline)) {
      constexpr int s = decltype(block)::value;
      static_for<EC>([&](auto x) __attribute__((always_inline)) {
        constexpr int r = decltype(step)::value * EC + decltype(x)::value;
        sc[s][r] = __builtin_amdgcn_exp2f(sc[s][r] * p.c);
        if (kMask) sc[s][r] = (uint32_t)(first[s] + 8 * (r >> 2) + (r & 3)) < see[s] ? sc[s][r] : 0.f;
      });
    };
    auto ds = [&](auto block, auto step) __attribute__((always_inline)) {
      constexpr int s = decltype(block)::value;
      static_for<EC>([&](auto x) __attribute__((always_inline)) {
        constexpr int r = decltype(step)::value * EC + decltype(x)::value;
        dp[s][r] *= kHalf ? sc[s][r] * factor : sc[s][r];
        if (kMask) dp[s][r] = sc[s][r] != 0.f ? dp[s][r] : 0.f;  // (a hidden key's dP may be anything)
        if constexpr (r % 8 == 7) df[s][r / 8] = pack_part<T>(dp[s], r - 7);
      });
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, NS - 1>;
    op[0] = ahead[0];
    op[1] = ahead[1];
    // S and dP of the blocks, one after the other: step i is product i / NK (S of each block, then dP of each).
    static_for<2 * NS * NK>([&](auto index) __attribute__((always_inline)) {
      constexpr int i = decltype(index)::value, kk = i % NK, s = i / NK % NS;
      constexpr bool kS = i < NS * NK;
      using Step = std::integral_constant<int, kk>;
      constexpr int at = kS ? kk : NK + kk;
      // what a first block reads two ahead: its own operands, then (at its end) nothing or the next product's
      if constexpr (s == 0 && kk + 2 < NK) read(std::integral_constant<int, at + 2>{});
      if constexpr (s == NS - 1 && kk + 2 >= NK) read(std::integral_constant<int, (kS ? NK : 2 * NK) + kk + 2 - NK>{});
      if constexpr (kS) {
        if constexpr (kk == 0)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[s][r] = nl[s];
        sc[s] = mfma32<T>(op[at], qf[s][kk], sc[s]);
        if constexpr (s > 0) exps(First{}, Step{});
      } else {
        if constexpr (kk == 0)
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[s][r] = nd[s];
        dp[s] = mfma32<T>(op[at], gf[s][kk], dp[s]);
        if constexpr (s == 0) exps(Second{}, Step{});
        else ds(First{}, Step{});
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    static_for<NK>([&](auto step) __attribute__((always_inline)) { ds(Second{}, step); });
    __builtin_amdgcn_sched_barrier(0);
    land();
    static_for<NK>([&](auto step) __attribute__((always_inline)) {
      constexpr int kk = decltype(step)::value;
      if constexpr (kk == NK - 2) read_first(after);
      read(std::integral_constant<int, 2 * NK + kk + 2>{});
#pragma unroll
      for (int s = 0; s < NS; ++s) mfma32_sum<T>(dq[s][kk % ND], op[2 * NK + kk], df[s][kk / ND]);
      static_for<LOADS>([&](auto x) __attribute__((always_inline)) {
        if constexpr (decltype(x)::value * NK / LOADS == kk) issue(x, to);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  for (int i = 0; i < NB - 1; ++i) static_for<LOADS>([&](auto x) __attribute__((always_inline)) { issue(x, i); });
  wait_vmem<(NB - 2) * LOADS>();
  barrier_lds();
  int b = 0;
  if (!work) {  // the loads and barriers alone
    for (int i = 0; i < steps; ++i) {
      land();
      static_for<LOADS>([&](auto x) __attribute__((always_inline)) { issue(x, b == 0 ? NB - 1 : b - 1); });
      b = b == NB - 1 ? 0 : b + 1;
    }
    wait_vmem<0>();
    return;
  }
  read_first(0);
  // `count` tiles of a run of keys from kb on, some hidden from a row or none.
  auto tiles = [&](auto masked, int run, int &kb, int count) __attribute__((always_inline)) {
    for (int n = 0; n < count; ++n) {
      compute(masked, kb, run, b);
      b = b == NB - 1 ? 0 : b + 1;
      kb += 32;
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(dq[s]);
  };
#pragma unroll 1
  for (int run = 0; run < 3; ++run) {
    const int count = run == 0 ? past_tiles : run == 1 ? trunk_tiles : steps - past_tiles - trunk_tiles;
    const int full = run == 0 ? un.past_len / 32 : run == 1 ? min(min(un.trunk, w0 + 1) / 32, count) : 0;
    int kb = run < 2 ? 0 : un.branch0;
    tiles(std::false_type{}, run, kb, full);
    tiles(std::true_type{}, run, kb, count - full);
  }
  wait_vmem<0>();
  const float f = kHalf ? p.scale / (factor * 16384.f) : p.scale;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    T *r = static_cast<T *>(p.dq) + (un.start + (int64_t)min(row[s], tend - 1)) * p.dq_st + head * p.dq_sh;
#pragma unroll
    for (int db = 0; db < ND; ++db) store_column<T>(r + 32 * db, dq[s][db], f, hl, row[s] < tend);
  }
}

// Both in one launch: the units of dK and dV, then those of dQ, each longest first. A work group fills a compute unit, and the last
// units of the one kind leave room for the first of the other: forward and backward pass of 3413 rows in four requests, fp16, 254 us in two
// launches and 244 in one, of 4099 in five behind 1024 keys, 16/2 heads x 256, 429 and 379 (with fewer parts of the heads); 8192 rows take as long.
template <typename T, int D, int KW>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads), amdgpu_waves_per_eu(1, 1)))
void grad_kernel(const GradParams p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int block = (int)blockIdx.x - p.key_groups;
  if (block < 0) grad_keys<T, D, KW>(p, blockIdx.x, smem);
  else grad_queries<T, D>(p, block, smem);
}

// ---------------------------------------------------------------- host
int wave_rows(int D) { return D == 256 ? 32 : 64; }
int heads_of_group(int rep) { return rep >= 3 ? 4 : rep; }

template <typename T, int D, int KW>
hipError_t launch_units(const GradParams &p, int64_t grid, hipStream_t s) {
  constexpr int bytes = std::max<int>(KeyLds<D, KW>::total, QueryLds<D>::total);
  const hipError_t err = allow_lds<&grad_kernel<T, D, KW>>(bytes);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((grad_kernel<T, D, KW>), dim3((uint32_t)grid), dim3(kThreads), bytes, s, p);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_all(const GradParams &p, int64_t grid, hipStream_t s) {
  hipLaunchKernelGGL((grad_rows_kernel<T, D>), dim3(p.partials), dim3(kThreads), 0, s, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  constexpr int KW = 64 / kWaveRows<D>;  // runs of a wave's keys in the smaller unit
  err = p.key_rows == 128 ? launch_units<T, D, 2 * KW>(p, grid, s) : launch_units<T, D, KW>(p, grid, s);
  if (err != hipSuccess || p.splits == 1) return err;
  constexpr int R = kThreads / (D / 8);
  hipLaunchKernelGGL((grad_sum_kernel<T, D>), dim3((p.num_tokens + R - 1) / R, p.num_kv_heads, 2), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace dan

extern "C" {

int dan_tree_grad_abi_version(void) { return DAN_TREE_GRAD_ABI_VERSION; }

int32_t dan_tree_grad_key_rows(int32_t head_dim, int32_t small) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return small ? 64 : 128;
}

int32_t dan_tree_grad_query_rows(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || !dan_tree_grad_key_rows(head_dim, 0)) return 0;
  return dan::wave_rows(head_dim) * 4 / dan::heads_of_group(num_heads / num_kv_heads);
}

// delta and the statistics, the bound's partials; then the parts of dK and dV.
static int64_t stats_bytes(int64_t H, int64_t N) { return (H * N * 8 + 3 * dan::kMaxPartials * 4 + dan::kAlign - 1) / dan::kAlign * dan::kAlign; }
int64_t dan_tree_grad_workspace_size(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_tokens, int32_t key_splits) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 || num_tokens <= 0 || key_splits < 1 || key_splits > num_heads / num_kv_heads) return 0;
  return stats_bytes(num_heads, num_tokens) + (key_splits > 1 ? (int64_t)key_splits * 2 * num_kv_heads * num_tokens * head_dim * 4 : 0);
}

int dan_tree_attn_bwd(const DanTreeGradArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_TREE_GRAD_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_TREE_GRAD_ABI_VERSION);
  const int H = a->num_heads, Hkv = a->num_kv_heads, D = a->head_dim, N = a->num_tokens;
  if (H <= 0 || Hkv <= 0 || H % Hkv)
    return fail(DAN_ERR_INVALID_ARGUMENT, "num_heads %d must be a positive multiple of num_kv_heads %d", H, Hkv);
  if (D != 64 && D != 128 && D != 256) return fail(DAN_ERR_UNSUPPORTED, "head_dim %d: only 64, 128 and 256 are built", D);
  if (a->dtype != DAN_DTYPE_BF16 && a->dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or fp16", a->dtype);
  if (N < 0 || a->num_key_units < 0 || a->num_query_units < 0 || a->num_pasts < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "negative count");
  // (-lse / scale has to be finite, too)
  if (!(a->scale >= 0x1p-100f && a->scale <= 0x1p100f)) return fail(DAN_ERR_INVALID_ARGUMENT, "scale must be from 2^-100 to 2^100");
  if (a->key_rows != dan_tree_grad_key_rows(D, 0) && a->key_rows != dan_tree_grad_key_rows(D, 1))
    return fail(DAN_ERR_INVALID_ARGUMENT, "key_rows %d: dan_tree_grad_key_rows", a->key_rows);
  if (a->key_splits < 1 || a->key_splits > H / Hkv) return fail(DAN_ERR_INVALID_ARGUMENT, "key_splits %d: 1 to the %d heads of a kv head", a->key_splits, H / Hkv);
  if (N == 0 || a->num_key_units == 0 || a->num_query_units == 0) return DAN_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->grad || !a->lse || !a->dq || !a->dk || !a->dv || !a->key_units || !a->query_units ||
      !a->row_lo || !a->row_end || (a->num_pasts > 0 && !a->pasts))
    return fail(DAN_ERR_INVALID_ARGUMENT, "NULL tensor or table pointer");
  const int64_t need = dan_tree_grad_workspace_size(H, Hkv, D, N, a->key_splits);
  if (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & (kAlign - 1)))
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace needs %lld bytes, 256-byte aligned", (long long)need);
  const int64_t strides[] = {a->q_stride_tok, a->q_stride_head, a->k_stride_tok, a->k_stride_head, a->v_stride_tok, a->v_stride_head,
                             a->o_stride_tok, a->o_stride_head, a->g_stride_tok, a->g_stride_head, a->dq_stride_tok, a->dq_stride_head,
                             a->dk_stride_tok, a->dk_stride_head, a->dv_stride_tok, a->dv_stride_head};
  for (int64_t s : strides)
    if (s % 8) return fail(DAN_ERR_INVALID_ARGUMENT, "strides must keep rows 16-byte aligned");
  const void *rows[] = {a->q, a->k, a->v, a->out, a->grad, a->dq, a->dk, a->dv};
  for (const void *r : rows)
    if ((uintptr_t)r & 15) return fail(DAN_ERR_INVALID_ARGUMENT, "q, k, v, out and the gradients must be 16-byte aligned");
  // Offsets within a tile and between the two planes of the workspace are kept in 32 bits.
  for (int64_t s : {a->q_stride_tok, a->k_stride_tok, a->v_stride_tok, a->g_stride_tok})
    if (s < 0 || s >= 1 << 25) return fail(DAN_ERR_UNSUPPORTED, "token stride %lld: fewer than 2^25", (long long)s);
  if ((int64_t)H * N * 4 >= (int64_t(1) << 31) - 4096) return fail(DAN_ERR_UNSUPPORTED, "%d heads x %d tokens: fewer than 2^29 rows", H, N);

  GradParams p;
  p.q = a->q; p.q_st = a->q_stride_tok; p.q_sh = a->q_stride_head;
  p.k = a->k; p.k_st = a->k_stride_tok; p.k_sh = a->k_stride_head;
  p.v = a->v; p.v_st = a->v_stride_tok; p.v_sh = a->v_stride_head;
  p.o = a->out; p.o_st = a->o_stride_tok; p.o_sh = a->o_stride_head;
  p.g = a->grad; p.g_st = a->g_stride_tok; p.g_sh = a->g_stride_head;
  p.dq = a->dq; p.dq_st = a->dq_stride_tok; p.dq_sh = a->dq_stride_head;
  p.dk = a->dk; p.dk_st = a->dk_stride_tok; p.dk_sh = a->dk_stride_head;
  p.dv = a->dv; p.dv_st = a->dv_stride_tok; p.dv_sh = a->dv_stride_head;
  p.lse = a->lse;
  p.stats = static_cast<float *>(a->workspace);
  p.partial = p.stats + 2 * (int64_t)H * N;
  p.key_units = a->key_units; p.query_units = a->query_units;
  p.row_lo = a->row_lo; p.row_end = a->row_end;
  p.pasts = a->pasts; p.num_pasts = a->num_pasts;
  p.num_tokens = N; p.num_heads = H; p.num_kv_heads = Hkv; p.rep = H / Hkv;
  p.hpw = heads_of_group(p.rep);
  p.groups = Hkv * ((p.rep + p.hpw - 1) / p.hpw);
  p.key_rows = a->key_rows;
  p.splits = a->key_splits;
  p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(a->workspace) + stats_bytes(H, N));
  const int64_t rows_a_block = kThreads / (D / 8);
  p.partials = (int)std::min<int64_t>(kMaxPartials, ((int64_t)H * N + rows_a_block - 1) / rows_a_block);
  p.scale = a->scale;
  p.c = a->scale * 1.4426950408889634f;
  const int64_t keys_grid = (int64_t)a->num_key_units * Hkv * p.splits, queries_grid = (int64_t)a->num_query_units * p.groups;
  if (p.splits > 1 && (Hkv > 65535 || (int64_t)Hkv * N * (D / 4) >= int64_t(1) << 31))
    return fail(DAN_ERR_UNSUPPORTED, "%d kv heads x %d tokens in parts: too many for one launch", Hkv, N);
  const int64_t grid = keys_grid + queries_grid;
  if (grid * kThreads >= int64_t(1) << 32)
    return fail(DAN_ERR_UNSUPPORTED, "%lld and %lld work groups: fewer than 2^24 together", (long long)keys_grid, (long long)queries_grid);
  p.key_groups = (int)keys_grid;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto by_d = [&](auto t) {
    using T = decltype(t);
    return D == 64 ? launch_all<T, 64>(p, grid, s) : D == 128 ? launch_all<T, 128>(p, grid, s) : launch_all<T, 256>(p, grid, s);
  };
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? by_d(__bf16{}) : by_d(_Float16{});
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "attention gradient launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
