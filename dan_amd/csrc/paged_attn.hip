// Attention of one new token per sequence over a paged key-value cache on
// gfx950 (MI355X, CDNA4):  o = sum_j e^{s_j} v_j / sum_j e^{s_j},  s_j = scale q . k_j,
// over the sequence's first lens[b] keys.
//
// HBM-bound: every key and value row is read once. The work is split over
// (sequence, kv head, range of keys): a work group of 4 or 8 waves takes one range, each
// of its waves every 4th or 8th tile of 32 keys, with a running maximum and sum of its
// own; the work group joins them in LDS, and where a sequence spans several
// ranges a second launch joins those (3 to 4 us: a launch behind another. The last work group of
// a sequence could join instead, but a counter that tells it so would have to be cleared
// for the next replay of a graph, and its partners' rows fetched from other dies' caches).
//
// A tile never passes through LDS. On the matrix core (16 x 16 x 32):
//   S^T [16 keys x 16 heads] = K [keys x D] Q^T: a lane's operand is 16 bytes of one key row per
//     step of 32 dims; the q heads of one kv head (up to 16) are the columns, so grouped
//     heads cost no second read of the keys;
//   O^T [D x 16 heads] += V^T [D x 32 keys] P^T: a lane loads D / 16 consecutive dims of
//     8 keys and takes the transpose in registers (one byte permute for two values).
// The keys of a lane's 8 contraction slots are the keys whose scores the same lane holds
// (4 g .. 4 g + 3 of both halves of the tile, g = lane / 16), so P goes from the score
// registers to the operand without an exchange. P keeps the bits of its fp32 weights: against bf16 values it is
// cut into three bf16 parts, which hold all 24 bits of a weight; against fp16 ones (e4m3 codes become
// fp16, which holds each of them) it is scaled by 2^15, so that small weights stay clear of fp16's subnormals, and
// is a rounded part and the rounded rest, off by 2^-24 of a weight. One product for each part. (Two bf16 parts
// leave 2^-17 of a weight: outputs next to a border of their own rounding then fall to the other side twice as
// often as fp32's own errors let them.)
//
// Measured, whole calls, us and TB/s of keys and values, 32/8 heads x 128 in bf16 if not said: 1 sequence of 277 keys
// 6.4 (of which 4 are a launch and its chain of dependent loads: length, page, keys), 1 of 131072 84.8
// (6.3), 64 of up to 8192 186 (6.0), 100 of up to 1000 (32/32 fp16) 128 (6.5), 37 of up to 4099 (16/2 x 256, e4m3) 22.4
// (2.9: a CU draws about 60 GB/s from HBM however many waves ask, so what holds a short launch of unequal
// sequences is the CU with the most keys, and then the join). A large copy moves 4.9.
// Two tiles in flight a wave (240 registers, 2 waves a SIMD) were 1 to 40 % slower; two parts
// of P in one product for up to 8 heads 0 to 3 %, and a third part costs nothing but 0.1 us of the shortest calls: the
// products are not what bounds it.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "cus.h"
#include "dan_paged.h"
#include "paged_index.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
bool finite_positive(float x);                // tree_attn.hip: decided from the float's bits
extern thread_local char g_err[512];
}  // namespace dan

namespace dan_pattn {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

#define DAN_GLOBAL __attribute__((address_space(1)))

constexpr int kTile = 32, kHeads = 16;
constexpr int kMaxLen = 1 << 30;  // places are 32-bit

template <typename T>
struct Ops;
template <>
struct Ops<__bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  typedef bf16x2 x2;
  static __device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ inline uint32_t from_e4m3(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};
template <>
struct Ops<_Float16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
  typedef f16x2 x2;
  static __device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ inline uint32_t from_e4m3(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};

// Two fp32 values as one register of T, rounded to nearest even, and back.
template <typename T>
__device__ inline uint32_t pack2(float a, float b) {
  const f32x2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, typename Ops<T>::x2));
}
template <typename T>
__device__ inline f32x2 unpack2(uint32_t w) {
  return __builtin_convertvector(__builtin_bit_cast(typename Ops<T>::x2, w), f32x2);
}

// The type that values and weights are multiplied in, the parts of a weight, and what the weights are scaled by.
template <typename T, bool FP8>
struct Weights {
  typedef typename std::conditional<FP8, _Float16, T>::type type;
  static constexpr bool bf16 = std::is_same<type, __bf16>::value;
  static constexpr int parts = bf16 ? 3 : 2;
  static constexpr float unit = bf16 ? 1.0f : 32768.0f;
};
// Two weights' parts, the largest last.
template <typename T, bool FP8>
__device__ inline void split_weights(float a, float b, uint32_t (&part)[Weights<T, FP8>::parts]) {
  typedef Weights<T, FP8> Wt;
  if constexpr (Wt::bf16) {
#pragma unroll
    for (int n = 2; n >= 0; --n) {
      const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
      part[n] = __builtin_amdgcn_perm(y, x, 0x07060302);
      a -= __builtin_bit_cast(float, x & 0xffff0000u);
      b -= __builtin_bit_cast(float, y & 0xffff0000u);
    }
  } else {
    a *= Wt::unit;
    b *= Wt::unit;
    part[1] = pack2<_Float16>(a, b);
    const f32x2 y = unpack2<_Float16>(part[1]);
    part[0] = pack2<_Float16>(a - y[0], b - y[1]);
  }
}

// A maximum that keeps a NaN out (v_max_f32): NaN scores reach the sum through their weights.
__device__ inline float max_across_groups(float x) {  // over the 4 lanes of one head (lane % 16)
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float sum_across_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The limits of a split (us on either side, 32/8 heads x 128 in bf16 if not said; here and at the rules below the sides of a pair
// ran on the same lengths, different pairs on different ones):
// - a range has at most kMaxChunk keys (a lane holds the address of one of a wave's 32 blocks of 16 keys):
//   64 sequences of up to 8192 194 with 2048, 199 with 1024; 128 of up to 2000 93 / 100; 1 of 131072 88 / 92;
// - one of kWideChunk keys or more takes 8 waves, 4 / 8: 64 of up to 8192 205 / 194, 128 of up to 2000
//   97 / 93, 100 of up to 1000 (32/32) 138 / 132, 16 of up to 8000 57 / 59; below it 4 to 8000 21 / 26, 16 to 1000
//   13.5 / 15.2 (few work groups: a range of 8 waves is twice as long);
// - keys and values of kDirectBytes or less are one range, one launch / several and the join: 1 of 277 6.4 / 7.5,
//   1 of 384 (192 KB) 7.0 / 7.5, 64 of up to 380 12.7 / 17.5.
constexpr int kMaxChunk = 2048;
constexpr int kWideChunk = 768;
constexpr int kDirectBytes = 192 * 1024;

struct Params {
  const void *q, *kc, *vc;
  void *out;
  float *lse;
  float *part;  // [B * H, splits, D] unnormalized outputs, then [B * H, splits, 2] (maximum q . k, sum)
  const float *ks, *vs;
  dan::PageTable table;
  const int32_t *lens;
  int64_t q_ss, q_sh, o_ss, o_sh, kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  int32_t B, H, Hkv, G, max_len, target, splits, waves, blocks, chunk;  // chunk: of a sequence of max_len
  float scale;
};

// The keys of sequence b, or -1 where its length is none the launch covers.
__device__ inline int length_of(const Params &p, int b) {
  const int n = p.lens[b];
  return (uint32_t)n <= (uint32_t)p.max_len ? n : -1;
}

// What a product q . k (of codes, from an e4m3 cache) is multiplied by to be a score. The largest product is subtracted
// before that, so that its weight is 1 whatever its size: the rounding of a maximum that is multiplied first would be part of every
// exponent, and at scores of 1e9 that is more than fp32 or fp16 hold.
__device__ inline float score_of(const Params &p) { return p.scale * (p.ks ? *p.ks : 1.0f); }
// The same for exponents of 2. A cache of scale 0 has scores of 0 and equal weights: a smallest value in place of 0, as what is
// masked has -inf to be multiplied.
__device__ inline float exponent_of(float to_score) { return to_score == 0.0f ? 0x1p-126f : to_score * 1.4426950408889634f; }

// Keys of a range of a sequence of `len`: a `target`-th of it, within limits, in whole rounds of the work
// group's tiles. By its own length alone, so that a sequence's result does not change with its
// neighbours', and a launch sized for max_len splits shorter ones well, too.
__host__ __device__ inline int chunk_of(int len, int target, int splits, int waves) {
  if (splits == 1) return len < 1 ? 1 : len;
  const int round = kTile * waves, share = (int)(((uint32_t)(len < 0 ? 0 : len) + (uint32_t)target - 1) / (uint32_t)target);
  const int chunk = (share + round - 1) / round * round;
  return chunk < round ? round : chunk > kMaxChunk ? kMaxChunk : chunk;
}

template <typename T, int D, bool FP8>
struct Tile {
  static constexpr int VE = D / 16;        // dims of a lane's value rows
  static constexpr int ES = FP8 ? 1 : 2;   // bytes of a cached value
  static constexpr int KR = D / 32 * (FP8 ? 2 : 4);  // registers of a 16-key block's K operand, as loaded
  static constexpr int VR = VE * ES / 4;   // registers of one value row, as loaded
  uint32_t k[2][KR];
  uint32_t v[2][4][VR];
};

// The dim of element j of lane i's (i = lane % 16) piece of a value row. A bf16 row of 256
// dims is loaded as two 16-byte pieces half a row apart.
template <int D, bool FP8>
__device__ inline int value_dim(int i, int j) {
  if constexpr (D == 256 && !FP8) return (j >> 3) * 128 + 8 * i + (j & 7);
  else return D / 16 * i + j;
}

// Keys. A unit is 64 bytes of a row: one step of 32 dims in 16 bits, two in 8. Where a row has
// several units they are loaded in pairs, 128 bytes of 8 rows in one instruction (whole cache lines, so
// the loads may pass the caches by), and dealt out to the lanes by key_unit. Offsets of a lane:
// first and second load of a pair.
struct KeyOffsets {
  uint32_t a, b;
};
// A load from the cache; STREAM: past the processor's caches.
template <bool STREAM, typename V>
__device__ inline V load(const uint8_t *p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const DAN_GLOBAL V *)p);
  else return *(const DAN_GLOBAL V *)p;
}
__device__ inline KeyOffsets key_offsets(int lane, uint32_t row, bool pairs) {
  const uint32_t i = lane & 15, g = lane >> 4, up = i >> 3;
  if (!pairs) return {i * row + 16 * g, 0};
  return {(i & 7) * row + 16 * g + 64 * up, (8 + (i & 7)) * row + 16 * g + 64 * (1 - up)};
}

template <bool STREAM, typename T, int D, bool FP8>
__device__ inline void load_k(Tile<T, D, FP8> &t, int u, const uint8_t *base, KeyOffsets off) {
  constexpr int KR = Tile<T, D, FP8>::KR;
  if constexpr (KR == 4) {
    const u32x4 x = load<STREAM, u32x4>(base + off.a);
#pragma unroll
    for (int c = 0; c < 4; ++c) t.k[u][c] = x[c];
  } else {
#pragma unroll
    for (int s = 0; s < KR / 8; ++s) {
      const u32x4 x = load<STREAM, u32x4>(base + off.a + 128 * s);
      const u32x4 y = load<STREAM, u32x4>(base + off.b + 128 * s);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        t.k[u][8 * s + c] = x[c];
        t.k[u][8 * s + 4 + c] = y[c];
      }
    }
  }
}

// Unit m of the lane's row i: of a pair, lanes 0 to 7 of each 16 have the first load's low half and
// lanes 8 to 15 the second's; the other halves belong to the lanes 8 further.
template <typename T, int D, bool FP8>
__device__ inline u32x4 key_unit(const Tile<T, D, FP8> &t, int u, int m, bool low) {
  u32x4 x;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (Tile<T, D, FP8>::KR == 4) {
      x[c] = t.k[u][c];
    } else {
      const uint32_t a = t.k[u][8 * (m / 2) + c], b = t.k[u][8 * (m / 2) + 4 + c];
      x[c] = m % 2 == 0 ? (low ? a : b) : (uint32_t)__builtin_amdgcn_mov_dpp((int)(low ? b : a), 0x128, 0xF, 0xF, false);  // row_ror:8
    }
  }
  return x;
}

template <bool STREAM, typename T, int D, bool FP8>
__device__ inline void load_v(Tile<T, D, FP8> &t, int u, const uint8_t *base, uint32_t off, uint32_t row) {
  constexpr int VR = Tile<T, D, FP8>::VR;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint8_t *p = base + off + r * row;
    if constexpr (VR == 8) {
      const u32x4 a = load<STREAM, u32x4>(p), b = load<STREAM, u32x4>(p + 256);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        t.v[u][r][c] = a[c];
        t.v[u][r][4 + c] = b[c];
      }
    } else if constexpr (VR == 4) {
      const u32x4 a = load<STREAM, u32x4>(p);
#pragma unroll
      for (int c = 0; c < 4; ++c) t.v[u][r][c] = a[c];
    } else if constexpr (VR == 2) {
      const u32x2 a = load<STREAM, u32x2>(p);
      t.v[u][r][0] = a[0];
      t.v[u][r][1] = a[1];
    } else {
      t.v[u][r][0] = load<STREAM, uint32_t>(p);
    }
  }
}

// The operand of 32 dims (step s) of a key block.
template <typename T, int D, bool FP8>
__device__ inline u32x4 k_operand(const Tile<T, D, FP8> &t, int u, int s, bool low) {
  if constexpr (!FP8) {
    return key_unit<T, D, FP8>(t, u, s, low);
  } else {
    const u32x4 x = key_unit<T, D, FP8>(t, u, s / 2, low);
    const uint32_t a = x[s % 2 * 2], b = x[s % 2 * 2 + 1];
    return (u32x4){Ops<T>::template from_e4m3<false>(a), Ops<T>::template from_e4m3<true>(a), Ops<T>::template from_e4m3<false>(b),
                   Ops<T>::template from_e4m3<true>(b)};
  }
}

// Elements 2 m and 2 m + 1 of a value row, as the weights' type has them.
template <typename T, int D, bool FP8>
__device__ inline uint32_t v_pair(const Tile<T, D, FP8> &t, int u, int r, int m) {
  if constexpr (!FP8) return t.v[u][r][m];
  else return m & 1 ? Ops<_Float16>::from_e4m3<true>(t.v[u][r][m >> 1]) : Ops<_Float16>::from_e4m3<false>(t.v[u][r][m >> 1]);
}

// W waves. LDS: the waves' results [W][heads][D + 4], their maxima and sums [2][W][heads];
// before that (D = 256) the q operand, in the order its steps read it.
template <typename T, int D, bool FP8, int W, bool STREAM>
__global__ __launch_bounds__(64 * W, 2) void paged_attn_kernel(const Params p) {
  typedef Tile<T, D, FP8> Tl;
  typedef Weights<T, FP8> Wt;
  constexpr int VE = Tl::VE, ES = Tl::ES, DP = D + 4, S = D / 32;
  constexpr bool kQLds = D == 256;  // 32 registers that the tile needs
  extern __shared__ __align__(16) float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  // (kv head, block of 16 q heads) fastest, then the sequence, then the range
  uint32_t at = blockIdx.x;
  const int hb = at % p.blocks;
  at /= p.blocks;
  const int hk = at % p.Hkv;
  at /= p.Hkv;
  const int b = at % p.B, split = at / p.B;
  const int heads = min(p.G - hb * kHeads, kHeads);  // of this block
  const int head0 = hk * p.G + hb * kHeads;
  const bool direct = p.splits == 1;

  // The length, q, and the pages that are this wave's if the sequence is of max_len, or this its first
  // range, are loaded side by side: lane n takes the wave's 16-key block n.
  const int mykey = kTile * (wave + W * (lane >> 1)) + 16 * (lane & 1);
  dan::PageRow from = dan::find_row(p.table, b, split * p.chunk + mykey);
  // q: column i is head min(i, heads - 1); dims as the key operand has them
  const T *qrow = static_cast<const T *>(p.q) + b * p.q_ss + (head0 + min(i, heads - 1)) * p.q_sh;
  auto q_step = [&](int s) { return *(const DAN_GLOBAL u32x4 *)(qrow + (FP8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g)); };
  u32x4 qf[kQLds ? S / W : S];  // in LDS: this wave's share of the steps, until it is written there
  u32x4 *ql = (u32x4 *)lds + lane;
#pragma unroll
  for (int s = 0; s < (kQLds ? S / W : S); ++s) qf[s] = q_step(kQLds ? W * s + wave : s);
  const float to_score = score_of(p), c = exponent_of(to_score);
  float vscale = 1.0f / Wt::unit;
  if constexpr (FP8) vscale *= *p.vs;
  const int len = length_of(p, b), chunk = chunk_of(len, p.target, p.splits, W), lo = split * chunk;
  if (lo >= len) {  // nothing here: the join leaves such ranges out (and takes wrong lengths to NaN)
    if (direct) {
      const float none = len < 0 ? __builtin_nanf("") : 0.0f;
      for (int e = threadIdx.x; e < heads * D; e += 64 * W) {
        static_cast<T *>(p.out)[b * p.o_ss + (head0 + e / D) * p.o_sh + e % D] = (T)none;
        if (p.lse && e % D == 0) p.lse[(int64_t)b * p.H + head0 + e / D] = len < 0 ? none : -INFINITY;
      }
    }
    return;
  }
  const int hi = min(len, lo + chunk);
  const int tiles = (hi - lo + kTile - 1) / kTile;
  const int mine = wave < tiles ? (tiles - wave + W - 1) / W : 0;  // at most 16 (kMaxChunk, kDirectBytes)

  f32x4 acc[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) acc[j] = (f32x4){0, 0, 0, 0};
  float m = -INFINITY, l = 0.f;

  Tl t;
  uint64_t bad = 0, kadr = 0, vadr = 0;
  const uint32_t krow = (uint32_t)(p.kc_st * ES), vrow = (uint32_t)(p.vc_st * ES);
  const KeyOffsets koff = key_offsets(lane, krow, Tl::KR > 4);
  const bool low = i < 8;
  const uint32_t voff = 4 * g * vrow + (D == 256 && !FP8 ? 16 * i : VE * ES * i);
  auto at_lane = [&](uint64_t x, int n) -> const uint8_t * {
    const uint32_t a = __builtin_amdgcn_readlane((uint32_t)x, n), h = __builtin_amdgcn_readlane((uint32_t)(x >> 32), n);
    return (const uint8_t *)((uint64_t)h << 32 | a);
  };
  auto fetch_k = [&](int n) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_k<STREAM, T, D, FP8>(t, u, at_lane(kadr, 2 * n + u), koff);
  };
  auto fetch_v = [&](int n) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_v<STREAM, T, D, FP8>(t, u, at_lane(vadr, 2 * n + u), voff, vrow);
  };
  if (mine > 0) {
    // Where the lane's block starts in the two caches. Page 0 stands in for a
    // block behind the end and for a page that does not exist. A block starts at a multiple of 16
    // rows, as a page's size is one, so all 16 lie in the page.
    if (lo != split * p.chunk) from = dan::find_row(p.table, b, lo + mykey);
    const bool there = lane < 2 * mine && lo + mykey < hi;
    bad = __ballot(there && from.page < 0);
    if (!there || from.page < 0) from = {0, 0};
    kadr = (uint64_t)p.kc + (from.page * p.kc_sp + hk * p.kc_sh + from.row * p.kc_st) * ES;
    vadr = (uint64_t)p.vc + (from.page * p.vc_sp + hk * p.vc_sh + from.row * p.vc_st) * ES;
    fetch_k(0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_v(0);
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (kQLds) {
#pragma unroll
    for (int s = 0; s < S / W; ++s) ql[64 * (W * s + wave)] = qf[s];
    __syncthreads();
  }

  if (mine > 0) {
    // One tile; the next one's keys are loaded once its own are spent, and its values likewise. The last tile
    // is a copy of its own: a load under a condition would make the wait in front of each product
    // one for all loads.
    auto tile = [&](int n, auto last) __attribute__((always_inline)) {
      f32x4 sc[2];  // scores of keys 16 u + 4 g + r and head i
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sc[u] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) sc[u] = Ops<T>::mfma(k_operand<T, D, FP8>(t, u, s, low), kQLds ? ql[64 * s] : qf[kQLds ? 0 : s], sc[u]);
      }
      if constexpr (!last.value) {
        fetch_k(n + 1);
        __builtin_amdgcn_sched_barrier(0);  // the scheduler would mix these loads with those of the values
      }
      if constexpr (last.value) {  // no weight, and no value either, behind the sequence's end
        const int key0 = lo + kTile * (wave + W * n) + 4 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * u + r >= hi) {
              sc[u][r] = -INFINITY;
#pragma unroll
              for (int e = 0; e < Tl::VR; ++e) t.v[u][r][e] = 0;
            }
      }
      float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])), fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      top = max_across_groups(top);
      if (__any(top > m)) {
        const float to = fmaxf(m, top);
        const float by = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - to) * c);
        m = to;
        l *= by;
#pragma unroll
        for (int j = 0; j < VE; ++j) acc[j] *= by;
      }
      const float sub = m == -INFINITY ? 0.0f : m;
      u32x4 pw[Wt::parts];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[r] = __builtin_amdgcn_exp2f((sc[u][r] - sub) * c);
          l += w[r];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t part[Wt::parts];
          split_weights<T, FP8>(w[2 * h], w[2 * h + 1], part);
#pragma unroll
          for (int n = 0; n < Wt::parts; ++n) pw[n][2 * u + h] = part[n];
        }
      }
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        uint32_t row[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) row[u][r] = v_pair<T, D, FP8>(t, u, r, e);
        u32x4 even, odd;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            even[2 * u + h] = __builtin_amdgcn_perm(row[u][2 * h + 1], row[u][2 * h], 0x05040100);
            odd[2 * u + h] = __builtin_amdgcn_perm(row[u][2 * h + 1], row[u][2 * h], 0x07060302);
          }
#pragma unroll
        for (int n = 0; n < Wt::parts; ++n) {
          acc[2 * e] = Ops<typename Wt::type>::mfma(even, pw[n], acc[2 * e]);
          acc[2 * e + 1] = Ops<typename Wt::type>::mfma(odd, pw[n], acc[2 * e + 1]);
        }
      }
      if constexpr (!last.value) {
        __builtin_amdgcn_sched_barrier(0);
        fetch_v(n + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int n = 0; n < mine - 1; ++n) tile(n, std::false_type());
    tile(mine - 1, std::true_type());
    l = sum_across_groups(l);
    if (bad) l = __builtin_nanf("");
  }

  // The waves' results into LDS: lane (i, g) holds head i, value lanes 4 g .. 4 g + 3.
  if constexpr (kQLds) __syncthreads();
  float *ml = lds + W * heads * DP;
  if (i < heads) {
    float *row = lds + (wave * heads + i) * DP;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
      for (int j = 0; j < VE; j += 4) {
        const f32x4 x = {acc[j][rr], acc[j + 1][rr], acc[j + 2][rr], acc[j + 3][rr]};
        *(f32x4 *)(row + value_dim<D, FP8>(4 * g + rr, j)) = x;
      }
    if (g == 0) {
      ml[wave * heads + i] = m;
      ml[(W + wave) * heads + i] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x * 4; e < heads * D; e += 256 * W) {
    const int h = e / D, d = e % D;
    float mw[W], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      mw[w] = ml[w * heads + h];
      top = fmaxf(top, mw[w]);
    }
    const float sub = top == -INFINITY ? 0.0f : top;
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float by = __builtin_amdgcn_exp2f((mw[w] - sub) * c);
      sum += by * ml[(W + w) * heads + h];
      o += by * *(const f32x4 *)(lds + (w * heads + h) * DP + d);
    }
    const int64_t row = (int64_t)b * p.H + head0 + h;
    if (direct) {
      const float inv = vscale / sum;
      typename Ops<T>::x4 y = __builtin_convertvector(o * inv, typename Ops<T>::x4);
      *(DAN_GLOBAL u32x2 *)(static_cast<T *>(p.out) + b * p.o_ss + (head0 + h) * p.o_sh + d) = __builtin_bit_cast(u32x2, y);
      if (p.lse && d == 0) p.lse[row] = sub * to_score + logf(sum);
    } else {
      *(DAN_GLOBAL f32x4 *)(p.part + (row * p.splits + split) * D + d) = o * vscale;
      if (d == 0) {
        float *s = p.part + (int64_t)p.B * p.H * p.splits * D + (row * p.splits + split) * 2;
        s[0] = top;
        s[1] = sum;
      }
    }
  }
}

// One work group joins the ranges of a (sequence, head): D / 4 lanes take every GR-th range with a running
// maximum, so a range's maximum, sum and row are loaded side by side, and the GR results meet in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const Params p) {
  constexpr int L = D / 4, GR = 256 / L;
  __shared__ float part[GR][D];
  __shared__ float tops[GR], sums[GR];
  const int64_t row = blockIdx.x;
  const int b = row / p.H, h = row % p.H;
  const int gr = threadIdx.x / L, d = threadIdx.x % L * 4;
  const float *ml = p.part + (int64_t)p.B * p.H * p.splits * D + row * p.splits * 2;
  const float *rows = p.part + row * p.splits * D + d;
  const int len = length_of(p, b);
  const int chunk = chunk_of(len, p.target, p.splits, p.waves), n = len <= 0 ? 0 : (len + chunk - 1) / chunk;
  const float to_score = score_of(p), c = exponent_of(to_score);
  f32x4 o = {0, 0, 0, 0};
  float top = -INFINITY, sum = 0.f;  // top: in products
#pragma unroll 4
  for (int s = gr; s < n; s += GR) {
    const f32x2 q = *(const DAN_GLOBAL f32x2 *)(ml + 2 * s);
    const f32x4 x = *(const DAN_GLOBAL f32x4 *)(rows + (int64_t)s * D);
    const float to = fmaxf(top, q[0]), sub = to == -INFINITY ? 0.0f : to;
    const float was = __builtin_amdgcn_exp2f((top - sub) * c), by = __builtin_amdgcn_exp2f((q[0] - sub) * c);
    top = to;
    sum = __builtin_fmaf(by, q[1], was * sum);
    o = was * o + by * x;
  }
  *(f32x4 *)&part[gr][d] = o;
  if (d == 0) {
    tops[gr] = top;
    sums[gr] = sum;
  }
  __syncthreads();
  if (threadIdx.x < L) {
#pragma unroll
    for (int w = 0; w < GR; ++w) top = fmaxf(top, tops[w]);
    const float sub = top == -INFINITY ? 0.0f : top;
    o = (f32x4){0, 0, 0, 0};
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < GR; ++w) {
      const float by = __builtin_amdgcn_exp2f((tops[w] - sub) * c);
      o += by * *(const f32x4 *)&part[w][d];
      sum += by * sums[w];
    }
    const float inv = len > 0 ? 1.0f / sum : len == 0 ? 0.0f : __builtin_nanf("");
    typename Ops<T>::x4 y = __builtin_convertvector(o * inv, typename Ops<T>::x4);
    *(DAN_GLOBAL u32x2 *)(static_cast<T *>(p.out) + b * p.o_ss + h * p.o_sh + d) = __builtin_bit_cast(u32x2, y);
    if (p.lse && d == 0) p.lse[row] = len > 0 ? sub * to_score + logf(sum) : len == 0 ? -INFINITY : __builtin_nanf("");
  }
}

// How a launch is split over the keys: work groups of `waves` waves, `splits` ranges of a
// sequence of max_len keys, a sequence's own number in proportion to its length up to `target`.
// Equal sequences would have one range for each CU in all; in a batch of unequal ones the long ones need
// more, the shorter the better, but each costs a work group's start and its row in the join. us with ranges
// for 1 / 2 / 4 times the CUs (32/8 x 128 in bf16 if not said): 1 of 131072 88 / 89 / 92, 1 of 32768 30 / 31 / 33;
// few sequences, 2: 4 to 8000 19.5 / 20.0 / 21.0, 2 to 20000 29.6 / 30.2 / 33.0, 32 to 3000 (8/2 x 64) 11.7 / 11.7 / 12.7;
// more, 4: 16 to 8000 63.6 / 58.3 / 58.6, 16 to 3000 27.7 / 27.4 / 24.7, 48 to 6000 120 / 118 / 116; of 256 dims, 2:
// 37 to 4099 (16/2, e4m3) 27.4 / 23.7 / 26.2, 64 to 4000 61.2 / 61.5 / 63.5. Where every CU has a sequence and a head
// and none is longer than a range may be, no join: 64 to 500 15.8 / 15.7 / 20.2, 64 to 1000 32 / 32 / 37,
// 32 to 1500 24.5 / 28.8 / 26.8 (a single sequence of 2000 among short ones then takes some 20 us of its own).
struct Split {
  int waves, target, splits, chunk;
};
Split split_of(int64_t seqs, int64_t groups, int max_len, int head_dim, int key_bytes, int cus) {
  if (cus <= 0) cus = 256;
  if (groups < 1) groups = 1;  // no sequences
  if ((int64_t)max_len * key_bytes <= kDirectBytes) return {4, 1, 1, chunk_of(max_len, 1, 1, 4)};
  const bool even = seqs == 1 || (groups >= cus && max_len <= kMaxChunk);
  const int64_t want = (even ? 1 : head_dim == 256 || 2 * groups < cus ? 2 : 4) * (int64_t)cus, shares = (want + groups - 1) / groups;
  auto of = [&](int waves) {
    const int64_t most = (max_len + kTile * waves - 1) / (kTile * waves);  // ranges of the shortest length
    const int target = (int)(shares < most ? shares : most), least = (max_len + kMaxChunk - 1) / kMaxChunk;
    const int splits = target > least ? target : least;
    return Split{waves, target, splits, chunk_of(max_len, target, splits, waves)};
  };
  const Split s = of(4);
  return s.chunk >= kWideChunk && head_dim <= 128 ? of(8) : s;
}

template <typename T, int D, bool FP8, int W, bool STREAM>
void launch_kernel(const Params &p, hipStream_t s) {
  const int heads = p.G < kHeads ? p.G : kHeads;
  const size_t out = sizeof(float) * W * heads * (D + 4 + 2), q = D == 256 ? 16 * 64 * (D / 32) : 0;
  auto kernel = paged_attn_kernel<T, D, FP8, W, STREAM>;
  // Beyond what a launch may have unasked, of 16 heads x 128 in 8 waves: asked of the current device each time.
  if (out > 64 * 1024) (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)out);
  const unsigned grid = (unsigned)((int64_t)p.splits * p.B * p.Hkv * p.blocks);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * W), out > q ? out : q, s, p);
}

// Keys and values of a launch that may read more than the last-level cache holds pass the caches by, which they would
// only sweep. us, through the caches / past them: 64 to 8192 (32/8 x 128; up to 2.1 GB) 216 / 194, 1 of 131072 99 / 88,
// 100 to 1000 (32/32) 146 / 132, 16 to 8000 (524 MB) 65 / 59; a smaller launch gains by the caches
// where a few layers' caches fit them (37 to 4099, 16/2 x 256 e4m3, 155 MB: 22.0 / 24.0 over 3 layers)
// and loses a little where they do not (25.6 / 24.7 over 12).
constexpr int64_t kStreamBytes = (int64_t)256 << 20;

template <typename T, int D, bool FP8, int W>
void launch_waves(const Params &p, hipStream_t s) {
  if ((double)p.B * p.max_len * p.Hkv * (2 * D * Tile<T, D, FP8>::ES) >= (double)kStreamBytes) launch_kernel<T, D, FP8, W, true>(p, s);
  else launch_kernel<T, D, FP8, W, false>(p, s);
}

template <typename T, int D, bool FP8>
void launch(const Params &p, hipStream_t s) {
  if constexpr (D <= 128) {
    if (p.waves == 8) launch_waves<T, D, FP8, 8>(p, s);
    else launch_waves<T, D, FP8, 4>(p, s);
  } else {
    launch_waves<T, D, FP8, 4>(p, s);
  }
  if (p.splits > 1) hipLaunchKernelGGL((paged_join_kernel<T, D>), dim3((unsigned)((int64_t)p.B * p.H)), dim3(256), 0, s, p);
}

template <typename T>
void by_dim(const Params &p, int d, bool fp8, hipStream_t s) {
  if (d == 64) fp8 ? launch<T, 64, true>(p, s) : launch<T, 64, false>(p, s);
  else if (d == 128) fp8 ? launch<T, 128, true>(p, s) : launch<T, 128, false>(p, s);
  else fp8 ? launch<T, 256, true>(p, s) : launch<T, 256, false>(p, s);
}

}  // namespace dan_pattn

extern "C" {

int64_t dan_paged_attn_workspace_size(int32_t cache_dtype, int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                      int32_t max_len) {
  using namespace dan_pattn;
  if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || max_len < 0 || max_len > kMaxLen ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) ||
      (cache_dtype != DAN_DTYPE_BF16 && cache_dtype != DAN_DTYPE_F16 && cache_dtype != DAN_DTYPE_E4M3))
    return -1;
  const int64_t blocks = (num_heads / num_kv_heads + kHeads - 1) / kHeads;
  const Split sp = split_of(num_seqs, (int64_t)num_seqs * num_kv_heads * blocks, max_len, head_dim, head_dim * (cache_dtype == DAN_DTYPE_E4M3 ? 2 : 4), dan::num_cus());
  return sp.splits > 1 ? (int64_t)num_seqs * num_heads * sp.splits * (head_dim + 2) * 4 : 0;
}

int dan_paged_attn(const DanPagedAttnArgs *a, void *stream) {
  using namespace dan_pattn;
  using dan::fail;
  dan::g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_PAGED_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, paged cache speaks %d", a->abi_version, DAN_PAGED_ABI_VERSION);
  const int B = a->num_seqs, H = a->num_heads, Hkv = a->num_kv_heads, D = a->head_dim;
  if (B < 0 || H <= 0 || Hkv <= 0 || H % Hkv)
    return fail(DAN_ERR_INVALID_ARGUMENT, "need num_seqs >= 0 and num_heads %d a positive multiple of num_kv_heads %d", H, Hkv);
  if (D != 64 && D != 128 && D != 256) return fail(DAN_ERR_UNSUPPORTED, "head_dim %d: only 64, 128 and 256 are built", D);
  if (a->dtype != DAN_DTYPE_BF16 && a->dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or f16", a->dtype);
  const bool fp8 = a->cache_dtype == DAN_DTYPE_E4M3;
  const int es = fp8 ? 1 : 2;
  if (!fp8 && a->cache_dtype != a->dtype) return fail(DAN_ERR_UNSUPPORTED, "cache_dtype %d: dtype's own or e4m3", a->cache_dtype);
  if (a->page_size <= 0 || a->page_size % DAN_PAGED_KEY_BLOCK)
    return fail(DAN_ERR_INVALID_ARGUMENT, "page_size %d must be a positive multiple of %d", a->page_size, DAN_PAGED_KEY_BLOCK);
  if (a->num_pages < 0 || a->table_width < 0) return fail(DAN_ERR_INVALID_ARGUMENT, "num_pages and table_width must be >= 0");
  if (a->max_len < 0 || a->max_len > kMaxLen || a->max_len > (int64_t)a->table_width * a->page_size)
    return fail(DAN_ERR_INVALID_ARGUMENT, "max_len %d: the table holds %lld keys a sequence", a->max_len, (long long)a->table_width * a->page_size);
  if (!dan::finite_positive(a->scale) || a->scale > 0x1p127f)  // (times log2 e it has to be finite, too)
    return fail(DAN_ERR_INVALID_ARGUMENT, "scale must be finite, > 0 and at most 2^127");
  if (B == 0) return DAN_OK;
  if (!a->q || !a->out || !a->lens) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
  if (a->max_len > 0 && (!a->k_cache || !a->v_cache || !a->table || a->num_pages == 0))
    return fail(DAN_ERR_INVALID_ARGUMENT, "a max_len of %d needs a cache with pages and a table", a->max_len);
  if (fp8 && (!a->k_scale || !a->v_scale)) return fail(DAN_ERR_INVALID_ARGUMENT, "an e4m3 cache needs k_scale and v_scale");
  for (int64_t st : {a->q_stride_seq, a->q_stride_head, a->o_stride_seq, a->o_stride_head})
    if (st % 8) return fail(DAN_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements (16-byte rows)");
  for (int64_t st : {a->kc_stride_page, a->kc_stride_head, a->kc_stride_tok, a->vc_stride_page, a->vc_stride_head, a->vc_stride_tok})
    if (st * es % 16) return fail(DAN_ERR_INVALID_ARGUMENT, "cache strides must be multiples of 16 bytes");
  for (int64_t st : {a->kc_stride_tok, a->vc_stride_tok})  // offsets inside a 16-key block are 32-bit
    if (st < D || st > (1 << 26)) return fail(DAN_ERR_INVALID_ARGUMENT, "cache token strides must lie in [head_dim, 2^26]");
  const void *ptrs[] = {a->q, a->out, a->k_cache, a->v_cache, a->workspace};
  for (const void *ptr : ptrs)
    if ((uintptr_t)ptr & 15) return fail(DAN_ERR_INVALID_ARGUMENT, "tensor pointers must be 16-byte aligned");

  Params p;
  p.q = a->q; p.kc = a->k_cache; p.vc = a->v_cache; p.out = a->out; p.lse = a->lse; p.part = static_cast<float *>(a->workspace);
  p.ks = fp8 ? a->k_scale : nullptr; p.vs = a->v_scale; p.table = {a->table, a->table_stride, B, a->table ? a->table_width : 0, a->page_size, a->num_pages}; p.lens = a->lens;
  p.q_ss = a->q_stride_seq; p.q_sh = a->q_stride_head; p.o_ss = a->o_stride_seq; p.o_sh = a->o_stride_head;
  p.kc_sp = a->kc_stride_page; p.kc_sh = a->kc_stride_head; p.kc_st = a->kc_stride_tok;
  p.vc_sp = a->vc_stride_page; p.vc_sh = a->vc_stride_head; p.vc_st = a->vc_stride_tok;
  p.B = B; p.H = H; p.Hkv = Hkv; p.G = H / Hkv;
  p.max_len = a->max_len; p.blocks = (p.G + kHeads - 1) / kHeads; p.scale = a->scale;
  const Split sp = split_of(B, (int64_t)B * Hkv * p.blocks, a->max_len, D, 2 * D * es, dan::num_cus());
  p.target = sp.target; p.splits = sp.splits; p.waves = sp.waves; p.chunk = sp.chunk;
  const int64_t threads = (int64_t)1 << 32;  // a launch has fewer
  if ((int64_t)sp.splits * B >= threads || (int64_t)sp.splits * B * Hkv * p.blocks * 64 * sp.waves >= threads || (int64_t)B * H * 256 >= threads)
    return fail(DAN_ERR_INVALID_ARGUMENT, "too many sequences and heads for one launch");
  if (sp.splits > 1) {
    const int64_t need = (int64_t)B * H * sp.splits * (D + 2) * 4;
    if (!a->workspace || a->workspace_bytes < need)
      return fail(DAN_ERR_INVALID_ARGUMENT, "workspace of %lld bytes, needs %lld", (long long)a->workspace_bytes, (long long)need);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == DAN_DTYPE_BF16) by_dim<__bf16>(p, D, fp8, s);
  else by_dim<_Float16>(p, D, fp8, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "paged attention launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
