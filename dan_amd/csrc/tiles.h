// Operand types and helpers of the kernels that feed 32x32 matrix products from tiles of
// 16-bit rows in LDS, and of what stands beside them (tree_attn_grad.hip, adapt.hip, add_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include <type_traits>
#include <utility>

namespace dan {
namespace tiles {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define DAN_TILE_GLOBAL __attribute__((address_space(1)))
#define DAN_TILE_LDS __attribute__((address_space(3)))

template <typename T>
__device__ inline u32x4 load16(const T *p) {
  return *(const DAN_TILE_GLOBAL u32x4 *)p;
}
template <typename T>
__device__ inline void store16(T *p, u32x4 x) {
  *(DAN_TILE_GLOBAL u32x4 *)p = x;
}
__device__ inline u32x4 lds_read16(uint32_t at) { return *(const DAN_TILE_LDS u32x4 *)(uintptr_t)at; }

// f(integral_constant 0), .. f(integral_constant N - 1): a loop that is always laid out in full, with indices that
// are constants, so that what they index stays in registers.
template <int... I, typename F>
__device__ __attribute__((always_inline)) inline void for_each(std::integer_sequence<int, I...>, F &&f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __attribute__((always_inline)) inline void static_for(F &&f) {
  for_each(std::make_integer_sequence<int, N>{}, f);
}

// 4 or 8 fp32 values rounded to T, packed.
template <typename T>
__device__ inline u32x4 pack8(f32x8 x) {
  if constexpr (std::is_same<T, __bf16>::value) return __builtin_bit_cast(u32x4, __builtin_convertvector(x, bf16x8));
  else return __builtin_bit_cast(u32x4, __builtin_convertvector(x, f16x8));
}
template <typename T>
__device__ inline u32x2 pack4(f32x4 x) {
  if constexpr (std::is_same<T, __bf16>::value) return __builtin_bit_cast(u32x2, __builtin_convertvector(x, bf16x4));
  else return __builtin_bit_cast(u32x2, __builtin_convertvector(x, f16x4));
}
template <typename T>
__device__ inline f32x8 unpack8(u32x4 x) {
  if constexpr (std::is_same<T, __bf16>::value) return __builtin_convertvector(__builtin_bit_cast(bf16x8, x), f32x8);
  else return __builtin_convertvector(__builtin_bit_cast(f16x8, x), f32x8);
}

// c += A B of a 32x32x16 product. Lane l holds row l % 32 of A (column of B) at k = 8 (l / 32) + 0..7, and
// of c column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4.
template <typename T>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The same with the result in accumulation registers, for sums that live through a loop: the compiler, asked for
// results in vector registers, would copy them there and back every time. The block waits by itself for operands that
// an instruction before it may have written; the sum may be read by other instructions only behind settle().
template <typename T>
__device__ inline void mfma32_sum(f32x16 &c, u32x4 a, u32x4 b) {
  if constexpr (std::is_same<T, __bf16>::value) asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <int N>
__device__ inline void settle(f32x16 (&c)[N]) {
  asm volatile("s_nop 15\n\ts_nop 15" : "+a"(c[0]));
#pragma unroll
  for (int i = 1; i < N; ++i) asm volatile("" : "+a"(c[i]));
}

// s_waitcnt vmcnt(N) (expcnt and lgkmcnt left alone).
template <int N>
__device__ inline void wait_vmem() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
  asm volatile("" ::: "memory");  // reads of what has landed stay behind
}
// A barrier that leaves the direct loads in flight alone: their completion is counted (wait_vmem).
__device__ inline void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A wave's own LDS reads end here (for a tile that it alone reads and refills).
__device__ inline void barrier_wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ inline int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename T>
__device__ inline const T *uniform_ptr(const T *p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const T *)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// Host: lets a kernel have `bytes` of dynamic LDS, once for each device.
template <auto kernel>
hipError_t allow_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  hipError_t err = hipGetDevice(&device);
  if (err != hipSuccess || ((done.load(std::memory_order_relaxed) >> (device & 63)) & 1)) return err;
  err = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == hipSuccess) done.fetch_or(uint64_t(1) << (device & 63), std::memory_order_relaxed);
  return err;
}

// Direct loads to LDS of 16 (4) bytes a lane: lane l's land at lds + 16 l (4 l). The address is a uniform
// base and a 32-bit byte offset of the lane. M0 holds the LDS address; its write needs one wait state, which
// the compiler does not see to inside the block. The loads are waited for with wait_vmem.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void dma16(const void *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(uniform_ptr((const char *)base)),
               "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory", "m0");
}
__device__ inline void dma16_at(const void *from, uint32_t lds) {  // (an address of each lane, read once: past the caches)
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}
__device__ inline void dma4(const void *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(uniform_ptr((const char *)base)),
               "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory", "m0");
}
#pragma clang diagnostic pop

// A tile of 32 rows of D values of 16 bits in LDS. Chunk c (16 bytes) of row r lies at slot c ^ swizzle(r):
// the 16 lanes that a 16-byte read serves together take one chunk of 16 rows, and the lanes of a transposing
// read take 64 bytes of each of 4 rows; both cover all 64 banks.
template <int D>
struct Tile {
  static constexpr int row = 2 * D, chunks = D / 8, bytes = 32 * row, blocks = bytes / 1024;
  __device__ static constexpr int swizzle(int r) {
    return D == 64 ? (((r >> 1) & 1) << 2 | ((r >> 2) & 3)) : ((r & 3) << 2 | ((r >> 2) & 3));
  }
  // Where a lane's operand pieces lie, as an offset from the tile's start.
  // Rows as the operand's rows: lane l row l % 32, k-step kk the values 16 kk + 8 (l / 32) + 0..7: rows_at(lane) ^ 32 kk.
  __device__ static uint32_t rows_at(int lane) {
    const int r = lane & 31;
    return (uint32_t)(r * row + (((lane >> 5) ^ swizzle(r)) << 4));
  }
  // Columns as the operand's rows, transposed as they are read: lane l column 32 db + l % 32, k-step ks its rows
  // 16 ks + 8 e + 4 (l / 32) + 0..3 for e = 0, 1 (as the products' results lie): two 8-byte reads,
  // (cols_at(lane) ^ 64 db ^ 32 e) + (16 ks + 8 e) rows.
  __device__ static uint32_t cols_at(int lane) {
    const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2);
    return (uint32_t)(r * row + (((2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ swizzle(r)) << 4) + 8 * (i & 1));
  }
  __device__ static u32x4 read_rows(uint32_t tile, uint32_t lane_at, int kk) { return lds_read16((tile + lane_at) ^ (uint32_t)(32 * kk)); }
  __device__ static u32x4 read_cols(uint32_t tile, uint32_t lane_at, int db, int ks) {
    const uint32_t at = (tile + lane_at) ^ (uint32_t)(64 * db);
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DAN_TILE_LDS i16x4 *)(uintptr_t)(at + (uint32_t)(16 * ks * row)));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DAN_TILE_LDS i16x4 *)(uintptr_t)((at ^ 32u) + (uint32_t)((16 * ks + 8) * row)));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
  // Direct loads of block b (1 KB, whole rows): the lane's row, and its chunk's byte in the row.
  __device__ static int block_row(int b, int lane) { return (b * 64 + lane) / chunks; }
  __device__ static uint32_t block_byte(int b, int lane) {
    const int at = b * 64 + lane;
    return (uint32_t)(((at % chunks) ^ swizzle(at / chunks)) << 4);
  }
};

}  // namespace tiles
}  // namespace dan
