// Where e4m3 codes lie in the tiled layout of include/dan_fp8.h, and what a row's scale is (fp8_quant.hip, add_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dan_fp8 {

constexpr float kE4m3Max = 448.0f;  // torch.finfo(torch.float8_e4m3fn).max (dan/quant.py:16)

// Byte offset of the 8 codes of row r, columns c .. c + 7 (c a multiple of 8), of rows of kt k-steps of 64 bytes:
// 256-row panels, each a run of 16 KB k-steps; a k-step is 16 blocks
// of 16 rows x 64 bytes, row i of a block at 64 i, its 16-byte chunk j at
// position j ^ (((i >> 1) & 3) ^ ((i >> 3) & 1)).
__device__ inline int64_t tiled_offset(int r, int c, int kt) {
  const int i = r & 15, chunk = (c >> 4) & 3;
  const int pos = chunk ^ (((i >> 1) & 3) ^ ((i >> 3) & 1));
  return ((((int64_t)(r >> 8) * kt + (c >> 6)) * 16 + ((r >> 4) & 15)) << 10) + 64 * i + 16 * pos + (c & 8);
}

// |x| as its fp32 bit pattern. Non-negative floats order as unsigned
// integers and every NaN pattern lies above +inf's, so an integer max over
// these propagates NaN as torch's amax does (dan/fused.py:88): a row holding
// a NaN gets a NaN scale and NaN codes. (A float max would skip the NaN.)
__device__ inline uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// max(amax, 1e-12) / 448 from amax's bits; a NaN amax gives a NaN scale
// (torch's clamp keeps NaN).
__device__ inline float scale_of(uint32_t amax_bits) {
  const float amax = __builtin_bit_cast(float, amax_bits);
  return amax_bits > 0x7f800000u ? amax : fmaxf(amax, 1e-12f) / kE4m3Max;
}

}  // namespace dan_fp8
