// fi8_i4q.cuh -- device code shared by the kernels that make FlatI4 rows and
// int8 queries: one warp quantizes one group of 32 values, or one query.
#pragma once

#include "fi8_device.cuh"
#include "fi8_i4.cuh"

namespace fi8 {

__device__ __forceinline__ float warp_absmax(float m) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = absmax_combine(m, __shfl_xor_sync(0xffffffffu, m, off));
  return m;
}

// A row's scale and the factor from a group's largest value to its multiplier.
// 1785 = 7 * 255. An all-zero row takes scale 1, as FlatI8's rows do.
__device__ __forceinline__ float i4_row_scale(float rmax, float* up) {
  if (rmax == 0.0f) {
    *up = 0.0f;
    return 1.0f;
  }
  *up = __fdiv_rn(255.0f, rmax);
  return __fdiv_rn(rmax, 1785.0f);
}

// A group's multiplier: its largest value in steps of rmax / 255, rounded up
// so that no code exceeds 7. Infinite rows (0 * inf) and overflow take 255.
__device__ __forceinline__ int i4_group_mult(float gmax, float up) {
  if (gmax == 0.0f) return 0;
  const float t = ceilf(__fmul_rn(gmax, up));
  return t <= 255.0f ? (int)t : 255;
}

// Round half away from zero, clamped to +-7; NaN and an empty group give 0.
__device__ __forceinline__ int i4_code(float x, int mult, float scale) {
  if (mult == 0) return 0;
  float t = roundf(__fmul_rn(x, __fdiv_rn(1.0f, __fmul_rn((float)mult, scale))));
  if (t > 7.0f) t = 7.0f;
  else if (t < -7.0f) t = -7.0f;
  return t == t ? (int)t : 0;
}

// One group by one warp, lane = value: writes its 16 bytes.
__device__ __forceinline__ void i4_store_group(float x, int mult, float scale, uint8_t* codes, int lane) {
  const uint32_t u = (uint32_t)(i4_code(x, mult, scale) + 8);
  uint32_t b = u | (__shfl_down_sync(0xffffffffu, u, 16) << 4);  // lanes 0..15: byte `lane`
  b |= __shfl_down_sync(0xffffffffu, b, 1) << 8;
  b |= __shfl_down_sync(0xffffffffu, b, 2) << 16;
  if (lane < 16 && (lane & 3) == 0) *reinterpret_cast<uint32_t*>(codes + lane) = b;
}

// One query by one warp: q8 [groups * 32] (zero past dim) and off [groups] =
// -8 * sum(q8), both in shared memory; returns the scale (0 for a zero query).
// load(i) gives value i as float32. FlatI8's quantizer, bit for bit.
template <typename Load>
__device__ __forceinline__ float i4_quantize_query(Load load, int dim, int groups, int8_t* q8, int* off, int lane) {
  float m = 0.0f;
  for (int i0 = lane; i0 < dim; i0 += 256) {  // eight loads in flight
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = i0 + 32 * u < dim ? load(i0 + 32 * u) : 0.0f;
#pragma unroll
    for (int u = 0; u < 8; u++) m = absmax_step(m, v[u]);
  }
  m = warp_absmax(m);
  const float sc = m == 0.0f ? 0.0f : __fdiv_rn(m, 127.0f);
  const float inv = m == 0.0f ? 0.0f : __fdiv_rn(1.0f, sc);
  for (int g = 0; g < groups; g++) {
    const int i = g * kI4Group + lane;
    const int8_t c = (m != 0.0f && i < dim) ? quant_code(load(i), inv) : (int8_t)0;
    q8[i] = c;
    const int sum = __reduce_add_sync(0xffffffffu, (int)c);
    if (lane == 0) off[g] = -8 * sum;
  }
  return sc;
}

}  // namespace fi8
