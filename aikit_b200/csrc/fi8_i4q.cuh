// fi8_i4q.cuh -- device code shared by the kernels that make FlatI4 rows and
// int8 queries and multiply them.
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

// One group by one warp, lane = value: put(t, w) for the words of its 16 bytes.
template <typename Put>
__device__ __forceinline__ void i4_store_group(float x, int mult, float scale, int lane, Put put) {
  const uint32_t u = (uint32_t)(i4_code(x, mult, scale) + 8);
  uint32_t b = u | (__shfl_down_sync(0xffffffffu, u, 16) << 4);  // lanes 0..15: byte `lane`
  b |= __shfl_down_sync(0xffffffffu, b, 1) << 8;
  b |= __shfl_down_sync(0xffffffffu, b, 2) << 16;
  if (lane < 16 && (lane & 3) == 0) put(lane >> 2, b);
}

// One query by one warp: q8 [groups * 32] (zero past dim) and off [groups] =
// -8 * sum(q8), both in shared memory; returns the scale (0 for a zero query).
// load(i) gives value i as float32. FlatI8's quantizer, bit for bit. Of several
// warps that share a query each takes the groups from g0 on in steps of gstep.
template <typename Load>
__device__ __forceinline__ float i4_quantize_query(Load load, int dim, int groups, int8_t* q8, int* off, int lane, int g0 = 0, int gstep = 1) {
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
  for (int g = g0; g < groups; g += gstep) {
    const int i = g * kI4Group + lane;
    const int8_t c = (m != 0.0f && i < dim) ? quant_code(load(i), inv) : (int8_t)0;
    q8[i] = c;
    const int sum = __reduce_add_sync(0xffffffffu, (int)c);
    if (lane == 0) off[g] = -8 * sum;
  }
  return sc;
}

// Word index, in its tile, of word t of group g of row r (0 .. 31).
__device__ __forceinline__ int i4_word_at(int g, int r, int t, int groups) {
  const int full = groups & ~3, block = r >> 3, lane = (r & 7) * 4 + t;
  return g < full ? (g >> 2) * 512 + (block * 32 + lane) * 4 + (g & 3)
                  : full * 128 + (block * (groups & 3) + g - full) * 32 + lane;
}

__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], const uint2 b, const int4 c) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}

// Shared memory of a query set, for each group and eight queries: the start
// values of the lanes' four results (int4), then their operands (uint2).
template <int NT>
__host__ __device__ constexpr size_t i4_frag_bytes(int groups) { return (size_t)groups * NT * 32 * 24; }
inline size_t i4_query_bytes(int groups, int nt) { return (size_t)8 * nt * groups * (kI4Group + 4); }

// The fragments of 8 NT quantized queries (q8 [8 NT][groups * 32], off [8 NT]
// [groups] in shared memory): lane 4 n + t gets query n's bytes 4t.. and 16 +
// 4t.. of the group, and the start values of queries 2t and 2t + 1. Begins and
// ends with a barrier of the CTA.
template <int NT>
__device__ __forceinline__ void i4_fragments(int groups, const int8_t* q8, const int* off, int4* starts, uint2* ops) {
  __syncthreads();
  for (int i = threadIdx.x; i < groups * NT * 32; i += blockDim.x) {
    const int l = i & 31, nt = (i >> 5) % NT, g = (i >> 5) / NT, n = nt * 8 + (l >> 2), t = l & 3;
    const int8_t* at = q8 + ((size_t)n * groups + g) * kI4Group + 4 * t;
    ops[i] = make_uint2(*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + 16));
    const int c0 = off[(nt * 8 + 2 * t) * groups + g], c1 = off[(nt * 8 + 2 * t + 1) * groups + g];
    starts[i] = make_int4(c0, c1, c0, c1);
  }
  __syncthreads();
}

// Quantize M queries q [M][dim] (a warp each) and lay out their fragments;
// queries past M are zero.
template <int NT>
__device__ __forceinline__ void i4_queries(const float* q, int M, int dim, int groups, unsigned char* scratch, int4* starts,
                                           uint2* ops, float* scales) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int8_t* q8 = reinterpret_cast<int8_t*>(scratch);
  int* off = reinterpret_cast<int*>(scratch + (size_t)8 * NT * groups * kI4Group);
  auto quantize = [&](int m, int dim_m, int g0, int gstep) {
    const float* qm = q + (size_t)m * dim;
    const float s = i4_quantize_query([&](int i) { return __ldg(qm + i); }, dim_m, groups, q8 + (size_t)m * groups * kI4Group, off + m * groups,
                                      lane, g0, gstep);
    if (lane == 0) scales[m] = s;
  };
  const int warps = blockDim.x >> 5;
  if (NT == 1) {
    // a few queries are shared by the warps, of which each finds the maximum for itself (one of 384 values: 8.4 us
    // with a warp for each query, 7.7 so)
    int shares = warps;
    while (shares > 1 && shares * M > warps) shares >>= 1;
    for (int m = warp / shares; m < M; m += warps / shares) quantize(m, dim, warp & (shares - 1), shares);
    // absent queries
    for (int i = threadIdx.x + M * groups * (kI4Group / 4); i < 8 * NT * groups * (kI4Group / 4); i += blockDim.x) reinterpret_cast<int*>(q8)[i] = 0;
    for (int i = threadIdx.x + M * groups; i < 8 * NT * groups; i += blockDim.x) off[i] = 0;
    for (int i = threadIdx.x + M; i < 8 * NT; i += blockDim.x) scales[i] = 0.0f;
  } else {
    for (int m = warp; m < 8 * NT; m += warps) quantize(m, m < M ? dim : 0, 0, 1);
  }
  i4_fragments<NT>(groups, q8, off, starts, ops);
}

// DEPTH groups of a quad into the totals of 32 rows.
template <int NT, int DEPTH>
__device__ __forceinline__ void i4_multiply(int (&tot)[2][NT][4], const uint32_t (&w)[4][4], const uint32_t (&mult)[4],
                                            const int4* starts, const uint2* ops) {
#pragma unroll
  for (int j = 0; j < DEPTH; j++) {
    int4 c[NT];
    uint2 b[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) c[n] = starts[(j * NT + n) * 32], b[n] = ops[(j * NT + n) * 32];
#pragma unroll
    for (int a = 0; a < 2; a++) {
      const uint32_t w0 = w[2 * a][j], w1 = w[2 * a + 1][j];
      const uint32_t op[4] = {w0 & 0x0F0F0F0Fu, w1 & 0x0F0F0F0Fu, (w0 >> 4) & 0x0F0F0F0Fu, (w1 >> 4) & 0x0F0F0F0Fu};
      const int m0 = (int)__byte_perm(mult[2 * a], 0, 0x4440 + j), m1 = (int)__byte_perm(mult[2 * a + 1], 0, 0x4440 + j);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        int d[4];
        mma_u8s8(d, op, b[n], c[n]);
        tot[a][n][0] += m0 * d[0];
        tot[a][n][1] += m0 * d[1];
        tot[a][n][2] += m1 * d[2];
        tot[a][n][3] += m1 * d[3];
      }
    }
  }
}

}  // namespace fi8
