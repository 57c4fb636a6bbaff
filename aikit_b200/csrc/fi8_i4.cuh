// fi8_i4.cuh -- FlatI4 rows: vectors in 4 bits a value, and the kernels over
// them (row quantization, scores, exact top-k of scores).
//
// Format. dim values are padded with zeros to G = ceil(dim / 32) groups of 32.
// A group's codes c in [-8, 7] are the nibbles c + 8 of 16 bytes (byte i: value
// i in the low nibble, value 16 + i in the high one), so that one mask of a
// 32-bit word yields the four bytes that face four consecutive query bytes. A
// group has a multiplier m in [0, 255], a row a float32 scale s; the row stands
// for s * m * c. Group scales s * m keep the group maxima apart as separate
// scales would (m is rounded up, so no code is clipped, and the step is at most
// 1/m wider than the group's own), but with whole m the dot with an int8 query,
//
//   dot = sum over the groups of m * sum(c * q8),
//
// is a whole number: any order of summation gives the same int32, every score
// float32(dot) * qscale * s has one value, and top-k ties are exact. |dot| is
// at most 8 * 255 * 127 * dim, so dim <= 4096 stays below 2^31 (8288 would).
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace fi8 {

constexpr int32_t kI4Group = 32;
constexpr int32_t kI4MaxDim = 4096;
constexpr int32_t kI4MaxBatch = 8;       // queries of one score launch (a pass over the rows)
constexpr int32_t kI4MaxK = 2048;
constexpr int32_t kI4SelectTile = 1024;  // scores a select CTA reads at a time
constexpr int32_t kI4SelectCtas = 296;   // select CTAs of a launch, all queries together (two an SM)

inline int32_t i4_groups(int32_t dim) { return (dim + kI4Group - 1) / kI4Group; }
// Bytes of a row's multipliers: whole words.
inline int32_t i4_mult_pitch(int32_t groups) { return (groups + 3) / 4 * 4; }

// Rows on the device. codes [n][groups * 16], mults [n][mpitch], scales [n].
struct I4Rows {
  uint8_t* codes;
  uint8_t* mults;
  float* scales;
  int64_t n;
  int32_t dim, groups, mpitch;
};

// Quantize float32 rows v [rows][dim] into rows [row0, row0 + rows).
cudaError_t i4_quantize_launch(const I4Rows& r, int64_t row0, const float* v, int64_t rows, cudaStream_t stream);

// Scores of M <= kI4MaxBatch queries q [M][dim] against rows [row0, row0 + rows):
// dst[m * ld + (row - row0)].
cudaError_t i4_score_launch(const I4Rows& r, int64_t row0, int64_t rows, const float* q, int32_t M, float* dst,
                            int64_t ld, int32_t sm_count, cudaStream_t stream);

// Top-k of M score rows, exact under (score desc, index asc), NaN excluded.
struct I4Select {
  const float* scores;   // [M][ld], 16-byte aligned, ld a multiple of 4
  int64_t ld, rows;
  uint32_t id0;          // global id of score 0
  const uint64_t* keep;  // optional keep bitmap over global ids
  int64_t keep_nbits;
  int32_t k, kp, cap, nslots;
  int32_t ctas;          // CTAs of a query
  unsigned long long* gthr;  // [M] shared threshold (zero at rest)
  unsigned int* counter;     // [M][blocks] (zero at rest)
  unsigned int* counter2;    // [M] (zero at rest)
  uint64_t* lvl1;            // [M][ctas][kp]
  uint64_t* lvl2;            // [M][blocks][kp]
  uint64_t* out;             // [M][k] sorted keys, 0 = empty
};

// Fills kp, cap, nslots and ctas for a shape; returns the dynamic shared memory.
size_t i4_select_plan(I4Select* s, int32_t M);
cudaError_t i4_select_launch(const I4Select& s, int32_t M, size_t smem, cudaStream_t stream);

#ifdef __CUDACC__

// Four codes of a word against four query bytes: the low nibbles face qlo, the
// high ones qhi. The bytes are c + 8; the caller starts acc at -8 * sum(q8).
__device__ __forceinline__ int i4_dot_word(uint32_t w, int qlo, int qhi, int acc) {
  acc = __dp4a((int)(w & 0x0F0F0F0Fu), qlo, acc);
  return __dp4a((int)((w >> 4) & 0x0F0F0F0Fu), qhi, acc);
}

__device__ __forceinline__ int i4_dot_group(const uint4 w, const int4 qlo, const int4 qhi, int acc) {
  acc = i4_dot_word(w.x, qlo.x, qhi.x, acc);
  acc = i4_dot_word(w.y, qlo.y, qhi.y, acc);
  acc = i4_dot_word(w.z, qlo.z, qhi.z, acc);
  return i4_dot_word(w.w, qlo.w, qhi.w, acc);
}

#endif  // __CUDACC__

}  // namespace fi8
