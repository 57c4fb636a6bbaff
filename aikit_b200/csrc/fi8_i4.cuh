// fi8_i4.cuh -- FlatI4 rows: vectors in 4 bits a value, and the kernels over
// them (row quantization, scores, exact top-k).
//
// Format. dim values are padded with zeros to G = ceil(dim / 32) groups of 32.
// A group's codes c in [-8, 7] are the nibbles c + 8 of 16 bytes (byte i: value
// i in the low nibble, value 16 + i in the high one), so that one mask of a
// 32-bit word yields the four bytes that face four consecutive query bytes. A
// group has a multiplier m in [0, 255], a row a float32 scale s; the row stands
// for s * m * c. Group scales s * m keep the group maxima apart as separate
// scales would (m is rounded up, so no code is clipped, and a group's step s * m
// is less than one row scale s above its own, a seventh of its maximum), but with
// whole m the dot with an int8 query,
//
//   dot = sum over the groups of m * sum(c * q8),
//
// is a whole number: any order of summation gives the same int32, every score
// float32(dot) * qscale * s has one value, and top-k ties are exact. |dot| is
// at most 8 * 255 * 127 * dim, so dim <= 4096 stays below 2^31 (8288 would).
//
// Device layout. Eight rows are interleaved word by word: lane l = 4 r + t of a
// warp owns word t of row r, as the operand of an 8-bit matrix instruction
// wants it, and its words of four groups are 16 neighbouring bytes. So a warp
// reads 8 rows x 4 groups with one 16-byte load a lane, 512 contiguous bytes,
// straight into operand registers.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace fi8 {

constexpr int32_t kI4Group = 32;
constexpr int32_t kI4MaxDim = 4096;
constexpr int32_t kI4MaxBatch = 16;  // queries of one pass over the rows
constexpr int32_t kI4MaxK = 2048;
constexpr int32_t kI4Tile = 32;      // rows that a warp scores together

// Queries of one pass over rows of that many groups: their fragments and the
// copies' rings fit in shared memory.
inline int32_t i4_batch(int32_t groups) { return groups <= 96 ? kI4MaxBatch : kI4MaxBatch / 2; }

inline int32_t i4_groups(int32_t dim) { return (dim + kI4Group - 1) / kI4Group; }

// Rows on the device, n rounded up to whole tiles of 32. A tile has
//   codes [groups / 4 quads][4 blocks of 8 rows][32 lanes][4 groups] words,
//         then, when groups is no multiple of 4, [4][groups % 4][32] words;
//   mults [(groups + 3) / 4 quads][32 rows] words, a byte a group.
struct I4Rows {
  uint32_t* codes;
  uint32_t* mults;
  float* scales;
  int64_t n;
  int32_t dim, groups;
};

inline int64_t i4_tiles(int64_t n) { return (n + kI4Tile - 1) / kI4Tile; }
inline size_t i4_code_bytes(int64_t n, int32_t groups) { return (size_t)i4_tiles(n) * kI4Tile * groups * 16; }
inline size_t i4_mult_bytes(int64_t n, int32_t groups) { return (size_t)i4_tiles(n) * kI4Tile * ((groups + 3) / 4) * 4; }

// Once on each device, before the first launch on it.
cudaError_t i4_init();

// Quantize float32 rows v [rows][dim] into rows [row0, row0 + rows).
cudaError_t i4_quantize_launch(const I4Rows& r, int64_t row0, const float* v, int64_t rows, cudaStream_t stream);

// Rows [row0, row0 + rows) from or to the row-major format: codes
// [rows][groups * 16], mults [rows][groups], scales [rows] (all on the device).
cudaError_t i4_pack_launch(const I4Rows& r, int64_t row0, int64_t rows, const uint8_t* codes, const uint8_t* mults,
                           const float* scales, cudaStream_t stream);
cudaError_t i4_unpack_launch(const I4Rows& r, int64_t row0, int64_t rows, uint8_t* codes, uint8_t* mults, float* scales,
                             cudaStream_t stream);

// Scores of M <= i4_batch(groups) queries q [M][dim] against rows [row0, row0 + rows),
// row0 a whole tile: dst[m * ld + (row - row0)].
cudaError_t i4_score_launch(const I4Rows& r, int64_t row0, int64_t rows, const float* q, int32_t M, float* dst,
                            int64_t ld, int32_t sm_count, cudaStream_t stream);

// Top-k of M <= i4_batch(groups) queries over all rows.
struct I4TopK {
  const float* q;        // [M][dim]
  int32_t M, k;
  uint32_t id_base;      // global id of row 0
  const uint64_t* keep;  // optional keep bitmap over global ids
  int64_t keep_nbits;
  uint32_t* best;        // [kI4MaxBatch][i4_best_ld(n)] scratch, zero at rest past the tiles: rank of each tile's best score
  uint32_t* list;        // [kI4MaxBatch][i4_picks(kI4MaxK)] scratch: tiles that hold the top k
  uint64_t* cand;        // [kI4MaxBatch][i4_cand(n)] scratch: their rows' keys
  uint64_t* out;         // [M][k] sorted keys, 0 = empty
};
// Ranks of a query's tiles, in whole fours.
inline int64_t i4_best_ld(int64_t n) { return (i4_tiles(n) + 3) / 4 * 4; }
// Tiles (or runs of tiles) that a top-k of k may look at: some more than k, so
// that the search for their threshold ends early.
__host__ __device__ constexpr int32_t i4_picks(int32_t k) { return k + k / 8 + 8; }
// Keys that a query's tiles can hold.
inline int64_t i4_cand(int64_t n) {
  const int64_t tiles = i4_tiles(n), most = i4_picks(kI4MaxK);
  return (tiles < most ? tiles : most) * kI4Tile;
}
cudaError_t i4_topk_launch(const I4Rows& r, const I4TopK& p, int32_t sm_count, cudaStream_t stream);

#ifdef __CUDACC__

// Four codes of a word against four query bytes: the low nibbles face qlo, the
// high ones qhi. The bytes are c + 8; the caller starts acc at -8 * sum(q8).
__device__ __forceinline__ int i4_dot_word(uint32_t w, int qlo, int qhi, int acc) {
  acc = __dp4a((int)(w & 0x0F0F0F0Fu), qlo, acc);
  return __dp4a((int)((w >> 4) & 0x0F0F0F0Fu), qhi, acc);
}

#endif  // __CUDACC__

}  // namespace fi8
