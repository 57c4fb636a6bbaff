// fi8_kb.cuh -- KeyBlocks: block-sparse attention over a key/value cache whose
// blocks are chosen by their FlatI4 rows.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "fi8_i4.cuh"

namespace fi8 {

constexpr int32_t kKbMaxHeadDim = 256;
constexpr int32_t kKbMaxGroup = 64;       // query heads of a key/value head
constexpr int32_t kKbMaxSelect = 1024;    // blocks a query row may read
constexpr int32_t kKbMaxBlocks = 36864;   // blocks of a slot: their ranks fit one CTA's shared memory
constexpr int32_t kKbMaxRows = 65535;     // query rows of a call

// Everything a launch needs. Strides in elements.
struct KbParams {
  const void* k;
  const void* v;
  int64_t slot_stride, head_stride, token_stride;
  int64_t capacity;
  int32_t slots, kv_heads, q_heads, head_dim, block, max_blocks;
  int32_t block_shift;  // block = 1 << block_shift
  bool f16;
  // FlatI4 rows, one a full block, a set of whole tiles a (slot, kv head)
  uint32_t* codes;
  uint32_t* mults;
  float* scales;
  int32_t groups, tiles;  // tiles of a set
  unsigned int* err;  // device error flags (kKbErrRow)
  // a call's query rows
  const void* q;
  int64_t q_stride;
  const int32_t* slot;
  const int32_t* len;
  int32_t rows, select, first, last;
  int32_t* sel;  // [rows][kv_heads][select]
  float scale;
  void* out;
  float* lse;
};

// The rows of (slot, kv head) pair i.
__host__ __device__ inline I4Rows kb_rows(const KbParams& p, int64_t i) {
  I4Rows r;
  r.codes = p.codes + i * p.tiles * p.groups * 128;
  r.mults = p.mults + i * p.tiles * ((p.groups + 3) / 4) * 32;
  r.scales = p.scales + i * p.tiles * kI4Tile;
  r.n = p.max_blocks;
  r.dim = p.head_dim;
  r.groups = p.groups;
  return r;
}

constexpr unsigned int kKbErrRow = 2u;  // a slot, length or range outside the cache

// Once on each device, before the first launch on it.
cudaError_t kb_init();

cudaError_t kb_update_launch(const KbParams& p, const int32_t* slot, const int32_t* from, const int32_t* to,
                             int32_t count, int32_t max_tokens, cudaStream_t stream);
cudaError_t kb_select_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream);
cudaError_t kb_attend_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream);
// Both, with the same results, in one launch or two.
cudaError_t kb_query_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream);

}  // namespace fi8
