// fi8_i4_api.cu -- the C entry points of FlatI4 (include/fi8.h, fi8_i4_*).
//
// The async forms allocate nothing: an index owns, from its creation on, the
// score scratch and the select lists that its largest call needs, so they can
// be captured into a graph and their addresses never change.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <new>

#include "fi8_device.cuh"
#include "fi8_host.h"
#include "fi8_i4.cuh"
#include "fi8_scan.cuh"
#include "fi8_stage.h"

using namespace fi8;

namespace {

// Scores of a top-k pass held at once. 64 MB stay in the 126 MB L2, so the
// select reads them from there; a larger pass runs as row ranges.
constexpr int64_t kScoreScratch = 16 << 20;

}  // namespace

struct fi8_i4 {
  fi8_ctx* ctx = nullptr;
  int device = 0, sm_count = 0;
  uint32_t id_base = 0;
  I4Rows rows{};
  cudaStream_t stream = nullptr;  // the host-pointer forms and the uploads
  std::mutex mu;

  // top-k scratch
  float* d_scores = nullptr;
  int64_t scores_cap = 0;
  uint64_t* d_lists = nullptr;  // sorted keys of the row ranges of a pass, null when there is one range
  uint64_t* d_lvl1 = nullptr;
  uint64_t* d_lvl2 = nullptr;
  unsigned long long* d_gthr = nullptr;  // [8], zero at rest
  unsigned int* d_counter = nullptr;     // zero at rest; the last 8 are the block tickets
  // staging of the host-pointer forms
  float* d_q = nullptr;
  size_t q_cap = 0;
  uint64_t* d_keys = nullptr;
  size_t keys_cap = 0;
  uint64_t* h_keys = nullptr;
  size_t h_keys_cap = 0;
  uint64_t* d_keep = nullptr;
  size_t keep_cap = 0;
};

namespace {

constexpr int32_t kCounters = kI4SelectCtas + kI4MaxBatch;  // block tickets of every query, then one a query

// Rows of one range of a pass of M queries.
int64_t range_rows(const fi8_i4* x, int32_t M) {
  const int64_t most = x->scores_cap / M / kI4SelectTile * kI4SelectTile;
  return std::min<int64_t>(x->rows.n, most);
}

void i4_free(fi8_i4* x) {
  DeviceGuard g(x->device);
  if (x->stream) cudaStreamSynchronize(x->stream);
  cudaFree(x->rows.codes);
  cudaFree(x->rows.mults);
  cudaFree(x->rows.scales);
  cudaFree(x->d_scores);
  cudaFree(x->d_lists);
  cudaFree(x->d_lvl1);
  cudaFree(x->d_lvl2);
  cudaFree(x->d_gthr);
  cudaFree(x->d_counter);
  cudaFree(x->d_q);
  cudaFree(x->d_keys);
  cudaFree(x->d_keep);
  if (x->h_keys) cudaFreeHost(x->h_keys);
  if (x->stream) cudaStreamDestroy(x->stream);
  delete x;
}

int i4_alloc(fi8_ctx* ctx, int64_t n, int32_t dim, int64_t id_base, const char* who, fi8_i4** out) {
  *out = nullptr;
  if (!ctx) return fail(FI8_ERR_ARG, "%s: null ctx", who);
  if (n <= 0 || dim <= 0) return fail(FI8_ERR_ARG, "gpu: empty 4-bit index (n=%lld dim=%d)", (long long)n, dim);
  if (id_base < 0 || n > 0x7FFFFFFFll || id_base > 0x7FFFFFFFll - n)
    return fail(FI8_ERR_ARG, "%s: global indices must fit in 31 bits (id_base=%lld n=%lld)", who, (long long)id_base,
                (long long)n);
  if (dim > kI4MaxDim) return fail(FI8_ERR_DECLINED, "%s: dim %d exceeds the supported %d", who, dim, kI4MaxDim);
  DeviceGuard g(ctx->device);
  fi8_i4* x = new (std::nothrow) fi8_i4;
  if (!x) return fail(FI8_ERR_OOM, "%s: host allocation", who);
  x->ctx = ctx;
  x->device = ctx->device;
  x->sm_count = ctx->sm_count;
  x->id_base = (uint32_t)id_base;
  I4Rows& r = x->rows;
  r.n = n;
  r.dim = dim;
  r.groups = i4_groups(dim);
  r.mpitch = i4_mult_pitch(r.groups);
  const int64_t n_tile = (n + kI4SelectTile - 1) / kI4SelectTile * kI4SelectTile;
  x->scores_cap = std::min<int64_t>(kI4MaxBatch * n_tile, kScoreScratch);
  size_t lists = 0;
  for (int32_t m = 1; m <= kI4MaxBatch; m++) {
    const int64_t per = range_rows(x, m), ranges = (n + per - 1) / per;
    if (ranges > 1) lists = std::max(lists, (size_t)ranges * m * kI4MaxK);
  }
  const size_t ctas = (size_t)std::min<int64_t>(kI4SelectCtas, kI4MaxBatch * (n_tile / kI4SelectTile));
  cudaError_t e = cudaStreamCreateWithFlags(&x->stream, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMalloc(&r.codes, (size_t)n * r.groups * 16);
  if (e == cudaSuccess) e = cudaMalloc(&r.mults, (size_t)n * r.mpitch);
  if (e == cudaSuccess) e = cudaMalloc(&r.scales, (size_t)n * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&x->d_scores, (size_t)x->scores_cap * sizeof(float));
  if (e == cudaSuccess && lists) e = cudaMalloc(&x->d_lists, lists * sizeof(uint64_t));
  if (e == cudaSuccess) e = cudaMalloc(&x->d_lvl1, ctas * kI4MaxK * sizeof(uint64_t));
  if (e == cudaSuccess) e = cudaMalloc(&x->d_lvl2, (ctas / 8 + kI4MaxBatch) * kI4MaxK * sizeof(uint64_t));
  if (e == cudaSuccess) e = cudaMalloc(&x->d_gthr, kI4MaxBatch * sizeof(unsigned long long));
  if (e == cudaSuccess) e = cudaMalloc(&x->d_counter, kCounters * sizeof(unsigned int));
  if (e == cudaSuccess) e = cudaMemsetAsync(r.codes, 0, (size_t)n * r.groups * 16, x->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(r.mults, 0, (size_t)n * r.mpitch, x->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(r.scales, 0, (size_t)n * sizeof(float), x->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(x->d_gthr, 0, kI4MaxBatch * sizeof(unsigned long long), x->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(x->d_counter, 0, kCounters * sizeof(unsigned int), x->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(x->stream);
  if (e != cudaSuccess) {
    const int rc = cuda_fail(e, "gpu: device allocation failed");
    i4_free(x);
    return rc;
  }
  *out = x;
  return FI8_OK;
}

int launch_scores(fi8_i4* x, const float* d_q, int32_t M, float* d_dst, cudaStream_t st) {
  for (int32_t m0 = 0; m0 < M; m0 += kI4MaxBatch) {
    const int32_t mm = std::min(kI4MaxBatch, M - m0);
    FI8_CUDA(i4_score_launch(x->rows, 0, x->rows.n, d_q + (size_t)m0 * x->rows.dim, mm,
                             d_dst + (size_t)m0 * x->rows.n, x->rows.n, x->sm_count, st),
             "i4_score_launch");
  }
  return FI8_OK;
}

int launch_topk(fi8_i4* x, const float* d_q, int32_t M, int32_t k, const uint64_t* d_keep, int64_t nbits,
                uint64_t* d_keys, cudaStream_t st) {
  const int64_t n = x->rows.n;
  for (int32_t m0 = 0; m0 < M; m0 += kI4MaxBatch) {
    const int32_t mm = std::min(kI4MaxBatch, M - m0);
    const int64_t per = range_rows(x, mm), ranges = (n + per - 1) / per;
    uint64_t* out = d_keys + (size_t)m0 * k;
    for (int64_t i = 0; i < ranges; i++) {
      const int64_t row0 = i * per, rows = std::min(per, n - row0);
      I4Select s{};
      s.scores = x->d_scores;
      s.ld = (rows + 3) / 4 * 4;
      s.rows = rows;
      s.id0 = x->id_base + (uint32_t)row0;
      s.keep = d_keep;
      s.keep_nbits = nbits;
      s.k = k;
      s.gthr = x->d_gthr;
      s.counter = x->d_counter;
      s.counter2 = x->d_counter + kI4SelectCtas;
      s.lvl1 = x->d_lvl1;
      s.lvl2 = x->d_lvl2;
      s.out = ranges == 1 ? out : x->d_lists + (size_t)i * mm * k;
      const size_t smem = i4_select_plan(&s, mm);
      FI8_CUDA(i4_score_launch(x->rows, row0, rows, d_q + (size_t)m0 * x->rows.dim, mm, x->d_scores, s.ld,
                               x->sm_count, st),
               "i4_score_launch");
      FI8_CUDA(i4_select_launch(s, mm, smem, st), "i4_select_launch");
    }
    if (ranges > 1)
      FI8_CUDA(merge_keys_launch(x->d_lists, (int32_t)ranges, mm, k, out, st), "merge_keys_launch");
  }
  return FI8_OK;
}

// Copy M host queries to the index's staging buffer.
int stage_queries(fi8_i4* x, const float* q, int32_t M) {
  const size_t count = (size_t)M * x->rows.dim;
  int rc = ensure_device(&x->d_q, &x->q_cap, count, "staging q");
  if (rc != FI8_OK) return rc;
  FI8_CUDA(cudaMemcpyAsync(x->d_q, q, count * sizeof(float), cudaMemcpyHostToDevice, x->stream), "H2D queries");
  return FI8_OK;
}

// Upload through pinned buffers; the host threads of the stager may throw.
template <typename F>
cudaError_t with_stager(F body) {
  try {
    PinnedStager stage;
    cudaError_t e = stage.init();
    if (e == cudaSuccess) e = body(stage);
    const cudaError_t f = stage.finish();
    return e == cudaSuccess ? f : e;
  } catch (...) {
    return cudaErrorMemoryAllocation;
  }
}

}  // namespace

extern "C" {

int fi8_i4_create_empty(fi8_ctx* ctx, int64_t n, int32_t dim, int64_t id_base, fi8_i4** out) {
  if (!out) return fail(FI8_ERR_ARG, "fi8_i4_create_empty: null out");
  return i4_alloc(ctx, n, dim, id_base, "fi8_i4_create_empty", out);
}

int fi8_i4_create(fi8_ctx* ctx, const uint8_t* codes, const uint8_t* mults, const float* scales, int64_t n, int32_t dim,
                  int64_t id_base, fi8_i4** out) {
  if (!out) return fail(FI8_ERR_ARG, "fi8_i4_create: null out");
  *out = nullptr;
  if (n > 0 && dim > 0 && (!codes || !mults || !scales)) return fail(FI8_ERR_ARG, "fi8_i4_create: null rows");
  fi8_i4* x = nullptr;
  int rc = i4_alloc(ctx, n, dim, id_base, "fi8_i4_create", &x);
  if (rc != FI8_OK) return rc;
  DeviceGuard g(x->device);
  const I4Rows& r = x->rows;
  const cudaError_t e = with_stager([&](PinnedStager& stage) {
    cudaError_t c = stage.put_rows(r.codes, (size_t)r.groups * 16, codes, (size_t)r.groups * 16, (size_t)r.groups * 16,
                                   n, x->stream);
    if (c == cudaSuccess) c = stage.put_rows(r.mults, r.mpitch, mults, r.groups, r.groups, n, x->stream);
    if (c == cudaSuccess) c = stage.put_rows(r.scales, 4, scales, 4, 4, n, x->stream);
    return c;
  });
  if (e != cudaSuccess) {
    rc = cuda_fail(e, "gpu: device upload failed");
    i4_free(x);
    return rc;
  }
  *out = x;
  return FI8_OK;
}

int fi8_i4_create_f32(fi8_ctx* ctx, const float* vecs, int64_t n, int32_t dim, int64_t id_base, fi8_i4** out) {
  if (!out) return fail(FI8_ERR_ARG, "fi8_i4_create_f32: null out");
  *out = nullptr;
  if (n > 0 && dim > 0 && !vecs) return fail(FI8_ERR_ARG, "fi8_i4_create_f32: null vectors");
  fi8_i4* x = nullptr;
  int rc = i4_alloc(ctx, n, dim, id_base, "fi8_i4_create_f32", &x);
  if (rc != FI8_OK) return rc;
  DeviceGuard g(x->device);
  const size_t rb = (size_t)dim * sizeof(float);
  const int64_t chunk = std::min<int64_t>(n, (int64_t)(PinnedStager::kBufBytes / rb));
  float* d_v = nullptr;
  cudaError_t e = cudaMalloc(&d_v, (size_t)chunk * rb);
  if (e == cudaSuccess)
    e = with_stager([&](PinnedStager& stage) {
      cudaError_t c = cudaSuccess;
      for (int64_t r0 = 0; c == cudaSuccess && r0 < n; r0 += chunk) {
        const int64_t rows = std::min(chunk, n - r0);
        // stream order keeps the next chunk's copy behind this chunk's kernel
        c = stage.put_rows(d_v, rb, vecs + (size_t)r0 * dim, rb, rb, rows, x->stream);
        if (c == cudaSuccess) c = i4_quantize_launch(x->rows, r0, d_v, rows, x->stream);
      }
      return c;
    });
  if (e == cudaSuccess) e = cudaStreamSynchronize(x->stream);
  cudaFree(d_v);
  if (e != cudaSuccess) {
    rc = cuda_fail(e, "gpu: device build failed");
    i4_free(x);
    return rc;
  }
  *out = x;
  return FI8_OK;
}

int fi8_i4_set_rows_async(fi8_i4* idx, int64_t row0, const float* d_vecs, int64_t rows, void* stream) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_set_rows_async: null index");
  if (rows == 0) return FI8_OK;
  if (rows < 0 || row0 < 0 || row0 > idx->rows.n - rows || !d_vecs)
    return fail(FI8_ERR_ARG, "fi8_i4_set_rows_async: rows [%lld, +%lld) outside [0, %lld) or null data",
                (long long)row0, (long long)rows, (long long)idx->rows.n);
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  FI8_CUDA(i4_quantize_launch(idx->rows, row0, d_vecs, rows, static_cast<cudaStream_t>(stream)), "i4_quantize_launch");
  return FI8_OK;
}

int fi8_i4_read_rows(fi8_i4* idx, uint8_t* codes, uint8_t* mults, float* scales) {
  if (!idx || !codes || !mults || !scales) return fail(FI8_ERR_ARG, "fi8_i4_read_rows: null argument");
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  const I4Rows& r = idx->rows;
  FI8_CUDA(cudaDeviceSynchronize(), "sync");  // rows set on any stream
  FI8_CUDA(cudaMemcpy(codes, r.codes, (size_t)r.n * r.groups * 16, cudaMemcpyDeviceToHost), "fi8_i4_read_rows");
  FI8_CUDA(cudaMemcpy2D(mults, r.groups, r.mults, r.mpitch, r.groups, (size_t)r.n, cudaMemcpyDeviceToHost),
           "fi8_i4_read_rows");
  FI8_CUDA(cudaMemcpy(scales, r.scales, (size_t)r.n * sizeof(float), cudaMemcpyDeviceToHost), "fi8_i4_read_rows");
  return FI8_OK;
}

int fi8_i4_destroy(fi8_i4* idx) {
  if (!idx) return FI8_OK;
  {
    std::lock_guard<std::mutex> lk(idx->mu);
  }
  i4_free(idx);
  return FI8_OK;
}

int fi8_i4_info(fi8_i4* idx, int64_t* n, int32_t* dim) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_info: null index");
  if (n) *n = idx->rows.n;
  if (dim) *dim = idx->rows.dim;
  return FI8_OK;
}

int fi8_i4_score_batch(fi8_i4* idx, const float* q, int32_t M, float* dst) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_score_batch: null index");
  if (M == 0) return FI8_OK;
  if (M < 0 || !q || !dst) return fail(FI8_ERR_ARG, "fi8_i4_score_batch: bad arguments");
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  fi8_i4* x = idx;
  const int64_t n = x->rows.n;
  int rc = stage_queries(x, q, M);
  if (rc != FI8_OK) return rc;
  for (int32_t m0 = 0; m0 < M; m0 += kI4MaxBatch) {
    const int32_t mm = std::min(kI4MaxBatch, M - m0);
    const int64_t per = range_rows(x, mm);
    for (int64_t row0 = 0; row0 < n; row0 += per) {
      const int64_t rows = std::min(per, n - row0);
      FI8_CUDA(i4_score_launch(x->rows, row0, rows, x->d_q + (size_t)m0 * x->rows.dim, mm, x->d_scores, rows,
                               x->sm_count, x->stream),
               "i4_score_launch");
      FI8_CUDA(cudaMemcpy2DAsync(dst + (size_t)m0 * n + row0, (size_t)n * 4, x->d_scores, (size_t)rows * 4,
                                 (size_t)rows * 4, mm, cudaMemcpyDeviceToHost, x->stream),
               "D2H scores");
    }
  }
  FI8_CUDA(cudaStreamSynchronize(x->stream), "sync");
  return FI8_OK;
}

int fi8_i4_score_async(fi8_i4* idx, const float* d_q, int32_t M, float* d_dst, void* stream) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_score_async: null index");
  if (M == 0) return FI8_OK;
  if (M < 0 || !d_q || !d_dst) return fail(FI8_ERR_ARG, "fi8_i4_score_async: bad arguments");
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  return launch_scores(idx, d_q, M, d_dst, static_cast<cudaStream_t>(stream));
}

int fi8_i4_topk_batch(fi8_i4* idx, const float* q, int32_t M, int32_t k, const uint64_t* keep, int64_t nbits,
                      int32_t* out_idx, float* out_score) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_topk_batch: null index");
  if (M == 0) return FI8_OK;
  if (M < 0 || !q || !out_idx || !out_score || nbits < 0) return fail(FI8_ERR_ARG, "fi8_i4_topk_batch: bad arguments");
  if (k <= 0 || (int64_t)k >= idx->rows.n || k > kI4MaxK)
    return fail(FI8_ERR_DECLINED, "gpu: TopKBatch declined (k=%d n=%lld batch=%d, k at most %d)", k,
                (long long)idx->rows.n, M, kI4MaxK);
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  fi8_i4* x = idx;
  const size_t nk = (size_t)M * k;
  int rc = stage_queries(x, q, M);
  if (rc == FI8_OK) rc = ensure_device(&x->d_keys, &x->keys_cap, nk, "staging keys");
  if (rc == FI8_OK) rc = ensure_host(&x->h_keys, &x->h_keys_cap, nk, "pinned keys");
  const uint64_t* d_keep = nullptr;
  if (rc == FI8_OK && keep) {
    const size_t words = (size_t)((nbits + 63) / 64);
    rc = ensure_device(&x->d_keep, &x->keep_cap, words, "keep bitmap");
    if (rc == FI8_OK && words)
      FI8_CUDA(cudaMemcpyAsync(x->d_keep, keep, words * 8, cudaMemcpyHostToDevice, x->stream), "H2D keep");
    d_keep = x->d_keep;
  }
  if (rc == FI8_OK) rc = launch_topk(x, x->d_q, M, k, d_keep, nbits, x->d_keys, x->stream);
  if (rc != FI8_OK) return rc;
  FI8_CUDA(cudaMemcpyAsync(x->h_keys, x->d_keys, nk * sizeof(uint64_t), cudaMemcpyDeviceToHost, x->stream),
           "D2H keys");
  FI8_CUDA(cudaStreamSynchronize(x->stream), "sync");
  return fi8_keys_unpack(x->h_keys, (int64_t)nk, out_idx, out_score);
}

int fi8_i4_topk_async(fi8_i4* idx, const float* d_q, int32_t M, int32_t k, const uint64_t* d_keep, int64_t nbits,
                      uint64_t* d_keys, void* stream) {
  if (!idx) return fail(FI8_ERR_ARG, "fi8_i4_topk_async: null index");
  if (M == 0) return FI8_OK;
  if (M < 0 || !d_q || !d_keys || nbits < 0) return fail(FI8_ERR_ARG, "fi8_i4_topk_async: bad arguments");
  if (k <= 0 || k > kI4MaxK)  // k >= n: a shard yields all of its rows, then empty keys
    return fail(FI8_ERR_DECLINED, "gpu: TopKBatch declined (k=%d, at most %d)", k, kI4MaxK);
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  return launch_topk(idx, d_q, M, k, d_keep, nbits, d_keys, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
