// fi8_i4_api.cu -- the C entry points of FlatI4 (include/fi8.h, fi8_i4_*).
//
// The async forms allocate nothing: an index owns, from its creation on, the
// scratch that its largest call needs (in one allocation with its rows), so
// they can be captured into a graph and their addresses never change.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <new>

#include "fi8_device.cuh"
#include "fi8_host.h"
#include "fi8_i4.cuh"
#include "fi8_stage.h"

using namespace fi8;

namespace {

// Scores that the host form of score_batch holds on the device at once.
constexpr int64_t kHostScores = 16 << 20;
// Bytes of packed rows that an upload or a read holds on the device at once.
constexpr size_t kPackBytes = (size_t)64 << 20;

}  // namespace

struct fi8_i4 {
  fi8_ctx* ctx = nullptr;
  int device = 0, sm_count = 0;
  uint32_t id_base = 0;
  I4Rows rows{};
  cudaStream_t stream = nullptr;  // the host-pointer forms and the uploads
  cudaEvent_t rows_set = nullptr;  // behind the last fi8_i4_set_rows_async
  std::mutex mu;

  unsigned char* d_base = nullptr;  // rows and top-k scratch
  uint32_t* d_best = nullptr;
  uint32_t* d_list = nullptr;
  uint64_t* d_cand = nullptr;
  // staging of the host-pointer forms
  float* d_q = nullptr;
  size_t q_cap = 0;
  uint64_t* d_keys = nullptr;
  size_t keys_cap = 0;
  uint64_t* h_keys = nullptr;
  size_t h_keys_cap = 0;
  uint64_t* d_keep = nullptr;
  size_t keep_cap = 0;
  float* d_scores = nullptr;
  size_t scores_cap = 0;
};

namespace {

void i4_free(fi8_i4* x) {
  DeviceGuard g(x->device);
  if (x->stream) cudaStreamSynchronize(x->stream);
  cudaFree(x->d_base);
  cudaFree(x->d_scores);
  cudaFree(x->d_q);
  cudaFree(x->d_keys);
  cudaFree(x->d_keep);
  if (x->h_keys) cudaFreeHost(x->h_keys);
  if (x->rows_set) cudaEventDestroy(x->rows_set);
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
  // one allocation: codes, multipliers, scales, then the scratch
  size_t at = 0;
  auto part = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t tiles = (size_t)i4_tiles(n);
  const size_t codes = part(i4_code_bytes(n, r.groups)), mults = part(i4_mult_bytes(n, r.groups));
  const size_t scales = part(tiles * kI4Tile * sizeof(float));
  const size_t best = part((size_t)kI4MaxBatch * i4_best_ld(n) * sizeof(uint32_t)), zero_end = at;
  const size_t list = part((size_t)kI4MaxBatch * i4_picks(kI4MaxK) * sizeof(uint32_t));
  const size_t cand = part((size_t)kI4MaxBatch * i4_cand(n) * sizeof(uint64_t));
  cudaError_t e = cudaStreamCreateWithFlags(&x->stream, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaEventCreateWithFlags(&x->rows_set, cudaEventDisableTiming);
  if (e == cudaSuccess) e = i4_init();
  if (e == cudaSuccess) e = cudaMalloc(&x->d_base, at);
  if (e == cudaSuccess) e = cudaMemsetAsync(x->d_base, 0, zero_end, x->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(x->stream);
  if (e != cudaSuccess) {
    const int rc = cuda_fail(e, "gpu: device allocation failed");
    i4_free(x);
    return rc;
  }
  r.codes = reinterpret_cast<uint32_t*>(x->d_base + codes);
  r.mults = reinterpret_cast<uint32_t*>(x->d_base + mults);
  r.scales = reinterpret_cast<float*>(x->d_base + scales);
  x->d_best = reinterpret_cast<uint32_t*>(x->d_base + best);
  x->d_list = reinterpret_cast<uint32_t*>(x->d_base + list);
  x->d_cand = reinterpret_cast<uint64_t*>(x->d_base + cand);
  *out = x;
  return FI8_OK;
}

int launch_scores(fi8_i4* x, const float* d_q, int32_t M, float* d_dst, cudaStream_t st) {
  for (int32_t m0 = 0, most = i4_batch(x->rows.groups); m0 < M; m0 += most) {
    const int32_t mm = std::min(most, M - m0);
    FI8_CUDA(i4_score_launch(x->rows, 0, x->rows.n, d_q + (size_t)m0 * x->rows.dim, mm,
                             d_dst + (size_t)m0 * x->rows.n, x->rows.n, x->sm_count, st),
             "i4_score_launch");
  }
  return FI8_OK;
}

int launch_topk(fi8_i4* x, const float* d_q, int32_t M, int32_t k, const uint64_t* d_keep, int64_t nbits,
                uint64_t* d_keys, cudaStream_t st) {
  for (int32_t m0 = 0, most = i4_batch(x->rows.groups); m0 < M; m0 += most) {
    I4TopK p{};
    p.q = d_q + (size_t)m0 * x->rows.dim;
    p.M = std::min(most, M - m0);
    p.k = k;
    p.id_base = x->id_base;
    p.keep = d_keep;
    p.keep_nbits = nbits;
    p.best = x->d_best;
    p.list = x->d_list;
    p.cand = x->d_cand;
    p.out = d_keys + (size_t)m0 * k;
    FI8_CUDA(i4_topk_launch(x->rows, p, x->sm_count, st), "i4_topk_launch");
  }
  return FI8_OK;
}

// Copy M host queries to the index's staging buffer, behind the rows set on
// other streams.
int stage_queries(fi8_i4* x, const float* q, int32_t M) {
  const size_t count = (size_t)M * x->rows.dim;
  int rc = ensure_device(&x->d_q, &x->q_cap, count, "staging q");
  if (rc != FI8_OK) return rc;
  FI8_CUDA(cudaStreamWaitEvent(x->stream, x->rows_set, 0), "wait for rows");
  FI8_CUDA(cudaMemcpyAsync(x->d_q, q, count * sizeof(float), cudaMemcpyHostToDevice, x->stream), "H2D queries");
  return FI8_OK;
}

// A part of the rows in the row-major format, on the device.
struct PackBuffer {
  int64_t rows = 0;
  unsigned char* base = nullptr;
  uint8_t* codes = nullptr;
  uint8_t* mults = nullptr;
  float* scales = nullptr;
  cudaError_t error;
  explicit PackBuffer(const I4Rows& r) {
    const size_t row = (size_t)r.groups * 17 + 4;
    rows = std::max<int64_t>(1, std::min<int64_t>(r.n, (int64_t)(kPackBytes / row)));
    error = cudaMalloc(&base, rows * row);
    if (error != cudaSuccess) return;
    scales = reinterpret_cast<float*>(base + rows * r.groups * 16);
    codes = base;
    mults = base + rows * (r.groups * 16 + 4);
  }
  ~PackBuffer() { cudaFree(base); }
  PackBuffer(const PackBuffer&) = delete;
  PackBuffer& operator=(const PackBuffer&) = delete;
};

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
  const PackBuffer b(x->rows);
  cudaError_t e = b.error;
  if (e == cudaSuccess)
    e = with_stager([&](PinnedStager& stage) {
      const size_t cb = (size_t)x->rows.groups * 16, mb = x->rows.groups;
      cudaError_t c = cudaSuccess;
      for (int64_t r0 = 0; c == cudaSuccess && r0 < n; r0 += b.rows) {
        // stream order keeps the next chunk's copies behind this chunk's kernel
        const int64_t rows = std::min(b.rows, n - r0);
        c = stage.put_rows(b.codes, cb, codes + (size_t)r0 * cb, cb, cb, rows, x->stream);
        if (c == cudaSuccess) c = stage.put_rows(b.mults, mb, mults + (size_t)r0 * mb, mb, mb, rows, x->stream);
        if (c == cudaSuccess) c = stage.put_rows(b.scales, 4, scales + r0, 4, 4, rows, x->stream);
        if (c == cudaSuccess) c = i4_pack_launch(x->rows, r0, rows, b.codes, b.mults, b.scales, x->stream);
      }
      return c;
    });
  if (e == cudaSuccess) e = cudaStreamSynchronize(x->stream);
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // One event for all streams: each call also waits for the one before. A captured
  // call has no place in that order.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  FI8_CUDA(cudaStreamIsCapturing(st, &capture), "cudaStreamIsCapturing");
  const bool ordered = capture == cudaStreamCaptureStatusNone;
  if (ordered) FI8_CUDA(cudaStreamWaitEvent(st, idx->rows_set, 0), "wait for rows");
  FI8_CUDA(i4_quantize_launch(idx->rows, row0, d_vecs, rows, st), "i4_quantize_launch");
  if (ordered) FI8_CUDA(cudaEventRecord(idx->rows_set, st), "cudaEventRecord");
  return FI8_OK;
}

int fi8_i4_read_rows(fi8_i4* idx, uint8_t* codes, uint8_t* mults, float* scales) {
  if (!idx || !codes || !mults || !scales) return fail(FI8_ERR_ARG, "fi8_i4_read_rows: null argument");
  std::lock_guard<std::mutex> lk(idx->mu);
  DeviceGuard g(idx->device);
  const I4Rows& r = idx->rows;
  const PackBuffer b(r);
  FI8_CUDA(b.error, "fi8_i4_read_rows");
  FI8_CUDA(cudaDeviceSynchronize(), "sync");  // rows set on any stream
  const size_t cb = (size_t)r.groups * 16, mb = r.groups;
  for (int64_t r0 = 0; r0 < r.n; r0 += b.rows) {
    const int64_t rows = std::min(b.rows, r.n - r0);
    FI8_CUDA(i4_unpack_launch(r, r0, rows, b.codes, b.mults, b.scales, idx->stream), "i4_unpack_launch");
    FI8_CUDA(cudaMemcpyAsync(codes + (size_t)r0 * cb, b.codes, rows * cb, cudaMemcpyDeviceToHost, idx->stream), "D2H codes");
    FI8_CUDA(cudaMemcpyAsync(mults + (size_t)r0 * mb, b.mults, rows * mb, cudaMemcpyDeviceToHost, idx->stream), "D2H mults");
    FI8_CUDA(cudaMemcpyAsync(scales + r0, b.scales, rows * 4, cudaMemcpyDeviceToHost, idx->stream), "D2H scales");
  }
  FI8_CUDA(cudaStreamSynchronize(idx->stream), "sync");
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
  const int64_t per = std::min<int64_t>(i4_tiles(n) * kI4Tile, kHostScores / kI4MaxBatch);
  rc = ensure_device(&x->d_scores, &x->scores_cap, (size_t)(std::min(M, kI4MaxBatch) * per), "staging scores");
  if (rc != FI8_OK) return rc;
  for (int32_t m0 = 0, most = i4_batch(x->rows.groups); m0 < M; m0 += most) {
    const int32_t mm = std::min(most, M - m0);
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
