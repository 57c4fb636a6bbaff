// fi8_kb_api.cu -- the C entry points of KeyBlocks (include/fi8.h, fi8_kb_*).
#include <cuda_runtime.h>

#include <cmath>
#include <mutex>
#include <new>

#include "fi8_host.h"
#include "fi8_kb.cuh"

using namespace fi8;

struct fi8_kb {
  fi8_ctx* ctx = nullptr;
  int device = 0, sm_count = 0;
  int32_t max_rows = 0, max_select = 0;
  KbParams p{};  // the cache and its block rows; a call fills in the rest
  unsigned char* base = nullptr;
  std::mutex mu;
};

namespace {

void kb_free(fi8_kb* b) {
  DeviceGuard g(b->device);
  cudaFree(b->base);
  delete b;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The arguments that select, attend and query share.
int fill_rows(fi8_kb* b, const char* who, const void* d_q, int64_t q_stride, const int32_t* d_slot, const int32_t* d_len,
              int32_t rows, int32_t k, int32_t* d_sel, KbParams* p) {
  if (!d_q || !d_slot || !d_len || !d_sel) return fail(FI8_ERR_ARG, "%s: null argument", who);
  if (rows < 0 || rows > b->max_rows) return fail(FI8_ERR_ARG, "%s: %d rows, made for at most %d", who, rows, b->max_rows);
  if (k <= 0 || k > b->max_select) return fail(FI8_ERR_ARG, "%s: k=%d outside [1, %d]", who, k, b->max_select);
  if (!aligned16(d_q) || q_stride % 8 != 0 || q_stride < (int64_t)b->p.q_heads * b->p.head_dim)
    return fail(FI8_ERR_ARG, "%s: query rows must be 16-byte aligned, a multiple of 8 and at least %lld values apart (got %lld)",
                who, (long long)b->p.q_heads * b->p.head_dim, (long long)q_stride);
  *p = b->p;
  p->q = d_q;
  p->q_stride = q_stride;
  p->slot = d_slot;
  p->len = d_len;
  p->rows = rows;
  p->select = k;
  p->sel = d_sel;
  return FI8_OK;
}

int fill_select(const char* who, int32_t first, int32_t last, KbParams* p) {
  if (first < 0 || last < 1 || first > p->select - last)
    return fail(FI8_ERR_ARG, "%s: first=%d and last=%d must leave first >= 0, last >= 1 and first + last <= k=%d", who, first,
                last, p->select);
  p->first = first;
  p->last = last;
  return FI8_OK;
}

int fill_attend(const char* who, float scale, void* d_out, float* d_lse, KbParams* p) {
  if (!d_out || !aligned16(d_out)) return fail(FI8_ERR_ARG, "%s: the output must be a 16-byte aligned device address", who);
  if (!std::isfinite(scale)) return fail(FI8_ERR_ARG, "%s: scale is not finite", who);
  p->scale = scale;
  p->out = d_out;
  p->lse = d_lse;
  return FI8_OK;
}

}  // namespace

extern "C" {

int fi8_kb_create(fi8_ctx* ctx, const fi8_kb_desc* desc, fi8_kb** out) {
  if (!out) return fail(FI8_ERR_ARG, "fi8_kb_create: null out");
  *out = nullptr;
  if (!ctx || !desc) return fail(FI8_ERR_ARG, "fi8_kb_create: null argument");
  const fi8_kb_desc& d = *desc;
  if (d.dtype != FI8_BF16 && d.dtype != FI8_F16) return fail(FI8_ERR_ARG, "fi8_kb_create: dtype %d", d.dtype);
  if (d.slots <= 0 || d.capacity <= 0 || d.kv_heads <= 0 || d.q_heads <= 0 || d.q_heads % d.kv_heads != 0)
    return fail(FI8_ERR_ARG, "fi8_kb_create: %d slots of %lld tokens, %d query heads over %d key/value heads", d.slots,
                (long long)d.capacity, d.q_heads, d.kv_heads);
  if (d.head_dim <= 0 || d.head_dim > kKbMaxHeadDim || d.head_dim % 16 != 0)
    return fail(FI8_ERR_DECLINED, "fi8_kb_create: head_dim %d is not a multiple of 16 up to %d", d.head_dim, kKbMaxHeadDim);
  if (d.block != 16 && d.block != 32 && d.block != 64 && d.block != 128)
    return fail(FI8_ERR_DECLINED, "fi8_kb_create: block %d is not 16, 32, 64 or 128", d.block);
  if (d.q_heads / d.kv_heads > kKbMaxGroup || d.kv_heads > 4096)
    return fail(FI8_ERR_DECLINED, "fi8_kb_create: at most %d query heads a key/value head and 4096 key/value heads", kKbMaxGroup);
  if (d.capacity > (int64_t)kKbMaxBlocks * d.block)
    return fail(FI8_ERR_DECLINED, "fi8_kb_create: capacity %lld exceeds %d blocks of %d", (long long)d.capacity,
                kKbMaxBlocks, d.block);
  if (d.max_rows <= 0 || d.max_rows > kKbMaxRows || d.max_select <= 0 || d.max_select > kKbMaxSelect)
    return fail(FI8_ERR_ARG, "fi8_kb_create: max_rows %d outside [1, %d] or max_select %d outside [1, %d]", d.max_rows,
                kKbMaxRows, d.max_select, kKbMaxSelect);
  if (!d.d_k || !d.d_v || !aligned16(d.d_k) || !aligned16(d.d_v))
    return fail(FI8_ERR_ARG, "fi8_kb_create: keys and values must be 16-byte aligned device addresses");
  if (d.slot_stride < 0 || d.head_stride < 0 || d.slot_stride % 8 || d.head_stride % 8 || d.token_stride % 8 ||
      d.token_stride < d.head_dim)
    return fail(FI8_ERR_ARG, "fi8_kb_create: strides must be non-negative multiples of 8 values, tokens at least head_dim apart");
  fi8_kb* b = new (std::nothrow) fi8_kb;
  if (!b) return fail(FI8_ERR_OOM, "fi8_kb_create: host allocation");
  b->ctx = ctx;
  b->device = ctx->device;
  b->sm_count = ctx->sm_count;
  b->max_rows = d.max_rows;
  b->max_select = d.max_select;
  KbParams& p = b->p;
  p.k = d.d_k;
  p.v = d.d_v;
  p.slot_stride = d.slot_stride;
  p.head_stride = d.head_stride;
  p.token_stride = d.token_stride;
  p.capacity = d.capacity;
  p.slots = d.slots;
  p.kv_heads = d.kv_heads;
  p.q_heads = d.q_heads;
  p.head_dim = d.head_dim;
  p.block = d.block;
  while ((1 << p.block_shift) < d.block) p.block_shift++;
  p.max_blocks = (int32_t)(d.capacity / d.block);
  p.f16 = d.dtype == FI8_F16;
  p.groups = i4_groups(d.head_dim);
  p.tiles = (int32_t)i4_tiles(p.max_blocks);
  // one allocation: codes, multipliers, scales, the error word
  const size_t sets = (size_t)d.slots * d.kv_heads;
  const size_t codes = sets * p.tiles * p.groups * 512, mults = sets * p.tiles * ((p.groups + 3) / 4) * 128;
  const size_t scales = sets * p.tiles * kI4Tile * sizeof(float), bytes = codes + mults + scales + 16;
  if ((double)sets * p.tiles * (p.groups * 512.0 + (p.groups + 3) / 4 * 128 + kI4Tile * 4) > 1e14) {
    kb_free(b);
    return fail(FI8_ERR_OOM, "fi8_kb_create: block rows of %d slots x %d heads x %d blocks", d.slots, d.kv_heads, p.max_blocks);
  }
  DeviceGuard g(b->device);
  unsigned char* base = nullptr;
  cudaError_t e = kb_init();
  if (e == cudaSuccess) e = cudaMalloc(&base, bytes);
  b->base = base;
  if (e == cudaSuccess) e = cudaMemset(base, 0, bytes);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    const int rc = cuda_fail(e, "gpu: device allocation failed");
    kb_free(b);
    return rc;
  }
  p.codes = reinterpret_cast<uint32_t*>(base);
  p.mults = reinterpret_cast<uint32_t*>(base + codes);
  p.scales = reinterpret_cast<float*>(base + codes + mults);
  p.err = reinterpret_cast<unsigned int*>(base + codes + mults + scales);
  *out = b;
  return FI8_OK;
}

int fi8_kb_destroy(fi8_kb* kb) {
  if (!kb) return FI8_OK;
  {
    std::lock_guard<std::mutex> lk(kb->mu);
  }
  kb_free(kb);
  return FI8_OK;
}

int fi8_kb_update_async(fi8_kb* kb, const int32_t* d_slot, const int32_t* d_from, const int32_t* d_to, int32_t count,
                        int32_t max_tokens, void* stream) {
  if (!kb) return fail(FI8_ERR_ARG, "fi8_kb_update_async: null handle");
  if (count == 0) return FI8_OK;
  if (count < 0 || count > 65535 || max_tokens < 0 || !d_slot || !d_from || !d_to)
    return fail(FI8_ERR_ARG, "fi8_kb_update_async: bad arguments (count=%d max_tokens=%d)", count, max_tokens);
  std::lock_guard<std::mutex> lk(kb->mu);
  DeviceGuard g(kb->device);
  FI8_CUDA(kb_update_launch(kb->p, d_slot, d_from, d_to, count, max_tokens, static_cast<cudaStream_t>(stream)),
           "kb_update_launch");
  return FI8_OK;
}

int fi8_kb_select_async(fi8_kb* kb, const void* d_q, int64_t q_stride, const int32_t* d_slot, const int32_t* d_len,
                        int32_t rows, int32_t k, int32_t first, int32_t last, int32_t* d_sel, void* stream) {
  static const char* who = "fi8_kb_select_async";
  if (!kb) return fail(FI8_ERR_ARG, "%s: null handle", who);
  if (rows == 0) return FI8_OK;
  std::lock_guard<std::mutex> lk(kb->mu);
  KbParams p;
  int rc = fill_rows(kb, who, d_q, q_stride, d_slot, d_len, rows, k, d_sel, &p);
  if (rc == FI8_OK) rc = fill_select(who, first, last, &p);
  if (rc != FI8_OK) return rc;
  DeviceGuard g(kb->device);
  FI8_CUDA(kb_select_launch(p, kb->sm_count, static_cast<cudaStream_t>(stream)), "kb_select_launch");
  return FI8_OK;
}

int fi8_kb_attend_async(fi8_kb* kb, const void* d_q, int64_t q_stride, const int32_t* d_slot, const int32_t* d_len,
                        int32_t rows, const int32_t* d_sel, int32_t k, float scale, void* d_out, float* d_lse,
                        void* stream) {
  static const char* who = "fi8_kb_attend_async";
  if (!kb) return fail(FI8_ERR_ARG, "%s: null handle", who);
  if (rows == 0) return FI8_OK;
  std::lock_guard<std::mutex> lk(kb->mu);
  KbParams p;
  int rc = fill_rows(kb, who, d_q, q_stride, d_slot, d_len, rows, k, const_cast<int32_t*>(d_sel), &p);
  if (rc == FI8_OK) rc = fill_attend(who, scale, d_out, d_lse, &p);
  if (rc != FI8_OK) return rc;
  DeviceGuard g(kb->device);
  FI8_CUDA(kb_attend_launch(p, kb->sm_count, static_cast<cudaStream_t>(stream)), "kb_attend_launch");
  return FI8_OK;
}

int fi8_kb_query_async(fi8_kb* kb, const void* d_q, int64_t q_stride, const int32_t* d_slot, const int32_t* d_len,
                       int32_t rows, int32_t k, int32_t first, int32_t last, float scale, int32_t* d_sel, void* d_out,
                       float* d_lse, void* stream) {
  static const char* who = "fi8_kb_query_async";
  if (!kb) return fail(FI8_ERR_ARG, "%s: null handle", who);
  if (rows == 0) return FI8_OK;
  std::lock_guard<std::mutex> lk(kb->mu);
  KbParams p;
  int rc = fill_rows(kb, who, d_q, q_stride, d_slot, d_len, rows, k, d_sel, &p);
  if (rc == FI8_OK) rc = fill_select(who, first, last, &p);
  if (rc == FI8_OK) rc = fill_attend(who, scale, d_out, d_lse, &p);
  if (rc != FI8_OK) return rc;
  DeviceGuard g(kb->device);
  FI8_CUDA(kb_query_launch(p, kb->sm_count, static_cast<cudaStream_t>(stream)), "kb_query_launch");
  return FI8_OK;
}

int fi8_kb_read_rows(fi8_kb* kb, int32_t slot, uint8_t* codes, uint8_t* mults, float* scales) {
  if (!kb || !codes || !mults || !scales) return fail(FI8_ERR_ARG, "fi8_kb_read_rows: null argument");
  const KbParams& p = kb->p;
  if (slot < 0 || slot >= p.slots) return fail(FI8_ERR_ARG, "fi8_kb_read_rows: slot %d of %d", slot, p.slots);
  std::lock_guard<std::mutex> lk(kb->mu);
  DeviceGuard g(kb->device);
  FI8_CUDA(cudaDeviceSynchronize(), "sync");
  const int64_t n = p.max_blocks;
  if (n == 0) return FI8_OK;
  const size_t cb = (size_t)p.groups * 16, mb = p.groups;
  unsigned char* tmp = nullptr;
  FI8_CUDA(cudaMalloc(&tmp, n * (cb + mb + 4)), "fi8_kb_read_rows");
  cudaError_t e = cudaSuccess;
  for (int32_t h = 0; e == cudaSuccess && h < p.kv_heads; h++) {
    uint8_t* d_mults = tmp + n * (cb + 4);
    float* d_scales = reinterpret_cast<float*>(tmp + n * cb);
    e = i4_unpack_launch(kb_rows(p, (int64_t)slot * p.kv_heads + h), 0, n, tmp, d_mults, d_scales, nullptr);
    if (e == cudaSuccess) e = cudaMemcpy(codes + h * n * cb, tmp, n * cb, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemcpy(mults + h * n * mb, d_mults, n * mb, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemcpy(scales + h * n, d_scales, n * 4, cudaMemcpyDeviceToHost);
  }
  cudaFree(tmp);
  if (e != cudaSuccess) return cuda_fail(e, "fi8_kb_read_rows");
  return FI8_OK;
}

int fi8_kb_sync(fi8_kb* kb) {
  if (!kb) return fail(FI8_ERR_ARG, "fi8_kb_sync: null handle");
  std::lock_guard<std::mutex> lk(kb->mu);
  DeviceGuard g(kb->device);
  FI8_CUDA(cudaDeviceSynchronize(), "sync");
  unsigned int err = 0;
  FI8_CUDA(cudaMemcpy(&err, kb->p.err, sizeof(err), cudaMemcpyDeviceToHost), "D2H err");
  if (err == 0) return FI8_OK;
  FI8_CUDA(cudaMemset(kb->p.err, 0, sizeof(unsigned int)), "clear err");
  FI8_CUDA(cudaDeviceSynchronize(), "clear err");  // not behind what a next call on another stream reports
  return fail(FI8_ERR_DEVICE, "fi8_kb: a slot, length or token range lay outside the cache; its row saw nothing");
}

}  // extern "C"
