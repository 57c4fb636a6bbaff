// fi8_i4.cu -- FlatI4: scores of 4-bit rows (a matrix-vector product with
// group scales), the row quantizer, and the exact top-k of a score row.
#include "fi8_i4.cuh"
#include "fi8_i4q.cuh"
#include "fi8_select.cuh"

namespace fi8 {

namespace {

constexpr int kWarps = 8;

// A warp per row: two passes over its groups, the second one from cache.
__global__ void __launch_bounds__(kWarps * 32) i4_quantize_kernel(I4Rows r, int64_t row0, const float* v, int64_t rows) {
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (i >= rows) return;
  const float* row = v + (size_t)i * r.dim;
  uint8_t* codes = r.codes + (size_t)(row0 + i) * r.groups * 16;
  uint8_t* mults = r.mults + (size_t)(row0 + i) * r.mpitch;
  float m = 0.0f;
  for (int j = lane; j < r.dim; j += 32) m = absmax_step(m, row[j]);
  m = warp_absmax(m);
  float up;
  const float scale = i4_row_scale(m, &up);
  for (int g = 0; g < r.groups; g++) {
    const int j = g * kI4Group + lane;
    const float x = j < r.dim ? row[j] : 0.0f;
    const int mult = i4_group_mult(warp_absmax(absmax_step(0.0f, x)), up);
    i4_store_group(x, mult, scale, codes + g * 16, lane);
    if (lane == 0) mults[g] = (uint8_t)mult;
  }
  if (lane < r.mpitch - r.groups) mults[r.groups + lane] = 0;
  if (lane == 0) r.scales[row0 + i] = scale;
}

// An 8-lane quarter-warp per row, a lane per group of 32 values. Bound by the
// rows' bytes.
template <int M>
__global__ void __launch_bounds__(kWarps * 32) i4_score_kernel(I4Rows r, int64_t row0, int64_t rows, const float* q,
                                                               float* dst, int64_t ld) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_scale[M];
  const int G = r.groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int8_t* q8 = reinterpret_cast<int8_t*>(smem);
  int* off = reinterpret_cast<int*>(smem + (size_t)M * G * kI4Group);
  if (warp < M) {
    const float* qm = q + (size_t)warp * r.dim;
    const float s = i4_quantize_query([&](int i) { return __ldg(qm + i); }, r.dim, G,
                                      q8 + (size_t)warp * G * kI4Group, off + warp * G, lane);
    if (lane == 0) s_scale[warp] = s;
  }
  __syncthreads();
  const int lane8 = lane & 7;
  const int64_t step = (int64_t)gridDim.x * kWarps * 4;
  for (int64_t base = ((int64_t)blockIdx.x * kWarps + warp) * 4; base < rows; base += step) {
    const int64_t i = base + (lane >> 3);
    const int64_t row = row0 + (i < rows ? i : rows - 1);
    const uint4* codes = reinterpret_cast<const uint4*>(r.codes + (size_t)row * G * 16);
    const uint8_t* mults = r.mults + (size_t)row * r.mpitch;
    int tot[M];
#pragma unroll
    for (int m = 0; m < M; m++) tot[m] = 0;
    for (int g = lane8; g < G; g += 8) {
      const uint4 w = __ldg(codes + g);
      const int mult = __ldg(mults + g);
#pragma unroll
      for (int m = 0; m < M; m++) {
        const int4* qg = reinterpret_cast<const int4*>(q8 + ((size_t)m * G + g) * kI4Group);
        tot[m] += mult * i4_dot_group(w, qg[0], qg[1], off[m * G + g]);
      }
    }
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) tot[m] += __shfl_xor_sync(0xffffffffu, tot[m], o);
    if (i < rows) {
#pragma unroll
      for (int m = 0; m < M; m++)
        if (lane8 == m) dst[(size_t)m * ld + i] = w8a8_score(tot[m], s_scale[m], r.scales[row]);
    }
  }
}

// Exact top-k of score rows. A CTA takes a contiguous part of a query's scores
// and keeps candidates above a threshold in shared memory; a full buffer is
// sorted and cut to the best k, which raises the threshold of every CTA of the
// query. Each threshold is the k-th best key of k real rows, so nothing of the
// top k is lost. The last CTA of a block of CTAs merges its lists, the last
// block merges the blocks' (tickets, returned to zero).
__global__ void __launch_bounds__(kGroupThreads) i4_select_kernel(I4Select p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_count;
  __shared__ unsigned long long s_local, s_thr;
  __shared__ int s_last;
  uint64_t* buf = reinterpret_cast<uint64_t*>(smem);
  const int tid = threadIdx.x, y = blockIdx.y, cta = blockIdx.x;
  const float* scores = p.scores + (size_t)y * p.ld;
  const int64_t tiles = (p.rows + kI4SelectTile - 1) / kI4SelectTile;
  const int64_t t0 = tiles * cta / p.ctas, t1 = tiles * (cta + 1) / p.ctas;
  if (tid == 0) {
    s_count = 0;
    s_local = 0;
  }
  for (int64_t t = t0; t < t1; t++) {
    if (tid == 0) s_thr = max(s_local, ld_relaxed_u64(p.gthr + y));
    __syncthreads();
    const unsigned long long thr = s_thr;
    const int64_t at = t * kI4SelectTile + tid * 4;
    float f[4];
    if (at < p.rows) {  // ld is a multiple of 4: a started four lies in the row's allocation
      const float4 v = __ldcg(reinterpret_cast<const float4*>(scores + at));
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      bool take = at + e < p.rows;
      uint64_t key = kEmptyKey;
      if (take) {
        const uint32_t id = p.id0 + (uint32_t)(at + e);
        key = make_key(f[e], id);
        take = f[e] == f[e] && key > thr && (!p.keep || keep_bit(p.keep, p.keep_nbits, id));
      }
      warp_append(take, key, buf, &s_count);
    }
    __syncthreads();
    const int cnt = s_count;
    if (cnt > p.cap - kI4SelectTile) group_compact(buf, cnt, p.k, &s_count, &s_local, p.gthr + y, tid, 1);
  }
  __syncthreads();
  group_compact(buf, s_count, p.k, &s_count, &s_local, p.gthr + y, tid, 1);
  const int kp = p.kp;
  for (int i = s_count + tid; i < kp; i += kGroupThreads) buf[i] = kEmptyKey;
  __syncthreads();
  const int nb = (p.ctas + 7) / 8, blk = cta / 8, members = min(8, p.ctas - blk * 8);
  uint64_t* mine = p.lvl1 + ((size_t)y * p.ctas + cta) * kp;
  for (int i = tid; i < kp; i += kGroupThreads) mine[i] = buf[i];
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.counter + (size_t)y * nb + blk, 1u) == (unsigned)(members - 1);
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  merge_global_lists(p.lvl1 + ((size_t)y * p.ctas + (size_t)blk * 8) * kp, members, kp, kp, kp, buf, p.nslots, tid, 1);
  uint64_t* list = p.lvl2 + ((size_t)y * nb + blk) * kp;
  for (int i = tid; i < kp; i += kGroupThreads) list[i] = buf[i];
  if (tid == 0) p.counter[(size_t)y * nb + blk] = 0u;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.counter2 + y, 1u) == (unsigned)(nb - 1);
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  merge_global_lists(p.lvl2 + (size_t)y * nb * kp, nb, kp, kp, kp, buf, p.nslots, tid, 1);
  for (int i = tid; i < p.k; i += kGroupThreads) p.out[(size_t)y * p.k + i] = buf[i];
  if (tid == 0) {
    p.counter2[y] = 0u;
    p.gthr[y] = 0ull;
  }
}

template <int M>
cudaError_t score_launch(const I4Rows& r, int64_t row0, int64_t rows, const float* q, float* dst, int64_t ld,
                         int32_t sm_count, cudaStream_t stream) {
  const size_t smem = (size_t)M * r.groups * (kI4Group + 4);
  cudaError_t e = cudaFuncSetAttribute(i4_score_kernel<M>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int64_t need = (rows + kWarps * 4 - 1) / (kWarps * 4);
  const unsigned grid = (unsigned)(need < (int64_t)sm_count * 4 ? need : (int64_t)sm_count * 4);
  i4_score_kernel<M><<<grid, kWarps * 32, smem, stream>>>(r, row0, rows, q, dst, ld);
  return cudaGetLastError();
}

}  // namespace

cudaError_t i4_quantize_launch(const I4Rows& r, int64_t row0, const float* v, int64_t rows, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  i4_quantize_kernel<<<(unsigned)((rows + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(r, row0, v, rows);
  return cudaGetLastError();
}

cudaError_t i4_score_launch(const I4Rows& r, int64_t row0, int64_t rows, const float* q, int32_t M, float* dst,
                            int64_t ld, int32_t sm_count, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  switch (M) {
    case 1: return score_launch<1>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 2: return score_launch<2>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 3: return score_launch<3>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 4: return score_launch<4>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 5: return score_launch<5>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 6: return score_launch<6>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 7: return score_launch<7>(r, row0, rows, q, dst, ld, sm_count, stream);
    case 8: return score_launch<8>(r, row0, rows, q, dst, ld, sm_count, stream);
    default: return cudaErrorInvalidValue;
  }
}

size_t i4_select_plan(I4Select* s, int32_t M) {
  int32_t kp = 1, cap = 1;
  while (kp < s->k) kp <<= 1;
  while (cap < s->k + kI4SelectTile) cap <<= 1;  // k survivors and a tile of new candidates
  if (cap < 2 * kp) cap = 2 * kp;                // the merges need two lists
  const int64_t tiles = (s->rows + kI4SelectTile - 1) / kI4SelectTile;
  const int32_t most = kI4SelectCtas / M;
  s->kp = kp;
  s->cap = cap;
  s->nslots = cap / kp;
  s->ctas = (int32_t)(tiles < most ? tiles : most);
  return (size_t)cap * sizeof(uint64_t);
}

cudaError_t i4_select_launch(const I4Select& s, int32_t M, size_t smem, cudaStream_t stream) {
  i4_select_kernel<<<dim3((unsigned)s.ctas, (unsigned)M), kGroupThreads, smem, stream>>>(s);
  return cudaGetLastError();
}

}  // namespace fi8
