// fi8_kb.cu -- KeyBlocks kernels: block rows from the cache's keys, the choice
// of blocks by their 4-bit scores, and attention over the chosen blocks.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "fi8_cluster.cuh"
#include "fi8_cp_async.cuh"
#include "fi8_i4q.cuh"
#include "fi8_kb.cuh"
#include "fi8_select.cuh"

namespace fi8 {

namespace {

template <bool F16>
struct Elem;
template <>
struct Elem<false> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Elem<true> {
  using T = __half;
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// A query row's slot and visible length; a row outside the cache is flagged
// and sees nothing.
__device__ __forceinline__ int kb_row(const KbParams& p, int r, int* slot) {
  const int s = __ldg(p.slot + r), n = __ldg(p.len + r);
  if (s < 0 || s >= p.slots || n < 0 || n > p.capacity) {
    if (threadIdx.x == 0) atomicOr(p.err, kKbErrRow);
    *slot = 0;
    return 0;
  }
  *slot = s;
  return n;
}

// ---------------------------------------------------------------------------
// Block rows. The mean of a full block's keys, per channel. The sum is taken
// in 64 bits: the values have at most 11 significant bits, so it is exact in
// any order (f16 always; bf16 unless values of one channel differ by 2^38),
// and the row has one value. Bound by the keys' bytes.
// A CTA per (block, head, entry); a thread holds 8 channels of one token in a
// few.
// ---------------------------------------------------------------------------
constexpr int kUpdateThreads = 256;

template <bool F16>
__global__ void __launch_bounds__(kUpdateThreads) kb_update_kernel(KbParams p, const int32_t* slots, const int32_t* from,
                                                                  const int32_t* to) {
  __shared__ double s_sum[8 * kKbMaxHeadDim];
  __shared__ float s_gmax[kKbMaxHeadDim / kI4Group];
  const int e = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = __ldg(slots + e), a = __ldg(from + e), b = __ldg(to + e);
  if (slot < 0 || slot >= p.slots || a < 0 || b < a || b > p.capacity) {
    if (tid == 0) atomicOr(p.err, kKbErrRow);
    return;
  }
  const int blk = a / p.block + (int)blockIdx.x;
  if (blk >= b / p.block) return;
  const int D = p.head_dim, chunks = D / 8;
  const uint4* base = reinterpret_cast<const uint4*>(
      static_cast<const uint16_t*>(p.k) + (int64_t)slot * p.slot_stride + (int64_t)h * p.head_stride +
      (int64_t)blk * p.block * p.token_stride);
  const int64_t pitch = p.token_stride / 8;  // in 16-byte chunks
  // s_sum [parts][D]: parts token subsets summed by different threads
  const int parts = min(8, kUpdateThreads / chunks);
  if (tid < parts * chunks) {
    const int part = tid / chunks, c = tid % chunks;
    double sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = 0.0;
    for (int t = part; t < p.block; t += parts) {
      const uint4 w = __ldg(base + (int64_t)t * pitch + c);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = Elem<F16>::unpack(u[i]);
        sum[2 * i] += (double)f.x;
        sum[2 * i + 1] += (double)f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) s_sum[part * D + c * 8 + i] = sum[i];
  }
  __syncthreads();
  // a warp per group of 32 channels
  float x = 0.0f;
  const int d = warp * kI4Group + lane;
  if (d < D) {
    double s = 0.0;
    for (int i = 0; i < parts; i++) s += s_sum[i * D + d];
    x = (float)(s / (double)p.block);
  }
  const float gmax = warp_absmax(absmax_step(0.0f, x));
  if (lane == 0) s_gmax[warp] = gmax;
  __syncthreads();
  if (warp >= p.groups) return;
  float rmax = 0.0f;
  for (int g = 0; g < p.groups; g++) rmax = absmax_combine(rmax, s_gmax[g]);
  float up;
  const float scale = i4_row_scale(rmax, &up);
  const int mult = i4_group_mult(gmax, up);
  const int64_t row = ((int64_t)slot * p.kv_heads + h) * p.max_blocks + blk;
  i4_store_group(x, mult, scale, p.codes + (row * p.groups + warp) * 16, lane);
  if (lane == 0) {
    p.mults[row * p.mpitch + warp] = (uint8_t)mult;
    if (warp == 0) p.scales[row] = scale;
  }
}

// ---------------------------------------------------------------------------
// Selection: the score of every visible block (the largest of the head group's
// FlatI4 scores), then the best by (score desc, index asc) with the first and
// last blocks always in: a radix select over the scores' order-preserving
// images, and a compaction in index order.
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 256;
constexpr uint32_t kForced = 0xFFFFFFFFu;  // above every score's image

// The smallest image t among the best `need` of n images, and how many of the
// best have exactly that image. All threads of the CTA call it.
__device__ void kb_threshold(const uint32_t* ord, int n, int need, uint32_t* hist, uint32_t* s_out, uint32_t* t,
                             int* ties) {
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSelectThreads)
      if (shift == 24 || (ord[i] >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(hist + ((ord[i] >> shift) & 255), 1u);
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds bins [255 - 8l - 7, 255 - 8l], counted from the top
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) sum += c[i] = hist[255 - threadIdx.x * 8 - i];
      uint32_t before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
        if ((int)threadIdx.x >= o) before += y;
      }
      before -= sum;
      if (before < (uint32_t)need && before + sum >= (uint32_t)need) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (before < (uint32_t)need && before + c[i] >= (uint32_t)need) {
            s_out[0] = 255 - threadIdx.x * 8 - i;
            s_out[1] = (uint32_t)need - before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= s_out[0] << shift;
    need = (int)s_out[1];
    __syncthreads();
  }
  *t = prefix;
  *ties = need;
}

template <bool F16>
__global__ void __launch_bounds__(kSelectThreads) kb_select_kernel(KbParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_out[2];
  __shared__ int s_gt[8], s_eq[8];
  const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = p.q_heads / p.kv_heads, G = p.groups, D = p.head_dim;
  int slot;
  const int len = kb_row(p, r, &slot);
  const int nb = (len + p.block - 1) / p.block;
  int32_t* sel = p.sel + ((int64_t)r * p.kv_heads + h) * p.select;
  if (nb <= p.select) {  // every visible block
    for (int i = tid; i < p.select; i += kSelectThreads) sel[i] = i < nb ? i : -1;
    return;
  }
  int8_t* q8 = reinterpret_cast<int8_t*>(smem);
  int* off = reinterpret_cast<int*>(q8 + (size_t)heads * G * kI4Group);
  float* qs = reinterpret_cast<float*>(off + heads * G);
  uint32_t* ord = reinterpret_cast<uint32_t*>(qs + heads);
  using T = typename Elem<F16>::T;
  for (int g = warp; g < heads; g += kSelectThreads / 32) {
    const T* q = static_cast<const T*>(p.q) + (int64_t)r * p.q_stride + (int64_t)(h * heads + g) * D;
    const float s = i4_quantize_query([&](int i) { return (float)q[i]; }, D, G, q8 + (size_t)g * G * kI4Group,
                                      off + g * G, lane);
    if (lane == 0) qs[g] = s;
  }
  __syncthreads();
  const int64_t row0 = ((int64_t)slot * p.kv_heads + h) * p.max_blocks;
  for (int b = tid; b < nb; b += kSelectThreads) {
    uint32_t best = 0;
    if (b < p.first || b >= nb - p.last) {
      best = kForced;
    } else {
      const uint4* codes = reinterpret_cast<const uint4*>(p.codes + (row0 + b) * G * 16);
      const uint8_t* mults = p.mults + (row0 + b) * p.mpitch;
      const float scale = __ldg(p.scales + row0 + b);
      for (int g = 0; g < heads; g++) {
        int dot = 0;
        for (int c = 0; c < G; c++) {
          const int4* qg = reinterpret_cast<const int4*>(q8 + ((size_t)g * G + c) * kI4Group);
          dot += (int)__ldg(mults + c) * i4_dot_group(__ldg(codes + c), qg[0], qg[1], off[g * G + c]);
        }
        const float s = w8a8_score(dot, qs[g], scale);
        if (s == s) best = max(best, score_to_ord(s));  // a NaN ranks below every score
      }
    }
    ord[b] = best;
  }
  __syncthreads();
  uint32_t t;
  int ties;
  kb_threshold(ord, nb, p.select, s_hist, s_out, &t, &ties);
  // each warp compacts a segment: counts first, then places
  const int seg = (nb + 255) / 256 * 32, b0 = min(nb, warp * seg), b1 = min(nb, b0 + seg);
  int gt = 0, eq = 0;
  for (int b = b0 + lane; b < b1; b += 32) {
    gt += ord[b] > t;
    eq += ord[b] == t;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < warp; w++) {
    gt += s_gt[w];
    eq += s_eq[w];
  }
  for (int base = b0; base < b1; base += 32) {
    const int b = base + lane;
    const uint32_t o = b < b1 ? ord[b] : 0;
    const bool is_gt = b < b1 && o > t, is_eq = b < b1 && o == t;
    const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt), meq = __ballot_sync(0xffffffffu, is_eq);
    const int my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
    if (is_gt || (is_eq && my_eq < ties)) sel[my_gt + min(my_eq, ties)] = b;
    gt += __popc(mgt);
    eq += __popc(meq);
  }
}

// ---------------------------------------------------------------------------
// Attention over the chosen blocks. One pass over the keys and values with the
// running maximum and sum of the softmax (in the log2 domain). The query heads
// that share a key/value head are the rows of one 16-row matrix product, so
// each key and value is read once for all of them; bound by those bytes.
// A cluster of CTAs per (query row, kv head, tile of 16 query heads); the
// selected blocks are dealt in pieces of 16 tokens to the cluster's warps, and
// each warp runs its own ring of asynchronous copies and its own softmax, so
// nothing but the end synchronizes. The warps' partial results are joined in
// shared memory, the CTAs' through the cluster's.
// ---------------------------------------------------------------------------
constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kPiece = 16;

// Shared memory of a head dimension up to DP.
template <int DP>
struct AttendSmem {
  static constexpr int kStages = DP == 64 ? 4 : DP == 128 ? 3 : 2;
  static constexpr size_t kStage = (size_t)2 * kPiece * DP * 2;  // a warp's stage: 16 keys, then 16 values
  static constexpr size_t kRing = kAttendWarps * kStages * kStage;
  // after the ring: the query tile, then the joined result (16 x DP f32) and its maxima and sums
  static constexpr size_t kBytes = kRing + 16 * DP * 2 + 16 * DP * 4 + 2 * 16 * 4;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kRing >= (size_t)kAttendWarps * 16 * (DP + 2) * 4, "the warps' partial results fit the ring");
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Byte offset of 16-byte chunk c of row r in a tile of DP-element rows; the
// chunk index is permuted by the row so that eight rows' equal chunks fall
// into different banks.
template <int DP>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * (DP * 2) + ((c ^ (r & 7)) << 4));
}

template <int DP, bool F16>
__global__ void __launch_bounds__(kAttendThreads) kb_attend_kernel(KbParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  constexpr int NS = AttendSmem<DP>::kStages;
  constexpr int kChunks = DP / 8;       // 16-byte chunks of a padded row
  constexpr int kSteps = DP / 16;
  constexpr bool kQInRegs = DP <= 128;  // else the query fragments are read again for each piece
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), nsplit = cluster_size();
  const int r = blockIdx.x / nsplit;
  const int heads = p.q_heads / p.kv_heads, mtiles = (heads + 15) / 16;
  const int h = blockIdx.y / mtiles, m0 = (blockIdx.y % mtiles) * 16;
  const int mrows = min(16, heads - m0);
  const int D = p.head_dim, chunks = D / 8, steps = D / 16;
  int slot;
  const int len = kb_row(p, r, &slot);
  const int nb = (len + p.block - 1) / p.block;
  const int32_t* sel = p.sel + ((int64_t)r * p.kv_heads + h) * p.select;

  unsigned char* s_q = smem + AttendSmem<DP>::kRing;
  float* s_o = reinterpret_cast<float*>(s_q + 16 * DP * 2);
  float* s_m = s_o + 16 * DP;
  float* s_l = s_m + 16;

  // the query tile: absent heads are zero rows
  const T* q = static_cast<const T*>(p.q) + (int64_t)r * p.q_stride + (int64_t)(h * heads + m0) * D;
  for (int i = tid; i < 16 * kChunks; i += kAttendThreads) {
    const int row = i / kChunks, c = i % kChunks;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < mrows && c < chunks) w = __ldg(reinterpret_cast<const uint4*>(q + (int64_t)row * D) + c);
    *reinterpret_cast<uint4*>(s_q + tile_at<DP>(row, c)) = w;
  }
  __syncthreads();
  const uint32_t q_base = smem_u32(s_q);
  // ldmatrix lane addresses: rows 0-7 / 8-15 by lane bit 3, chunk +1 by bit 4
  const int a_row = (lane & 7) + (lane & 8), a_chunk = lane >> 4;
  // keys: rows by lane bit 4, chunk by bit 3
  const int b_row = (lane & 7) + ((lane & 16) >> 1), b_chunk = (lane >> 3) & 1;
  uint32_t qf[kQInRegs ? kSteps : 1][4];
  if (kQInRegs) {
#pragma unroll
    for (int s = 0; s < kSteps; s++)
      if (s < steps) ldmatrix4(qf[s], q_base + tile_at<DP>(a_row, 2 * s + a_chunk));
  }

  const int per_block = p.block / kPiece, pieces = p.select * per_block;
  const int stride = (int)nsplit * kAttendWarps;
  const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + (int64_t)slot * p.slot_stride +
                                                    (int64_t)h * p.head_stride);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + (int64_t)slot * p.slot_stride +
                                                    (int64_t)h * p.head_stride);
  const int64_t pitch = p.token_stride * 2;
  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * NS * AttendSmem<DP>::kStage);

  // tokens of piece i that the row sees (0: the piece is skipped), from token *t0
  auto visible = [&](int i, int* t0) {
    if (i >= pieces) return 0;
    const int b = __ldg(sel + i / per_block);
    if (b < 0 || b >= nb) return 0;
    *t0 = b * p.block + (i % per_block) * kPiece;
    return max(0, min(kPiece, len - *t0));
  };
  auto load = [&](int i, int stage) {
    int t0 = 0;
    const int n = visible(i, &t0);
    if (n > 0) {
      const uint32_t dst = ring + (uint32_t)(stage * AttendSmem<DP>::kStage);
      for (int j = lane; j < kPiece * kChunks; j += 32) {
        const int row = j / kChunks, c = j % kChunks;
        if (c >= chunks) continue;
        const bool ok = row < n;  // hidden tokens are zeros: 0 * their weight 0 stays 0
        const int64_t at = (int64_t)(t0 + (ok ? row : 0)) * pitch + c * 16;
        cp_async16(dst + tile_at<DP>(row, c), kbase + at, ok);
        cp_async16(dst + kPiece * DP * 2 + tile_at<DP>(row, c), vbase + at, ok);
      }
    }
    cp_async_commit();
    return n;
  };

  float o[kSteps * 2][4];
#pragma unroll
  for (int i = 0; i < kSteps * 2; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  const float c2 = p.scale * 1.4426950408889634f;  // log2(e)

  int i = (int)rank * kAttendWarps + warp;
  int have[NS];
#pragma unroll
  for (int s = 0; s < NS; s++) have[s] = 0;
#pragma unroll
  for (int s = 0; s < NS - 1; s++) have[s] = load(i + s * stride, s);
  for (; i < pieces; i += NS * stride) {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int at = i + s * stride;
      if (at >= pieces) break;
      have[(s + NS - 1) % NS] = load(at + (NS - 1) * stride, (s + NS - 1) % NS);
      cp_async_wait<NS - 1>();
      __syncwarp();
      const int n = have[s];
      if (n > 0) {
        const uint32_t kt = ring + (uint32_t)(s * AttendSmem<DP>::kStage), vt = kt + kPiece * DP * 2;
        float sc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int t = 0; t < kSteps; t++) {
          if (t >= steps) break;
          uint32_t kf[4];
          ldmatrix4(kf, kt + tile_at<DP>(b_row, 2 * t + b_chunk));
          if (kQInRegs) {
            E::mma(sc[0], qf[kQInRegs ? t : 0], kf[0], kf[1]);
            E::mma(sc[1], qf[kQInRegs ? t : 0], kf[2], kf[3]);
          } else {
            uint32_t a[4];
            ldmatrix4(a, q_base + tile_at<DP>(a_row, 2 * t + a_chunk));
            E::mma(sc[0], a, kf[0], kf[1]);
            E::mma(sc[1], a, kf[2], kf[3]);
          }
        }
        // hidden tokens out, then the maximum of the four lanes that share a row
        float pm[2] = {mx[0], mx[1]};
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int token = j * 8 + (lane & 3) * 2 + (e & 1);
            sc[j][e] = token < n ? sc[j][e] * c2 : -INFINITY;
            pm[e >> 1] = fmaxf(pm[e >> 1], sc[j][e]);
          }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          pm[e] = fmaxf(pm[e], __shfl_xor_sync(0xffffffffu, pm[e], 1));
          pm[e] = fmaxf(pm[e], __shfl_xor_sync(0xffffffffu, pm[e], 2));
        }
        if (__any_sync(0xffffffffu, pm[0] != mx[0] || pm[1] != mx[1])) {
          const float f0 = pm[0] == mx[0] ? 1.0f : exp2_fast(mx[0] - pm[0]);
          const float f1 = pm[1] == mx[1] ? 1.0f : exp2_fast(mx[1] - pm[1]);
#pragma unroll
          for (int t = 0; t < kSteps * 2; t++) {
            o[t][0] *= f0, o[t][1] *= f0;
            o[t][2] *= f1, o[t][3] *= f1;
          }
          sum[0] *= f0, sum[1] *= f1;
          mx[0] = pm[0], mx[1] = pm[1];
        }
        // a row that has seen nothing but -inf keeps weights of 0
        const float base0 = mx[0] == -INFINITY ? 0.0f : mx[0], base1 = mx[1] == -INFINITY ? 0.0f : mx[1];
        uint32_t pf[4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const float p0 = exp2_fast(sc[j][0] - base0), p1 = exp2_fast(sc[j][1] - base0);
          const float p2 = exp2_fast(sc[j][2] - base1), p3 = exp2_fast(sc[j][3] - base1);
          sum[0] += p0 + p1;
          sum[1] += p2 + p3;
          // the weights enter the product in the cache's type (a relative 2^-9 or 2^-12 each; the sums stay 32 bits)
          pf[2 * j] = E::pack(p0, p1);
          pf[2 * j + 1] = E::pack(p2, p3);
        }
#pragma unroll
        for (int t = 0; t < kSteps; t++) {
          if (t >= steps) break;
          uint32_t vf[4];
          ldmatrix4_trans(vf, vt + tile_at<DP>(a_row, 2 * t + a_chunk));
          E::mma(o[2 * t], pf, vf[0], vf[1]);
          E::mma(o[2 * t + 1], pf, vf[2], vf[3]);
        }
      }
      __syncwarp();  // the stage may be filled again
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
    sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
  }
  __syncthreads();  // every warp is done with the ring: it holds the warps' partial results now

  float* w_o = reinterpret_cast<float*>(smem);             // [warps][16][DP]
  float* w_m = w_o + (size_t)kAttendWarps * 16 * DP;       // [warps][16]
  float* w_l = w_m + kAttendWarps * 16;
  {
    const int row = lane >> 2, col = (lane & 3) * 2;
    float* mine = w_o + (size_t)warp * 16 * DP;
#pragma unroll
    for (int t = 0; t < kSteps * 2; t++) {
      if (t * 8 >= D) break;
      *reinterpret_cast<float2*>(mine + row * DP + t * 8 + col) = make_float2(o[t][0], o[t][1]);
      *reinterpret_cast<float2*>(mine + (row + 8) * DP + t * 8 + col) = make_float2(o[t][2], o[t][3]);
    }
    if ((lane & 3) == 0) {
      w_m[warp * 16 + row] = mx[0], w_m[warp * 16 + row + 8] = mx[1];
      w_l[warp * 16 + row] = sum[0], w_l[warp * 16 + row + 8] = sum[1];
    }
  }
  __syncthreads();
  for (int j = tid; j < mrows * D; j += kAttendThreads) {
    const int row = j / D, d = j % D;
    float m = w_m[row];
#pragma unroll
    for (int w = 1; w < kAttendWarps; w++) m = fmaxf(m, w_m[w * 16 + row]);
    const float base = m == -INFINITY ? 0.0f : m;
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttendWarps; w++) {
      const float f = exp2_fast(w_m[w * 16 + row] - base);
      acc += f * w_o[((size_t)w * 16 + row) * DP + d];
      l += f * w_l[w * 16 + row];
    }
    s_o[row * DP + d] = acc;
    if (d == 0) {
      s_m[row] = m;
      s_l[row] = l;
    }
  }
  __syncthreads();
  if (nsplit > 1) cluster_sync();
  // the cluster's CTAs share out the joined tile
  T* out = static_cast<T*>(p.out) + ((int64_t)r * p.q_heads + h * heads + m0) * D;
  float* lse = p.lse ? p.lse + (int64_t)r * p.q_heads + h * heads + m0 : nullptr;
  const uint32_t o_at = smem_u32(s_o), m_at = smem_u32(s_m), l_at = smem_u32(s_l);
  for (int j = (int)rank * kAttendThreads + tid; j < mrows * D; j += (int)nsplit * kAttendThreads) {
    const int row = j / D, d = j % D;
    float m = -INFINITY, acc = 0.0f, l = 0.0f;
    for (uint32_t c = 0; c < nsplit; c++) m = fmaxf(m, ld_cluster(m_at + row * 4, c));
    const float base = m == -INFINITY ? 0.0f : m;
    for (uint32_t c = 0; c < nsplit; c++) {
      const float f = exp2_fast(ld_cluster(m_at + row * 4, c) - base);
      acc += f * ld_cluster(o_at + (row * DP + d) * 4, c);
      l += f * ld_cluster(l_at + row * 4, c);
    }
    out[(int64_t)row * D + d] = T(l > 0.0f || l != l ? acc / l : 0.0f);
    if (lse && d == 0) lse[row] = l > 0.0f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
  if (nsplit > 1) cluster_sync();  // the others' shared memory is read until here
}

template <int DP, bool F16>
cudaError_t attend_launch(const KbParams& p, int32_t splits, cudaStream_t stream) {
  auto fn = kb_attend_kernel<DP, F16>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AttendSmem<DP>::kBytes);
  if (e != cudaSuccess) return e;
  const int heads = p.q_heads / p.kv_heads, mtiles = (heads + 15) / 16;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * splits), (unsigned)(p.kv_heads * mtiles));
  cfg.blockDim = dim3(kAttendThreads);
  cfg.dynamicSmemBytes = AttendSmem<DP>::kBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace

cudaError_t kb_update_launch(const KbParams& p, const int32_t* slot, const int32_t* from, const int32_t* to,
                             int32_t count, int32_t max_tokens, cudaStream_t stream) {
  const int64_t most = (int64_t)max_tokens / p.block + 1;  // blocks that a range of max_tokens can complete
  const dim3 grid((unsigned)(most < p.max_blocks ? most : p.max_blocks), (unsigned)p.kv_heads, (unsigned)count);
  if (grid.x == 0) return cudaSuccess;
  if (p.f16) kb_update_kernel<true><<<grid, kUpdateThreads, 0, stream>>>(p, slot, from, to);
  else kb_update_kernel<false><<<grid, kUpdateThreads, 0, stream>>>(p, slot, from, to);
  return cudaGetLastError();
}

cudaError_t kb_select_launch(const KbParams& p, cudaStream_t stream) {
  const int heads = p.q_heads / p.kv_heads;
  const int64_t blocks = (p.capacity + p.block - 1) / p.block;
  const size_t smem = (size_t)heads * (p.groups * (kI4Group + 4) + 4) + (size_t)blocks * 4;
  auto fn = p.f16 ? kb_select_kernel<true> : kb_select_kernel<false>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  fn<<<dim3((unsigned)p.rows, (unsigned)p.kv_heads), kSelectThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t kb_attend_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream) {
  // Splits of a (row, kv head): enough CTAs for two an SM, at least two pieces
  // a warp, eight at most (the portable cluster size).
  const int heads = p.q_heads / p.kv_heads, mtiles = (heads + 15) / 16;
  const int64_t units = (int64_t)p.rows * p.kv_heads * mtiles;
  const int64_t pieces = (int64_t)p.select * (p.block / kPiece);
  int32_t splits = 1;
  while (splits < 8 && units * splits < 2 * (int64_t)sm_count && pieces >= (int64_t)splits * 2 * kAttendWarps * 2) splits *= 2;
  const int d = p.head_dim;
  if (p.f16) return d <= 64 ? attend_launch<64, true>(p, splits, stream)
                  : d <= 128 ? attend_launch<128, true>(p, splits, stream) : attend_launch<256, true>(p, splits, stream);
  return d <= 64 ? attend_launch<64, false>(p, splits, stream)
         : d <= 128 ? attend_launch<128, false>(p, splits, stream) : attend_launch<256, false>(p, splits, stream);
}

}  // namespace fi8
