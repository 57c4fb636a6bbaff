// fi8_kb.cu -- KeyBlocks kernels: block rows from the cache's keys, the choice
// of blocks by their 4-bit scores, and attention over the chosen blocks.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "fi8_cluster.cuh"
#include "fi8_cp_async.cuh"
#include "fi8_i4q.cuh"
#include "fi8_kb.cuh"
#include "fi8_kth.cuh"
#include "fi8_select.cuh"

namespace fi8 {

namespace {

// kLift: what a softmax weight is multiplied by before it is rounded to the type.
template <bool F16>
struct Elem;
template <>
struct Elem<false> {
  using T = __nv_bfloat16;
  static constexpr float kLift = 1.0f;
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
  static constexpr float kLift = 32768.0f;
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
__device__ __forceinline__ int kb_row_at(const KbParams& p, int r, int* slot) {
  const int s = __ldg(p.slot + r), n = __ldg(p.len + r);
  if (s < 0 || s >= p.slots || n < 0 || n > p.capacity) {
    atomicOr(p.err, kKbErrRow);
    *slot = 0;
    return 0;
  }
  *slot = s;
  return n;
}

// w8a8_score where a NaN's bits do not matter.
__device__ __forceinline__ float kb_score(int dot, float qscale, float rowscale) {
  const float s = __fmul_rn(__fmul_rn(__int2float_rn(dot), qscale), rowscale);
  return qscale == 0.0f ? 0.0f : s;
}

// ---------------------------------------------------------------------------
// Block rows. The mean of a full block's keys, per channel. The sum is taken
// in 64 bits: the values have at most 11 significant bits, so it is exact in
// any order and the row has one value (f16 always; bf16 unless values of one
// channel differ by 2^38: such sums are rounded to 53 bits, in an order that
// head_dim alone decides). A CTA per (block, head, entry); a thread adds 8
// channels of one token in a few. 17 us for the 256 new blocks of a 16,384-token
// prompt, 8 heads of 128 (33 MB, 2 TB/s): bound by the latency of a CTA's few
// loads and barriers, beside the keys' bytes.
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
  const I4Rows r = kb_rows(p, (int64_t)slot * p.kv_heads + h);
  const int tile = blk / kI4Tile, in_tile = blk % kI4Tile, quads = (p.groups + 3) / 4;
  uint32_t* codes = r.codes + (size_t)tile * p.groups * 128;
  i4_store_group(x, mult, scale, lane, [&](int t, uint32_t w) { codes[i4_word_at(warp, in_tile, t, p.groups)] = w; });
  if (lane == 0) {
    reinterpret_cast<uint8_t*>(r.mults + ((size_t)tile * quads + (warp >> 2)) * 32 + in_tile)[warp & 3] = (uint8_t)mult;
    if (warp == 0) r.scales[blk] = scale;
  }
}

// ---------------------------------------------------------------------------
// Selection: the rank of every visible block (the largest of the head group's
// FlatI4 scores), then the best by (score desc, index asc) with the first and
// last blocks always in.
// The query vectors of a head group, eight or more columns, are the right operand
// of the score kernel's matrix product, 32 block rows the left one. The ranks lie
// in shared memory. There are two kernels. In one a CTA has one query row; with
// very many blocks a cluster scores them and its rank 0 picks. In the other a
// CTA has several rows, and those that share a slot, a prompt's chunk, read its
// block rows once; there a warp picks a row's blocks from registers, up to 1023.
// Bound by the latency of dependent steps (loads, quantization, products, picks):
// 3.2 us for one row over 64 blocks a head, 6.1 us for sixteen over up to 512,
// 11.4 us for two over up to 7,813; 83 us for 2,048 rows over 256 (there by the
// instructions of the warps' picks and of the ranks' updates).
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kWarpPicks = 1024;  // a warp picks from fewer blocks

// One row's picks by a warp: ranks ord[0 .. n) of the inner blocks, n <= 32 E
// and below 1024; `need` of them, behind `first` and before `last` blocks that are
// always in. As kth_rank does, with the ranks in registers: 256 bins of equal
// spans of the scores (hist), then the ranks of the bin that holds the need-th
// one, found from the top bit down, two bits a step, by three counts of at most
// 1023 in one word.
template <int E>
__device__ void kb_warp_picks(const uint32_t* ord, int n, int need, int first, int last, int32_t* sel, uint32_t* hist) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < first; i += 32) sel[i] = i;
  for (int i = lane; i < last; i += 32) sel[first + need + i] = first + n + i;
  if (need == 0) return;
  uint32_t v[E], top = 0, low = 0xFFFFFFFFu;
  for (int i = lane; i < 256; i += 32) hist[i] = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int i = e * 32 + lane;
    v[e] = i < n ? ord[i] : 0u;  // past n: 0, which no count below takes in
    top = max(top, v[e]);
    low = min(low, v[e] - 1u);  // the smallest score that is one
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  __syncwarp();
  const ScoreBins bins(ord_to_score(low + 1u), ord_to_score(top), 256);
#pragma unroll
  for (int e = 0; e < E; e++)
    if (e * 32 + lane < n) atomicAdd(hist + bins(v[e]), 1u);
  __syncwarp();
  uint32_t c8[8], mine = 0;  // the highest first
  const uint4* at = reinterpret_cast<const uint4*>(hist + 248 - lane * 8);
  const uint4 lo = at[0], hi = at[1];
  c8[0] = hi.w, c8[1] = hi.z, c8[2] = hi.y, c8[3] = hi.x, c8[4] = lo.w, c8[5] = lo.z, c8[6] = lo.y, c8[7] = lo.x;
#pragma unroll
  for (int i = 0; i < 8; i++) mine += c8[i];
  uint32_t before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  before -= mine;
  const bool here = before < (uint32_t)need && before + mine >= (uint32_t)need;
  uint32_t bin = 0, count = 0;
  if (here) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (!found) {
        bin = (uint32_t)(255 - lane * 8 - i);
        count = before + c8[i];
        found = count >= (uint32_t)need;
        if (!found) before = count;
      }
    }
  }
  const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  bin = __shfl_sync(0xffffffffu, bin, from);
  count = __shfl_sync(0xffffffffu, count, from);               // ranks in that bin or above
  uint32_t above = __shfl_sync(0xffffffffu, before, from);
  // the bin's ranks stay, those above it become the largest, the others 0
  uint32_t in_top = 0, in_low = 0xFFFFFFFFu;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int b = e * 32 + lane < n ? bins(v[e]) : -1;
    if (b == (int)bin) in_top = max(in_top, v[e]), in_low = min(in_low, v[e]);
    else v[e] = b > (int)bin ? 0xFFFFFFFFu : 0u;
  }
  in_top = __reduce_max_sync(0xffffffffu, in_top);
  in_low = __reduce_min_sync(0xffffffffu, in_low);
  uint32_t t = in_low, ties = 0xFFFFFFFFu;
  if (count != (uint32_t)need) {
    int bits = 32 - __clz(in_top ^ in_low);
    t = bits == 32 ? 0u : in_top >> bits << bits;
    while (bits > 0 && count > (uint32_t)need) {
      bits = max(0, bits - 2);  // an odd last bit: t + 2 and t + 3 count the ranks known to be above
      const uint32_t t1 = t + (1u << bits), t2 = t + (2u << bits), t3 = t + (3u << bits);
      uint32_t c = 0;
#pragma unroll
      for (int e = 0; e < E; e++) c += (v[e] >= t1 ? 1u : 0u) + (v[e] >= t2 ? 1u << 10 : 0u) + (v[e] >= t3 ? 1u << 20 : 0u);
      c = __reduce_add_sync(0xffffffffu, c);
      const uint32_t c1 = c & 1023u, c2 = (c >> 10) & 1023u, c3 = c >> 20;
      if (c3 >= (uint32_t)need) t = t3, count = c3;
      else if (c2 >= (uint32_t)need) t = t2, count = c2, above = c3;
      else if (c1 >= (uint32_t)need) t = t1, count = c1, above = c2;
      else above = c1;
    }
    // of the ranks equal to t the first, when they are too many
    if (count != (uint32_t)need) ties = (uint32_t)need - above;
  }
  uint32_t gt = 0, eq = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int i = e * 32 + lane;
    const bool is_gt = i < n && v[e] > t, is_eq = i < n && v[e] == t;
    const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt), meq = __ballot_sync(0xffffffffu, is_eq);
    const uint32_t my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
    if (is_gt || (is_eq && my_eq < ties)) sel[first + my_gt + min(my_eq, ties)] = first + i;
    gt += __popc(mgt);
    eq += __popc(meq);
  }
}

// One row's picks of a short list, n at most the CTA's threads: a rank's place
// is the number of larger ones, and of equal ones before it. No search, one
// barrier. ord is 16-byte aligned and 0 from n to a multiple of 32. (Eight wide
// loads at a time: rolled loops over single ranks took four times as long.)
// pick(place, i) takes the picks.
template <typename Pick>
__device__ __forceinline__ void kb_count_picks(const uint32_t* ord, int n, int need, uint32_t* part, Pick pick) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t place = 0;
  if (warp * 32 < n) {
    const uint32_t mine = ord[tid];
#pragma unroll 1
    for (int b = 0; b * 32 < n; b++) {
      uint4 v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const uint4*>(ord + b * 32)[j];
      if (b == warp) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          place += (v[j].x >= mine + (4 * j >= lane)) + (v[j].y >= mine + (4 * j + 1 >= lane)) + (v[j].z >= mine + (4 * j + 2 >= lane)) +
                   (v[j].w >= mine + (4 * j + 3 >= lane));
      } else {
        const uint32_t least = mine + (b > warp);  // a rank is never the largest 32-bit number
#pragma unroll
        for (int j = 0; j < 8; j++) place += (v[j].x >= least) + (v[j].y >= least) + (v[j].z >= least) + (v[j].w >= least);
      }
    }
  }
  const uint32_t mask = __ballot_sync(0xffffffffu, tid < n && place < (uint32_t)need);
  if (lane == 0) part[warp] = __popc(mask);
  __syncthreads();
  const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? part[lane] : 0u);
  if ((mask >> lane) & 1u) pick(before + __popc(mask & lanemask_lt()), tid);
}

// One row's picks, by the CTA. Of a long list the few ranks that reach a floor
// are gathered first, in order; where they are many, the ranks are searched.
__device__ void kb_pick_row(const uint32_t* ord, int n, int need, int first, int last, int32_t* sel, KthShared* s) {
  for (int i = threadIdx.x; i < first + last; i += kSelectThreads) sel[i < first ? i : need + i] = i < first ? i : n + i;
  if (need == 0) return;
  if (n <= kSelectThreads) {
    kb_count_picks(ord, n, need, s->warp_a, [&](uint32_t at, int i) { sel[first + at] = first + i; });
    return;
  }
  auto get = [&](int i) { return ord[i]; };
  if (need <= kKthFew) {
    uint32_t* few = s->hist;  // ranks, zeros behind them, then where they stood
    int* where = reinterpret_cast<int*>(s->hist + kSelectThreads + 32);
    const Kth floor{kth_floor(get, n, (uint32_t)need, s), 0xFFFFFFFFu, 0, -1, ScoreBins(0.0f, 0.0f, 1)};
    const uint32_t found = kth_place(get, n, floor, s, [&](uint32_t at, int i) {
      if (at < kSelectThreads) few[at] = ord[i], where[at] = i;
    });
    if (found <= kSelectThreads) {
      if (threadIdx.x < 32) few[found + threadIdx.x] = 0;
      __syncthreads();
      kb_count_picks(few, (int)found, need, s->warp_a, [&](uint32_t at, int i) { sel[first + at] = first + where[i]; });
      return;
    }
  }
  const Kth kth = kth_rank(get, n, (uint32_t)need, (uint32_t)need, s);
  kth_place(get, n, kth, s, [&](uint32_t at, int i) { sel[first + at] = first + i; });
}

// Quantize the query vectors of `columns` (row, head) pairs (LANES lanes each,
// eight values a lane, all loads in flight together) and lay out their
// fragments. Columns without a pair are zero and have a scale that makes their
// scores NaN, which lose. between() runs while the loads travel.
template <bool F16, int NT, int LANES, bool SHARED, int THREADS = kSelectThreads, typename Between>
__device__ __forceinline__ void kb_queries(const KbParams& p, int row0, int columns, int heads, int h, unsigned char* scratch, int4* starts,
                                           uint2* ops, float* scales, Between between) {
  constexpr int kAtOnce = THREADS / LANES, kRounds = (8 * NT + kAtOnce - 1) / kAtOnce;
  const int G = p.groups, D = p.head_dim, sub = threadIdx.x % LANES;
  int8_t* q8 = reinterpret_cast<int8_t*>(scratch);
  int* off = reinterpret_cast<int*>(scratch + (size_t)8 * NT * G * kI4Group);
  uint4 w[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; k++) {
    const int m = k * kAtOnce + threadIdx.x / LANES;
    w[k] = make_uint4(0, 0, 0, 0);
    if (m < columns && sub * 8 < D) {
      const int row = SHARED ? m / heads : 0, head = m - row * heads;
      w[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (int64_t)(row0 + row) * p.q_stride +
                                                  (int64_t)(h * heads + head) * D) + sub);
    }
  }
  between();
#pragma unroll
  for (int k = 0; k < kRounds; k++) {
    const int m = k * kAtOnce + threadIdx.x / LANES;
    const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
    float x[8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = Elem<F16>::unpack(u[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
      top = absmax_step(absmax_step(top, f.x), f.y);
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) top = absmax_combine(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = top == 0.0f ? 0.0f : __fdiv_rn(top, 127.0f), inv = top == 0.0f ? 0.0f : __fdiv_rn(1.0f, scale);
    int sum = 0;
    uint32_t b[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int c = top == 0.0f ? 0 : (int)quant_code(x[i], inv);
      sum += c;
      b[i >> 2] |= (uint32_t)(c & 255) << (8 * (i & 3));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);  // four lanes hold a group
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (m < 8 * NT && sub * 8 < G * kI4Group) {
      *reinterpret_cast<uint2*>(q8 + (size_t)m * G * kI4Group + sub * 8) = make_uint2(b[0], b[1]);
      if ((sub & 3) == 0) off[m * G + (sub >> 2)] = -8 * sum;
      if (sub == 0) scales[m] = m < columns ? scale : __uint_as_float(0x7FFFFFFFu);
    }
  }
  i4_fragments<NT>(G, q8, off, starts, ops);
}

// The words, multipliers and scales of a quad (four groups) of a tile.
struct KbQuad {
  uint32_t w[4][4], mult[4];
  float scale[4];
};

__device__ __forceinline__ void kb_load(KbQuad& d, const I4Rows& rows, int tile, int quad, int lane) {
  const int G = rows.groups, quads = (G + 3) / 4, depth = G - quad * 4;
  const uint32_t* at = rows.codes + (size_t)tile * G * 128 + quad * 512;
  const uint32_t* mults = rows.mults + ((size_t)tile * quads + quad) * 32 + (lane >> 2);
#pragma unroll
  for (int b = 0; b < 4; b++) d.mult[b] = __ldg(mults + b * 8);
#pragma unroll
  for (int b = 0; b < 4; b++) d.scale[b] = __ldg(rows.scales + tile * kI4Tile + b * 8 + (lane >> 2));
  if (depth >= 4) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(at) + b * 32 + lane);
      d.w[b][0] = v.x, d.w[b][1] = v.y, d.w[b][2] = v.z, d.w[b][3] = v.w;
    }
  } else {
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
      for (int j = 0; j < 3; j++) d.w[b][j] = j < depth ? __ldg(at + (b * depth + j) * 32 + lane) : 0u;
  }
}

template <int NT>
__device__ __forceinline__ void kb_multiply(int (&tot)[2][NT][4], const KbQuad& d, int quad, int groups, const int4* starts, const uint2* ops) {
  const int depth = groups - quad * 4;
  const int4* c = starts + quad * 4 * NT * 32;
  const uint2* o = ops + quad * 4 * NT * 32;
  if (depth >= 4) i4_multiply<NT, 4>(tot, d.w, d.mult, c, o);
  else if (depth == 1) i4_multiply<NT, 1>(tot, d.w, d.mult, c, o);
  else if (depth == 2) i4_multiply<NT, 2>(tot, d.w, d.mult, c, o);
  else i4_multiply<NT, 3>(tot, d.w, d.mult, c, o);
}

// The ranks of the tiles from `tile` on in steps of `step`: store(block, rank). A
// tile's words travel during the products of the one before where registers
// allow; `next` holds the first one's first quad.
template <int NT, typename Store>
__device__ __forceinline__ void kb_score_tiles(const I4Rows& rows, int tile, int step, int tiles, KbQuad& next, const int4* starts, const uint2* ops,
                                               const float* s_scale, Store store) {
  constexpr bool kAhead = NT <= 2;
  const int lane = threadIdx.x & 31, G = rows.groups, quads = (G + 3) / 4;
  starts += lane;
  ops += lane;
  float qscale[NT][2];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int c = 0; c < 2; c++) qscale[n][c] = s_scale[n * 8 + 2 * (lane & 3) + c];
  KbQuad now;
  for (bool first = true; tile < tiles; tile += step, first = false) {
    int tot[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) tot[a][n][e] = 0;
    for (int quad = 0; quad < quads; quad++) {
      if (kAhead || (first && quad == 0)) now = next;
      else kb_load(now, rows, tile, quad, lane);
      if (kAhead) {
        if (quad + 1 < quads) kb_load(next, rows, tile, quad + 1, lane);
        else if (tile + step < tiles) kb_load(next, rows, tile + step, 0, lane);
      }
      kb_multiply<NT>(tot, now, quad, G, starts, ops);
    }
    // lane 4 r + t: blocks r, r + 8, r + 16, r + 24 of the tile, columns 2t and 2t + 1 of each eight
    float best[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
      best[b] = __uint_as_float(0x7FFFFFFFu);  // a NaN loses
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) best[b] = fmaxf(best[b], kb_score(tot[b >> 1][n][(b & 1) * 2 + c], qscale[n][c], now.scale[b]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
#pragma unroll
      for (int b = 0; b < 4; b++) best[b] = fmaxf(best[b], __shfl_xor_sync(0xffffffffu, best[b], o));
    // lane 4 r + t stores block 8 t + r
    const float mine = (lane & 2) ? (lane & 1) ? best[3] : best[2] : (lane & 1) ? best[1] : best[0];
    store(tile * kI4Tile + (lane & 3) * 8 + (lane >> 2), mine == mine ? score_to_ord(mine) : 0u);
  }
}

// A query row a CTA or cluster (grid: rows * cluster size, kv heads). Its first
// tile's words travel while the queries are quantized.
template <bool F16, int NT>
__global__ void __launch_bounds__(kSelectThreads, NT == 1 ? 3 : NT == 8 ? 1 : 2) kb_select_kernel(KbParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ KthShared s_kth;
  __shared__ float s_scale[8 * NT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.y, G = p.groups, heads = p.q_heads / p.kv_heads;
  const uint32_t rank = cluster_rank(), nranks = cluster_size();
  const int row = (int)(blockIdx.x / nranks);
  int4* starts = reinterpret_cast<int4*>(smem);
  uint2* ops = reinterpret_cast<uint2*>(starts + (size_t)G * NT * 32);
  unsigned char* scratch = smem + i4_frag_bytes<NT>(G);
  // the ranks; the first that is chosen from is 16-byte aligned
  uint32_t* ord = reinterpret_cast<uint32_t*>(scratch + (((size_t)8 * NT * G * (kI4Group + 4) + 15) & ~(size_t)15)) + ((-p.first) & 3);
  if (nranks > 1) cluster_arrive();
  pdl_wait_prior();         // queries, lengths and block rows may come from the kernel before
  pdl_launch_dependents();  // after the wait: the attention reads queries and lengths as it starts
  int nb = 0, tiles = 0, tile = (int)rank * kSelectWarps + warp;
  I4Rows rows;
  KbQuad next;
  auto start = [&] {
    int slot;
    nb = (kb_row_at(p, row, &slot) + p.block - 1) >> p.block_shift;
    rows = kb_rows(p, (int64_t)slot * p.kv_heads + h);
    // a row that sees no more blocks than it may take needs no ranks
    tiles = nb > p.select ? (nb - p.last + kI4Tile - 1) / kI4Tile : 0;
    if (tile < tiles) kb_load(next, rows, tile, 0, lane);
    if (nb > p.select && rank == 0 && tid < 32) ord[nb - p.last + tid] = 0;
  };
  if (p.head_dim <= 128) kb_queries<F16, NT, 16, false>(p, row, heads, heads, h, scratch, starts, ops, s_scale, start);
  else kb_queries<F16, NT, 32, false>(p, row, heads, heads, h, scratch, starts, ops, s_scale, start);
  if (nranks > 1) cluster_wait();
  kb_score_tiles<NT>(rows, tile, (int)nranks * kSelectWarps, tiles, next, starts, ops, s_scale, [&](int i, uint32_t o) {
    if (i >= nb - p.last) return;
    if (nranks > 1) st_cluster_u32(smem_u32(ord + i), 0, o);
    else ord[i] = o;
  });
  if (nranks > 1) cluster_sync();
  else __syncthreads();
  if (rank != 0) return;

  const int n = nb - p.first - p.last, need = p.select - p.first - p.last;
  int32_t* sel = p.sel + ((int64_t)row * p.kv_heads + h) * p.select;
  const uint32_t* o = ord + p.first;
  if (nb <= p.select) {  // every visible block
    for (int i = tid; i < p.select; i += kSelectThreads) sel[i] = i < nb ? i : -1;
  } else {
    kb_pick_row(o, n, need, p.first, p.last, sel, &s_kth);
  }
}

// Rows share a CTA: rt of them, of which those of one slot share the scoring of
// its block rows.
template <bool F16, int NT>
__global__ void __launch_bounds__(kSelectThreads, 2) kb_select_shared_kernel(KbParams p, int rt, int stride) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ KthShared s_kth;
  __shared__ float s_scale[8 * NT];
  __shared__ int s_slot[32], s_len[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.y, G = p.groups;
  const int heads = p.q_heads / p.kv_heads, quads = (G + 3) / 4;
  const int row0 = (int)blockIdx.x * rt, nrows = min(rt, p.rows - row0);
  int4* starts = reinterpret_cast<int4*>(smem);
  uint2* ops = reinterpret_cast<uint2*>(starts + (size_t)G * NT * 32);
  unsigned char* scratch = smem + i4_frag_bytes<NT>(G);
  uint32_t* ord = reinterpret_cast<uint32_t*>(scratch + (((size_t)8 * NT * G * (kI4Group + 4) + 15) & ~(size_t)15));
  pdl_wait_prior();         // queries, lengths and block rows may come from the kernel before
  pdl_launch_dependents();  // after the wait: the attention reads queries and lengths as it starts
  auto start = [&] {
    if (tid < nrows) {
      int slot;
      s_len[tid] = kb_row_at(p, row0 + tid, &slot);
      s_slot[tid] = slot;
    }
    for (int i = tid; i < nrows * stride; i += kSelectThreads) ord[i] = 0;  // several columns meet in one rank
  };
  if (p.head_dim <= 128) kb_queries<F16, NT, 16, true>(p, row0, nrows * heads, heads, h, scratch, starts, ops, s_scale, start);
  else kb_queries<F16, NT, 32, true>(p, row0, nrows * heads, heads, h, scratch, starts, ops, s_scale, start);
  auto blocks_of = [&](int r) { return (s_len[r] + p.block - 1) >> p.block_shift; };
  starts += lane;
  ops += lane;
  // runs of rows that share a slot; rows that see no more blocks than they may take need no ranks
  for (int r0 = 0; r0 < nrows;) {
    const int slot = s_slot[r0];
    int r1 = r0, most = 0;
    for (; r1 < nrows && s_slot[r1] == slot; r1++)
      if (blocks_of(r1) > p.select) most = max(most, blocks_of(r1));
    const int tiles = (max(0, most - p.last) + kI4Tile - 1) / kI4Tile;
    const I4Rows rows = kb_rows(p, (int64_t)slot * p.kv_heads + h);
    for (int tile = warp; tile < tiles; tile += kSelectWarps) {
      int tot[2][NT][4];
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) tot[a][n][e] = 0;
      KbQuad d;
      for (int quad = 0; quad < quads; quad++) {
        kb_load(d, rows, tile, quad, lane);
        kb_multiply<NT>(tot, d, quad, G, starts, ops);
      }
      // lane 4 r + t: blocks r, r + 8, r + 16, r + 24 of the tile, columns 2t and 2t + 1 of each eight
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int m = n * 8 + 2 * (lane & 3), row = m / heads, next = (m + 1) / heads;
        const float qs0 = s_scale[m], qs1 = s_scale[m + 1];
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const int i = tile * kI4Tile + b * 8 + (lane >> 2);
          float s0 = kb_score(tot[b >> 1][n][(b & 1) * 2], qs0, d.scale[b]);
          const float s1 = kb_score(tot[b >> 1][n][(b & 1) * 2 + 1], qs1, d.scale[b]);
          if (i >= stride) continue;
          if (next == row) s0 = fmaxf(s0, s1);
          else if (next >= r0 && next < r1 && s1 == s1) atomicMax(ord + next * stride + i, score_to_ord(s1));
          if (row >= r0 && row < r1 && s0 == s0) atomicMax(ord + row * stride + i, score_to_ord(s0));
        }
      }
    }
    r0 = r1;
  }
  __syncthreads();

  for (int r = 0; r < nrows; r++) {
    const int nb = blocks_of(r), n = nb - p.first - p.last, need = p.select - p.first - p.last;
    int32_t* sel = p.sel + ((int64_t)(row0 + r) * p.kv_heads + h) * p.select;
    const uint32_t* o = ord + r * stride + p.first;
    if (nb <= p.select) {  // every visible block
      if (r % kSelectWarps == warp)
        for (int i = lane; i < p.select; i += 32) sel[i] = i < nb ? i : -1;
    } else if (n < kWarpPicks) {
      if (r % kSelectWarps == warp) {
        uint32_t* hist = s_kth.hist + warp * 256;
        if (n <= 256) kb_warp_picks<8>(o, n, need, p.first, p.last, sel, hist);
        else kb_warp_picks<32>(o, n, need, p.first, p.last, sel, hist);
      }
    } else {
      __syncthreads();  // warps may be picking for rows before this one
      kb_pick_row(o, n, need, p.first, p.last, sel, &s_kth);
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Attention over the chosen blocks. One pass over the keys and values with the
// running maximum and sum of the softmax (in the log2 domain). The query heads
// that share a key/value head share one read of each key and value; bound by
// those bytes. They are the columns of the matrix products, eight or sixteen,
// and the tokens and channels their rows: S' = K Q', O' = V' P'. (With the heads
// as the rows a tile has sixteen of them whether they are there or not: twice
// the products, results and exponentials for up to eight heads.)
// A cluster of CTAs per (query row, kv head, tile of heads); the selected blocks
// are dealt in pieces of 16 tokens to the cluster's warps, and each warp runs
// its own ring of asynchronous copies and its own softmax, so nothing but the
// end synchronizes. The warps' partial results are joined in shared memory, the
// CTAs' through the cluster's.
// Measured, 32 heads of 128 over 8: sixteen rows of 32 blocks of 64 24.0 to 24.4 us
// (132 MB, 5.5 TB/s); one row of 16 blocks 5.1 us, latency; 2,048 rows of 16
// blocks 541 us: each row reads its own blocks, 8.6 GB at 16 TB/s, near the 64
// bytes a clock that an SM takes from L2.
// ---------------------------------------------------------------------------
constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kPiece = 16;

// Shared memory of a head dimension up to DP and 8 NT heads: the warps' rings
// (each holds, at the end, its warp's result, rows of kRow floats; the CTA's
// joined result replaces the first), the query tile, maxima and sums, the chosen
// blocks. Three CTAs an SM up to 128.
template <int DP, int NT>
struct AttendSmem {
  static constexpr int kStages = DP == 64 ? 4 : 2, kHeads = 8 * NT;
  static constexpr uint32_t kStage = 2 * kPiece * DP * 2;  // 16 keys, then 16 values
  static constexpr uint32_t kRing = kStages * kStage;      // of a warp
  static constexpr uint32_t kRow = DP + 4;                 // eight channels of four even heads fall into different banks
  static constexpr uint32_t kQuery = kAttendWarps * kRing, kStats = kQuery + kHeads * DP * 2;
  static_assert(kRing >= kHeads * kRow * 4, "a warp's result fits its ring");
  static constexpr uint32_t kSel = kStats + (2 + 2 * kAttendWarps) * kHeads * 4;
  static size_t bytes(int select) { return kSel + (size_t)select * 4; }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// With a constant offset, which costs no instruction.
template <bool TRANS, int AT>
__device__ __forceinline__ void ldmatrix4_at(uint32_t (&r)[4], uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(AT)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(AT)
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// Byte offset of 16-byte chunk c of row r in a tile of DP-element rows; the
// chunk index is permuted by the row so that eight rows' equal chunks fall
// into different banks.
template <int DP>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * (DP * 2) + ((c ^ (r & 7)) << 4));
}

// The running state of 8 NT heads over the tokens of a warp (log2 domain): lane
// 4 g + t holds channels 16 i + g and 16 i + g + 8 of heads 2t and 2t + 1 of each
// eight, times kLift; the lane's sums are those of its own tokens.
template <int DP, int NT>
struct AttendState {
  float o[NT][DP / 16][4];
  float mx[NT][2], sum[NT][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < DP / 16; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
      mx[n][0] = mx[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.0f;
    }
  }
};

// Steps t = 0 .. STEPS - 1 as compile-time constants: f(Int<t>{}).
template <int N>
struct Int {
  static constexpr int value = N;
};
template <int STEPS, int T = 0, typename F>
__device__ __forceinline__ void for_steps(F f) {
  if constexpr (T < STEPS) {
    f(Int<T>{});
    for_steps<STEPS, T + 1>(f);
  }
}

// An 8 x 8 matrix of 16-bit values, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// The 16 tokens of stage S (`n` of them visible) into the state. c2 >= 0 is the
// softmax scale times log2(e). ka and va are the lane's ldmatrix addresses in
// stage 0 for the steps 0 .. 3 of 16 channels, whose two bits are permuted by
// the row; further steps and stages are constant offsets.
template <int DP, int NT, bool F16, bool FULL, int S>
__device__ __forceinline__ void attend_piece(AttendState<DP, NT>& st, const uint32_t (&qf)[NT][DP / 16][2], const uint32_t (&ka)[4],
                                             const uint32_t (&va)[4], int n, float c2, int steps) {
  constexpr int kAt = S * (int)AttendSmem<DP, NT>::kStage, kValues = kAt + kPiece * DP * 2;
  using E = Elem<F16>;
  const int lane = threadIdx.x & 31;
  // tokens g and g + 8 by heads 2t and 2t + 1
  float sc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; i++) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
  for_steps<DP / 16>([&](auto step) {
    constexpr int t = decltype(step)::value;
    if (!FULL && t >= steps) return;
    uint32_t kf[4];
    ldmatrix4_at<false, kAt + (t >> 2) * 128>(kf, ka[t & 3]);
#pragma unroll
    for (int i = 0; i < NT; i++) E::mma(sc[i], kf, qf[i][t][0], qf[i][t][1]);
  });
  if (n < kPiece) {
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if ((lane >> 2) + (e & 2) * 4 >= n) sc[i][e] = -INFINITY;
  }
  // the heads' maxima: the eight lanes that share their columns
  float pm[NT][2];
  bool up = false;
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float m = fmaxf(sc[i][e], sc[i][e + 2]);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
      // scaled after the maximum; a scale of 0 must not meet -inf
      pm[i][e] = fmaxf(st.mx[i][e], m == -INFINITY ? -INFINITY : __fmul_rn(m, c2));
      up |= pm[i][e] != st.mx[i][e];
    }
  if (__any_sync(0xffffffffu, up)) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        f[e] = pm[i][e] == st.mx[i][e] ? 1.0f : exp2_fast(st.mx[i][e] - pm[i][e]);
        st.sum[i][e] *= f[e];
        st.mx[i][e] = pm[i][e];
      }
#pragma unroll
      for (int t = 0; t < DP / 16; t++) {
        st.o[i][t][0] *= f[0], st.o[i][t][1] *= f[1];
        st.o[i][t][2] *= f[0], st.o[i][t][3] *= f[1];
      }
    }
  }
  uint32_t pf[NT][2];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      // a head that has seen nothing but -inf keeps weights of 0
      const float base = st.mx[i][e & 1] == -INFINITY ? 0.0f : -st.mx[i][e & 1];
      // the product is rounded as the maximum's was, so that no weight passes 1 however large the scores are (fused, it
      // differs from the maximum by up to half a step of it, thousands from 2^36 on)
      w[e] = exp2_fast(__fadd_rn(__fmul_rn(sc[i][e], c2), base));
      if (n < kPiece && (lane >> 2) + (e & 2) * 4 >= n) w[e] = 0.0f;  // hidden: a scale of 0 times -inf is none
      st.sum[i][e & 1] += w[e];
    }
    // The weights enter the product in the cache's type (half a step, a relative 2^-8 or 2^-11, each; the sums stay 32
    // bits). Weights of f16 are lifted by 2^15: they keep those 2^-11 down to 2^-29 and an absolute 2^-40 below, where
    // without it a long tail of tokens under 2^-25 of the largest weight, up to 2^-8 of the sum, left the result.
    pf[i][0] = transpose8(E::pack(w[0] * E::kLift, w[1] * E::kLift));
    pf[i][1] = transpose8(E::pack(w[2] * E::kLift, w[3] * E::kLift));
  }
  for_steps<DP / 16>([&](auto step) {
    constexpr int t = decltype(step)::value;
    if (!FULL && t >= steps) return;
    uint32_t vf[4];
    ldmatrix4_at<true, kValues + (t >> 2) * 128>(vf, va[t & 3]);
#pragma unroll
    for (int i = 0; i < NT; i++) E::mma(st.o[i][t], vf, pf[i][0], pf[i][1]);
  });
}

// Two packed values of the query tile, negated when the scale is negative (the
// rest then works with its absolute value).
__device__ __forceinline__ uint4 flip_sign(uint4 w, bool flip) {
  const uint32_t f = flip ? 0x80008000u : 0u;
  return make_uint4(w.x ^ f, w.y ^ f, w.z ^ f, w.w ^ f);
}

// The choice of row r's blocks for head h by the attention's own CTA, over up to
// kAttendThreads blocks: into s_sel, and into p.sel if write. Works in smem.
template <bool F16, int LANES>
__device__ __forceinline__ void kb_choose(const KbParams& p, int r, int h, bool write, unsigned char* smem, int* s_sel) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = p.groups, heads = p.q_heads / p.kv_heads;
  float* s_scale = reinterpret_cast<float*>(smem);                    // [8]
  uint32_t* part = reinterpret_cast<uint32_t*>(smem + 32);            // [kAttendWarps]
  uint32_t* ord = reinterpret_cast<uint32_t*>(smem + 64) + ((-p.first) & 3);  // [kAttendThreads + 35]
  int4* starts = reinterpret_cast<int4*>(smem + 1024);
  uint2* ops = reinterpret_cast<uint2*>(starts + (size_t)G * 32);
  static_assert(64 + (kAttendThreads + 36) * 4 <= 1024, "the ranks fit");
  int nb = 0, tiles = 0;
  I4Rows rows;
  KbQuad next;
  kb_queries<F16, 1, LANES, false, kAttendThreads>(p, r, heads, heads, h, smem + 1024 + i4_frag_bytes<1>(G), starts, ops, s_scale, [&] {
    int slot;
    nb = (kb_row_at(p, r, &slot) + p.block - 1) >> p.block_shift;
    rows = kb_rows(p, (int64_t)slot * p.kv_heads + h);
    tiles = nb > p.select ? (nb - p.last + kI4Tile - 1) / kI4Tile : 0;
    if (warp < tiles) kb_load(next, rows, warp, 0, lane);
    if (nb > p.select && tid < 32) ord[nb - p.last + tid] = 0;
  });
  kb_score_tiles<1>(rows, warp, kAttendWarps, tiles, next, starts, ops, s_scale, [&](int i, uint32_t o) {
    if (i < nb - p.last) ord[i] = o;
  });
  __syncthreads();
  if (nb <= p.select) {  // every visible block
    for (int i = tid; i < p.select; i += kAttendThreads) s_sel[i] = i < nb ? i : -1;
  } else {
    const int n = nb - p.first - p.last, need = p.select - p.first - p.last;
    for (int i = tid; i < p.first + p.last; i += kAttendThreads) s_sel[i < p.first ? i : need + i] = i < p.first ? i : n + i;
    kb_count_picks(ord + p.first, n, need, part, [&](uint32_t at, int i) { s_sel[p.first + at] = p.first + i; });
  }
  __syncthreads();  // smem is the rings' from here on
  if (write) {
    int32_t* sel = p.sel + ((int64_t)r * p.kv_heads + h) * p.select;
    for (int i = tid; i < p.select; i += kAttendThreads) sel[i] = s_sel[i];
  }
}

// FULL: head_dim is DP itself. CHOOSE: every CTA of a row chooses its blocks, too.
template <int DP, int NT, bool F16, bool FULL, bool CHOOSE>
__global__ void __launch_bounds__(kAttendThreads, DP <= 128 ? 3 : 1) kb_attend_kernel(KbParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using S = AttendSmem<DP, NT>;
  constexpr int NS = S::kStages;
  constexpr int kChunks = DP / 8;             // 16-byte chunks of a padded row
  constexpr int kRowStep = 32 / kChunks;      // rows that a warp copies at once
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), nsplit = cluster_size();
  const int r = blockIdx.x / nsplit;
  const int heads = p.q_heads / p.kv_heads, mtiles = (heads + S::kHeads - 1) / S::kHeads;
  const int h = blockIdx.y / mtiles, m0 = (blockIdx.y % mtiles) * S::kHeads;
  const int mrows = min(S::kHeads, heads - m0);
  const int D = FULL ? DP : p.head_dim, chunks = D / 8, steps = D / 16;
  const uint32_t base = smem_u32(smem);
  float* s_o = reinterpret_cast<float*>(smem);  // each value replaces the first warp's, which the same thread has read
  float* s_m = reinterpret_cast<float*>(smem + S::kStats);  // maxima, then the sums
  float* w_m = s_m + 2 * S::kHeads;                         // the warps', then their sums
  float* w_l = w_m + kAttendWarps * S::kHeads;
  int* s_sel = reinterpret_cast<int*>(smem + S::kSel);

  if constexpr (CHOOSE) {
    pdl_wait_prior();
    pdl_launch_dependents();
    kb_choose<F16, DP <= 128 ? 16 : 32>(p, r, h, rank == 0, smem, s_sel);
  }
  // the query tile: absent heads are zero rows
  const T* q = static_cast<const T*>(p.q) + (int64_t)r * p.q_stride + (int64_t)(h * heads + m0) * D;
#pragma unroll
  for (int i0 = 0; i0 < S::kHeads * kChunks; i0 += kAttendThreads) {
    const int i = i0 + tid, row = i / kChunks, c = i % kChunks;
    if (S::kHeads * kChunks < kAttendThreads && i >= S::kHeads * kChunks) break;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < mrows && c < chunks) w = flip_sign(__ldg(reinterpret_cast<const uint4*>(q + (int64_t)row * D) + c), p.scale < 0.0f);
    *reinterpret_cast<uint4*>(smem + S::kQuery + tile_at<DP>(row, c)) = w;
  }
  int slot;
  const int len = kb_row_at(p, r, &slot);
  const int nb = (len + p.block - 1) >> p.block_shift;
  if constexpr (!CHOOSE) {
    pdl_wait_prior();  // the chosen blocks may come from the kernel before
    const int32_t* sel = p.sel + ((int64_t)r * p.kv_heads + h) * p.select;
    for (int i = tid; i < p.select; i += kAttendThreads) s_sel[i] = __ldcg(sel + i);
  }
  __syncthreads();
  // ldmatrix lane addresses. Keys: tokens 0-7 / 8-15 by lane bit 3, chunk + 1 by bit 4; values: the other way round
  const uint32_t koff = tile_at<DP>(lane & 15, lane >> 4), voff = tile_at<DP>((lane & 7) + ((lane & 16) >> 1), (lane >> 3) & 1);
  uint32_t qf[NT][DP / 16][2];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int t = 0; t < DP / 16; t += 2) {
      uint32_t f[4];
      ldmatrix4(f, base + S::kQuery + tile_at<DP>(n * 8 + (lane & 7), 2 * t + (lane >> 3)));
      qf[n][t][0] = f[0], qf[n][t][1] = f[1], qf[n][t + 1][0] = f[2], qf[n][t + 1][1] = f[3];
    }

  const int shift = p.block_shift - 4, pieces = p.select << shift;
  const int stride = (int)nsplit * kAttendWarps;
  const int64_t pitch = p.token_stride * 2;
  const int lane_row = lane / kChunks, lane_chunk = lane % kChunks;
  const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + (int64_t)slot * p.slot_stride +
                                                    (int64_t)h * p.head_stride) + lane_row * pitch + lane_chunk * 16;
  const int64_t to_values = static_cast<const char*>(p.v) - static_cast<const char*>(p.k);
  const uint32_t ring = base + warp * S::kRing;
  const bool copies = FULL || lane_chunk < chunks;
  // where a warp's first rows go; rows further on by multiples of kRowStep flip chunk bits
  uint32_t to[8 / kRowStep];
#pragma unroll
  for (int i = 0; i < 8 / kRowStep; i++) to[i] = ring + (tile_at<DP>(lane_row, lane_chunk) ^ ((i * kRowStep) << 4));
  uint32_t ka[4], va[4];
#pragma unroll
  for (int t = 0; t < 4; t++) ka[t] = ring + (koff ^ (t * 32)), va[t] = ring + (voff ^ (t * 32));
  const int64_t row_step = kRowStep * pitch;

  // starts the copies of piece i into a stage; the tokens of it that the row sees (0: skipped)
  auto load = [&](int i, auto stage) {
    constexpr int kAt = decltype(stage)::value * (int)S::kStage;
    int n = 0;
    const int b = i < pieces ? s_sel[i >> shift] : -1;
    if (b >= 0 && b < nb) {
      const int t0 = b * p.block + (i & ((1 << shift) - 1)) * kPiece;
      n = max(0, min(kPiece, len - t0));
      const char* from = kbase + t0 * pitch;
      if (copies && n > 0) {
        if (n == kPiece) {
#pragma unroll
          for (int row = 0; row < kPiece; row += kRowStep) {
            const uint32_t at = to[(row & 7) / kRowStep] + kAt + row * (DP * 2);
            cp_async16(at, from, true);
            cp_async16(at + kPiece * DP * 2, from + to_values, true);
            from += row_step;
          }
        } else {
#pragma unroll 1
          for (int row = 0; row < kPiece; row += kRowStep) {
            // hidden tokens are zeros: 0 * their weight 0 stays 0
            const bool ok = row + lane_row < n;
            const uint32_t at = ring + (tile_at<DP>(lane_row, lane_chunk) ^ ((row & 7) << 4)) + kAt + row * (DP * 2);
            cp_async16(at, ok ? from : kbase, ok);
            cp_async16(at + kPiece * DP * 2, (ok ? from : kbase) + to_values, ok);
            from += row_step;
          }
        }
      }
    }
    cp_async_commit();
    return n;
  };

  AttendState<DP, NT> st;
  st.clear();
  const float c2 = fabsf(p.scale) * 1.4426950408889634f;  // log2(e)
  int i = (int)rank * kAttendWarps + warp;
  int have[NS];
  for_steps<NS - 1>([&](auto s) { have[decltype(s)::value] = load(i + decltype(s)::value * stride, s); });
  for (; i < pieces; i += NS * stride) {
    for_steps<NS>([&](auto stage) {
      constexpr int s = decltype(stage)::value, before = (s + NS - 1) % NS;
      const int at = i + s * stride;
      if (at >= pieces) return;
      have[before] = load(at + (NS - 1) * stride, Int<before>{});
      cp_async_wait<NS - 1>();
      __syncwarp();
      if (have[s] > 0)
        attend_piece<DP, NT, F16, FULL, s>(st, qf, ka, va, have[s], c2, steps);
      __syncwarp();  // the stage may be filled again
    });
  }
  cp_async_wait<0>();
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) st.sum[n][e] += __shfl_xor_sync(0xffffffffu, st.sum[n][e], x);
  __syncwarp();
  {  // the warp's result over its own ring
    float* mine = reinterpret_cast<float*>(smem + warp * S::kRing);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int head = n * 8 + (lane & 3) * 2 + e;
        if (head >= mrows) continue;
#pragma unroll
        for (int t = 0; t < DP / 16; t++) {
          if (!FULL && t >= steps) break;
          mine[head * S::kRow + t * 16 + (lane >> 2)] = st.o[n][t][e];
          mine[head * S::kRow + t * 16 + (lane >> 2) + 8] = st.o[n][t][e + 2];
        }
        if (lane < 4) w_m[warp * S::kHeads + head] = st.mx[n][e], w_l[warp * S::kHeads + head] = st.sum[n][e];
      }
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + ((int64_t)r * p.q_heads + h * heads + m0) * D;
  float* lse = p.lse ? p.lse + (int64_t)r * p.q_heads + h * heads + m0 : nullptr;
  // four channels of a row, of the whole softmax
  auto finish = [&](int row, int d, float4 acc, float m, float l) {
    const bool some = l > 0.0f || l != l;
    const float f = some ? 1.0f / l * (1.0f / E::kLift) : 0.0f;
    *reinterpret_cast<uint2*>(out + (int64_t)row * D + d) = make_uint2(E::pack(acc.x * f, acc.y * f), E::pack(acc.z * f, acc.w * f));
    if (lse && d == 0) lse[row] = some ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  };
  for (int j = tid; j < mrows * (DP / 4); j += kAttendThreads) {
    const int row = j / (DP / 4), d = j % (DP / 4) * 4;
    if (d >= D) continue;
    float m = w_m[row];
#pragma unroll
    for (int w = 1; w < kAttendWarps; w++) m = fmaxf(m, w_m[w * S::kHeads + row]);
    const float zero = m == -INFINITY ? 0.0f : m;
    float4 acc = make_float4(0, 0, 0, 0);
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttendWarps; w++) {
      const float f = exp2_fast(w_m[w * S::kHeads + row] - zero);
      const float4 v = *reinterpret_cast<const float4*>(smem + w * S::kRing + (row * S::kRow + d) * 4);
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      l += f * w_l[w * S::kHeads + row];
    }
    if (nsplit == 1) {
      finish(row, d, acc, m, l);
    } else {
      *reinterpret_cast<float4*>(s_o + row * S::kRow + d) = acc;
      if (d == 0) s_m[row] = m, s_m[S::kHeads + row] = l;
    }
  }
  if (nsplit == 1) return;
  cluster_sync();
  // the cluster's CTAs share out the channels of the joined tile
  for (int j = tid * (int)nsplit + (int)rank; j < mrows * (DP / 4); j += kAttendThreads * (int)nsplit) {
    const int row = j / (DP / 4), d = j % (DP / 4) * 4;
    if (d >= D) continue;
    const uint32_t at = base + S::kStats + row * 4;
    float m = -INFINITY;
    for (uint32_t c = 0; c < nsplit; c++) m = fmaxf(m, ld_cluster(at, c));
    const float zero = m == -INFINITY ? 0.0f : m;
    float4 acc = make_float4(0, 0, 0, 0);
    float l = 0.0f;
    for (uint32_t c = 0; c < nsplit; c++) {
      const float f = exp2_fast(ld_cluster(at, c) - zero);
      const float4 v = ld_cluster_v4(base + (row * S::kRow + d) * 4, c);
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      l += f * ld_cluster(at + S::kHeads * 4, c);
    }
    finish(row, d, acc, m, l);
  }
  cluster_sync_relaxed();  // the others' shared memory is read until here
}

// A launch in clusters, as a programmatic dependent of the one before if pdl.
template <typename... Args>
cudaError_t launch_cluster(void (*kernel)(Args...), dim3 grid, int threads, int cluster, bool pdl, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// What an attention is launched with: behind what it takes its blocks from.
enum class Blocks { kGiven, kSelectBefore, kChoose };

template <int DP, int NT, bool F16, bool FULL>
cudaError_t attend_launch(const KbParams& p, int32_t splits, Blocks from, cudaStream_t stream) {
  const int heads = p.q_heads / p.kv_heads, mtiles = (heads + 8 * NT - 1) / (8 * NT);
  auto fn = kb_attend_kernel<DP, NT, F16, FULL, false>;
  if constexpr (NT == 1) fn = from == Blocks::kChoose ? kb_attend_kernel<DP, NT, F16, FULL, true> : fn;
  // Given blocks: queries and lengths are read before the wait for the launch before, which must not be.
  return launch_cluster(fn, dim3((unsigned)(p.rows * splits), (unsigned)(p.kv_heads * mtiles)), kAttendThreads, splits, from != Blocks::kGiven,
                        AttendSmem<DP, NT>::bytes(p.select), stream, p);
}

template <int DP, int NT, bool F16>
cudaError_t attend_full(const KbParams& p, int32_t splits, Blocks from, cudaStream_t stream) {
  return p.head_dim == DP ? attend_launch<DP, NT, F16, true>(p, splits, from, stream) : attend_launch<DP, NT, F16, false>(p, splits, from, stream);
}

template <bool F16, int NT>
cudaError_t attend_any(const KbParams& p, int32_t splits, Blocks from, cudaStream_t stream) {
  return p.head_dim <= 64    ? attend_full<64, NT, F16>(p, splits, from, stream)
         : p.head_dim <= 128 ? attend_full<128, NT, F16>(p, splits, from, stream)
                             : attend_full<256, NT, F16>(p, splits, from, stream);
}

template <int DP, int NT, bool F16, bool FULL, bool CHOOSE>
cudaError_t attend_init() {
  auto fn = kb_attend_kernel<DP, NT, F16, FULL, CHOOSE>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AttendSmem<DP, NT>::bytes(kKbMaxSelect));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <int NT, bool CHOOSE>
cudaError_t attend_init_all() {
  cudaError_t e = cudaSuccess;
  for (auto init : {attend_init<64, NT, false, false, CHOOSE>, attend_init<64, NT, false, true, CHOOSE>, attend_init<64, NT, true, false, CHOOSE>,
                    attend_init<64, NT, true, true, CHOOSE>, attend_init<128, NT, false, false, CHOOSE>, attend_init<128, NT, false, true, CHOOSE>,
                    attend_init<128, NT, true, false, CHOOSE>, attend_init<128, NT, true, true, CHOOSE>, attend_init<256, NT, false, false, CHOOSE>,
                    attend_init<256, NT, false, true, CHOOSE>, attend_init<256, NT, true, false, CHOOSE>, attend_init<256, NT, true, true, CHOOSE>})
    if (e == cudaSuccess) e = init();
  return e;
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

namespace {

template <bool F16>
cudaError_t select_any(int nt, int rt, int stride, int cluster, const KbParams& p, size_t smem, cudaStream_t stream) {
  if (rt > 1)
    return launch_cluster(kb_select_shared_kernel<F16, 4>, dim3((unsigned)((p.rows + rt - 1) / rt), (unsigned)p.kv_heads), kSelectThreads, 1,
                          true, smem, stream, p, rt, stride);
  const auto fn = nt == 1 ? kb_select_kernel<F16, 1> : nt == 2 ? kb_select_kernel<F16, 2> : nt == 4 ? kb_select_kernel<F16, 4> : kb_select_kernel<F16, 8>;
  return launch_cluster(fn, dim3((unsigned)(p.rows * cluster), (unsigned)p.kv_heads), kSelectThreads, cluster, true, smem, stream, p);
}

}  // namespace

cudaError_t kb_init() {
  const int most = 227 * 1024 - 12 * 1024;  // beside the select kernels' static shared memory
  const auto kind = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaSuccess;
  auto set = [&](auto fn, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, kind, bytes);
  };
  set(kb_select_kernel<false, 1>, most), set(kb_select_kernel<true, 1>, most);
  set(kb_select_kernel<false, 2>, most), set(kb_select_kernel<true, 2>, most);
  set(kb_select_kernel<false, 4>, most), set(kb_select_kernel<true, 4>, most);
  set(kb_select_kernel<false, 8>, most), set(kb_select_kernel<true, 8>, most);
  set(kb_select_shared_kernel<false, 4>, most), set(kb_select_shared_kernel<true, 4>, most);
  if (e == cudaSuccess) e = attend_init_all<1, false>();
  if (e == cudaSuccess) e = attend_init_all<1, true>();
  if (e == cudaSuccess) e = attend_init_all<2, false>();
  return e;
}

cudaError_t kb_select_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream) {
  const int heads = p.q_heads / p.kv_heads;
  const int64_t blocks = (p.capacity + p.block - 1) / p.block;
  const int stride = (int)((blocks + 31) / 32 * 32);  // ranks held for a row
  int rt = 1;  // query rows of a CTA
  int nt = heads <= 8 ? 1 : heads <= 16 ? 2 : heads <= 32 ? 4 : 8, cluster = 1;
  // Rows that can share slots (two or more a slot on average) and fill the GPU
  // without it share a CTA: up to 32 query vectors and 96 KB of ranks.
  if (heads <= 16 && p.rows >= 2 * p.slots && (int64_t)p.rows * p.kv_heads >= 8 * (int64_t)sm_count) {
    const int64_t fit = 96 * 1024 / ((int64_t)stride * 4);
    rt = std::max(1, (int)std::min<int64_t>(fit, 32 / heads));
    if (rt > 1) nt = 4;
  }
  // Very many blocks and few rows: a cluster of up to eight, while there are SMs
  // for it and every warp keeps two tiles (two rows over 7,813 blocks: 18.6 us for
  // the query with eight, 20.0 with sixteen; sixteen rows over 512: 30.8 without
  // one, 32.0 with two).
  if (rt == 1)
    while (cluster < 8 && (int64_t)p.rows * p.kv_heads * cluster * 2 <= 2 * (int64_t)sm_count &&
           blocks >= (int64_t)cluster * 4 * kSelectWarps * kI4Tile)
      cluster *= 2;
  const size_t smem = (size_t)p.groups * nt * 32 * 24 + (((size_t)8 * nt * p.groups * (kI4Group + 4) + 15) & ~(size_t)15) +
                      ((size_t)rt * stride + 36) * 4;  // zeros behind a row's ranks, and their alignment
  return p.f16 ? select_any<true>(nt, rt, stride, cluster, p, smem, stream) : select_any<false>(nt, rt, stride, cluster, p, smem, stream);
}

namespace {

// The attention's CTAs can choose the blocks, one a thread.
bool short_cache(const KbParams& p) { return p.capacity <= (int64_t)kAttendThreads * p.block; }

// The attention's CTAs that run at once, in clusters: three an SM up to 128
// channels, one above, less what the parts of the chip have left over beside
// whole clusters. Of 148 SMs' 444 CTAs 416, 384 and 336 run in clusters of 4, 8
// and 16; of 148 CTAs 132, 120 and 112 (what the runtime says of these kernels).
int64_t attend_at_once(const KbParams& p, int32_t cluster, int32_t sm_count) {
  const int64_t sms = sm_count;
  if (p.head_dim <= 128) return cluster <= 2 ? 3 * sms : cluster == 4 ? sms * 104 / 37 : cluster == 8 ? sms * 96 / 37 : sms * 84 / 37;
  return cluster <= 2 ? sms : cluster == 4 ? sms * 33 / 37 : cluster == 8 ? sms * 30 / 37 : sms * 28 / 37;
}

// Splits of a (row, kv head): as many as still run at once, while every warp has
// a piece; at most 16 (8 above 128 channels, and over a short cache, where one row
// of 32 heads over 64 blocks takes 7.6 us with 8 and 8.3 with 16), and a power of
// two: clusters of other sizes pack badly (16 rows x 8 heads over 32k tokens: 37 us
// with 2, 47 with 3, 44 with 4, 47 with 8).
int32_t attend_splits(const KbParams& p, int32_t sm_count) {
  const int heads = p.q_heads / p.kv_heads, tile = heads <= 8 ? 8 : 16, mtiles = (heads + tile - 1) / tile;
  const int64_t units = (int64_t)p.rows * p.kv_heads * mtiles;
  const int64_t pieces = (int64_t)p.select * (p.block / kPiece);
  int32_t splits = 1;
  const int32_t most = p.head_dim <= 128 && !short_cache(p) ? 16 : 8;
  while (splits < most && units * splits * 2 <= attend_at_once(p, splits * 2, sm_count) && pieces >= (int64_t)splits * 2 * kAttendWarps)
    splits *= 2;
  return splits;
}

cudaError_t attend_from(const KbParams& p, int32_t splits, Blocks from, cudaStream_t stream) {
  if (p.q_heads / p.kv_heads <= 8)
    return p.f16 ? attend_any<true, 1>(p, splits, from, stream) : attend_any<false, 1>(p, splits, from, stream);
  return p.f16 ? attend_any<true, 2>(p, splits, from, stream) : attend_any<false, 2>(p, splits, from, stream);
}

}  // namespace

cudaError_t kb_attend_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream) {
  return attend_from(p, attend_splits(p, sm_count), Blocks::kGiven, stream);
}

cudaError_t kb_query_launch(const KbParams& p, int32_t sm_count, cudaStream_t stream) {
  const int32_t splits = attend_splits(p, sm_count);
  // Short caches and rows whose CTAs all run at once: one launch, in which every
  // CTA of a row chooses its blocks. A call with two launches and with one, 32
  // heads of 128 over 8, 16 of 128 blocks of 64: one row 11.4 and 8.9 us, six 17.9
  // and 12.7 (the choice's CTAs still hold what the last clusters need), 16 19.5
  // and 20.2, 48 39.4 and 37.9. A head group of one: 11.4 and 8.9, 16.9 and 12.2,
  // 19.2 and 19.9, 39.1 and 37.4. Heads of 256, 8 over 1, 32 of 128 blocks of 128:
  // one row 16.7 and 16.3, 16 23.9 and 23.6. Over some hundred shapes one launch
  // was between 32 % faster and 4 % slower, but for calls of 256 CTAs with more than 64
  // MB to read, where it was 3 to 16 % slower (32 rows of 64 blocks of 64: 89 and
  // 101) and with some more or fewer CTAs was not.
  if (p.q_heads / p.kv_heads <= 8 && short_cache(p) && (int64_t)p.rows * p.kv_heads * splits <= attend_at_once(p, splits, sm_count))
    return attend_from(p, splits, Blocks::kChoose, stream);
  const cudaError_t e = kb_select_launch(p, sm_count, stream);
  return e == cudaSuccess ? attend_from(p, splits, Blocks::kSelectBefore, stream) : e;
}

}  // namespace fi8
