// fi8_kth.cuh -- the threshold of a top-k over ranks (order-preserving images
// of float32 scores, 0 for none), and the picks in index order.
//
// The scores are counted in equal bins between the smallest and the largest: a
// digit of the rank would put scores of one size, or all those away from zero,
// into a few bins, whose atomics queue and which decide nothing. The bins are
// scanned from the top; the few ranks of the bin that holds the need-th one are
// placed by counting, and a bin of many (equal scores, or infinite ones, which
// all share one) is searched by the ranks themselves.
#pragma once

#include "fi8_device.cuh"
#include "fi8_select.cuh"

namespace fi8 {

#ifdef __CUDACC__

constexpr int kKthBins = 2048;
constexpr int kKthList = 256;

struct KthShared {
  uint32_t hist[kKthBins];
  uint32_t list[kKthList];
  uint32_t warp_a[32], warp_b[32];
  uint32_t bin, above, in_bin, listed;
};

// The score of a rank (0: a NaN).
__device__ __forceinline__ float ord_to_score(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

// Scores to bins, monotone. Without a finite span all share bin 0.
struct ScoreBins {
  float low, scale;
  int last;
  __device__ __forceinline__ ScoreBins(float low_, float high, int bins) : low(low_), last(bins - 1) {
    scale = (float)bins / (high - low);
    if (!(high - low < 3.0e38f) || !(scale < 3.0e38f)) scale = 0.0f;
  }
  __device__ __forceinline__ int operator()(uint32_t o) const {
    return min(max((int)((ord_to_score(o) - low) * scale), 0), last);  // a NaN converts to 0
  }
  // A rank that none of bin b is below: half a bin under its edge, far more than
  // the roundings.
  __device__ __forceinline__ uint32_t below(int b) const {
    return b > 0 ? score_to_ord(low + ((float)b - 0.5f) / scale) : 0u;
  }
};

// The picks: ranks in bin `bin` or above, or, with bin < 0, the ranks above t and
// the first `ties` ranks equal to t.
struct Kth {
  uint32_t t;  // with a bin, a rank that no pick is below
  uint32_t ties;
  uint32_t count;  // picks
  int bin;
  ScoreBins bins;
  __device__ __forceinline__ bool above(uint32_t o) const { return bin < 0 ? o > t : o >= t && bins(o) >= bin; }
  __device__ __forceinline__ bool equal(uint32_t o) const { return bin < 0 && o == t; }
  __device__ __forceinline__ bool unordered() const { return bin >= 0 || ties == 0xFFFFFFFFu; }  // no tie is left out
};

// need in [1, n]: between need and limit picks, or, where no threshold gives
// so many (ranks tie), need. All threads of the CTA (kKthList to kKthBins, a
// power of two) call it, behind a barrier after which get(0 .. n) is ready.
template <typename Get>
__device__ Kth kth_rank(Get get, int n, uint32_t need, uint32_t limit, KthShared* s) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5, per = kKthBins / nt;
  uint32_t top = 0, low = 0xFFFFFFFFu;  // the smallest score that is one
#pragma unroll 4
  for (int i = tid; i < n; i += nt) {
    const uint32_t o = get(i);
    top = max(top, o);
    low = min(low, o - 1u);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) s->warp_a[warp] = top, s->warp_b[warp] = low;
  for (int i = tid; i < kKthBins; i += nt) s->hist[i] = 0;
  if (tid == 0) s->listed = 0;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s->warp_a[lane] : 0u);
  low = __reduce_min_sync(0xffffffffu, lane < warps ? s->warp_b[lane] : 0xFFFFFFFFu) + 1u;
  const ScoreBins bins(ord_to_score(low), ord_to_score(top), kKthBins);
  if ((uint32_t)n <= limit) return Kth{0u, 0xFFFFFFFFu, (uint32_t)n, -1, bins};
  int chosen = -1;  // the bin that the ranks are searched in; -1: none yet
  uint32_t base = 0, above = 0;  // in the bin: ranks from base + 2^bits on are all picks, `above` in all
  int bits = 32;
  for (;;) {
    const int shift = max(0, bits - 11);
#pragma unroll 4
    for (int i = tid; i < n; i += nt) {
      const uint32_t o = get(i);
      const int b = bins(o);
      if (chosen < 0) atomicAdd(s->hist + b, 1u);
      else if (b == chosen && o >= base && (bits == 32 || ((o - base) >> bits) == 0)) atomicAdd(s->hist + ((o - base) >> shift), 1u);
    }
    __syncthreads();
    // thread 0 holds the highest bins; counts run from the top
    uint32_t mine = 0;
#pragma unroll 4
    for (int i = 0; i < per; i++) mine += s->hist[kKthBins - 1 - tid * per - i];
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) s->warp_a[warp] = before;
    __syncthreads();
    before += above - mine + __reduce_add_sync(0xffffffffu, lane < warp ? s->warp_a[lane] : 0u);
    if (before < need && before + mine >= need) {
      for (int i = 0; i < per; i++) {
        const uint32_t c = s->hist[kKthBins - 1 - tid * per - i];
        if (before + c >= need) {
          s->bin = (uint32_t)(kKthBins - 1 - tid * per - i);
          s->above = before;
          s->in_bin = c;
          break;
        }
        before += c;
      }
    }
    __syncthreads();
    const uint32_t bin = s->bin, in_bin = s->in_bin;
    above = s->above;
    const uint32_t t = chosen < 0 ? 0u : base + (bin << shift);
    if (above + in_bin <= limit || (chosen >= 0 && shift == 0)) {
      __syncthreads();  // the shared memory may be used again
      if (chosen < 0) return Kth{bins.below((int)bin), 0xFFFFFFFFu, above + in_bin, (int)bin, bins};
      return above + in_bin <= limit ? Kth{t, 0xFFFFFFFFu, above + in_bin, -1, bins} : Kth{t, need - above, need, -1, bins};
    }
    if (in_bin <= (uint32_t)kKthList) {
      // ranks well below the bin are passed over without their bins
      const uint32_t edge = chosen < 0 ? bins.below((int)bin) : t;
#pragma unroll 4
      for (int i = tid; i < n; i += nt) {
        const uint32_t o = get(i);
        if (o >= edge && (chosen < 0 ? bins(o) == (int)bin : bins(o) == chosen && ((o - t) >> shift) == 0))
          s->list[atomicAdd(&s->listed, 1u)] = o;
      }
      __syncthreads();
      if (tid < (int)in_bin) {
        const uint32_t mine = s->list[tid];
        uint32_t gt = above, eq = 0;
#pragma unroll 4
        for (int i = 0; i < (int)in_bin; i++) {
          gt += s->list[i] > mine;
          eq += s->list[i] == mine;
        }
        if (gt < need && gt + eq >= need) {  // equal ranks write the same
          s->bin = mine;
          s->above = gt;
          s->in_bin = eq;
        }
      }
      __syncthreads();
      const uint32_t count = s->above + s->in_bin;
      const Kth k = count <= limit ? Kth{s->bin, 0xFFFFFFFFu, count, -1, bins} : Kth{s->bin, need - s->above, need, -1, bins};
      __syncthreads();
      return k;
    }
    if (chosen < 0) {
      chosen = (int)bin;
    } else {
      base = t;
      bits = shift;
    }
    for (int i = tid; i < kKthBins; i += nt) s->hist[i] = 0;
    __syncthreads();
  }
}

// Calls put(position, i) for the picks, in index order.
template <typename Get, typename Put>
__device__ void kth_place(Get get, int n, const Kth& k, KthShared* s, Put put) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int seg = (n + warps * 32 - 1) / (warps * 32) * 32, i0 = min(n, warp * seg), i1 = min(n, i0 + seg);
  uint32_t gt = 0, eq = 0;
#pragma unroll 4
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t o = get(i);
    gt += k.above(o);
    eq += k.equal(o);
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  const bool any = gt + eq > 0;
  if (lane == 0) s->warp_a[warp] = gt, s->warp_b[warp] = eq;
  __syncthreads();
  gt = __reduce_add_sync(0xffffffffu, lane < warp ? s->warp_a[lane] : 0u);
  eq = __reduce_add_sync(0xffffffffu, lane < warp ? s->warp_b[lane] : 0u);
  for (int base = any ? i0 : i1; base < i1; base += 128) {
    bool is_gt[4], is_eq[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = base + 32 * u + lane;
      const uint32_t o = i < i1 ? get(i) : 0u;
      is_gt[u] = i < i1 && k.above(o);
      is_eq[u] = i < i1 && k.equal(o);
    }
    if (!__any_sync(0xffffffffu, is_gt[0] || is_eq[0] || is_gt[1] || is_eq[1] || is_gt[2] || is_eq[2] || is_gt[3] || is_eq[3])) continue;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt[u]), meq = __ballot_sync(0xffffffffu, is_eq[u]);
      const uint32_t my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
      if (is_gt[u] || (is_eq[u] && my_eq < k.ties)) put(my_gt + min(my_eq, k.ties), base + 32 * u + lane);
      gt += __popc(mgt);
      eq += __popc(meq);
    }
  }
  __syncthreads();
}

// The same in any order, where no tie is left out.
template <typename Get, typename Put>
__device__ void kth_list(Get get, int n, const Kth& k, KthShared* s, Put put) {
  if (threadIdx.x == 0) s->listed = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint32_t o = get(i);
    if (k.above(o) || k.equal(o)) put(atomicAdd(&s->listed, 1u), i);
  }
  __syncthreads();
}

#endif  // __CUDACC__

}  // namespace fi8
