// fi8_kth.cuh -- the threshold of a top-k over 32-bit ranks by one CTA, and the
// picks in index order.
//
// A histogram of 2048 equal bins between the smallest and the largest rank (a
// radix digit from the top would put scores of one size into one bin, where
// their atomics queue), a scan from the top, and the same again inside the bin
// that holds the need-th rank. A caller that takes a few picks more than it
// needs is mostly done after the first one: the best ranks lie apart.
#pragma once

#include "fi8_device.cuh"
#include "fi8_select.cuh"

namespace fi8 {

#ifdef __CUDACC__

constexpr int kKthBins = 2048;

struct KthShared {
  uint32_t hist[kKthBins];
  uint32_t warp_a[32], warp_b[32];
  uint32_t bin, above, in_bin;
};

struct Kth {
  uint32_t t;      // picks are the ranks above t and the first `ties` ranks equal to t
  uint32_t ties;
  uint32_t count;  // picks
};

// need in [1, n]: between need and limit picks, or, where no threshold gives
// so many (ranks tie), need. All threads of the CTA (a multiple of 32 that
// divides kKthBins) call it, behind a barrier after which get(0 .. n) is ready.
template <typename Get>
__device__ Kth kth_rank(Get get, int n, uint32_t need, uint32_t limit, KthShared* s) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5, per = kKthBins / nt;
  uint32_t top = 0, low = 0xFFFFFFFFu;
#pragma unroll 4
  for (int i = tid; i < n; i += nt) {
    const uint32_t o = get(i);
    top = max(top, o);
    low = min(low, o);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) s->warp_a[warp] = top, s->warp_b[warp] = low;
  for (int i = tid; i < kKthBins; i += nt) s->hist[i] = 0;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s->warp_a[lane] : 0u);
  low = __reduce_min_sync(0xffffffffu, lane < warps ? s->warp_b[lane] : 0xFFFFFFFFu);
  if ((uint32_t)n <= limit) return Kth{low, 0xFFFFFFFFu, (uint32_t)n};
  uint32_t base = low, above = 0;  // ranks from base + 2^bits on: `above` of them, all picks
  int bits = 32 - __clz(top - low);
  for (;;) {
    const int shift = max(0, bits - 11);
#pragma unroll 4
    for (int i = tid; i < n; i += nt) {
      const uint32_t o = get(i) - base;  // below base: wraps to at least 2^bits
      if ((o >> shift) < (uint32_t)kKthBins && (bits == 32 || (o >> bits) == 0)) atomicAdd(s->hist + (o >> shift), 1u);
    }
    __syncthreads();
    // thread 0 holds the highest bins; counts run from the top
    uint32_t mine = 0;
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
    const uint32_t t = base + (s->bin << shift);
    above = s->above;
    const uint32_t count = above + s->in_bin;
    if (count <= limit || shift == 0) {
      __syncthreads();  // the shared memory may be used again
      return count <= limit ? Kth{t, 0xFFFFFFFFu, count} : Kth{t, need - above, need};
    }
    base = t;
    bits = shift;
    for (int i = tid; i < kKthBins; i += nt) s->hist[i] = 0;
    __syncthreads();
  }
}

// Calls put(position, i) for the picks, in index order. With all ties taken, t
// is a lower bound: the picks are the ranks from t on.
template <typename Get, typename Put>
__device__ void kth_place(Get get, int n, const Kth& k, KthShared* s, Put put) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int seg = (n + warps * 32 - 1) / (warps * 32) * 32, i0 = min(n, warp * seg), i1 = min(n, i0 + seg);
  uint32_t gt = 0, eq = 0;
#pragma unroll 8
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t o = get(i);
    gt += o > k.t;
    eq += o == k.t;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  const bool any = gt + eq > 0;
  if (lane == 0) s->warp_a[warp] = gt, s->warp_b[warp] = eq;
  __syncthreads();
  gt = __reduce_add_sync(0xffffffffu, lane < warp ? s->warp_a[lane] : 0u);
  eq = __reduce_add_sync(0xffffffffu, lane < warp ? s->warp_b[lane] : 0u);
  for (int base = any ? i0 : i1; base < i1; base += 128) {
    uint32_t o[4];
#pragma unroll
    for (int u = 0; u < 4; u++) o[u] = base + 32 * u + lane < i1 ? get(base + 32 * u + lane) : 0u;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = base + 32 * u + lane;
      const bool is_gt = i < i1 && o[u] > k.t, is_eq = i < i1 && o[u] == k.t;
      const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt), meq = __ballot_sync(0xffffffffu, is_eq);
      if ((mgt | meq) == 0) continue;
      const uint32_t my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
      if (is_gt || (is_eq && my_eq < k.ties)) put(my_gt + min(my_eq, k.ties), i);
      gt += __popc(mgt);
      eq += __popc(meq);
    }
  }
  __syncthreads();
}

#endif  // __CUDACC__

}  // namespace fi8
