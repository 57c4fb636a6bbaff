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
constexpr int kKthGroups = 128;
constexpr int kKthFew = 64;  // what kth_floor is asked for at most

struct KthShared {
  alignas(16) uint32_t hist[kKthBins];
  alignas(16) uint32_t list[kKthList];
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
    scale = __fdividef((float)bins, high - low);  // 0 for the widest spans; any scale is monotone
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

// The picks: ranks in bin `bin` or above (all of them at least t), or, with bin < 0,
// the ranks above t and the first `ties` ranks equal to t (0xFFFFFFFF: all).
struct Kth {
  uint32_t t;
  uint32_t ties;
  uint32_t count;  // picks
  int bin;
  ScoreBins bins;
};

// f(rank) for the thread's share of get(0 .. n), four loads in flight.
template <typename Get, typename F>
__device__ __forceinline__ void kth_each(Get get, int n, F f) {
  const int nt = blockDim.x;
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * nt) {
    uint32_t o[4];
#pragma unroll
    for (int u = 0; u < 4; u++) o[u] = i0 + u * nt < n ? get(i0 + u * nt) : 0u;
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (i0 + u * nt < n) f(o[u]);
  }
}

// need in [1, n], limit >= need: between need and limit picks, or, where no
// threshold gives so many (ranks tie), need. All threads of the CTA (kKthList to 1024, a power
// of two) call it, behind a barrier after which get(0 .. n) is ready.
template <typename Get>
__device__ Kth kth_rank(Get get, int n, uint32_t need, uint32_t limit, KthShared* s) {
  // all of them: before any shared word is touched, so that no barrier has to follow
  if ((uint32_t)n <= limit) return Kth{0u, 0xFFFFFFFFu, (uint32_t)n, -1, ScoreBins(0.0f, 0.0f, 1)};
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5, per = kKthBins / nt;
  uint32_t top = 0, low = 0xFFFFFFFFu;  // the smallest score that is one
  kth_each(get, n, [&](uint32_t o) {
    top = max(top, o);
    low = min(low, o - 1u);
  });
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) s->warp_a[warp] = top, s->warp_b[warp] = low;
  for (int i = tid; i < kKthBins / 4; i += nt) reinterpret_cast<uint4*>(s->hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) s->listed = 0;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s->warp_a[lane] : 0u);
  low = __reduce_min_sync(0xffffffffu, lane < warps ? s->warp_b[lane] : 0xFFFFFFFFu) + 1u;
  const ScoreBins bins(ord_to_score(low), ord_to_score(top), kKthBins);
  int chosen = -1;  // the bin that the ranks are searched in; -1: none yet
  uint32_t base = 0, above = 0;  // in the bin: ranks from base + 2^bits on are all picks, `above` in all
  int bits = 32;
  for (;;) {
    const int shift = max(0, bits - 11);
    if (chosen < 0)
      kth_each(get, n, [&](uint32_t o) { atomicAdd(s->hist + bins(o), 1u); });
    else
      kth_each(get, n, [&](uint32_t o) {
        if (bins(o) == chosen && o >= base && (bits == 32 || ((o - base) >> bits) == 0)) atomicAdd(s->hist + ((o - base) >> shift), 1u);
      });
    __syncthreads();
    // thread 0 holds the highest bins, c[0] the highest of them; counts run from the top
    uint32_t c[8], mine = 0;
    const uint32_t* at = s->hist + kKthBins - (tid + 1) * per;
    if (per == 8) {
      const uint4 lo = *reinterpret_cast<const uint4*>(at), hi = *reinterpret_cast<const uint4*>(at + 4);
      c[0] = hi.w, c[1] = hi.z, c[2] = hi.y, c[3] = hi.x, c[4] = lo.w, c[5] = lo.z, c[6] = lo.y, c[7] = lo.x;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = i < per ? at[per - 1 - i] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) mine += c[i];
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
      bool found = false;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (!found && before + c[i] >= need) {
          found = true;
          s->bin = (uint32_t)(kKthBins - 1 - tid * per - i);
          s->above = before;
          s->in_bin = c[i];
        }
        before += c[i];
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
      kth_each(get, n, [&](uint32_t o) {
        if (o >= edge && (chosen < 0 ? bins(o) == (int)bin : bins(o) == chosen && ((o - t) >> shift) == 0))
          s->list[atomicAdd(&s->listed, 1u)] = o;
      });
      __syncthreads();
      if (tid < (int)in_bin) {
        const uint32_t mine = s->list[tid];
        uint32_t gt = above, eq = 0;
#pragma unroll 8
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

// A rank that at least need (at most kKthFew) of get(0 .. n) reach, n > 256, and
// few more than need where the ranks lie in no order: the need-th largest of the
// maxima of 128 groups, in which few of the largest ranks fall together. (-ln(1 -
// need / 128) * 128 ranks reach it on average: 34 for 30, 84 for 62.) All threads
// of a CTA of 256 to 1024 call it, behind a barrier after which get is ready.
template <typename Get>
__device__ uint32_t kth_floor(Get get, int n, uint32_t need, KthShared* s) {
  const int tid = threadIdx.x, lane = tid & 31, per = blockDim.x / kKthGroups;
  uint32_t top = 0;
  kth_each(get, n, [&](uint32_t o) { top = max(top, o); });
  for (int o = 1; o < per; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane % per == 0) s->list[tid / per] = top;
  if (tid == 0) s->bin = 0;
  __syncthreads();
  if (tid < kKthGroups) {
    const uint32_t mine = s->list[tid];
    uint32_t ge = 0;
#pragma unroll 1
    for (int b = 0; b < kKthGroups / 4; b += 8) {
      uint4 v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const uint4*>(s->list)[b + j];
#pragma unroll
      for (int j = 0; j < 8; j++) ge += (v[j].x >= mine) + (v[j].y >= mine) + (v[j].z >= mine) + (v[j].w >= mine);
    }
    const uint32_t best = __reduce_max_sync(0xffffffffu, ge >= need ? mine : 0u);
    if (lane == 0) atomicMax(&s->bin, best);
  }
  __syncthreads();
  return s->bin;
}

// Calls put(position, i) for the picks, in index order, and returns their
// number. A warp takes a run of ranks, 1024 at a time: a lane's picks and ties
// among its 32 of them are bits.
template <typename Get, typename Put>
__device__ uint32_t kth_place(Get get, int n, const Kth& k, KthShared* s, Put put) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int seg = (n + warps * 32 - 1) / (warps * 32) * 32, i0 = min(n, warp * seg), i1 = min(n, i0 + seg);
  const bool all = k.ties == 0xFFFFFFFFu;
  uint32_t picks = 0, ties = 0;
  auto look = [&](int base) {
    picks = ties = 0;
    const int left = i1 - base - lane, steps = min(32, (i1 - base + 31) >> 5);
    const uint32_t there = left <= 0 ? 0u : left > 31 * 32 ? 0xFFFFFFFFu : (1u << ((left + 31) >> 5)) - 1u;
#pragma unroll
    for (int e0 = 0; e0 < 32; e0 += 8) {
      if (e0 >= steps) break;
      uint32_t o[8];
#pragma unroll
      for (int u = 0; u < 8; u++) o[u] = (e0 + u) * 32 < left ? get(base + (e0 + u) * 32 + lane) : 0u;
#pragma unroll
      for (int u = 0; u < 8; u++) picks |= o[u] >= k.t ? 1u << (e0 + u) : 0u;
    }
    picks &= there;
    if (!all) {
      for (uint32_t m = picks; m; m &= m - 1) {
        const int e = __ffs(m) - 1;
        if (get(base + e * 32 + lane) == k.t) ties |= 1u << e;
      }
      picks &= ~ties;
    }
    if (k.bin >= 0)  // t lies a little under the bin
      for (uint32_t m = picks; m; m &= m - 1) {
        const int e = __ffs(m) - 1;
        if (k.bins(get(base + e * 32 + lane)) < k.bin) picks &= ~(1u << e);
      }
  };
  uint32_t gt = 0, eq = 0;
  for (int base = i0; base < i1; base += 1024) {
    look(base);
    gt += __popc(picks);
    eq += __popc(ties);
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  const bool any = gt + eq > 0;
  if (lane == 0) s->warp_a[warp] = gt, s->warp_b[warp] = eq;
  __syncthreads();
  const uint32_t a = lane < warps ? s->warp_a[lane] : 0u, b = lane < warps ? s->warp_b[lane] : 0u;
  const uint32_t total = __reduce_add_sync(0xffffffffu, a) + min(__reduce_add_sync(0xffffffffu, b), k.ties);
  gt = __reduce_add_sync(0xffffffffu, lane < warp ? a : 0u);
  eq = __reduce_add_sync(0xffffffffu, lane < warp ? b : 0u);
  for (int base = any ? i0 : i1; base < i1; base += 1024) {
    if (seg > 1024) look(base);
    for (uint32_t m = __reduce_or_sync(0xffffffffu, picks | ties); m; m &= m - 1) {
      const int e = __ffs(m) - 1;
      const bool is_gt = (picks >> e) & 1u, is_eq = (ties >> e) & 1u;
      if (all) {
        const uint32_t mask = __ballot_sync(0xffffffffu, is_gt);
        if (is_gt) put(gt + __popc(mask & lanemask_lt()), base + e * 32 + lane);
        gt += __popc(mask);
        continue;
      }
      const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt), meq = __ballot_sync(0xffffffffu, is_eq);
      const uint32_t my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
      if (is_gt || (is_eq && my_eq < k.ties)) put(my_gt + min(my_eq, k.ties), base + e * 32 + lane);
      gt += __popc(mgt);
      eq += __popc(meq);
    }
  }
  __syncthreads();
  return total;
}

// The same in any order, where no tie is left out; positions may pass what put has room for.
template <typename Get, typename Put>
__device__ uint32_t kth_list(Get get, int n, const Kth& k, KthShared* s, Put put) {
  const int nt = blockDim.x;
  if (threadIdx.x == 0) s->listed = 0;
  __syncthreads();
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * nt) {
    uint32_t o[4];
#pragma unroll
    for (int u = 0; u < 4; u++) o[u] = i0 + u * nt < n ? get(i0 + u * nt) : 0u;
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (i0 + u * nt < n && o[u] >= k.t && (k.bin < 0 || k.bins(o[u]) >= k.bin)) put(atomicAdd(&s->listed, 1u), i0 + u * nt);
  }
  __syncthreads();
  return s->listed;
}

#endif  // __CUDACC__

}  // namespace fi8
