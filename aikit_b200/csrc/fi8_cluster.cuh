// fi8_cluster.cuh -- thread-block clusters: rank, barrier and remote shared
// loads, and the threshold of a top-k over 32-bit ranks that a cluster's CTAs
// hold in parts.
#pragma once

#include "fi8_device.cuh"
#include "fi8_select.cuh"

namespace fi8 {

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The word at this CTA's shared address `addr`, in the CTA of rank `rank`.
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  return __uint_as_float(ld_cluster_u32(addr, rank));
}

// Shared memory of cluster_kth, and the counts that place a cluster's picks.
struct KthShared {
  uint32_t hist[2][256];
  uint32_t total[256];
  uint32_t out[2];
  uint32_t warp_gt[32], warp_eq[32];
  uint32_t gt, eq;  // this CTA's
};

__device__ __forceinline__ void cluster_or_cta_sync(uint32_t nranks) {
  if (nranks > 1) cluster_sync();
  else __syncthreads();
}

// The image t of the need-th largest of the ranks get(0 .. n) that all CTAs of
// the cluster hold, and how many picks have exactly t (need <= their number).
// A radix select, eight bits a pass: every CTA counts its own values, then all
// sum all counts and come to the same digit. Two histograms alternate, so that
// one barrier a pass is enough: a CTA that clears the other one has passed the
// barrier behind which everyone had read it.
template <typename Get>
__device__ void cluster_kth(Get get, int n, uint32_t need, KthShared* s, uint32_t nranks, uint32_t* t, uint32_t* ties) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  for (int pass = 0; pass < 4; pass++) {
    const int shift = 24 - 8 * pass;
    uint32_t* hist = s->hist[pass & 1];
    for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
      const uint32_t o = get(i);
      if (pass == 0 || (o >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(hist + ((o >> shift) & 255u), 1u);
    }
    cluster_or_cta_sync(nranks);
    for (int i = tid; i < 256; i += blockDim.x) {
      uint32_t sum = hist[i];
      if (nranks > 1) {
        const uint32_t at = smem_u32(hist + i);
        sum = 0;
        for (uint32_t c = 0; c < nranks; c++) sum += ld_cluster_u32(at, c);
      }
      s->total[i] = sum;
    }
    __syncthreads();
    if (tid < 32) {  // lane l holds bins 255 - 8l .. 255 - 8l - 7, the largest first
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) sum += c[i] = s->total[255 - tid * 8 - i];
      uint32_t before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
        if (tid >= o) before += y;
      }
      before -= sum;
      if (before < need && before + sum >= need) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (before < need && before + c[i] >= need) {
            s->out[0] = 255u - tid * 8 - i;
            s->out[1] = need - before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= s->out[0] << shift;
    need = s->out[1];
  }
  *t = prefix;
  *ties = need;
}

// Write the picks (rank above t, and the first `ties` with rank t) of the
// cluster's values in index order: put(position, i). CTA c holds the values
// behind those of the CTAs before it.
template <typename Get, typename Put>
__device__ void cluster_place(Get get, int n, uint32_t t, uint32_t ties, KthShared* s, uint32_t rank, uint32_t nranks, Put put) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int seg = (n + warps * 32 - 1) / (warps * 32) * 32, i0 = min(n, warp * seg), i1 = min(n, i0 + seg);
  uint32_t gt = 0, eq = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t o = get(i);
    gt += o > t;
    eq += o == t;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    s->warp_gt[warp] = gt;
    s->warp_eq[warp] = eq;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t a = 0, b = 0;
    for (int w = 0; w < warps; w++) a += s->warp_gt[w], b += s->warp_eq[w];
    s->gt = a;
    s->eq = b;
  }
  cluster_or_cta_sync(nranks);
  gt = eq = 0;
  for (uint32_t c = 0; c < rank; c++) {
    gt += ld_cluster_u32(smem_u32(&s->gt), c);
    eq += ld_cluster_u32(smem_u32(&s->eq), c);
  }
  for (int w = 0; w < warp; w++) gt += s->warp_gt[w], eq += s->warp_eq[w];
  for (int base = i0; base < i1; base += 32) {
    const int i = base + lane;
    const uint32_t o = i < i1 ? get(i) : 0;
    const bool is_gt = i < i1 && o > t, is_eq = i < i1 && o == t;
    const uint32_t mgt = __ballot_sync(0xffffffffu, is_gt), meq = __ballot_sync(0xffffffffu, is_eq);
    const uint32_t my_gt = gt + __popc(mgt & lanemask_lt()), my_eq = eq + __popc(meq & lanemask_lt());
    if (is_gt || (is_eq && my_eq < ties)) put(my_gt + min(my_eq, ties), i);
    gt += __popc(mgt);
    eq += __popc(meq);
  }
}

#endif  // __CUDACC__

}  // namespace fi8
