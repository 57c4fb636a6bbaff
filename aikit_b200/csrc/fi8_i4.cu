// fi8_i4.cu -- FlatI4: scores of 4-bit rows (a matrix-vector product with
// group scales), the row quantizer, and the exact top-k.
#include "fi8_cluster.cuh"
#include "fi8_i4.cuh"
#include "fi8_i4q.cuh"

namespace fi8 {

namespace {

constexpr int kWarps = 8;

// Word index of lane l's word of group g in its block of 8 rows.
__device__ __forceinline__ int i4_word_at(int g, int lane, int groups) {
  const int full = groups & ~3;
  return g < full ? (g >> 2) * 128 + lane * 4 + (g & 3) : full * 32 + lane * (groups & 3) + (g - full);
}

// ---------------------------------------------------------------------------
// Row quantization and the row-major format.
// ---------------------------------------------------------------------------

// A CTA per block of 8 rows, a warp a row: its codes and multipliers are
// gathered in shared memory in the row-major format, then written interleaved.
// Rows of the block outside [row0, row0 + rows) stay as they are.
template <typename Row>
__device__ __forceinline__ void i4_write_block(const I4Rows& r, int64_t row0, int64_t rows, unsigned char* smem, Row fill) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = r.groups, quads = (G + 3) / 4;
  const int64_t block = row0 / 8 + blockIdx.x, row = block * 8 + warp;
  uint32_t* s_codes = reinterpret_cast<uint32_t*>(smem);                    // [8][G * 4]
  uint8_t* s_mults = reinterpret_cast<uint8_t*>(s_codes + (size_t)8 * G * 4);  // [8][quads * 4]
  const bool mine = row >= row0 && row < row0 + rows;
  if (mine) {
    const float scale = fill(row, reinterpret_cast<uint8_t*>(s_codes + (size_t)warp * G * 4), s_mults + warp * quads * 4);
    if (lane < quads * 4 - G) s_mults[warp * quads * 4 + G + lane] = 0;
    if (lane == 0) r.scales[row] = scale;
  }
  __syncthreads();
  uint32_t* codes = r.codes + (size_t)block * G * 32;
  uint32_t* mults = r.mults + (size_t)block * quads * 8;
  for (int i = threadIdx.x; i < G * 32; i += kWarps * 32) {
    const int g = i >> 5, l = i & 31;
    const int64_t at = block * 8 + (l >> 2);
    if (at >= row0 && at < row0 + rows) codes[i4_word_at(g, l, G)] = s_codes[(l >> 2) * G * 4 + g * 4 + (l & 3)];
  }
  for (int i = threadIdx.x; i < quads * 8; i += kWarps * 32) {
    const int64_t at = block * 8 + (i & 7);
    if (at >= row0 && at < row0 + rows) mults[i] = reinterpret_cast<const uint32_t*>(s_mults)[(i & 7) * quads + (i >> 3)];
  }
}

__global__ void __launch_bounds__(kWarps * 32) i4_quantize_kernel(I4Rows r, int64_t row0, const float* v, int64_t rows) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31;
  i4_write_block(r, row0, rows, smem, [&](int64_t row, uint8_t* codes, uint8_t* mults) {
    const float* x = v + (size_t)(row - row0) * r.dim;
    float m = 0.0f;
    for (int j = lane; j < r.dim; j += 32) m = absmax_step(m, x[j]);
    m = warp_absmax(m);
    float up;
    const float scale = i4_row_scale(m, &up);
    for (int g = 0; g < r.groups; g++) {  // the row again, from cache
      const int j = g * kI4Group + lane;
      const float y = j < r.dim ? x[j] : 0.0f;
      const int mult = i4_group_mult(warp_absmax(absmax_step(0.0f, y)), up);
      i4_store_group(y, mult, scale, codes + g * 16, lane);
      if (lane == 0) mults[g] = (uint8_t)mult;
    }
    return scale;
  });
}

__global__ void __launch_bounds__(kWarps * 32) i4_pack_kernel(I4Rows r, int64_t row0, int64_t rows, const uint8_t* codes,
                                                              const uint8_t* mults, const float* scales) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31;
  i4_write_block(r, row0, rows, smem, [&](int64_t row, uint8_t* c, uint8_t* m) {
    const size_t at = (size_t)(row - row0) * r.groups;
    for (int i = lane; i < r.groups * 4; i += 32)
      reinterpret_cast<uint32_t*>(c)[i] = reinterpret_cast<const uint32_t*>(codes + at * 16)[i];
    for (int i = lane; i < r.groups; i += 32) m[i] = mults[at + i];
    return scales[row - row0];
  });
}

__global__ void __launch_bounds__(kWarps * 32) i4_unpack_kernel(I4Rows r, int64_t row0, int64_t rows, uint8_t* codes,
                                                                uint8_t* mults, float* scales) {
  const int lane = threadIdx.x & 31, G = r.groups, quads = (G + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (i >= rows) return;
  const int64_t row = row0 + i, block = row / 8;
  const int rr = (int)(row & 7);
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + (size_t)i * G * 16);
  for (int j = lane; j < G * 4; j += 32) out[j] = r.codes[(size_t)block * G * 32 + i4_word_at(j >> 2, rr * 4 + (j & 3), G)];
  for (int g = lane; g < G; g += 32)
    mults[(size_t)i * G + g] = (uint8_t)(r.mults[((size_t)block * quads + (g >> 2)) * 8 + rr] >> (8 * (g & 3)));
  if (lane == 0) scales[i] = r.scales[row];
}

// ---------------------------------------------------------------------------
// Scores. A warp scores 32 rows at a time on the 8-bit matrix instruction: the
// rows' codes (as unsigned nibbles) are its left operand, eight queries its
// right one, one group of 32 values its depth. Each group's whole dots start
// at -8 * sum(q8), the nibbles' offset, and enter the totals times the rows'
// multipliers: a row's 16 bytes cost the same few instructions for one query
// as for eight, and the rows' bytes bound the kernel. The queries' fragments
// lie in shared memory, 16 bytes a lane and group. The words of the next four
// groups are loaded while the present ones are multiplied.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c0, int c1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1));
}

// Four blocks of 8 rows, up to four groups: the lane's words and multipliers.
struct I4Frag {
  uint32_t w[4][4];
  uint32_t m[4];
};

__device__ __forceinline__ void i4_load(I4Frag& f, const I4Rows& r, int64_t tile, int quad, int lane) {
  const int G = r.groups, full = G >> 2, quads = (G + 3) >> 2;
  const uint32_t* codes = r.codes + (size_t)tile * 4 * G * 32 + quad * 128;
  const uint32_t* mults = r.mults + ((size_t)tile * 4 * quads + quad) * 8 + (lane >> 2);
#pragma unroll
  for (int b = 0; b < 4; b++) {
    const uint32_t* at = codes + (size_t)b * G * 32;
    if (quad < full) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(at) + lane);
      f.w[b][0] = v.x, f.w[b][1] = v.y, f.w[b][2] = v.z, f.w[b][3] = v.w;
    } else {
      const int rest = G & 3;
#pragma unroll
      for (int j = 0; j < 3; j++) f.w[b][j] = j < rest ? __ldg(at + lane * rest + j) : 0u;
    }
    f.m[b] = __ldg(mults + (size_t)b * quads * 8);
  }
}

// Shared memory of a query set: fragments [groups][NT][32 lanes] uint4, scales.
template <int NT>
__host__ __device__ constexpr size_t i4_frag_bytes(int groups) { return (size_t)groups * NT * 512; }
inline size_t i4_query_bytes(int groups, int nt) { return (size_t)8 * nt * groups * (kI4Group + 4); }

// Quantize the M queries of a launch (a warp each) and lay out their fragments:
// lane 4 n + t gets query n's bytes 4t.. and 16 + 4t.. of the group, and the
// start values of queries 2t and 2t + 1. Queries past M are zero.
template <int NT>
__device__ __forceinline__ void i4_queries(const float* q, int M, int dim, int groups, unsigned char* scratch, uint4* frags,
                                           float* scales) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int8_t* q8 = reinterpret_cast<int8_t*>(scratch);
  int* off = reinterpret_cast<int*>(scratch + (size_t)8 * NT * groups * kI4Group);
  for (int m = warp; m < 8 * NT; m += kWarps) {
    const float* qm = q + (size_t)m * dim;
    const int d = m < M ? dim : 0;
    const float s = i4_quantize_query([&](int i) { return __ldg(qm + i); }, d, groups, q8 + (size_t)m * groups * kI4Group,
                                      off + m * groups, lane);
    if (lane == 0) scales[m] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < groups * NT * 32; i += kWarps * 32) {
    const int l = i & 31, nt = (i >> 5) % NT, g = (i >> 5) / NT, n = nt * 8 + (l >> 2), t = l & 3;
    const int8_t* at = q8 + ((size_t)n * groups + g) * kI4Group + 4 * t;
    frags[i] = make_uint4(*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + 16),
                          (uint32_t)off[(nt * 8 + 2 * t) * groups + g], (uint32_t)off[(nt * 8 + 2 * t + 1) * groups + g]);
  }
  __syncthreads();
}

struct I4ScoreArgs {
  I4Rows r;
  int64_t tile0, tiles, rows;  // tiles [tile0, tile0 + tiles), of which `rows` rows are real
  const float* q;
  int M;
  float* dst;  // scores
  int64_t ld;
  uint32_t* best;  // or the tiles' best ranks [M][tiles]
  uint32_t id_base;
  const uint64_t* keep;
  int64_t keep_nbits;
};

template <int NT, bool TOPK>
__global__ void __launch_bounds__(kWarps * 32) i4_score_kernel(I4ScoreArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_scale[8 * NT];
  const I4Rows& r = p.r;
  const int G = r.groups, quads = (G + 3) >> 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* frags = reinterpret_cast<uint4*>(smem);
  if (TOPK) pdl_launch_dependents();
  i4_queries<NT>(p.q, p.M, r.dim, G, smem + i4_frag_bytes<NT>(G), frags, s_scale);

  const int64_t step = (int64_t)gridDim.x * kWarps;
  int64_t tile = (int64_t)blockIdx.x * kWarps + warp;
  if (tile >= p.tiles) return;
  I4Frag next;
  i4_load(next, r, p.tile0 + tile, 0, lane);
  for (; tile < p.tiles; tile += step) {
    int tot[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) tot[a][n][e] = 0;
    for (int quad = 0; quad < quads; quad++) {
      const I4Frag f = next;
      const bool more = quad + 1 < quads;
      if (more || tile + step < p.tiles) i4_load(next, r, p.tile0 + (more ? tile : tile + step), more ? quad + 1 : 0, lane);
      const int depth = min(4, G - quad * 4);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (j >= depth) break;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint4 b = frags[((quad * 4 + j) * NT + n) * 32 + lane];
#pragma unroll
          for (int a = 0; a < 2; a++) {
            const uint32_t w0 = f.w[2 * a][j], w1 = f.w[2 * a + 1][j];
            const uint32_t op[4] = {w0 & 0x0F0F0F0Fu, w1 & 0x0F0F0F0Fu, (w0 >> 4) & 0x0F0F0F0Fu, (w1 >> 4) & 0x0F0F0F0Fu};
            int d[4];
            mma_u8s8(d, op, b.x, b.y, (int)b.z, (int)b.w);
            const int m0 = (int)((f.m[2 * a] >> (8 * j)) & 255u), m1 = (int)((f.m[2 * a + 1] >> (8 * j)) & 255u);
            tot[a][n][0] += m0 * d[0];
            tot[a][n][1] += m0 * d[1];
            tot[a][n][2] += m1 * d[2];
            tot[a][n][3] += m1 * d[3];
          }
        }
      }
    }
    // lane 4 r + t: rows r, r + 8, r + 16, r + 24 of the tile, queries 2t and 2t + 1
    const int64_t row0 = tile * kI4Tile;
    float scale[4];
#pragma unroll
    for (int b = 0; b < 4; b++) scale[b] = __ldg(r.scales + p.tile0 * kI4Tile + row0 + b * 8 + (lane >> 2));
    uint32_t alive = p.rows - row0 >= kI4Tile ? 0xFFFFFFFFu : (1u << (int)(p.rows - row0)) - 1u;
    if (TOPK && p.keep) alive &= keep_bits32(p.keep, p.keep_nbits, (uint64_t)p.id_base + (uint64_t)row0);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int m = n * 8 + 2 * (lane & 3) + c;
        const float qs = s_scale[m];
        uint32_t best = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float s = w8a8_score(tot[b >> 1][n][(b & 1) * 2 + c], qs, scale[b]);
          const int i = b * 8 + (lane >> 2);
          if (TOPK) {
            if (((alive >> i) & 1u) && s == s) best = max(best, score_to_ord(s));
          } else if (m < p.M && ((alive >> i) & 1u)) {
            p.dst[(size_t)m * p.ld + row0 + i] = s;
          }
        }
        if (TOPK) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
          if (lane < 4 && m < p.M) p.best[(size_t)m * p.tiles + tile] = best;
        }
      }
  }
}

// ---------------------------------------------------------------------------
// Top-k. Rank the tiles by (best score desc, tile asc), which is the order of
// their best rows' (score desc, index asc). The k best tiles hold the top k:
// their best rows are k rows, so the k-th best row is no worse than the k-th
// tile's best, and a row that good lies in a tile that good. So the score pass
// writes one rank for 32 rows instead of 32 scores, and these k tiles are
// scored again, row by row: k * 32 rows at most, whatever n is and however
// many scores are equal.
// A cluster per query: the threshold among the tiles, the list of tiles, their
// rows' keys, and the last sort, by the CTA of rank 0.
// ---------------------------------------------------------------------------
constexpr int kTopThreads = 512;
constexpr int kTopCluster = 8;
constexpr int kTopSort = 4096;        // keys that a sort takes: two lists of the largest k
constexpr int kTopHeld = 24 * 1024;   // tile ranks a CTA keeps in shared memory (more are read again in each pass)

struct I4SelectArgs {
  I4Rows r;
  int64_t tiles;
  int M, k;
  const float* q;
  uint32_t id_base;
  const uint64_t* keep;
  int64_t keep_nbits;
  const uint32_t* best;
  uint32_t* list;
  uint64_t* cand;
  int64_t cand_cap;
  uint64_t* out;
  int held;  // whether a CTA's ranks fit in shared memory
};

__global__ void __launch_bounds__(kTopThreads) i4_select_kernel(I4SelectArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ KthShared s_kth;
  __shared__ float s_scale;
  __shared__ uint32_t s_count;
  const I4Rows& r = p.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, y = blockIdx.y, G = r.groups;
  const uint32_t rank = cluster_rank(), nranks = cluster_size();
  int8_t* q8 = reinterpret_cast<int8_t*>(smem);             // [G * 32]
  int* off = reinterpret_cast<int*>(q8 + G * kI4Group);     // [G]
  // the held ranks, later the sort's keys
  uint32_t* held = reinterpret_cast<uint32_t*>(smem + ((G * (kI4Group + 4) + 15) & ~15));
  if (warp == 0) {
    const float* q = p.q + (size_t)y * r.dim;
    const float s = i4_quantize_query([&](int i) { return __ldg(q + i); }, r.dim, G, q8, off, lane);
    if (lane == 0) s_scale = s;
  }
  if (tid == 0) s_count = 0;
  pdl_wait_prior();  // the tiles' ranks
  const int64_t t0 = p.tiles * rank / nranks, t1 = p.tiles * (rank + 1) / nranks;
  const int n = (int)(t1 - t0);
  const uint32_t* mine = p.best + (size_t)y * p.tiles + t0;
  uint32_t some = 0;
  for (int i = tid; i < n; i += kTopThreads) {
    const uint32_t o = __ldcg(mine + i);
    some += o != 0;
    if (p.held) held[i] = o;
  }
  some = __reduce_add_sync(0xffffffffu, some);
  if (lane == 0) s_kth.warp_gt[warp] = some;
  __syncthreads();
  if (tid == 0) {
    uint32_t sum = 0;
    for (int w = 0; w < kTopThreads / 32; w++) sum += s_kth.warp_gt[w];
    s_kth.gt = sum;
  }
  cluster_sync();
  uint32_t all = 0;  // tiles with a row to offer
  for (uint32_t c = 0; c < nranks; c++) all += ld_cluster_u32(smem_u32(&s_kth.gt), c);
  const uint32_t need = min((uint32_t)p.k, all);
  uint32_t* list = p.list + (size_t)y * kI4MaxK;
  uint32_t t = 0, ties = 0;
  cluster_sync();  // s_kth.gt is written again
  if (need > 0) {
    auto get = [&](int i) { return p.held ? held[i] : __ldcg(mine + i); };
    cluster_kth(get, n, need, &s_kth, nranks, &t, &ties);
    cluster_place(get, n, t, ties, &s_kth, rank, nranks, [&](uint32_t at, int i) { list[at] = (uint32_t)(t0 + i); });
  }
  cluster_sync();  // the list is complete
  // k tiles bound the top k from below; fewer tiles offer every row they have
  const uint32_t floor = need == (uint32_t)p.k ? t : 0u;

  // a warp per tile, a lane per row
  const uint32_t count_at = smem_u32(&s_count);
  uint64_t* cand = p.cand + (size_t)y * p.cand_cap;
  const int quads = (G + 3) / 4;
  for (uint32_t i = rank * (kTopThreads / 32) + warp; i < need; i += nranks * (kTopThreads / 32)) {
    const int64_t tile = __ldcg(list + i), row = tile * kI4Tile + lane, block = row / 8;
    const uint32_t* codes = r.codes + (size_t)block * G * 32;
    const uint32_t* mults = r.mults + (size_t)block * quads * 8 + (lane & 7);
    int dot = 0;
    for (int g = 0; g < G; g++) {
      int acc = off[g];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const uint32_t word = __ldg(codes + i4_word_at(g, (lane & 7) * 4 + w, G));
        const int* qg = reinterpret_cast<const int*>(q8 + g * kI4Group);
        acc = i4_dot_word(word, qg[w], qg[4 + w], acc);
      }
      dot += (int)((__ldg(mults + (g >> 2) * 8) >> (8 * (g & 3))) & 255u) * acc;
    }
    const float s = w8a8_score(dot, s_scale, __ldg(r.scales + row));
    const uint64_t id = (uint64_t)p.id_base + (uint64_t)row;
    const bool ok = row < r.n && s == s && score_to_ord(s) >= floor && (!p.keep || keep_bit(p.keep, p.keep_nbits, id));
    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
    if (mask) {
      uint32_t base = 0;
      if (lane == 0) {
        uint32_t a;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(count_at));
        asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(base) : "r"(a), "r"((uint32_t)__popc(mask)) : "memory");
      }
      base = __shfl_sync(0xffffffffu, base, 0);
      if (ok) cand[base + __popc(mask & lanemask_lt())] = make_key(s, (uint32_t)id);
    }
  }
  cluster_sync();  // the candidates are complete; no CTA reads another's shared memory after this
  if (rank != 0) return;

  // sort what there is, at most kTopSort keys at a time behind the best k so far
  uint64_t* keys = reinterpret_cast<uint64_t*>(held);
  const int total = (int)s_count;
  int have = 0;
  for (int at = 0; at < total || have == 0;) {
    const int take = min(total - at, kTopSort - have);
    int n2 = 2;
    while (n2 < have + take) n2 <<= 1;
    for (int i = tid; i < n2 - have; i += kTopThreads) keys[have + i] = i < take ? __ldcg(cand + at + i) : kEmptyKey;
    __syncthreads();
    bitonic_sort_desc(keys, n2);
    at += take;
    have = min(have + take, p.k);
    if (at >= total) break;
  }
  for (int i = tid; i < p.k; i += kTopThreads) p.out[(size_t)y * p.k + i] = i < have ? keys[i] : kEmptyKey;
}

template <int NT, bool TOPK>
cudaError_t score_launch(const I4ScoreArgs& p, int32_t sm_count, cudaStream_t stream) {
  const size_t smem = i4_frag_bytes<NT>(p.r.groups) + i4_query_bytes(p.r.groups, NT);
  auto fn = i4_score_kernel<NT, TOPK>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  int ctas = 0;
  e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, fn, kWarps * 32, smem);
  if (e != cudaSuccess) return e;
  const int64_t need = (p.tiles + kWarps - 1) / kWarps, most = (int64_t)sm_count * (ctas > 0 ? ctas : 1);
  fn<<<(unsigned)(need < most ? need : most), kWarps * 32, smem, stream>>>(p);
  return cudaGetLastError();
}

size_t block_smem(int groups) { return (size_t)8 * groups * 16 + (size_t)8 * ((groups + 3) / 4) * 4; }

}  // namespace

cudaError_t i4_quantize_launch(const I4Rows& r, int64_t row0, const float* v, int64_t rows, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const int64_t blocks = (row0 + rows + 7) / 8 - row0 / 8;
  i4_quantize_kernel<<<(unsigned)blocks, kWarps * 32, block_smem(r.groups), stream>>>(r, row0, v, rows);
  return cudaGetLastError();
}

cudaError_t i4_pack_launch(const I4Rows& r, int64_t row0, int64_t rows, const uint8_t* codes, const uint8_t* mults,
                           const float* scales, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const int64_t blocks = (row0 + rows + 7) / 8 - row0 / 8;
  i4_pack_kernel<<<(unsigned)blocks, kWarps * 32, block_smem(r.groups), stream>>>(r, row0, rows, codes, mults, scales);
  return cudaGetLastError();
}

cudaError_t i4_unpack_launch(const I4Rows& r, int64_t row0, int64_t rows, uint8_t* codes, uint8_t* mults, float* scales,
                             cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  i4_unpack_kernel<<<(unsigned)((rows + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(r, row0, rows, codes, mults, scales);
  return cudaGetLastError();
}

cudaError_t i4_score_launch(const I4Rows& r, int64_t row0, int64_t rows, const float* q, int32_t M, float* dst,
                            int64_t ld, int32_t sm_count, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  if (row0 % kI4Tile != 0 || M <= 0 || M > kI4MaxBatch) return cudaErrorInvalidValue;
  I4ScoreArgs p{};
  p.r = r;
  p.tile0 = row0 / kI4Tile;
  p.tiles = i4_tiles(rows);
  p.rows = rows;
  p.q = q;
  p.M = M;
  p.dst = dst;
  p.ld = ld;
  return M <= 8 ? score_launch<1, false>(p, sm_count, stream) : score_launch<2, false>(p, sm_count, stream);
}

cudaError_t i4_topk_launch(const I4Rows& r, const I4TopK& p, int32_t sm_count, cudaStream_t stream) {
  if (p.M <= 0 || p.M > kI4MaxBatch || p.k <= 0 || p.k > kI4MaxK) return cudaErrorInvalidValue;
  I4ScoreArgs a{};
  a.r = r;
  a.tiles = i4_tiles(r.n);
  a.rows = r.n;
  a.q = p.q;
  a.M = p.M;
  a.best = p.best;
  a.id_base = p.id_base;
  a.keep = p.keep;
  a.keep_nbits = p.keep_nbits;
  cudaError_t e = p.M <= 8 ? score_launch<1, true>(a, sm_count, stream) : score_launch<2, true>(a, sm_count, stream);
  if (e != cudaSuccess) return e;
  I4SelectArgs s{};
  s.r = r;
  s.tiles = a.tiles;
  s.M = p.M;
  s.k = p.k;
  s.q = p.q;
  s.id_base = p.id_base;
  s.keep = p.keep;
  s.keep_nbits = p.keep_nbits;
  s.best = p.best;
  s.list = p.list;
  s.cand = p.cand;
  s.cand_cap = i4_cand(r.n);
  s.out = p.out;
  s.held = a.tiles <= (int64_t)kTopHeld * kTopCluster;
  const size_t smem = (((size_t)r.groups * (kI4Group + 4) + 15) & ~(size_t)15) + (size_t)kTopHeld * 4;
  static_assert(kTopHeld * 4 >= kTopSort * 8, "the sort reuses the held ranks");
  e = cudaFuncSetAttribute(i4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kTopCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kTopCluster, (unsigned)p.M);
  cfg.blockDim = dim3(kTopThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, i4_select_kernel, s);
}

}  // namespace fi8
