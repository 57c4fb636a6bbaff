// fi8_i4.cu -- FlatI4: scores of 4-bit rows (a matrix-vector product with
// group scales), the row quantizer, and the exact top-k.
#include <algorithm>

#include "fi8_cluster.cuh"
#include "fi8_cp_async.cuh"
#include "fi8_i4.cuh"
#include "fi8_i4q.cuh"
#include "fi8_kth.cuh"

namespace fi8 {

namespace {

constexpr int kWarps = 8;

// ---------------------------------------------------------------------------
// Row quantization and the row-major format.
// ---------------------------------------------------------------------------

// A CTA per block of 8 rows, a warp a row: its codes and multipliers are
// gathered in shared memory in the row-major format, then written interleaved.
// Rows of the block outside [row0, row0 + rows) stay as they are.
// The quantizer is bound by its instructions, some 130 a warp for a group of 32
// values (a lane a value: shuffles for the group's maximum and for its bytes, a
// division): 262,144 rows of 256 values 269 us (1.1 TB/s, 5.7 times what the bytes
// take), of 1024 values 908 us (1.3 TB/s, 4.8 times). Packing and unpacking move
// 1.0 to 1.3 TB/s for rows of 256 values and 2.7 of 1024, latency; the copies over
// the host link beside them are tens of times slower.
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
  uint32_t* codes = r.codes + (size_t)(block >> 2) * G * 128;
  uint32_t* mults = r.mults + (size_t)(block >> 2) * quads * 32;
  const int in_tile = (int)(block & 3) * 8;
  for (int i = threadIdx.x; i < G * 32; i += kWarps * 32) {
    const int g = i >> 5, rr = (i & 31) >> 2, t = i & 3;
    const int64_t at = block * 8 + rr;
    if (at >= row0 && at < row0 + rows) codes[i4_word_at(g, in_tile + rr, t, G)] = s_codes[rr * G * 4 + g * 4 + t];
  }
  for (int i = threadIdx.x; i < quads * 8; i += kWarps * 32) {
    const int rr = i & 7, quad = i >> 3;
    const int64_t at = block * 8 + rr;
    if (at >= row0 && at < row0 + rows)
      mults[quad * 32 + in_tile + rr] = reinterpret_cast<const uint32_t*>(s_mults)[rr * quads + quad];
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
      i4_store_group(y, mult, scale, lane, [&](int t, uint32_t w) { reinterpret_cast<uint32_t*>(codes)[g * 4 + t] = w; });
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
  const int64_t row = row0 + i, tile = row / kI4Tile;
  const int rr = (int)(row % kI4Tile);
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + (size_t)i * G * 16);
  for (int j = lane; j < G * 4; j += 32) out[j] = r.codes[(size_t)tile * G * 128 + i4_word_at(j >> 2, rr, j & 3, G)];
  for (int g = lane; g < G; g += 32)
    mults[(size_t)i * G + g] = (uint8_t)(r.mults[((size_t)tile * quads + (g >> 2)) * 32 + rr] >> (8 * (g & 3)));
  if (lane == 0) scales[i] = r.scales[row];
}

// ---------------------------------------------------------------------------
// Scores. A warp scores 32 rows at a time on the 8-bit matrix instruction: the
// rows' codes (as unsigned nibbles) are its left operand, eight queries its
// right one, one group of 32 values its depth. Each group's whole dots start
// at -8 * sum(q8), the nibbles' offset, and enter the totals times the rows'
// multipliers: a row's 16 bytes cost the same few instructions for one query
// as for eight, and the rows' bytes bound the kernel. The queries' fragments
// lie in shared memory, 16 bytes a lane and group. A warp's words pass through
// a ring of its own, a few quads (four groups) deep, filled by asynchronous
// copies; nothing but the warp itself waits for it.
// Measured, on several GPUs: 3 queries over 1,000,003 x 300 38 to 41 us (4.5 to 4.8
// TB/s), 8 queries over 2M x 1024 196 to 210 us (5.5 to 5.9 TB/s; a plain copy
// reaches 6.4), 16 queries over 1.5M x 256 57 us in a top-k (3.7 TB/s: there the
// products' instructions bound it), one over 100k x 384 7.8 us, of which launch and
// quantization are most.
// ---------------------------------------------------------------------------
// CTAs an SM at most, and quads of a warp's ring. Up to eight queries three CTAs
// of two quads keep the memory busy; with sixteen the products' registers leave
// room for two (measured, CTAs x quads: 8 queries 3 x 2 208 us, 3 x 3 220, 2 x 4
// 212 over 2M x 1024; 16 queries 2 x 4 78 us, 3 x 2 86 over 1.5M x 256).
template <int NT>
constexpr int kScoreCtas = NT == 1 ? 3 : 2;
template <int NT>
constexpr int kScoreStages = NT == 1 ? 2 : 4;
constexpr size_t kSmemSm = 228 * 1024;  // an SM's shared memory; a CTA takes 1 KB more than it asks for

// One quad of a tile: the lanes' words of four blocks of 8 rows (a tile's last
// quad may have fewer groups, [4 blocks][groups][32 lanes] words from the start
// of w), the rows' multipliers.
struct I4Stage {
  uint4 w[4][32];
  uint32_t m[32];
};

// The next quad to fetch for a warp: where its words and multipliers lie.
struct I4Cursor {
  const uint32_t* codes;  // of the quad, at the lane's first 16 bytes
  const uint32_t* mults;
  int quad;
};

__device__ __forceinline__ void i4_fetch(I4Stage& s, const I4Cursor& at, int G, int lane) {
  const int pieces = min(4, G - at.quad * 4);  // of 32 x 16 bytes: a group of four blocks each
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i < pieces) cp_async16(smem_u32(&s.w[i][lane]), at.codes + i * 128, true);
  if (lane < 8) cp_async16(smem_u32(&s.m[4 * lane]), at.mults, true);
}

struct I4ScoreArgs {
  I4Rows r;
  int64_t tile0, tiles, rows;  // tiles [tile0, tile0 + tiles), of which `rows` rows are real
  const float* q;
  int M;
  float* dst;  // scores
  int64_t ld;
  uint32_t* best;  // or the tiles' best ranks [M][best_ld]
  int64_t best_ld;
  uint32_t id_base;
  const uint64_t* keep;
  int64_t keep_nbits;
  uint32_t ring_at;  // byte offset of the rings in shared memory
};

template <int NT, bool TOPK>
__global__ void __launch_bounds__(kWarps * 32, kScoreCtas<NT>) i4_score_kernel(I4ScoreArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_scale[8 * NT];
  const I4Rows& r = p.r;
  const int G = r.groups, quads = (G + 3) >> 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int4* starts = reinterpret_cast<int4*>(smem);
  uint2* ops = reinterpret_cast<uint2*>(starts + (size_t)G * NT * 32);
  constexpr int kStages = kScoreStages<NT>;
  I4Stage* ring = reinterpret_cast<I4Stage*>(smem + p.ring_at) + warp * kStages;
  pdl_wait_prior();           // queries and rows may come from the kernel before
  pdl_launch_dependents();    // after the wait: what starts early now may read the queries

  // the copies run kStages - 1 quads ahead of the products, over the ends of tiles
  const int64_t step = (int64_t)gridDim.x * kWarps;
  int64_t tile = (int64_t)blockIdx.x * kWarps + warp, ahead = tile;
  const int64_t next_codes = (step - 1) * G * 128 + (G & 3) * 128 + ((G & 3) ? 0 : 512), next_mults = (step - 1) * quads * 32 + 32;
  I4Cursor cursor{r.codes + (size_t)(p.tile0 + tile) * G * 128 + lane * 4,
                  r.mults + (size_t)(p.tile0 + tile) * quads * 32 + 4 * lane, 0};
  int to = 0, from = 0;
  auto fetch = [&]() {
    if (ahead < p.tiles) i4_fetch(ring[to], cursor, G, lane);
    cp_async_commit();
    to = (to + 1) % kStages;
    if (++cursor.quad == quads) {  // from a tile's last quad to the next tile's first
      cursor.quad = 0;
      ahead += step;
      cursor.codes += next_codes;
      cursor.mults += next_mults;
    } else {
      cursor.codes += 512;
      cursor.mults += 32;
    }
  };
  // the first copies travel while the queries are quantized, unless the rings lie over that work's scratch
  const bool early = p.ring_at > i4_frag_bytes<NT>(G);
  if (early)
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) fetch();
  i4_queries<NT>(p.q, p.M, r.dim, G, smem + i4_frag_bytes<NT>(G), starts, ops, s_scale);
  starts += lane;
  ops += lane;
  if (!early)
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) fetch();
  for (; tile < p.tiles; tile += step) {
    // lane 4 r + t ends with rows r, r + 8, r + 16, r + 24 of the tile, queries 2t and 2t + 1
    const int64_t row0 = tile * kI4Tile;
    float scale[4];
#pragma unroll
    for (int b = 0; b < 4; b++) scale[b] = __ldg(r.scales + p.tile0 * kI4Tile + row0 + b * 8 + (lane >> 2));
    int tot[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) tot[a][n][e] = 0;
    for (int quad = 0; quad < quads; quad++) {
      fetch();
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const I4Stage& s = ring[from];
      uint32_t w[4][4], mult[4];
#pragma unroll
      for (int b = 0; b < 4; b++) mult[b] = s.m[b * 8 + (lane >> 2)];
      const int4* c = starts + quad * 4 * NT * 32;
      const uint2* b = ops + quad * 4 * NT * 32;
      const int depth = G - quad * 4;
      if (depth >= 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint4 v = s.w[i][lane];
          w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
        }
        __syncwarp();  // the stage may be filled again
        i4_multiply<NT, 4>(tot, w, mult, c, b);
      } else {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(s.w) + lane;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 3; j++) w[i][j] = j < depth ? words[(i * depth + j) * 32] : 0u;
        __syncwarp();
        if (depth == 1) i4_multiply<NT, 1>(tot, w, mult, c, b);
        else if (depth == 2) i4_multiply<NT, 2>(tot, w, mult, c, b);
        else i4_multiply<NT, 3>(tot, w, mult, c, b);
      }
      from = (from + 1) % kStages;
    }
    uint32_t alive = p.rows - row0 >= kI4Tile ? 0xFFFFFFFFu : (1u << (int)(p.rows - row0)) - 1u;
    if (TOPK && p.keep) alive &= keep_bits32(p.keep, p.keep_nbits, (uint64_t)p.id_base + (uint64_t)row0);
    alive >>= lane >> 2;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int m = n * 8 + 2 * (lane & 3) + c;
        const float qs = s_scale[m];
        // a NaN, and a row that is not there, loses against every score
        float best = __uint_as_float(0x7FFFFFFFu);
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const int dot = tot[b >> 1][n][(b & 1) * 2 + c];
          const bool there = (alive >> (b * 8)) & 1u;
          float s = __fmul_rn(__fmul_rn(__int2float_rn(dot), qs), scale[b]);
          if (qs == 0.0f) s = 0.0f;
          if (TOPK) {
            best = fmaxf(best, there ? s : best);
          } else if (m < p.M && there) {
            p.dst[(size_t)m * p.ld + row0 + b * 8 + (lane >> 2)] = s == s ? s : w8a8_score(dot, qs, scale[b]);
          }
        }
        if (TOPK) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
          if (lane < 4 && m < p.M) p.best[(size_t)m * p.best_ld + tile] = best == best ? score_to_ord(best) : 0u;
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
// The same holds for runs of tiles: the k best runs hold the k best tiles. So
// a cluster per query reduces the tiles' ranks to runs (all its CTAs), the CTA
// of rank 0 picks the runs and then the tiles, all CTAs score the tiles' rows,
// and rank 0 sorts what is left. Few tiles need no runs; and where few of few
// tiles are picked, a CTA alone does it all, without a cluster's meetings.
// Bound by the latency of its dependent steps, not by bytes or operations. With
// the score pass: 14 us over 100k rows of 384 values, k = 10 (scores alone 8;
// a cluster took 2.8 longer), 280 to 304 us over 4M rows of 768, k = 100 (the scores' floor 256).
// ---------------------------------------------------------------------------
constexpr int kTopThreads = 512;  // of a CTA of a cluster
constexpr int kTopCluster = 8;
constexpr int kTopAlone = 1024;   // of a CTA that works alone: at most kTopDirect tiles, of which kTopAlonePicks are scored
constexpr int kTopAlonePicks = 64;
constexpr int kTopSort = 4096;        // keys that a sort takes: two lists of the largest k
constexpr int kTopHeld = 48 * 1024;   // ranks that rank 0 can hold in shared memory (more are read again in each step)
constexpr int kTopDirect = 8 * 1024;  // tiles that it picks from without runs
static_assert(kTopAlonePicks * kI4Tile <= kTopSort, "one sort, in place, of a lone CTA's candidates");

struct I4SelectArgs {
  I4Rows r;
  int64_t tiles;
  int k;
  const float* q;
  uint32_t id_base;
  const uint64_t* keep;
  int64_t keep_nbits;
  const uint32_t* best;  // [M][best_ld]
  int64_t best_ld;
  uint32_t* list;
  uint64_t* cand;
  int64_t cand_cap;
  uint64_t* out;
  int run;   // tiles of a run, a power of two from 8; 0: none
  int held;  // ranks held in shared memory
};

template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) i4_select_kernel(I4SelectArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ KthShared s_kth;
  __shared__ float s_scale;
  __shared__ uint32_t s_count, s_floor, s_picks;
  __shared__ uint32_t s_list[CLUSTER ? 1 : kTopAlonePicks];
  const I4Rows& r = p.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, y = blockIdx.y, G = r.groups;
  const uint32_t rank = CLUSTER ? cluster_rank() : 0, nranks = CLUSTER ? cluster_size() : 1;
  auto sync = [] {
    if (CLUSTER) cluster_sync();
    else __syncthreads();
  };
  int8_t* q8 = reinterpret_cast<int8_t*>(smem);             // [G * 32]
  int* off = reinterpret_cast<int*>(q8 + G * kI4Group);     // [G], 16-byte aligned
  // the runs' or tiles' ranks, later the sort's keys
  uint32_t* held = reinterpret_cast<uint32_t*>(smem + ((G * (kI4Group + 4) + 15) & ~15));
  uint32_t* s_runs = held + p.held;  // [i4_picks(kI4MaxK)]
  if (CLUSTER && p.run) cluster_arrive();
  __syncwarp();
  {
    const float* q = p.q + (size_t)y * r.dim;
    const float s = i4_quantize_query([&](int i) { return __ldg(q + i); }, r.dim, G, q8, off, lane, warp, THREADS / 32);
    if (tid == 0) s_scale = s;
  }
  if (tid == 0) s_count = 0;
  pdl_wait_prior();  // the tiles' ranks
  const uint32_t* best = p.best + (size_t)y * p.best_ld;
  const int runs = p.run ? (int)((p.tiles + p.run - 1) / p.run) : 0;
  if (CLUSTER && p.run) {
    // a few lanes reduce a run; the first of them writes to rank 0
    cluster_wait();
    const int lanes = min(8, p.run >> 2), per = p.run / (4 * lanes), sub = tid & (lanes - 1);
    const int step = (int)nranks * (THREADS / lanes);
    for (int base = (int)rank * (THREADS / lanes) + tid / lanes; base - tid / lanes < runs; base += 4 * step) {
      uint32_t top[4] = {0, 0, 0, 0};
      for (int i = 0; i < per; i++) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int run = base + u * step;
          const int64_t at = (int64_t)run * p.run + (i * lanes + sub) * 4;
          v[u] = run < runs && at < p.tiles ? __ldcg(reinterpret_cast<const uint4*>(best + at)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 4; u++) top[u] = max(top[u], max(max(v[u].x, v[u].y), max(v[u].z, v[u].w)));
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        for (int o = 1; o < lanes; o <<= 1) top[u] = max(top[u], __shfl_xor_sync(0xffffffffu, top[u], o));
        if (base + u * step < runs && sub == 0) st_cluster_u32(smem_u32(held + base + u * step), 0, top[u]);
      }
    }
    cluster_sync();
  }
  const uint32_t need = (uint32_t)min((int64_t)p.k, p.tiles);
  uint32_t* list = CLUSTER ? p.list + (size_t)y * i4_picks(kI4MaxK) : s_list;
  if (rank == 0) {
    uint32_t picks, t;
    // in any order where no tie is left out
    auto choose = [&](auto get, int n, auto put) {
      const uint32_t limit = (uint32_t)i4_picks((int)need);
      if (need <= kKthFew / 2 && n > kKthList) {
        t = kth_floor(get, n, need, &s_kth);
        const Kth kth{t, 0xFFFFFFFFu, 0, -1, ScoreBins(0.0f, 0.0f, 1)};
        picks = kth_list(get, n, kth, &s_kth, [&](uint32_t at, int i) {
          if (at < limit) put(at, i);
        });
        if (picks <= limit) return;
        __syncthreads();  // more ranks reach the floor than may be picked
      }
      const Kth kth = kth_rank(get, n, need, limit, &s_kth);
      if (kth.ties == 0xFFFFFFFFu) kth_list(get, n, kth, &s_kth, put);
      else kth_place(get, n, kth, &s_kth, put);
      picks = kth.count;
      t = kth.t;
    };
    if (CLUSTER && p.run) {
      const uint32_t best_runs = (uint32_t)min(p.k, runs);
      auto get_run = [&](int i) { return held[i]; };
      // some more where their tiles' ranks can be held
      const uint32_t most_runs = max(best_runs, min((uint32_t)i4_picks((int)best_runs), (uint32_t)p.held / p.run));
      const Kth kth = kth_rank(get_run, runs, best_runs, most_runs, &s_kth);
      kth_place(get_run, runs, kth, &s_kth, [&](uint32_t at, int i) { s_runs[at] = (uint32_t)i; });
      const int n = (int)kth.count * p.run, shift = __ffs(p.run) - 1;
      auto tile_of = [&](int i) { return (int64_t)s_runs[i >> shift] * p.run + (i & (p.run - 1)); };
      auto rank_of = [&](int i) {
        const int64_t tile = tile_of(i);
        return tile < p.tiles ? __ldcg(best + tile) : 0u;
      };
      const bool fits = n <= p.held;
      if (fits) {
        for (int i0 = tid; i0 < n; i0 += 8 * THREADS) {  // eight loads in flight
          uint32_t v[8];
#pragma unroll
          for (int u = 0; u < 8; u++) v[u] = i0 + u * THREADS < n ? rank_of(i0 + u * THREADS) : 0u;
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (i0 + u * THREADS < n) held[i0 + u * THREADS] = v[u];
        }
        __syncthreads();
      }
      auto get = [&](int i) { return fits ? held[i] : rank_of(i); };
      choose(get, n, [&](uint32_t at, int i) { list[at] = (uint32_t)tile_of(i); });
    } else {
      const int n = (int)p.tiles;
      for (int i0 = tid * 4; i0 < n; i0 += 4 * THREADS * 4) {  // four loads in flight
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int i = i0 + u * THREADS * 4;
          v[u] = i < n ? __ldcg(reinterpret_cast<const uint4*>(best + i)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (i0 + u * THREADS * 4 < n) *reinterpret_cast<uint4*>(held + i0 + u * THREADS * 4) = v[u];
      }
      __syncthreads();
      auto get = [&](int i) { return held[i]; };
      choose(get, n, [&](uint32_t at, int i) { list[at] = (uint32_t)i; });
    }
    if (tid == 0) {
      s_floor = need == (uint32_t)p.k ? t : 0u;  // fewer tiles than k offer every row
      s_picks = picks;
    }
  }
  sync();  // the list is complete
  const uint32_t floor = CLUSTER ? ld_cluster_u32(smem_u32(&s_floor), 0) : s_floor;
  const uint32_t picks = CLUSTER ? ld_cluster_u32(smem_u32(&s_picks), 0) : s_picks;

  // a warp per tile; lane 4 r + t has word t of rows r, r + 8, r + 16, r + 24
  const uint32_t count_at = smem_u32(&s_count);
  // a CTA alone keeps its candidates where the ranks were
  uint64_t* cand = CLUSTER ? p.cand + (size_t)y * p.cand_cap : reinterpret_cast<uint64_t*>(held);
  const int quads = (G + 3) / 4, t = lane & 3;
  for (uint32_t i = rank * (THREADS / 32) + warp; i < picks; i += nranks * (THREADS / 32)) {
    const int64_t tile = CLUSTER ? __ldcg(list + i) : list[i], row = tile * kI4Tile + t * 8 + (lane >> 2);
    if (tile >= p.tiles) continue;  // behind the last run's tiles, picked where nothing better was left
    const uint32_t* codes = r.codes + (size_t)tile * G * 128 + lane * 4;
    const uint32_t* mults = r.mults + (size_t)tile * quads * 32 + (lane >> 2);
    const float scale = __ldg(r.scales + row);
    int dot[4] = {0, 0, 0, 0};
    auto group = [&](uint32_t w, uint32_t m, int g, int& dot) {
      const int* qg = reinterpret_cast<const int*>(q8 + g * kI4Group) + t;
      dot += (int)m * i4_dot_word(w, qg[0], qg[4], t == 0 ? off[g] : 0);
    };
#pragma unroll 2
    for (int quad = 0; quad < G >> 2; quad++) {
      uint4 w[4];
      uint32_t m[4];
#pragma unroll
      for (int b = 0; b < 4; b++) w[b] = __ldg(reinterpret_cast<const uint4*>(codes + quad * 512 + b * 128));
#pragma unroll
      for (int b = 0; b < 4; b++) m[b] = __ldg(mults + quad * 32 + b * 8);
#pragma unroll
      for (int b = 0; b < 4; b++) {
        group(w[b].x, m[b] & 255u, quad * 4, dot[b]);
        group(w[b].y, (m[b] >> 8) & 255u, quad * 4 + 1, dot[b]);
        group(w[b].z, (m[b] >> 16) & 255u, quad * 4 + 2, dot[b]);
        group(w[b].w, m[b] >> 24, quad * 4 + 3, dot[b]);
      }
    }
    for (int g = G & ~3; g < G; g++)
#pragma unroll
      for (int b = 0; b < 4; b++)
        group(__ldg(codes - lane * 4 + i4_word_at(g, b * 8 + (lane >> 2), t, G)),
              (__ldg(mults + (g >> 2) * 32 + b * 8) >> (8 * (g & 3))) & 255u, g, dot[b]);
#pragma unroll
    for (int b = 0; b < 4; b++) {
      dot[b] += __shfl_xor_sync(0xffffffffu, dot[b], 1);
      dot[b] += __shfl_xor_sync(0xffffffffu, dot[b], 2);
    }
    const float s = w8a8_score(t == 0 ? dot[0] : t == 1 ? dot[1] : t == 2 ? dot[2] : dot[3], s_scale, scale);
    const uint64_t id = (uint64_t)p.id_base + (uint64_t)row;
    const bool ok = row < r.n && s == s && score_to_ord(s) >= floor && (!p.keep || keep_bit(p.keep, p.keep_nbits, id));
    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
    if (mask) {
      uint32_t base = 0;
      if (lane == 0) {
        base = CLUSTER ? atom_cluster_add(count_at, 0, (uint32_t)__popc(mask)) : atomicAdd(&s_count, (uint32_t)__popc(mask));
      }
      base = __shfl_sync(0xffffffffu, base, 0);
      if (ok) cand[base + __popc(mask & lanemask_lt())] = make_key(s, (uint32_t)id);
    }
  }
  sync();  // the candidates are complete; no CTA reads another's shared memory after this
  if (rank != 0) return;

  uint64_t* keys = reinterpret_cast<uint64_t*>(held);
  uint64_t* out = p.out + (size_t)y * p.k;
  const int total = (int)s_count;
  if (total <= THREADS) {
    // one key a thread: its place is the number of larger keys
    const uint64_t mine = tid < total ? CLUSTER ? __ldcg(cand + tid) : cand[tid] : kEmptyKey;
    if (CLUSTER) {
      keys[tid] = mine;
      __syncthreads();
    }
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < total; i++) place += keys[i] > mine;
    if (tid < total && place < p.k) out[place] = mine;
    for (int i = total + tid; i < p.k; i += THREADS) out[i] = kEmptyKey;
    return;
  }
  // sort what there is, at most kTopSort keys at a time behind the best k so far
  int have = 0;
  for (int at = 0; at < total || have == 0;) {
    const int take = min(total - at, kTopSort - have);
    int n2 = 2;
    while (n2 < have + take) n2 <<= 1;
    for (int i = tid; i < n2 - have; i += THREADS) keys[have + i] = i < take ? CLUSTER ? __ldcg(cand + at + i) : cand[at + i] : kEmptyKey;
    __syncthreads();
    bitonic_sort_desc(keys, n2);
    at += take;
    have = min(have + take, p.k);
    if (at >= total) break;
  }
  for (int i = tid; i < p.k; i += THREADS) out[i] = i < have ? keys[i] : kEmptyKey;
}

template <int NT, bool TOPK>
cudaError_t score_launch(I4ScoreArgs p, int32_t sm_count, cudaStream_t stream) {
  // Fragments, the queries' scratch, the rings; over the scratch where the CTAs
  // would not fit otherwise.
  const size_t frags = i4_frag_bytes<NT>(p.r.groups), scratch = i4_query_bytes(p.r.groups, NT), ring = sizeof(I4Stage) * kScoreStages<NT> * kWarps;
  const size_t apart = frags + (scratch + 15) / 16 * 16 + ring;
  const bool early = apart + 1024 <= kSmemSm / kScoreCtas<NT>;
  p.ring_at = (uint32_t)(early ? apart - ring : frags);
  const size_t smem = early ? apart : frags + (ring > scratch ? ring : scratch);
  const int64_t fit = (int64_t)(kSmemSm / (smem + 1024)), ctas = std::min<int64_t>(fit, kScoreCtas<NT>);
  const int64_t need = (p.tiles + kWarps - 1) / kWarps, most = (int64_t)sm_count * ctas;
  return launch_pdl(i4_score_kernel<NT, TOPK>, dim3((unsigned)(need < most ? need : most)), dim3(kWarps * 32), smem, stream, p);
}

size_t block_smem(int groups) { return (size_t)8 * groups * 16 + (size_t)8 * ((groups + 3) / 4) * 4; }

}  // namespace

// The limit is a property of the function on a device, so every index sets the
// same one.
cudaError_t i4_init() {
  const int most = 227 * 1024 - 1024;  // beside the score kernels' static shared memory
  cudaError_t e = cudaFuncSetAttribute(i4_score_kernel<1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(i4_score_kernel<1, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(i4_score_kernel<2, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(i4_score_kernel<2, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  const int beside = 227 * 1024 - 12 * 1024;  // beside the select kernels' static shared memory
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(i4_select_kernel<kTopThreads, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, beside);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(i4_select_kernel<kTopAlone, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, beside);
  return e;
}

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
  if (row0 % kI4Tile != 0 || M <= 0 || M > i4_batch(r.groups)) return cudaErrorInvalidValue;
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
  if (p.M <= 0 || p.M > i4_batch(r.groups) || p.k <= 0 || p.k > kI4MaxK) return cudaErrorInvalidValue;
  I4ScoreArgs a{};
  a.r = r;
  a.tiles = i4_tiles(r.n);
  a.rows = r.n;
  a.q = p.q;
  a.M = p.M;
  a.best = p.best;
  a.best_ld = i4_best_ld(r.n);
  a.id_base = p.id_base;
  a.keep = p.keep;
  a.keep_nbits = p.keep_nbits;
  cudaError_t e = p.M <= 8 ? score_launch<1, true>(a, sm_count, stream) : score_launch<2, true>(a, sm_count, stream);
  if (e != cudaSuccess) return e;
  I4SelectArgs s{};
  s.r = r;
  s.tiles = a.tiles;
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
  s.best_ld = a.best_ld;
  // Runs of about sqrt(tiles / k) tiles: as many runs to pick from as tiles in
  // the picked runs. Fewer and longer ones where the runs would not fit.
  if (a.tiles > kTopDirect)
    for (s.run = 8; a.tiles > (int64_t)s.run * s.run * 2 * p.k || a.tiles > (int64_t)s.run * kTopHeld;) s.run *= 2;
  int64_t held = s.run ? (a.tiles + s.run - 1) / s.run : (a.tiles + 3) / 4 * 4;
  if (s.run) held = std::max<int64_t>(held, std::min<int64_t>((int64_t)i4_picks(p.k) * s.run, kTopHeld));
  s.held = (int)std::max<int64_t>(held, kTopSort * 2);
  const size_t smem = (((size_t)r.groups * (kI4Group + 4) + 15) & ~(size_t)15) + ((size_t)s.held + (s.run ? i4_picks(p.k) : 0)) * 4;
  if (!s.run && i4_picks(p.k) <= kTopAlonePicks) {
    // few tiles to look at: their rows are scored before a cluster would have met
    return launch_pdl(i4_select_kernel<kTopAlone, false>, dim3(1, (unsigned)p.M), dim3(kTopAlone), smem, stream, s);
  }
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
  return cudaLaunchKernelEx(&cfg, i4_select_kernel<kTopThreads, true>, s);
}

}  // namespace fi8
