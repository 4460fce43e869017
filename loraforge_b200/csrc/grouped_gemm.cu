// Matrix products grouped by expert, 16-bit operands, on tcgen05 + TMEM.  Rows r of group e
// (offsets[e] <= r < offsets[e+1]) belong to expert e:
//
//   forward   y[r, n]     = sum_k W[e, n, k] x[i(r), k]          i(r) = rows[r], or r
//   input     dx[r, k]    = sum_n W[e, n, k] dy[r, n]
//   weight    dW[e, n, k] = sum_{r of e} dy[r, n] x[i(r), k]
//
// One kernel for the three: D[feature, column] with 128 output features on the TMEM lanes (256
// in a CTA pair) and up to kNT columns, rows of the group (forward, input) or the N features of
// dy (weight).  Rows on the MMA's N side cost in steps of 16, so a ragged group pays at most 15
// rows of padding, and a lane's neighbours are neighbours in the output row: a warp stores 32
// adjacent features of one row at a time.
//
//   mode      A (lanes)                     B (columns)          contraction
//   forward   W[e], K-major                 x rows, K-major      K
//   input     W[e], MN-major (k on lanes)   dy rows, K-major     N
//   weight    x rows, MN-major              dy rows, MN-major    the group's rows
//
// Nothing is transposed in memory: MN-major operands are read as they lie through the
// shared-memory descriptor.  Steps past K, N or a group's last row read zeros (out of bounds for
// the tensor map, or a row index that is), so a neighbouring group's infinities never reach a
// sum.  x's rows by token: with few rows a group gather4 loads fetch them.  Those move about one
// 128-byte row per 20 cycles and SM, a third of what the wide tiles take (8 experts, 16384 rows,
// 4096 -> 14336: 4340 us against 1475 with rows in order), so for more rows gather_rows_kernel
// copies them into the caller's workspace first (2 x 134 MB there, 35 us).
//
// Per CTA: warp 0 loads 64-deep stages into a ring, warp 1 issues the MMAs and owns the TMEM
// (two accumulators, so a tile's stores overlap the next tile's MMAs), warps 2-5 store (2-9 for short
// contractions).  The grid is persistent and computes its tile list from `offsets` on the device.
//
//   wide    CTA pairs (cta_group::2), 256 x 256 tiles: each CTA loads half of both operands.
//   narrow  one CTA, up to 128 features x up to 32 or 64 rows, for groups of few rows, where the
//           weights' bytes are the cost (32: three more stages of weights in flight); the
//           contraction can be split over a cluster of CTAs, whose partial sums are added in
//           rank order through distributed shared memory.
//
// Measured: 8 x 2048 rows, 4096 -> 14336: 1262 us (1524 TFLOP/s; later calls 1345-1480 under the
// power cap, as a dense library product of that size), input gradient 1455, weight gradient 1333;
// 64 experts of 2048 x 2048, 2 rows each: 83 us (537 MB of weights at 6.4 TB/s); dW of 64 experts of
// 1536 x 2048, 64 rows each: 136 us (403 MB written at 3.0 TB/s; a plain fill of them takes 105).
//
// Every wait is bounded (tma.cuh): an expiry stops every role at its next wait.
#include "experts.cuh"
#include "grouped.cuh"

namespace lfb {
namespace {

using namespace grouped;

enum Mode { kForward = 0, kInput = 1, kWeight = 2 };

constexpr int kStep = 64;             // contraction per stage: 128 bytes
constexpr int kABytes = 128 * 128;    // 128 features x 128 bytes (K-major), or two 64-feature boxes of 64 steps

struct GParams {
  const int32_t* offsets;  // [E + 1]
  const int32_t* rows;     // [R] or null
  Output out;
  int E, R, x_rows;
  int M, C;  // output features, contraction (forward K, input N; weight: the groups' rows)
  int N;     // weight: columns of D (dy's features)
  int elem_bf16, height, split, store_sets;
  int prepared;  // the grid before this one only put x's rows in order: all else can be read before it ends
  Bands bands;
  CUtensorMap a_map;     // forward: W boxes 64 k x 128 n; input: 64 k x 64 n; weight: x boxes 64 k x 64 rows
  CUtensorMap a_small;   // weight: 64 k x 8 rows
  CUtensorMap a_gather;  // weight: single x rows of 64 k
  CUtensorMap b_map;     // weight: dy boxes 64 n x 64 rows
  CUtensorMap b_small;   // weight: 64 n x 8 rows
  CUtensorMap b_gather;  // forward: single x rows; weight: single dy rows
  CUtensorMap b_rows[8]; // forward / input: rows of x or dy, 64 wide x 16, 32, .. 128 rows
};

template <int kCtas, int kNT>
struct Shape {
  static constexpr int kBRows = kNT / kCtas;  // a CTA's share of the columns
  static constexpr int kStageBytes = kABytes + kBRows * 128;
  static constexpr int kStoreSets = kCtas == 1 ? 1 : 2;     // at most
  static constexpr int kThreads = 64 + 128 * kStoreSets;  // warp 0 loads, warp 1 MMA, then sets of four that store
  static constexpr int kPartBytes = kCtas == 1 ? kNT * 128 * 4 : kStoreSets * 4 * kChunkBytes;  // sums, or the stores' staging
  static constexpr int kStages = stages_of(kStageBytes, kPartBytes);  // what is in flight hides some 2 us a load
  static constexpr int kColumns = 2 * kNT;  // TMEM
};

// Descriptor of an MN-major tile: boxes of 64 elements (128 bytes, swizzled) x kStep rows,
// the boxes 8 KiB apart, groups of 8 rows 1024 bytes apart.  16 steps are 2048 bytes.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t((kStep * 128) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

__device__ __forceinline__ uint32_t instruction(int bf16, int a_mn, int b_mn, int m, int n) {
  return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

struct Tile {
  int e, m0, end, n0, nt, valid, steps;  // features m0 .. end - 1; n0: first row (forward, input) or feature of dy
  int lo, hi;                            // the group's rows
};

// A role's walk over its CTA's tiles.
template <int kMode, int kCtas, int kNT>
struct Tiles {
  Walk walk;
  int each;  // rows of the group's column tiles
  __device__ __forceinline__ Tile at(const GParams& p, const int* bounds, const int* starts, int t) {
    if (walk.go(p.bands, bounds, starts, p.E, t, [&](int rows) { return ceil_div(kMode == kWeight ? p.N : rows, kNT); }))
      each = round_up(walk.nt == 1 ? walk.hi - walk.lo : ceil_div(walk.hi - walk.lo, walk.nt), 16);  // the group's rows in even tiles
    Tile x;
    x.e = walk.e, x.lo = walk.lo, x.hi = walk.hi;
    x.m0 = walk.m * p.height * kCtas;
    x.end = min(p.M, x.m0 + p.height * kCtas);
    if (kMode == kWeight) {
      x.n0 = walk.n * kNT;
      x.valid = min(kNT, p.N - x.n0);
      x.nt = round_up(x.valid, kNT / 2);  // whole 64-feature boxes in each CTA
      x.steps = ceil_div(x.hi - x.lo, kStep);
    } else {
      x.n0 = x.lo + walk.n * each;
      x.valid = min(each, x.hi - x.n0);
      x.nt = round_up(x.valid, 16);
      x.steps = ceil_div(p.C, kStep);
    }
    return x;
  }
};

template <int kMode, int kCtas, int kNT>
__global__ void __launch_bounds__((Shape<kCtas, kNT>::kThreads), 1) grouped_kernel(const __grid_constant__ GParams p) {
  using S = Shape<kCtas, kNT>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = smem;
  float* part = reinterpret_cast<float*>(ring + kStages * S::kStageBytes);  // narrow: [kNT][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * S::kStageBytes + S::kPartBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* part_full = acc_empty + 2;
  uint64_t* part_empty = part_full + 1;
  uint64_t* fin = part_empty + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(fin + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);
  int* scan = reinterpret_cast<int*>(tslot + 2);  // one int a warp
  int* bounds = scan + kMaxWarps;                         // [E + 1]
  int* starts = bounds + p.E + 1;                 // [E + 1]

  // Pair: rank 0 issues the MMAs of both CTAs.  Split: the cluster's CTAs share the contraction.
  const int cluster = kCtas == 2 ? 2 : p.split;
  const int rank = cluster > 1 ? int(cluster_rank()) : 0;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4 * p.store_sets * kCtas);
    }
    mbar_init(part_full, 4 * cluster);
    mbar_init(part_empty, 4 * cluster);
    mbar_init(fin, 1);
    fence_mbar_init();
    *abort = 0;
  }
  Tiles<kMode, kCtas, kNT> walk;
  if (!p.prepared) pdl_wait();
  if (warp == 1) alloc_tmem<kCtas>(tslot, S::kColumns);  // not while waiting for a grid that may want some too
  const int mtiles = p.bands.mt;
  list_tiles(p.offsets, p.E, p.R, bounds, starts, scan, [&](int rows) {
    return mtiles * ceil_div(kMode == kWeight ? p.N : rows, kNT);
  });
  tc_fence_before();
  __syncthreads();
  if (cluster > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  const int tiles = starts[p.E];
  const int first = int(blockIdx.x) / cluster, stride = int(gridDim.x) / cluster;

  if (kMode != kWeight) zero_rows(p.out, bounds[0], bounds[p.E], p.R);

  // The steps of a tile that this CTA takes.
  auto my_steps = [&](const Tile& x, int* ks0, int* ks1) {
    if (kCtas == 1 && cluster > 1) {
      const int each = ceil_div(x.steps, cluster);
      *ks0 = min(x.steps, rank * each);
      *ks1 = min(x.steps, *ks0 + each);
    } else {
      *ks0 = 0;
      *ks1 = x.steps;
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    const bool elected = elect_one();
    if (p.prepared) {
      if (kMode == kForward && lane == 0 && first < tiles) {
        const Tile x = walk.at(p, bounds, starts, first);
        for (int ks = 0; ks < min(x.steps, kAhead); ++ks)
          prefetch_3d(&p.a_map, ks * kStep, x.m0 + (kCtas == 2 ? rank * 128 : 0), x.e);
      }
      __syncwarp();
      walk = {};
      pdl_wait();
    }
    int it = 0;
    for (int t = first; t < tiles; t += stride) {
      const Tile x = walk.at(p, bounds, starts, t);
      const int m_cta = x.m0 + (kCtas == 2 ? rank * 128 : 0);
      const int share = x.nt / kCtas;  // columns this CTA loads
      const int n_cta = x.n0 + (kCtas == 2 ? rank * share : 0);
      int ks0, ks1;
      my_steps(x, &ks0, &ks1);
      // Forward: this lane's four rows of the tile (fixed over the steps).
      int row4[4];
      if (kMode == kForward && kCtas == 1 && p.rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = n_cta + 4 * lane + i;
          const int src = 4 * lane + i < share && r < x.hi ? p.rows[r] : -1;
          row4[i] = src >= 0 && src < p.x_rows ? src : p.x_rows;
        }
      }
      const bool boxed = kMode != kWeight && !(kMode == kForward && kCtas == 1 && p.rows);
      const int loaded = kMode == kWeight ? share : boxed ? round_up(share, 16) : round_up(x.valid, 4);
      const uint32_t whole = kCtas * uint32_t(p.height + loaded) * 128u;
      const CUtensorMap* b_rows = &p.b_rows[kMode == kWeight ? 0 : ceil_div(share, 16) - 1];
      bool ok = true;
      for (int ks = ks0; ks < ks1; ++ks, ++it) {
        const int st = it % kStages;
        ok = __all_sync(0xffffffffu, wait_here(&empty[st], (uint32_t(it / kStages) & 1u) ^ 1u, abort));
        if (!ok) break;
        const uint32_t a = smem_u32(ring + st * S::kStageBytes), b = a + kABytes;
        const uint32_t bar = kCtas == 2 ? mapa(&full[st], 0) : smem_u32(&full[st]);
        const int c = ks * kStep;
        // Weight: the rows of this step; the last one is loaded by 8 rows up to a multiple of 16.
        const int left = kMode == kWeight ? min(kStep, x.hi - x.lo - c) : kStep;
        const uint32_t bytes = left == kStep ? whole : whole / kStep * uint32_t(round_up(left, 16));
        const bool by_row = kMode == kForward && kCtas == 1 && p.rows;
        if (elected) {
          if (rank * (kCtas - 1) == 0) mbar_arrive_expect_tx(&full[st], bytes);
          if (kMode == kForward) {
            load_3d<kCtas>(a, &p.a_map, c, m_cta, x.e, bar);
          } else if (kMode == kInput) {
            load_3d<kCtas>(a, &p.a_map, m_cta, c, x.e, bar);
            load_3d<kCtas>(a + 8192, &p.a_map, m_cta + 64, c, x.e, bar);
          } else if (left == kStep) {
            load_2d<kCtas>(a, &p.a_map, m_cta, x.lo + c, bar);
            load_2d<kCtas>(a + 8192, &p.a_map, m_cta + 64, x.lo + c, bar);
            load_2d<kCtas>(b, &p.b_map, n_cta, x.lo + c, bar);
            if (share > 64) load_2d<kCtas>(b + 8192, &p.b_map, n_cta + 64, x.lo + c, bar);
          }
          // One box of the share's rows in steps of 16: small boxes cost the copy engine near 0.1 us
          // each, whatever their size (rows past the share are loaded and not used).
          if (kMode != kWeight && !by_row) load_2d<kCtas>(b, b_rows, c, n_cta, bar);
        }
        __syncwarp();
        if (by_row && 4 * lane < x.valid) gather4<kCtas>(b + lane * 512, &p.b_gather, c, row4, bar);
        if (kMode == kWeight && left < kStep) {
          // Boxes of 64 features x 8 rows: two of x (lanes 0-15), one or two of dy (lanes 16-31).
          const bool is_x = lane < 16;
          const int box = lane >> 3 & 1, unit = lane & 7;
          const int col = (is_x ? m_cta : n_cta) + 64 * box;
          const uint32_t dst = (is_x ? a : b) + box * 8192 + unit * 1024;
          const int r = x.lo + c + 8 * unit;
          if (is_x || box * 64 < share) {
            if (8 * unit + 8 <= left) {
              load_2d<kCtas>(dst, is_x ? &p.a_small : &p.b_small, col, r, bar);
            } else if (8 * unit < round_up(left, 16)) {  // rows past the group's last read zeros
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                int r4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) r4[i] = r + 4 * q + i < x.hi ? r + 4 * q + i : is_x ? p.x_rows : p.R;
                gather4<kCtas>(dst + q * 512, is_x ? &p.a_gather : &p.b_gather, col, r4, bar);
              }
            }
          }
          __syncwarp();
        }
      }
      if (!ok) break;
    }
    // A pair's CTA stays until the commits that arrive here from the other CTA have.
    if (kCtas == 2)
      for (int j = max(0, it - kStages); j < it; ++j) wait_here(&empty[j % kStages], uint32_t(j / kStages) & 1u, abort);
    // No load may still be landing when the CTA exits (only an expired wait leaves any).
    if (*abort && elected && rank * (kCtas - 1) == 0)
      for (int j = max(0, it - kStages); j < it; ++j) mbar_wait(&full[j % kStages], uint32_t(j / kStages) & 1u);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    if (rank * (kCtas - 1) == 0) {
      const bool elected = elect_one();
      int it = 0, count = 0;
      for (int t = first; t < tiles; t += stride) {
        const Tile x = walk.at(p, bounds, starts, t);
        int ks0, ks1;
        my_steps(x, &ks0, &ks1);
        if (ks0 >= ks1) continue;
        const int ab = count & 1;
        if (!__all_sync(0xffffffffu, wait_cluster(&acc_empty[ab], (uint32_t(count >> 1) & 1u) ^ 1u, abort))) break;
        ++count;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(ab * kNT);
        const uint32_t idesc = instruction(p.elem_bf16, kMode != kForward, kMode == kWeight, 128 * kCtas, x.nt);
        bool ok = true;
        for (int ks = ks0; ks < ks1; ++ks, ++it) {
          const int st = it % kStages;
          ok = __all_sync(0xffffffffu, wait_here(&full[st], uint32_t(it / kStages) & 1u, abort));
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(ring + st * S::kStageBytes);
          const uint64_t ad = kMode == kForward ? sw128_desc(sa) : mn_desc(sa);
          const uint64_t bd = kMode == kWeight ? mn_desc(sa + kABytes) : sw128_desc(sa + kABytes);
          constexpr int kAStep = kMode == kForward ? 2 : 128, kBStep = kMode == kWeight ? 128 : 2;
          const int subs = kMode == kWeight ? min(kStep, round_up(x.hi - x.lo - ks * kStep, 16)) / 16 : kStep / 16;
          if (elected) {
#pragma unroll
            for (int k = 0; k < kStep / 16; ++k)
              if (kMode != kWeight || k < subs)
                mma_f16<kCtas>(d, ad + kAStep * k, bd + kBStep * k, idesc, (ks > ks0 || k > 0) ? 1u : 0u);
            commit<kCtas>(&empty[st]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elected) commit<kCtas>(&acc_full[ab]);
        __syncwarp();
      }
      if (*abort && elected) {  // every MMA has retired before the TMEM columns are released
        commit<kCtas>(fin);
        mbar_wait(fin, 0);
      }
    }
  } else {
    // ------------------------------------------------------------ stores
    const int quarter = warp & 3;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t staging = smem_u32(part) + uint32_t((warp - 2) * kChunkBytes);
    int count = 0, parts = 0;
    for (int t = first; t < tiles; t += stride) {
      const Tile x = walk.at(p, bounds, starts, t);
      int ks0, ks1;
      my_steps(x, &ks0, &ks1);
      const bool live = ks1 > ks0;
      const int ab = count & 1;
      if (live) {
        if (!__all_sync(0xffffffffu, wait_here(&acc_full[ab], uint32_t(count >> 1) & 1u, abort))) break;
        ++count;
        tc_fence_after();
      }
      const uint32_t d = tmem + lanes + uint32_t(ab * kNT);
      const int f0 = x.m0 + (kCtas == 2 ? rank * 128 : 0) + quarter * 32;
      const int64_t row0 = kMode == kWeight ? int64_t(x.e) * p.N + x.n0 : x.n0;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (live && lane == 0) {
          if (kCtas == 2) arrive_cluster(mapa(&acc_empty[ab], 0));
          else mbar_arrive(&acc_empty[ab]);
        }
      };
      if (kCtas == 1 && cluster > 1) {
        if (!store_split(p.out, d, live, f0, x.end, row0, x.nt, x.valid, part, part_full, part_empty, parts, cluster, rank,
                         quarter, lane, abort, release))
          break;
        ++parts;
      } else {
        store_whole(p.out, d, live, f0, x.end, row0, x.nt, x.valid, staging, lane, (warp - 2) >> 2,
                    p.store_sets);
        release();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (cluster > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    free_tmem<kCtas>(tmem, S::kColumns);
  }
}

// out[r] = x[rows[r]], eight rows a block (a thread that divides its way to row and column for every
// 16 bytes took 8 us for 6000 rows of 4 KB).
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint4* x, int64_t stride, int x_rows,
                                                          const int32_t* rows, int words, int64_t R, uint4* out) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t r = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (r < R) copy_row(x, stride, x_rows, rows, r, words, out, threadIdx.x & 31);
}

int gather_rows(const void* x, int64_t x_stride, int64_t x_rows, const int32_t* rows, int64_t R, int64_t width,
                void* out, void* stream, const char* what) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  config.gridDim = dim3(unsigned((R + 7) / 8));
  config.blockDim = dim3(256);
  config.stream = static_cast<cudaStream_t>(stream);
  return launch_status(cudaLaunchKernelEx(&config, gather_rows_kernel, static_cast<const uint4*>(x), x_stride / 8,
                                          int(x_rows), rows, int(width / 8), R, static_cast<uint4*>(out)),
                       what);
}

template <int kCtas, int kNT>
int smem_of(int E) {
  using S = Shape<kCtas, kNT>;
  return 1024 + S::kStages * S::kStageBytes + S::kPartBytes + 512 + int(sizeof(int)) * (kMaxWarps + 2 + 2 * (E + 1));
}

template <int kMode, int kCtas, int kNT>
int clusters_at_once(Clusters* out) {
  const auto kernel = grouped_kernel<kMode, kCtas, kNT>;
  static int flags[64] = {};
  if (int rc = ensure_smem(kernel, smem_of<kCtas, kNT>(kMaxExperts), flags)) return rc;
  return clusters_of(kernel, (Shape<kCtas, kNT>::kThreads), smem_of<kCtas, kNT>(kMaxExperts), out);
}

// Pairs with a contraction of up to kShort store with eight warps a CTA instead of four, which do not
// keep up with the MMAs of so few steps.  16 experts, dW of 4096 x 2048: 128 rows each 94 us against
// 107, 768 rows 175 against 190, but 1024 rows 234 against 224, as the stores then come in the way of
// the loads; forward to 4096 features, 1024 rows each: 512 wide 94 against 98, 2048 wide 236 against 228.
constexpr int kShort = 768;

template <int kMode, int kCtas, int kNT>
int launch_grouped(GParams& p, int64_t tiles, void* stream, const char* what) {
  p.bands = bands_of(ceil_div(p.M, p.height * kCtas));
  const int cluster = kCtas == 2 ? 2 : p.split;
  p.store_sets = kCtas == 2 && (kMode == kWeight ? p.R / (p.E < p.R ? p.E : p.R) : p.C) <= kShort ? 2 : 1;
  Clusters clusters;
  if (int rc = clusters_at_once<kMode, kCtas, kNT>(&clusters)) return rc;
  const int grid = grid_of(clusters, tiles, cluster, what);
  if (!grid) return LF_E_CUDA;
  return launch_clusters(grouped_kernel<kMode, kCtas, kNT>, grid, 64 + 128 * p.store_sets, cluster,
                         smem_of<kCtas, kNT>(p.E), stream, what, p);
}

constexpr int kWideRows = 256, kNarrowRows = 64, kFewRows = 32;
constexpr char kNoWorkspace[] = "expert_linear: workspace missing, too small or not 16-byte aligned (see lf_expert_linear_workspace_bytes)";

// Groups of up to 24 rows on average take the narrow tiles.  64 experts of 2048 x 2048: 20 rows each
// 89 us against 91 in pairs, 40 rows 99 against 95, and 40 on average but unequal (the first expert
// has 580) 116 against 99, as narrow tiles read the weights again for every 64 rows.
bool narrow(int64_t E, int64_t R) { return R <= 24 * (E < R ? E : R); }

// Rows by index: with up to eight a group on average the loads gather them, else they are put in
// order first.  Two gather4 a stage, of four rows each, cost next to nothing beside the weights (64
// experts of 2048 x 2048, 2 rows each: 84 us against 83 with rows in order), four do (16 rows: 97
// against 86).
bool gather_in_loads(int64_t E, int64_t R) { return R <= 8 * (E < R ? E : R); }

int check_sizes(const char* what, int dtype, int E, int64_t R, int64_t N, int64_t K) {
  const int64_t limit = int64_t(1) << 31;
  if (dtype != LF_BF16 && dtype != LF_F16)
    return fail(LF_E_INVALID, (std::string(what) + ": operands must be BF16 or FP16").c_str());
  if (E < 1 || E > kMaxExperts || R < 0 || R >= limit - 256 || N < 1 || K < 1 || N % 8 || K % 8 || N >= limit - 256 ||
      K >= limit - 256)
    return fail(LF_E_INVALID,
                (std::string(what) + ": needs 1..1024 experts, widths that are multiples of 8, and rows that fit int32").c_str());
  // Tiles are counted in int32, also those of narrow tiles.
  const int64_t m = (N > K ? N : K) / 64 + 1;
  if ((R / kFewRows + E + 1) * m >= limit || (N / kWideRows + 1) * (K / 256 + 1) * int64_t(E) >= limit)
    return fail(LF_E_INVALID, (std::string(what) + ": too many tiles").c_str());
  return LF_OK;
}

bool good_rows(const void* p, int64_t stride, int64_t width) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= width;
}

bool encode_rows(CUtensorMap* map, CUtensorMapDataType type, const void* p, int64_t width, int64_t rows,
                 int64_t stride, int box_rows) {
  const cuuint64_t dims[2] = {cuuint64_t(width), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(stride) * 2};
  const cuuint32_t box[2] = {64, cuuint32_t(box_rows)};
  return encode_map(map, type, 2, p, dims, strides, box);
}

bool encode_row_boxes(CUtensorMap (&maps)[8], CUtensorMapDataType type, const void* p, int64_t width, int64_t rows,
                      int64_t stride, bool few) {
  bool ok = true;
  for (int i = 0; i < (few ? kNarrowRows / 16 : 8) && ok; ++i) ok = encode_rows(&maps[i], type, p, width, rows, stride, 16 * (i + 1));
  return ok;
}

bool encode_weights(CUtensorMap* map, CUtensorMapDataType type, const void* w, int64_t K, int64_t N, int64_t E,
                    int64_t row_stride, int64_t expert_stride, int box_rows) {
  const cuuint64_t dims[3] = {cuuint64_t(K), cuuint64_t(N), cuuint64_t(E)};
  const cuuint64_t strides[2] = {cuuint64_t(row_stride) * 2, cuuint64_t(expert_stride) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), 1};
  return encode_map(map, type, 3, w, dims, strides, box);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == LF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

struct Weights {
  const void* data;
  int64_t K, N, row_stride, expert_stride;
};

template <int kMode>
int launch_rows(GParams& p, CUtensorMapDataType type, const Weights& w, void* stream, const char* what) {
  const int64_t groups = p.E < p.R ? p.E : p.R;
  if (narrow(p.E, p.R)) {
    Clusters clusters;
    if (int rc = clusters_at_once<kMode, 1, kNarrowRows>(&clusters)) return rc;
    const int steps = ceil_div(p.C, kStep);
    const Cut cut = choose_cut(clusters, groups, p.M, steps, 1, kMode == kForward);  // input: boxes of 64 features
    p.height = cut.height, p.split = cut.split;
    if (kMode == kForward && !encode_weights(&p.a_map, type, w.data, w.K, w.N, p.E, w.row_stride, w.expert_stride, cut.height))
      return fail(LF_E_CUDA, (std::string(what) + ": cuTensorMapEncodeTiled failed").c_str());
    const int64_t mt = ceil_div(p.M, cut.height);  // tiles: at most
    // Tiles of 32 rows up to 16 on average: 20 rows each took 95 us in them against 89 in tiles of 64.
    if (p.R <= kFewRows / 2 * groups)
      return launch_grouped<kMode, 1, kFewRows>(p, mt * (groups + p.R / kFewRows), stream, what);
    return launch_grouped<kMode, 1, kNarrowRows>(p, mt * (groups + p.R / kNarrowRows), stream, what);
  }
  p.height = 128, p.split = 1;
  if (kMode == kForward && !encode_weights(&p.a_map, type, w.data, w.K, w.N, p.E, w.row_stride, w.expert_stride, 128))
    return fail(LF_E_CUDA, (std::string(what) + ": cuTensorMapEncodeTiled failed").c_str());
  const int64_t tiles = int64_t(ceil_div(p.M, 256)) * (groups + p.R / kWideRows);
  return launch_grouped<kMode, 2, kWideRows>(p, tiles, stream, what);
}

}  // namespace

int grouped_wait_timeouts(unsigned int* value, int reset) {
  if (cudaMemcpyFromSymbol(value, g_lf_wait_timeouts, sizeof(*value)) != cudaSuccess)
    return check_launch("device_wait_timeouts (expert products)");
  if (reset && *value) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_lf_wait_timeouts, &zero, sizeof(zero)) != cudaSuccess)
      return check_launch("device_wait_timeouts (expert products)");
  }
  return LF_OK;
}

}  // namespace lfb

using namespace lfb;

extern "C" int64_t lf_expert_linear_workspace_bytes(int32_t num_experts, int64_t num_rows, int64_t width,
                                                    int32_t weight_grad) {
  if (num_experts < 1 || num_rows < 0 || width < 1) return -1;
  return weight_grad || !gather_in_loads(num_experts, num_rows) ? num_rows * width * 2 : 0;
}

extern "C" int lf_expert_linear(int32_t dtype, const void* x, int64_t x_stride, int64_t x_rows, const int32_t* rows,
                                const void* w, int64_t w_expert_stride, int64_t w_row_stride, const int32_t* offsets,
                                int32_t num_experts, int64_t num_rows, int64_t out_width, int64_t width, void* y,
                                int64_t y_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "expert_linear";
  if (int rc = check_sizes(what, dtype, num_experts, num_rows, out_width, width)) return rc;
  if (num_rows == 0) return LF_OK;
  if (!offsets || !y || y_stride < out_width || !good_rows(w, w_row_stride, width) || w_expert_stride % 8 ||
      w_expert_stride < (out_width - 1) * w_row_stride + width)
    return fail(LF_E_INVALID, "expert_linear: W must be 16-byte aligned with strides that are multiples of 8, y's rows must not overlap");
  if (x_rows < 1 || x_rows >= (int64_t(1) << 31) - 1 || (!rows && x_rows < num_rows) || !good_rows(x, x_stride, width))
    return fail(LF_E_INVALID, "expert_linear: x must have rows, 16-byte aligned, with a stride that is a multiple of 8");
  int prepared = 0;
  if (rows) {
    const int64_t need = lf_expert_linear_workspace_bytes(num_experts, num_rows, width, 0);
    if (need) {
      if (!workspace || workspace_bytes < need || !aligned16(workspace)) return fail(LF_E_INVALID, kNoWorkspace);
      if (int rc = gather_rows(x, x_stride, x_rows, rows, num_rows, width, workspace, stream, what)) return rc;
      x = workspace, x_stride = width, x_rows = num_rows, rows = nullptr, prepared = 1;
    }
  }
  GParams p{};
  p.prepared = prepared;
  p.offsets = offsets, p.rows = rows, p.out = {y, y_stride, int(out_width), dtype};
  p.E = num_experts, p.R = int(num_rows), p.x_rows = int(x_rows);
  p.M = int(out_width), p.C = int(width), p.elem_bf16 = dtype == LF_BF16;
  const CUtensorMapDataType type = map_type(dtype);
  if ((rows ? !encode_rows(&p.b_gather, type, x, width, x_rows, x_stride, 1)
            : !encode_row_boxes(p.b_rows, type, x, width, x_rows, x_stride, narrow(num_experts, num_rows))))
    return fail(LF_E_CUDA, "expert_linear: cuTensorMapEncodeTiled failed");
  return launch_rows<kForward>(p, type, {w, width, out_width, w_row_stride, w_expert_stride}, stream, what);
}

extern "C" int lf_expert_linear_input_grad(int32_t dtype, const void* dy, int64_t dy_stride, const void* w,
                                           int64_t w_expert_stride, int64_t w_row_stride, const int32_t* offsets,
                                           int32_t num_experts, int64_t num_rows, int64_t out_width, int64_t width,
                                           void* dx, int64_t dx_stride, void* stream) {
  const char* what = "expert_linear_input_grad";
  if (int rc = check_sizes(what, dtype, num_experts, num_rows, out_width, width)) return rc;
  if (num_rows == 0) return LF_OK;
  if (!offsets || !dx || dx_stride < width || !good_rows(w, w_row_stride, width) || w_expert_stride % 8 ||
      w_expert_stride < (out_width - 1) * w_row_stride + width || !good_rows(dy, dy_stride, out_width))
    return fail(LF_E_INVALID, "expert_linear_input_grad: W and dy must be 16-byte aligned with strides that are multiples of 8, dx's rows must not overlap");
  GParams p{};
  p.offsets = offsets, p.out = {dx, dx_stride, int(width), dtype};
  p.E = num_experts, p.R = int(num_rows), p.x_rows = int(num_rows);
  p.M = int(width), p.C = int(out_width), p.elem_bf16 = dtype == LF_BF16;
  const CUtensorMapDataType type = map_type(dtype);
  if (!encode_weights(&p.a_map, type, w, width, out_width, num_experts, w_row_stride, w_expert_stride, 64) ||
      !encode_row_boxes(p.b_rows, type, dy, out_width, num_rows, dy_stride, narrow(num_experts, num_rows)))
    return fail(LF_E_CUDA, "expert_linear_input_grad: cuTensorMapEncodeTiled failed");
  return launch_rows<kInput>(p, type, {w, width, out_width, w_row_stride, w_expert_stride}, stream, what);
}

extern "C" int lf_expert_linear_weight_grad(int32_t dtype, const void* dy, int64_t dy_stride, const void* x,
                                            int64_t x_stride, int64_t x_rows, const int32_t* rows,
                                            const int32_t* offsets, int32_t num_experts, int64_t num_rows,
                                            int64_t out_width, int64_t width, int32_t out_dtype, void* dw,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "expert_linear_weight_grad";
  if (int rc = check_sizes(what, dtype, num_experts, num_rows, out_width, width)) return rc;
  if (out_dtype != dtype && out_dtype != LF_F32)
    return fail(LF_E_INVALID, "expert_linear_weight_grad: dW is of the operands' type or FP32");
  if (!dw) return fail(LF_E_INVALID, "expert_linear_weight_grad: null buffer");
  if (num_rows == 0) {
    const size_t bytes = size_t(num_experts) * out_width * width * (out_dtype == LF_F32 ? 4 : 2);
    if (cudaMemsetAsync(dw, 0, bytes, static_cast<cudaStream_t>(stream)) != cudaSuccess) return check_launch(what);
    return LF_OK;
  }
  if (!offsets || x_rows < 1 || x_rows >= (int64_t(1) << 31) - 1 || (!rows && x_rows < num_rows) ||
      !good_rows(x, x_stride, width) || !good_rows(dy, dy_stride, out_width))
    return fail(LF_E_INVALID, "expert_linear_weight_grad: x and dy must have rows, 16-byte aligned, with strides that are multiples of 8");
  if (rows) {
    if (!workspace || workspace_bytes < num_rows * width * 2 || !aligned16(workspace)) return fail(LF_E_INVALID, kNoWorkspace);
    if (int rc = gather_rows(x, x_stride, x_rows, rows, num_rows, width, workspace, stream, what)) return rc;
    x = workspace, x_stride = width, x_rows = num_rows;
  }
  GParams p{};
  p.prepared = rows != nullptr;
  p.offsets = offsets, p.out = {dw, width, int(width), out_dtype};
  p.E = num_experts, p.R = int(num_rows), p.x_rows = int(x_rows);
  p.M = int(width), p.N = int(out_width), p.elem_bf16 = dtype == LF_BF16, p.height = 128, p.split = 1;
  const CUtensorMapDataType type = map_type(dtype);
  if (!encode_rows(&p.a_map, type, x, width, x_rows, x_stride, 64) ||
      !encode_rows(&p.a_small, type, x, width, x_rows, x_stride, 8) ||
      !encode_rows(&p.a_gather, type, x, width, x_rows, x_stride, 1) ||
      !encode_rows(&p.b_map, type, dy, out_width, num_rows, dy_stride, 64) ||
      !encode_rows(&p.b_small, type, dy, out_width, num_rows, dy_stride, 8) ||
      !encode_rows(&p.b_gather, type, dy, out_width, num_rows, dy_stride, 1))
    return fail(LF_E_CUDA, "expert_linear_weight_grad: cuTensorMapEncodeTiled failed");
  const int64_t tiles = int64_t(ceil_div(p.M, 256)) * ceil_div(p.N, kWideRows) * num_experts;
  return launch_grouped<kWeight, 2, kWideRows>(p, tiles, stream, what);
}
