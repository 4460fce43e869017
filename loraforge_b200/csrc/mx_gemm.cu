// Expert products of MXFP4 activations and weights on the block-scaled tensor cores:
//
//   y[r, n] = sum over blocks b of 32 of 2^(sx[i(r), b] + sw[e, n, b] - 254)
//             sum over k in b of qx[i(r), k] qw[e, n, k]
//
// for rows offsets[e] <= r < offsets[e+1], i(r) = rows[r] or r.  tcgen05.mma kind::mxf4 takes
// the 4-bit codes as they lie (K-major, 64 a step) and one scale byte for 32 of them, and sums
// in FP32; a product of two codes and two powers of two is exact.
//
// The tiles are those of the 16-bit products (grouped_gemm.cu): features on the TMEM lanes,
// rows on the columns, CTA pairs with 256 features x up to 208 rows, or single CTAs with up to
// 128 x 32 whose contraction may be split over a cluster.  208, not 256, rows: two
// accumulators of 208 columns leave 96 TMEM columns for four sets of scales.
//
// Scales.  The tensor core wants them in TMEM: for 128 operand rows and 128 codes a row, four
// columns in which lane l of column j holds the four bytes of row 32 j + l, the same in every
// quarter of the lanes.  Four warps, one a quarter, write them there, to several sets of columns
// in turn (a stage each), and tell the MMA warp.  (Copied by tcgen05.cp from the MMA warp, each block
// of 512 bytes held the MMAs up for some 33 ns, and a wide stage has six.)
//   wide    the warps read them from shared memory, where a stage's come by bulk copies from
//           blocks that pack_kernel laid out in the workspace before (the scales of
//           28672 x 4096 weights: 3.7 MB each way).  Row by row from global memory, the warps
//           were slower than the MMAs.
//   narrow  every warp reads all rows itself (three of four times from a cache): 32 bytes, a
//           whole sector, of each row for four stages, one such group ahead, also across tiles.
//
// Per CTA: warp 0 loads (TMA), warp 1 MMA and TMEM, warps 2-5 store (10-13 too for short
// contractions), warps 6-9 scales.  Measured on eight experts of 14336 x 4096: 8 x 2048 rows
// 396-478 us by the power cap (4.0-4.9 PFLOP/s, packing included; 338 without the stores; on 8 x 624
// rows the tensor pipe is active in 66 % of the cycles and no other unit at its limit), 8 x 2 rows 50 us
// (5.0 TB/s).
// Every wait is bounded (tma.cuh): an expiry stops every role at its next wait.
#include "experts.cuh"
#include "grouped.cuh"

namespace lfb {
namespace {

using namespace grouped;

constexpr int kStep = 256;           // codes per stage: 128 bytes a row
constexpr int kABytes = 128 * 128;
constexpr int kSuper = 4;            // stages whose scales a thread loads at once (32 bytes a row)

struct MxParams {
  const int32_t* offsets;  // [E + 1]
  const int32_t* rows;     // [R] or null: row of x (and of its scales)
  Output out;
  const uint8_t* x_scales;  // [x_rows][blocks]
  const uint8_t* w_scales;  // [E][N][blocks]
  int E, R, x_rows, N, K, blocks;
  int x_align, w_align;  // 16, 8 or 1: alignment of every row of the scales
  const uint8_t* w_blocks;  // wide: packed scales
  const uint8_t* x_blocks;
  int groups;            // of 128 codes in them, an even number
  int height, split, store_sets;
  Bands bands;
  CUtensorMap w_map;      // 128 bytes x 128 rows
  CUtensorMap x_map[7];   // 128 bytes x 16, 32, .. 112 rows
  CUtensorMap x_gather;   // single rows
};

template <int kCtas, int kNT>
struct Shape {
  static constexpr int kBRows = round_up(kNT / kCtas, 16);  // a CTA's share of the rows, loaded by 16
  static constexpr int kHalves = (kNT + 127) / 128;              // scale blocks of 128 rows of x
  static constexpr int kScaleBytes = kCtas == 2 ? 2 * 512 * (1 + kHalves) : 0;  // blocks of two groups of 128 codes
  static constexpr int kStageBytes = (kABytes + kBRows * 128 + kScaleBytes + 1023) / 1024 * 1024;
  static constexpr int kStoreSets = kCtas == 1 ? 1 : 2;  // of four warps, at most
  static constexpr int kThreads = 192 + 128 * kStoreSets;
  static constexpr int kPartBytes = kCtas == 1 ? kNT * 128 * 4 : kStoreSets * 4 * kChunkBytes;
  static constexpr int kStages = stages_of(kStageBytes, kPartBytes);
  static constexpr int kScaleColumns = 2 * (4 + 4 * kHalves);  // a set of TMEM columns for a stage's scales
  static constexpr int kSets = kCtas == 2 ? 4 : kStages;       // that the stages use in turn
  static constexpr int kColumns = 512;                         // TMEM
  static_assert(2 * kNT + kSets * kScaleColumns <= kColumns, "TMEM");
};

__device__ __forceinline__ uint32_t instruction(int m, int n, int scale_id) {
  return (uint32_t(scale_id) << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) |
         (uint32_t(m >> 7) << 27) | (uint32_t(scale_id) << 29);
}

template <int kCtas>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accumulate) {
  if constexpr (kCtas == 1) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  }
}

// Columns taddr .. taddr + 4 n - 1 of this warp's lane quarter from n blocks of 512 bytes, lane l's
// 16 bytes at l * 16.
template <int n>
__device__ __forceinline__ void store_scales(uint32_t taddr, uint32_t blocks, int lane) {
  static_assert(n == 4 || n == 6, "two groups of one block of W and one or two of x");
#pragma unroll
  for (int i = 0; i < n; i += 2) {
    const uint4 a = lds16(blocks + i * 512 + lane * 16), b = lds16(blocks + i * 512 + 512 + lane * 16);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr + 4 * i),
                 "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// Arrive on a barrier of the cluster after tcgen05 operations (which the fence before it orders).
__device__ __forceinline__ void arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

struct Tile {
  int e, m0, end, n0, nt, valid, hi;
  int row_tile;  // among the row tiles of all groups
};

// A role's walk over its CTA's tiles.
template <int kCtas, int kNT>
struct Tiles {
  Walk walk;
  int each, row_tiles;  // rows of the group's row tiles; row tiles of the groups before it
  __device__ __forceinline__ Tile at(const MxParams& p, const int* bounds, const int* starts, int t) {
    if (walk.go(p.bands, bounds, starts, p.E, t, [](int rows) { return ceil_div(rows, kNT); })) {
      each = round_up(walk.nt == 1 ? walk.hi - walk.lo : ceil_div(walk.hi - walk.lo, walk.nt), 16);
      if (kCtas == 2) row_tiles = walk.start / p.bands.mt;
    }
    Tile x;
    x.e = walk.e, x.hi = walk.hi;
    x.m0 = walk.m * p.height * kCtas;
    x.end = min(p.N, x.m0 + p.height * kCtas);
    x.row_tile = row_tiles + walk.n;
    x.n0 = walk.lo + walk.n * each;
    x.valid = min(each, x.hi - x.n0);
    x.nt = round_up(x.valid, 16);
    return x;
  }
};

// 32 scale bytes from byte k0 of a row of `blocks`; zeros past the row and where row is null.
__device__ __forceinline__ void load_scales(const uint8_t* row, int k0, int blocks, int align, uint32_t (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0;
  if (!row) return;
  if (align == 16 && k0 + 32 <= blocks) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + k0), b = *reinterpret_cast<const uint4*>(row + k0 + 16);
    s[0] = a.x, s[1] = a.y, s[2] = a.z, s[3] = a.w, s[4] = b.x, s[5] = b.y, s[6] = b.z, s[7] = b.w;
  } else if (align >= 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k0 + 8 * i < blocks) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + k0 + 8 * i);
        s[2 * i] = v.x, s[2 * i + 1] = v.y;
      }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (k0 + i < blocks) s[i >> 2] |= uint32_t(row[k0 + i]) << (8 * (i & 3));
  }
}

template <int kCtas, int kNT>
__global__ void __launch_bounds__((Shape<kCtas, kNT>::kThreads), 1) mx_kernel(const __grid_constant__ MxParams p) {
  using S = Shape<kCtas, kNT>;
  constexpr int kStages = S::kStages, kSets = S::kSets;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = smem;  // stage: W codes, x codes, scales of W (two groups), of x (two groups x halves)
  float* part = reinterpret_cast<float*>(ring + kStages * S::kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * S::kStageBytes + S::kPartBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* blocks_full = acc_empty + 2;      // wide: a stage's scale blocks are here
  uint64_t* set_full = blocks_full + kStages;  // a set of scale columns is written, in both CTAs
  uint64_t* part_full = set_full + kSets;
  uint64_t* part_empty = part_full + 1;
  uint64_t* fin = part_empty + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(fin + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);
  int* scan = reinterpret_cast<int*>(tslot + 2);
  int* bounds = scan + kMaxWarps;  // [E + 1]
  int* starts = bounds + p.E + 1;  // [E + 1]

  const int cluster = kCtas == 2 ? 2 : p.split;
  const int rank = cluster > 1 ? int(cluster_rank()) : 0;
  const bool leader = rank * (kCtas - 1) == 0;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&blocks_full[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4 * p.store_sets * kCtas);
    }
    for (int i = 0; i < kSets; ++i) mbar_init(&set_full[i], 4 * kCtas);
    mbar_init(part_full, 4 * cluster);
    mbar_init(part_empty, 4 * cluster);
    mbar_init(fin, 1);
    fence_mbar_init();
    *abort = 0;
  }
  Tiles<kCtas, kNT> walk;
  // Wide: the grid before is pack_kernel, and all but what it packs can be read before it ends.
  if (kCtas == 1) pdl_wait();
  if (warp == 1) alloc_tmem<kCtas>(tslot, S::kColumns);  // not while waiting for a grid that may want some too
  const int mtiles = p.bands.mt;
  list_tiles(p.offsets, p.E, p.R, bounds, starts, scan, [&](int rows) { return mtiles * ceil_div(rows, kNT); });
  tc_fence_before();
  __syncthreads();
  if (cluster > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  const int tiles = starts[p.E];
  const int first = int(blockIdx.x) / cluster, stride = int(gridDim.x) / cluster;
  zero_rows(p.out, bounds[0], bounds[p.E], p.R);

  // The steps this CTA takes of every tile, in whole groups of kSuper.
  const int steps = ceil_div(p.K, kStep);
  int ks0 = 0, ks1 = steps;
  if (kCtas == 1 && cluster > 1) {
    const int each = round_up(ceil_div(steps, cluster), kSuper);
    ks0 = min(steps, rank * each);
    ks1 = min(steps, ks0 + each);
  }
  const bool live = ks1 > ks0;

  if (warp == 0) {
    // ------------------------------------------------------------ codes
    const bool elected = elect_one();
    if (kCtas == 2) {
      if (lane == 0 && first < tiles) {
        const Tile x = walk.at(p, bounds, starts, first);
        for (int ks = 0; ks < min(steps, kAhead); ++ks) prefetch_3d(&p.w_map, ks * 128, x.m0 + rank * 128, x.e);
      }
      __syncwarp();
      walk = {};
      pdl_wait();
    }
    int it = 0;
    for (int t = first; t < tiles && live; t += stride) {
      const Tile x = walk.at(p, bounds, starts, t);
      const int m_cta = x.m0 + (kCtas == 2 ? rank * 128 : 0);
      const int share = kCtas == 1 ? x.valid : x.nt / kCtas;
      const int n_cta = x.n0 + (kCtas == 2 ? rank * share : 0);
      const bool by_row = kCtas == 1 && p.rows;
      int row4[4];
      if (by_row) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = n_cta + 4 * lane + i;
          const int src = 4 * lane + i < share && r < x.hi ? p.rows[r] : -1;
          row4[i] = src >= 0 && src < p.x_rows ? src : p.x_rows;
        }
      }
      const uint32_t bytes = kCtas * uint32_t(p.height + (by_row ? round_up(x.valid, 4) : round_up(share, 16))) * 128u;
      bool ok = true;
      if (!by_row) {
        // Addresses kept from step to step (64 groups of 94 rows, 1416 x 2048: 38.2 us, 39.4 shared out
        // over the lanes).  One box of the share's rows in steps of 16, as small boxes cost the copy
        // engine near 0.1 us each, whatever their size (rows past the share are loaded and not used).
        const CUtensorMap* x_map = &p.x_map[ceil_div(share, 16) - 1];
        const uint8_t *w_blocks = nullptr, *x_blocks = nullptr;
        if (kCtas == 2) {
          w_blocks = p.w_blocks + (int64_t(x.e * ceil_div(p.N, 256) * 2 + m_cta / 128) * p.groups + 2 * ks0) * 512;
          x_blocks = p.x_blocks + (int64_t(x.row_tile) * p.groups + 2 * ks0) * 1024;
        }
        for (int ks = ks0; ks < ks1; ++ks, ++it) {
          const int st = it % kStages;
          ok = __all_sync(0xffffffffu, wait_here(&empty[st], (uint32_t(it / kStages) & 1u) ^ 1u, abort));
          if (!ok) break;
          uint8_t* stage = ring + st * S::kStageBytes;
          const uint32_t a = smem_u32(stage);
          const uint32_t bar = kCtas == 2 ? mapa(&full[st], 0) : smem_u32(&full[st]);
          if (elected) {
            if (leader) mbar_arrive_expect_tx(&full[st], bytes);
            load_3d<kCtas>(a, &p.w_map, ks * 128, m_cta, x.e, bar);
            load_2d<kCtas>(a + kABytes, x_map, ks * 128, n_cta, bar);
            if (kCtas == 2) {
              uint8_t* sc = stage + kABytes + S::kBRows * 128;
              mbar_arrive_expect_tx(&blocks_full[st], S::kScaleBytes);
              bulk_g2s(sc, w_blocks, 1024, &blocks_full[st]);
              bulk_g2s(sc + 1024, x_blocks, 2048, &blocks_full[st]);
            }
          }
          __syncwarp();
          if (kCtas == 2) w_blocks += 1024, x_blocks += 2048;
        }
      } else {
        for (int ks = ks0; ks < ks1; ++ks, ++it) {
          const int st = it % kStages;
          ok = __all_sync(0xffffffffu, wait_here(&empty[st], (uint32_t(it / kStages) & 1u) ^ 1u, abort));
          if (!ok) break;
          const uint32_t a = smem_u32(ring + st * S::kStageBytes), bar = smem_u32(&full[st]);
          if (elected) {
            mbar_arrive_expect_tx(&full[st], bytes);
            load_3d<1>(a, &p.w_map, ks * 128, m_cta, x.e, bar);
          }
          __syncwarp();
          if (4 * lane < x.valid) gather4<1>(a + kABytes + lane * 512, &p.x_gather, ks * 128, row4, bar);
        }
      }
      if (!ok) break;
    }
    // A pair's CTA stays until the commits that arrive here from the other CTA have.
    if (kCtas == 2)
      for (int j = max(0, it - kStages); j < it; ++j) wait_here(&empty[j % kStages], uint32_t(j / kStages) & 1u, abort);
    // No load may still be landing when the CTA exits: after an expired wait, give them time.
    if (*abort && elected)
      for (int j = max(0, it - kStages); j < it; ++j) {
        if (leader) mbar_wait(&full[j % kStages], uint32_t(j / kStages) & 1u);
        if (kCtas == 2) mbar_wait(&blocks_full[j % kStages], uint32_t(j / kStages) & 1u);
      }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    if (leader) {
      const bool elected = elect_one();
      int it = 0, count = 0;
      for (int t = first; t < tiles && live; t += stride) {
        const Tile x = walk.at(p, bounds, starts, t);
        const int ab = count & 1;
        if (!__all_sync(0xffffffffu, wait_cluster(&acc_empty[ab], (uint32_t(count >> 1) & 1u) ^ 1u, abort))) break;
        ++count;
        const uint32_t d = tmem + uint32_t(ab * kNT);
        const uint32_t idesc0 = instruction(128 * kCtas, x.nt, 0), idesc1 = instruction(128 * kCtas, x.nt, 2);
        bool ok = true;
        for (int ks = ks0; ks < ks1; ++ks, ++it) {
          const int st = it % kStages, set = it % kSets;
          ok = wait_here(&full[st], uint32_t(it / kStages) & 1u, abort) &&
               wait_cluster(&set_full[set], uint32_t(it / kSets) & 1u, abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(ring + st * S::kStageBytes);
          const uint32_t ts = tmem + uint32_t(2 * kNT + set * S::kScaleColumns);  // W: 2 x 4 columns, then x
          const uint64_t ad = sw128_desc(sa), bd = sw128_desc(sa + kABytes);
          if (elected) {
#pragma unroll
            for (int k = 0; k < kStep / 64; ++k)
              mma_mxf4<kCtas>(d, ad + 2 * k, bd + 2 * k, k & 1 ? idesc1 : idesc0, ts + 4 * (k >> 1),
                              ts + 8 + 4 * S::kHalves * (k >> 1), (ks > ks0 || k > 0) ? 1u : 0u);
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
  } else if (warp < 6 || warp >= 10) {
    // ------------------------------------------------------------ stores
    const int quarter = warp & 3;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const int set = warp >= 10 ? 1 : 0;
    const uint32_t staging = smem_u32(part) + uint32_t((set * 4 + quarter) * kChunkBytes);
    int count = 0;
    for (int t = first; t < tiles; t += stride, ++count) {
      const Tile x = walk.at(p, bounds, starts, t);
      const int ab = count & 1;
      if (live) {
        if (!__all_sync(0xffffffffu, wait_here(&acc_full[ab], uint32_t(count >> 1) & 1u, abort))) break;
        tc_fence_after();
      }
      const uint32_t d = tmem + lanes + uint32_t(ab * kNT);
      const int f0 = x.m0 + (kCtas == 2 ? rank * 128 : 0) + quarter * 32;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (live && lane == 0) {
          if (kCtas == 2) arrive_cluster(mapa(&acc_empty[ab], 0));
          else mbar_arrive(&acc_empty[ab]);
        }
      };
      if (kCtas == 1 && cluster > 1) {
        if (!store_split(p.out, d, live, f0, x.end, x.n0, x.nt, x.valid, part, part_full, part_empty, count, cluster, rank,
                         quarter, lane, abort, release))
          break;
      } else {
        store_whole(p.out, d, live, f0, x.end, x.n0, x.nt, x.valid, staging, lane, set, p.store_sets);
        release();
      }
    }
  } else {
    // ------------------------------------------------------------ scales
    const uint32_t quarter_set = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(2 * kNT);
    if constexpr (kCtas == 2) {
      const int mine = first < tiles ? (tiles - first + stride - 1) / stride : 0;
      for (int it = 0; it < mine * steps; ++it) {
        const int before = it - kSets, st = it % kStages, set = it % kSets;
        bool ready = wait_here(&blocks_full[st], uint32_t(it / kStages) & 1u, abort);
        if (before >= 0) ready = ready && wait_here(&empty[before % kStages], uint32_t(before / kStages) & 1u, abort);
        if (!__all_sync(0xffffffffu, ready)) break;
        tc_fence_after();
        store_scales<2 * (1 + S::kHalves)>(quarter_set + uint32_t(set * S::kScaleColumns),
                                           smem_u32(ring + st * S::kStageBytes) + kABytes + S::kBRows * 128, lane);
        tc_fence_before();
        if (lane == 0) arrive_cluster_relaxed(mapa(&set_full[set], 0));
      }
    } else {
      constexpr int kXRows = kNT / 32;
      const uint8_t *w_row[4], *x_row[kXRows];  // this lane's of every 32 rows
      auto rows_of = [&](int t) {
        const Tile x = walk.at(p, bounds, starts, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = x.m0 + 32 * j + lane;
          w_row[j] = n < x.end ? p.w_scales + (int64_t(x.e) * p.N + n) * p.blocks : nullptr;
        }
#pragma unroll
        for (int j = 0; j < kXRows; ++j) {
          const int r = 32 * j + lane;
          const int src = r < x.valid ? (p.rows ? p.rows[x.n0 + r] : x.n0 + r) : -1;
          x_row[j] = src >= 0 && src < p.x_rows ? p.x_scales + int64_t(src) * p.blocks : nullptr;
        }
      };
      uint32_t w_next[4][8], x_next[kXRows][8];
      auto load = [&](int k0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load_scales(w_row[j], k0 * 8, p.blocks, p.w_align, w_next[j]);
#pragma unroll
        for (int j = 0; j < kXRows; ++j) load_scales(x_row[j], k0 * 8, p.blocks, p.x_align, x_next[j]);
      };
      int it = 0, t = first, k0 = ks0;
      bool ok = live && t < tiles;
      if (ok) {
        rows_of(t);
        load(k0);
      }
      while (ok) {
        uint32_t w_now[4][8], x_now[kXRows][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w_now[j][i] = w_next[j][i];
#pragma unroll
          for (int j = 0; j < kXRows; ++j) x_now[j][i] = x_next[j][i];
        }
        const int todo = min(kSuper, ks1 - k0);
        k0 += kSuper;
        if (k0 >= ks1) {
          k0 = ks0;
          t += stride;
          if (t < tiles) rows_of(t);
        }
        if (t < tiles) load(k0);
#pragma unroll
        for (int j = 0; j < kSuper; ++j) {
          if (j >= todo || !ok) continue;
          const int set = it % kSets;  // free when the MMAs of its stage are done
          ok = __all_sync(0xffffffffu, wait_here(&empty[set], (uint32_t(it / kSets) & 1u) ^ 1u, abort));
          if (!ok) continue;
          tc_fence_after();
          // Groups 2 j and 2 j + 1 of W, then of x; columns past the tile's rows are not read.
          asm volatile(
              "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %11, %12, "
              "%13, %14, %14};\n tcgen05.wait::st.sync.aligned;" ::"r"(quarter_set + uint32_t(set * S::kScaleColumns)),
              "r"(w_now[0][2 * j]), "r"(w_now[1][2 * j]), "r"(w_now[2][2 * j]), "r"(w_now[3][2 * j]),
              "r"(w_now[0][2 * j + 1]), "r"(w_now[1][2 * j + 1]), "r"(w_now[2][2 * j + 1]), "r"(w_now[3][2 * j + 1]),
              "r"(x_now[0][2 * j]), "r"(x_now[kXRows - 1][2 * j]), "r"(0), "r"(x_now[0][2 * j + 1]),
              "r"(x_now[kXRows - 1][2 * j + 1]), "r"(0)
              : "memory");
          tc_fence_before();
          if (lane == 0) mbar_arrive(&set_full[set]);
          ++it;
        }
        ok = ok && t < tiles;
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

constexpr int kWideRows = 208, kNarrowRows = 32;

// Groups of up to 16 rows on average take the narrow tiles, whose loads gather rows by index; the
// others' codes are put in order and the scales packed first.  64 experts of 2048 x 2048: 9 rows each
// 34 us against 36, 17 rows 41 against 38, 40 unequal ones 51 against 43.
bool narrow(int64_t E, int64_t R) { return R <= 16 * (E < R ? E : R); }

// The wide tiles' workspace: W's scales as blocks [expert][128 features][group of 128 codes],
// x's as [row tile][group][half], and x's codes in the rows' order.
struct PackParams {
  const int32_t* offsets;
  const int32_t* rows;
  const uint8_t* x_scales;
  const uint8_t* w_scales;
  const uint4* x_codes;  // null: in order already
  uint8_t *w_blocks, *x_blocks;
  uint4* codes;
  int E, R, x_rows, N, blocks, groups, words;  // words: 16-byte words of a row of codes
  int w_tasks, x_tasks;                        // CUDA blocks for each part
  int align;                                   // 16, 4 or 1: alignment of every row of the scales
};

// Four bytes each of groups g .. g + 3 of a row; zeros past it and where row is null.
__device__ __forceinline__ uint4 scale_words(const uint8_t* row, int g, int blocks, int align) {
  uint32_t v[4] = {0, 0, 0, 0};
  const int k = 4 * g;
  if (!row) return make_uint4(0, 0, 0, 0);
  if (align == 16 && k + 16 <= blocks) return *reinterpret_cast<const uint4*>(row + k);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (align >= 4) {
      if (k + 4 * i < blocks) v[i] = *reinterpret_cast<const uint32_t*>(row + k + 4 * i);
    } else {
      for (int j = 0; j < 4; ++j)
        if (k + 4 * i + j < blocks) v[i] |= uint32_t(row[k + 4 * i + j]) << (8 * j);
    }
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Blocks of groups g .. g + 3 (`pitch` uint4 apart, those below `groups`): lane l takes rows l, l + 32,
// l + 64 and l + 96, 16 bytes of each, and writes their words for each group.
__device__ __forceinline__ void pack_groups(const uint8_t* const (&row)[4], int g, int blocks, int align, int groups,
                                            uint4* out, int pitch) {
  const uint4 a = scale_words(row[0], g, blocks, align), b = scale_words(row[1], g, blocks, align);
  const uint4 c = scale_words(row[2], g, blocks, align), d = scale_words(row[3], g, blocks, align);
  out[0] = make_uint4(a.x, b.x, c.x, d.x);
  if (g + 1 < groups) out[pitch] = make_uint4(a.y, b.y, c.y, d.y);
  if (g + 2 < groups) out[2 * pitch] = make_uint4(a.z, b.z, c.z, d.z);
  if (g + 3 < groups) out[3 * pitch] = make_uint4(a.w, b.w, c.w, d.w);
}

constexpr int kPackThreads = 256;

// One CUDA block writes the scale blocks of 128 features, or of a row tile (2 x 128 rows), a warp
// those of four groups at a time.  Or it moves eight rows of codes.
template <int kNT>
__global__ void __launch_bounds__(kPackThreads) pack_kernel(const __grid_constant__ PackParams p) {
  __shared__ int scan[kMaxWarps];
  extern __shared__ int tables[];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int task = blockIdx.x;
  if (task < p.w_tasks) {
    const int mb = ceil_div(p.N, 256) * 2, e = task / mb, n0 = (task % mb) * 128 + lane;
    const uint8_t* row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      row[j] = n0 + 32 * j < p.N ? p.w_scales + (int64_t(e) * p.N + n0 + 32 * j) * p.blocks : nullptr;
    uint4* out = reinterpret_cast<uint4*>(p.w_blocks + int64_t(task) * p.groups * 512) + lane;
    for (int g = 4 * warp; g < p.groups; g += kPackThreads / 8)
      pack_groups(row, g, p.blocks, p.align, p.groups, out + g * 32, 32);
    return;
  }
  task -= p.w_tasks;
  if (task < p.x_tasks) {
    int* bounds = tables;
    int* starts = bounds + p.E + 1;
    list_tiles(p.offsets, p.E, p.R, bounds, starts, scan, [](int rows) { return ceil_div(rows, kNT); });
    if (task >= starts[p.E]) return;
    const int e = group_of(starts, p.E, task), lo = bounds[e], hi = bounds[e + 1];
    const int each = round_up(ceil_div(hi - lo, ceil_div(hi - lo, kNT)), 16);
    const int n0 = lo + (task - starts[e]) * each, valid = min(each, hi - n0);
    const uint8_t* row[2][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = lane + 32 * j;
      const int src = r < valid ? (p.rows ? p.rows[n0 + r] : n0 + r) : -1;
      row[j >> 2][j & 3] = src >= 0 && src < p.x_rows ? p.x_scales + int64_t(src) * p.blocks : nullptr;
    }
    uint4* out = reinterpret_cast<uint4*>(p.x_blocks + int64_t(task) * p.groups * 1024) + lane;
    for (int g = 4 * warp; g < p.groups; g += kPackThreads / 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) pack_groups(row[h], g, p.blocks, p.align, p.groups, out + (g * 2 + h) * 32, 64);
    }
    return;
  }
  task -= p.x_tasks;
  const int64_t r = int64_t(task) * (kPackThreads / 32) + warp;
  if (r < p.R) copy_row(p.x_codes, p.words, p.x_rows, p.rows, r, p.words, p.codes, lane);
}

template <int kCtas, int kNT>
int smem_of(int E) {
  using S = Shape<kCtas, kNT>;
  return 1024 + S::kStages * S::kStageBytes + S::kPartBytes + 512 + int(sizeof(int)) * (kMaxWarps + 2 + 2 * (E + 1));
}

template <int kCtas, int kNT>
int clusters_at_once(Clusters* out) {
  const auto kernel = mx_kernel<kCtas, kNT>;
  static int flags[64] = {};
  if (int rc = ensure_smem(kernel, smem_of<kCtas, kNT>(kMaxExperts), flags)) return rc;
  return clusters_of(kernel, (Shape<kCtas, kNT>::kThreads), smem_of<kCtas, kNT>(kMaxExperts), out);
}

// Pairs with a contraction of up to kShort store with eight warps a CTA instead of four, which do not
// keep up with the MMAs of so few steps.  8 experts, 2048 rows each to 14336 features: 1024 wide 197 us
// against 234, 2048 wide 272 against 308, but 4096 wide 485 against 477; 16 experts, 1024 rows each
// to 4096 features: 2048 wide 83 against 92, 3040 wide 138 against 131.
constexpr int kShort = 2048;

template <int kCtas, int kNT>
int launch_mx(MxParams& p, int64_t tiles, void* stream) {
  p.bands = bands_of(ceil_div(p.N, p.height * kCtas));
  const int cluster = kCtas == 2 ? 2 : p.split;
  p.store_sets = kCtas == 2 && p.blocks * 32 <= kShort ? 2 : 1;
  Clusters clusters;
  if (int rc = clusters_at_once<kCtas, kNT>(&clusters)) return rc;
  const int grid = grid_of(clusters, tiles, cluster, "expert_linear_mxfp4");
  if (!grid) return LF_E_CUDA;
  return launch_clusters(mx_kernel<kCtas, kNT>, grid, 192 + 128 * p.store_sets, cluster,
                         smem_of<kCtas, kNT>(p.E), stream, "expert_linear_mxfp4", p);
}

bool encode_codes(CUtensorMap* map, const void* p, int64_t bytes, int64_t rows, int box_rows) {
  const cuuint64_t dims[2] = {cuuint64_t(bytes), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(bytes)};
  const cuuint32_t box[2] = {128, cuuint32_t(box_rows)};
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims, strides, box);
}

// Sizes of the wide tiles' workspace: 512-byte blocks of W's and of x's scales, then codes.
struct Workspace {
  int groups;
  int64_t row_tiles, w_blocks, x_blocks, bytes;
};
Workspace workspace_of(int64_t E, int64_t R, int64_t N, int64_t K, bool by_rows) {
  Workspace w{};
  if (narrow(E, R)) return w;
  w.groups = 2 * int((K + kStep - 1) / kStep);
  w.row_tiles = (E < R ? E : R) + R / kWideRows;  // at most
  w.w_blocks = E * ((N + 255) / 256) * 2 * w.groups;
  w.x_blocks = w.row_tiles * w.groups * 2;
  w.bytes = (w.w_blocks + w.x_blocks) * 512 + (by_rows ? R * (K / 2) : 0);
  return w;
}

int row_alignment(const void* p, int blocks) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | uintptr_t(blocks);
  return bits & 7 ? 1 : bits & 15 ? 8 : 16;
}

}  // namespace

int mx_wait_timeouts(unsigned int* value, int reset) {
  if (cudaMemcpyFromSymbol(value, g_lf_wait_timeouts, sizeof(*value)) != cudaSuccess)
    return check_launch("device_wait_timeouts (MXFP4 products)");
  if (reset && *value) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_lf_wait_timeouts, &zero, sizeof(zero)) != cudaSuccess)
      return check_launch("device_wait_timeouts (MXFP4 products)");
  }
  return LF_OK;
}

}  // namespace lfb

using namespace lfb;

extern "C" int64_t lf_expert_linear_mxfp4_workspace_bytes(int32_t num_experts, int64_t num_rows, int64_t out_width,
                                                          int64_t width, int32_t by_rows) {
  if (num_experts < 1 || num_rows < 0 || out_width < 1 || width < 1) return -1;
  return workspace_of(num_experts, num_rows, out_width, width, by_rows != 0).bytes;
}

extern "C" int lf_expert_linear_mxfp4(int32_t out_dtype, const uint8_t* x_codes, const uint8_t* x_scales,
                                      int64_t x_rows, const int32_t* rows, const uint8_t* w_codes,
                                      const uint8_t* w_scales, const int32_t* offsets, int32_t num_experts,
                                      int64_t num_rows, int64_t out_width, int64_t width, void* y, int64_t y_stride,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t limit = int64_t(1) << 31;
  if (out_dtype < LF_F32 || out_dtype > LF_BF16) return fail(LF_E_INVALID, "expert_linear_mxfp4: unknown output type");
  if (num_experts < 1 || num_experts > kMaxExperts || num_rows < 0 || num_rows >= limit - 256 || out_width < 1 ||
      out_width >= limit - 256 || width < 32 || width % 32 || width >= limit - 256 ||
      (num_rows / kNarrowRows + num_experts + 1) * (out_width / 64 + 1) >= limit)
    return fail(LF_E_INVALID, "expert_linear_mxfp4: needs 1..1024 experts, a width that is a multiple of 32, and rows and tiles that fit int32");
  if (num_rows == 0) return LF_OK;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !offsets || !y || y_stride < out_width || !aligned16(x_codes) ||
      !aligned16(w_codes))
    return fail(LF_E_INVALID, "expert_linear_mxfp4: null buffer, codes not 16-byte aligned, or y's rows overlap");
  if (x_rows < 1 || x_rows >= limit - 1 || (!rows && x_rows < num_rows))
    return fail(LF_E_INVALID, "expert_linear_mxfp4: x has too few rows");
  MxParams p{};
  p.offsets = offsets, p.rows = rows, p.out = {y, y_stride, int(out_width), out_dtype};
  p.x_scales = x_scales, p.w_scales = w_scales;
  p.E = num_experts, p.R = int(num_rows), p.x_rows = int(x_rows), p.N = int(out_width), p.K = int(width);
  p.blocks = int(width / 32);
  p.x_align = row_alignment(x_scales, p.blocks), p.w_align = row_alignment(w_scales, p.blocks);
  const bool few = narrow(num_experts, num_rows);
  int64_t code_rows = x_rows;
  if (!few) {
    const Workspace w = workspace_of(num_experts, num_rows, out_width, width, rows != nullptr);
    if (!workspace || workspace_bytes < w.bytes || !aligned16(workspace))
      return fail(LF_E_INVALID, "expert_linear_mxfp4: workspace missing, too small or not 16-byte aligned "
                                "(see lf_expert_linear_mxfp4_workspace_bytes)");
    if (w.w_blocks >= limit || w.x_blocks >= limit)
      return fail(LF_E_INVALID, "expert_linear_mxfp4: too many scale blocks");
    PackParams k{};
    k.offsets = offsets, k.rows = rows, k.x_scales = x_scales, k.w_scales = w_scales;
    k.w_blocks = static_cast<uint8_t*>(workspace), k.x_blocks = k.w_blocks + w.w_blocks * 512;
    k.codes = reinterpret_cast<uint4*>(k.x_blocks + w.x_blocks * 512);
    k.x_codes = reinterpret_cast<const uint4*>(x_codes);
    k.E = p.E, k.R = p.R, k.x_rows = p.x_rows, k.N = p.N, k.blocks = p.blocks, k.groups = w.groups;
    k.words = int(width / 32), k.w_tasks = int(w.w_blocks / w.groups), k.x_tasks = int(w.row_tiles);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales) | uintptr_t(p.blocks);
    k.align = bits & 3 ? 1 : bits & 15 ? 4 : 16;
    const int64_t moves = rows ? (num_rows + kPackThreads / 32 - 1) / (kPackThreads / 32) : 0;
    if (int rc = launch_clusters(pack_kernel<kWideRows>, int(k.w_tasks + k.x_tasks + moves), kPackThreads, 1,
                                 int(sizeof(int)) * 2 * (p.E + 1), stream, "expert_linear_mxfp4 (scales)", k))
      return rc;
    if (rows) x_codes = reinterpret_cast<const uint8_t*>(k.codes), code_rows = num_rows;
    p.groups = w.groups, p.w_blocks = k.w_blocks, p.x_blocks = k.x_blocks;
  }
  const cuuint64_t dims[3] = {cuuint64_t(width / 2), cuuint64_t(out_width), cuuint64_t(num_experts)};
  const cuuint64_t strides[2] = {cuuint64_t(width / 2), cuuint64_t(width / 2) * cuuint64_t(out_width)};
  const int64_t groups = num_experts < num_rows ? num_experts : num_rows;
  Cut cut{128, 1};
  if (few) {
    Clusters clusters;
    if (int rc = clusters_at_once<1, kNarrowRows>(&clusters)) return rc;
    cut = choose_cut(clusters, groups, p.N, ceil_div(p.K, kStep), kSuper, true);
  }
  p.height = cut.height, p.split = cut.split;
  const cuuint32_t box[3] = {128, cuuint32_t(cut.height), 1};
  bool ok = encode_map(&p.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, w_codes, dims, strides, box);
  if (rows && few) ok = ok && encode_codes(&p.x_gather, x_codes, width / 2, code_rows, 1);
  else
    for (int i = 0; i < (few ? kNarrowRows / 16 : 7) && ok; ++i)
      ok = encode_codes(&p.x_map[i], x_codes, width / 2, code_rows, 16 * (i + 1));
  if (!ok) return fail(LF_E_CUDA, "expert_linear_mxfp4: cuTensorMapEncodeTiled failed");
  if (few) return launch_mx<1, kNarrowRows>(p, ceil_div(p.N, cut.height) * (groups + num_rows / kNarrowRows), stream);
  return launch_mx<2, kWideRows>(p, int64_t(ceil_div(p.N, 256)) * (groups + num_rows / kWideRows), stream);
}
