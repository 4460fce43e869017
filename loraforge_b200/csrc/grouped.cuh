// Pieces shared by the expert products (16-bit and MXFP4): CTA pairs and clusters on tcgen05,
// gathered TMA rows, and the tile list over ragged groups of rows.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <string>

#include "launch.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace lfb {
namespace grouped {

using namespace tc;

constexpr int kMaxExperts = 1024;
constexpr int kMaxWarps = 14;

// Stages that fit beside `other` bytes of shared memory (and the tables of kMaxExperts groups).
constexpr int stages_of(int stage_bytes, int other) {
  return (227 * 1024 - 1024 - 512 - 4 * (kMaxWarps + 2 + 2 * (kMaxExperts + 1)) - other) / stage_bytes;
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Called by a kernel that prepares the next one's operands, after its own pdl_wait: the next one
// starts, may read whatever was complete before this kernel, and waits before it reads the rest.
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------ clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The shared::cluster address of `p` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float lds_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));  // the barriers around order it
  return v;
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Wait for the phase of `bar` with parity `parity`; false, with the CTA's abort word set, when it has
// not come after kWaitLimitNs, or when another role gave up.  kCluster: other CTAs arrive on it.  The
// abort word is read only when there is something to wait for: these waits stand between MMAs.
template <bool kCluster>
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (kCluster ? try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
  const uint64_t start = global_timer_ns();
  while (!(kCluster ? try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity))) {
    if (*abort) return false;
    if (global_timer_ns() - start > kWaitLimitNs) {
      atomicAdd(&g_lf_wait_timeouts, 1u);
      *abort = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_here(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return wait_for<false>(bar, parity, abort);
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return wait_for<true>(bar, parity, abort);
}
// One thread of a converged warp.  The MMA warp runs its loop whole and issues through this one, so
// that the descriptors are computed once for the warp (in one thread's branch each MMA cost some
// 100 cycles to issue, as much as it takes to run).
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(chosen));
  return chosen != 0;
}

// ------------------------------------------------------------------ tcgen05 on one CTA or a pair
template <int kCtas>
__device__ __forceinline__ void alloc_tmem(uint32_t* slot, uint32_t columns) {
  if constexpr (kCtas == 1) {
    tc_alloc(slot, columns);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int kCtas>
__device__ __forceinline__ void free_tmem(uint32_t addr, uint32_t columns) {
  if constexpr (kCtas == 1) {
    tc_dealloc(addr, columns);
  } else {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
  }
}
// D (+)= A . B^T, 16-bit operands (both of one type), FP32 sums.
template <int kCtas>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kCtas == 1) {
    tc_mma(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// Arrive on `bar`, in both CTAs of a pair, when this thread's MMAs so far are complete.
template <int kCtas>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (kCtas == 1) {
    tc_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
  }
}

// ------------------------------------------------------------------ TMA; `bar` may be the pair's first CTA's
template <int kCtas>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (kCtas == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  }
}
template <int kCtas>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if constexpr (kCtas == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
  }
}
// A box on its way into L2.
__device__ __forceinline__ void prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
constexpr int kAhead = 16;  // stages of W asked into L2 while the operands' other half is prepared
// Four rows of one box width, from columns c0 on; a row index past the tensor reads zeros.
template <int kCtas>
__device__ __forceinline__ void gather4(uint32_t dst, const CUtensorMap* map, int c0, const int (&r)[4], uint32_t bar) {
  if constexpr (kCtas == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
        "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
        : "memory");
  }
}

// 32 TMEM lanes x 32 columns as two halves of 16 lanes (r[0..15], r[16..31]): r[4j], r[4j+1] are
// lane t / 4, columns 8j + 2 (t % 4) and the next; r[4j+2], r[4j+3] the lane eight further.
__device__ __forceinline__ void ld_fragments(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr), "r"(taddr + (16u << 16)));
}

// Rows of `words` 16-byte words to `out` in the order of `rows`, zeros for an index outside x: one
// warp a row, eight words a lane in flight.
__device__ __forceinline__ void copy_row(const uint4* x, int64_t stride, int x_rows, const int32_t* rows, int64_t r,
                                         int words, uint4* out, int lane) {
  const int src = rows[r];
  const bool live = src >= 0 && src < x_rows;
  const uint4* from = x + (live ? src * stride : 0);
  uint4* to = out + r * words;
  for (int c = lane; c < words; c += 256) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c + 32 * u < words) v[u] = live ? from[c + 32 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c + 32 * u < words) to[c + 32 * u] = v[u];
  }
}

// ------------------------------------------------------------------ tiles of ragged groups
__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ constexpr int round_up(int a, int b) { return (a + b - 1) / b * b; }

// Inclusive scan over the CTA's threads of `v` under `op`, going on from `*carry`, which ends
// as the scan's last value.  `part`: one int a warp.  Two barriers.
template <typename Op>
__device__ __forceinline__ int scan_threads(int v, int* carry, int* part, Op&& op) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v = op(v, up);
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  int before = *carry, all = *carry;
  for (int w = 0; w < int(blockDim.x) / 32; ++w) {
    if (w < warp) before = op(before, part[w]);
    all = op(all, part[w]);
  }
  __syncthreads();
  *carry = all;
  return op(before, v);
}

// Fills bounds[0..E] with the groups' row bounds, ascending and in [0, R] whatever `offsets`
// holds, and starts[0..E] with the first tile of each group, `tiles_of(rows)` tiles a group.
// All threads of the CTA; ends with a barrier.
template <typename F>
__device__ void list_tiles(const int32_t* offsets, int E, int R, int* bounds, int* starts, int* part, F&& tiles_of) {
  const int tid = threadIdx.x;
  int largest = 0, total = 0;
  for (int e0 = 0; e0 <= E; e0 += int(blockDim.x)) {
    const int e = e0 + tid;
    const int v = scan_threads(e <= E ? min(max(offsets[e], 0), R) : 0, &largest, part,
                               [](int a, int b) { return max(a, b); });
    if (e <= E) bounds[e] = v;
  }
  __syncthreads();
  for (int e0 = 0; e0 < E; e0 += int(blockDim.x)) {
    const int e = e0 + tid;
    const int n = e < E ? tiles_of(bounds[e + 1] - bounds[e]) : 0;
    const int v = scan_threads(n, &total, part, [](int a, int b) { return a + b; });
    if (e < E) starts[e] = v - n;
  }
  if (tid == 0) starts[E] = total;
  __syncthreads();
}

// The group of tile t, e at least: the last with starts[e] <= t (empty groups share their
// successor's start).
__device__ __forceinline__ int group_of(const int* starts, int E, int t, int e = 0) {
  int lo = e, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Walks one CTA's tiles t = first, first + stride, ...: a group's mt feature tiles x nt column tiles in
// bands of up to eight column tiles, inside a band column tiles fastest, so that the CTAs of a
// wave share both operands in L2.  What holds for a group is kept from tile to tile and the
// divisions are multiplications by a reciprocal: between two tiles nothing covers this.
constexpr int kBand = 8;
struct Bands {
  int mt;            // feature tiles
  uint64_t by_band;  // 2^64 / (kBand * mt), rounded up: exact for dividends below 2^32
};
inline Bands bands_of(int mt) { return {mt, ~0ull / (uint64_t(kBand) * uint64_t(mt)) + 1}; }

struct Walk {
  int e, m, n;         // group, feature tile, column tile
  int lo, hi, nt;      // the group's rows, its column tiles
  int start, end;      // its first tile, and the tile after its last
  uint32_t by_last;    // 2^32 / the columns of its last band, rounded up: exact for dividends below 2^29

  __device__ __forceinline__ Walk() : e(-1), end(-1) {}
  // Moves to tile t; true when it is the first one here of its group.  columns_of(rows): the number
  // of column tiles.
  template <typename F>
  __device__ __forceinline__ bool go(const Bands& bands, const int* bounds, const int* starts, int E, int t,
                                     F&& columns_of) {
    const bool moved = t >= end;
    if (moved) {
      e = group_of(starts, E, t, e + 1);
      lo = bounds[e];
      hi = bounds[e + 1];
      start = starts[e];
      end = starts[e + 1];
      nt = columns_of(hi - lo);
      if (nt % kBand > 1) by_last = 0xffffffffu / uint32_t(nt % kBand) + 1;
    }
    const uint32_t q = uint32_t(t - start), band = nt <= kBand ? 0 : uint32_t(__umul64hi(q, bands.by_band));
    const uint32_t w = q - band * uint32_t(kBand * bands.mt);
    const int width = min(kBand, nt - int(band) * kBand);
    m = width == kBand ? int(w / kBand) : width == 1 ? int(w) : int(__umulhi(w, by_last));
    n = int(band) * kBand + int(w) - m * width;
    return moved;
  }
};

// ------------------------------------------------------------------ host
inline PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static std::mutex mutex;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::lock_guard<std::mutex> lock(mutex);
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &status) == cudaSuccess &&
        status == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }
  return fn;
}

// A map of `ndim` dimensions (innermost first, strides in bytes from the second on) with
// 128-byte swizzle; false when the driver refuses it.
inline bool encode_map(CUtensorMap* map, CUtensorMapDataType type, int ndim, const void* base, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = map_encoder();
  const cuuint32_t ones[3] = {1, 1, 1};
  return encode && encode(map, type, ndim, const_cast<void*>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ------------------------------------------------------------------ stores
constexpr int kMaxSplit = 8;
constexpr int kChunkBytes = 32 * 64;  // 32 columns x 32 features of a warp, 16 bits

// Rows of `features` values, `stride` apart, of type LF_F32, LF_F16 or LF_BF16.
struct Output {
  void* data;
  int64_t stride;
  int features, type;
};

__device__ __forceinline__ void store_value(const Output& o, int64_t at, float v) {
  if (o.type == LF_BF16) static_cast<__nv_bfloat16*>(o.data)[at] = __float2bfloat16_rn(v);
  else if (o.type == LF_F16) static_cast<__half*>(o.data)[at] = __float2half_rn(v);
  else static_cast<float*>(o.data)[at] = v;
}

// Zeros to the rows of no group, [0, first) and [last, R), spread over the grid.  `first` is above 0
// where the groups are part of a longer table, as on a rank that holds some of the experts.
__device__ __forceinline__ void zero_rows(const Output& o, int first, int last, int R) {
  const int size = o.type == LF_F32 ? 4 : 2;
  const int64_t bytes = int64_t(o.features) * size;
  const int64_t none = int64_t(first) + (R - last);
  for (int64_t i = blockIdx.x; i < none; i += gridDim.x) {
    const int64_t r = i < first ? i : i - first + last;
    uint8_t* row = static_cast<uint8_t*>(o.data) + r * o.stride * size;
    if (((reinterpret_cast<uintptr_t>(row) | uintptr_t(bytes)) & 15) == 0) {
      for (int64_t b = threadIdx.x * 16; b < bytes; b += blockDim.x * 16)
        *reinterpret_cast<uint4*>(row + b) = make_uint4(0, 0, 0, 0);
    } else {
      for (int64_t b = threadIdx.x * 2; b < bytes; b += blockDim.x * 2) *reinterpret_cast<uint16_t*>(row + b) = 0;
    }
  }
}

// Columns c0 .. c0 + 31 of this warp's 32 features as 16-bit values to global memory.  The
// accumulator is read in the fragment shape whose transpose stmatrix writes, so that a column's
// 32 features (64 bytes) lie together in the warp's staging, 16-byte chunks swizzled by column;
// each store instruction then writes eight columns.  `dst`: feature 0 of column c0.
__device__ __forceinline__ void store_chunk(uint32_t taddr, bool live, uint32_t staging, int bf16, uint8_t* dst,
                                            int64_t pitch, int columns, int features, int lane) {
  uint32_t r[32];
  if (live) {
    ld_fragments(taddr, r);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = 0;
  }
  __syncwarp();  // the previous chunk has left the staging
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // eight columns each
    uint32_t m[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // eight features each
      const uint32_t lo = r[(h >> 1) * 16 + 4 * j + 2 * (h & 1)], hi = r[(h >> 1) * 16 + 4 * j + 2 * (h & 1) + 1];
      if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(m[h]) : "f"(__uint_as_float(hi)), "f"(__uint_as_float(lo)));
      else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(m[h]) : "f"(__uint_as_float(hi)), "f"(__uint_as_float(lo)));
    }
    const int col = 8 * j + (lane & 7), chunk = lane >> 3;
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     staging + uint32_t(col * 64 + ((chunk ^ (col >> 1 & 3)) << 4))),
                 "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3])
                 : "memory");
  }
  __syncwarp();
  const int chunk = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = 8 * i + (lane >> 2);
    const uint4 v = lds16(staging + uint32_t(col * 64 + ((chunk ^ (col >> 1 & 3)) << 4)));
    if (col < columns && 8 * chunk < features) *reinterpret_cast<uint4*>(dst + col * pitch + 16 * chunk) = v;
  }
}

// A tile's columns 0 .. valid - 1 of this warp's features f0 .. f0 + 31, those below `end` (TMEM
// address `d`; zeros unless live), to rows row0 + column; of `parts` warps this one takes chunk `part`,
// part + parts, ...
__device__ __forceinline__ void store_whole(const Output& o, uint32_t d, bool live, int f0, int end, int64_t row0, int nt,
                                            int valid, uint32_t staging, int lane, int part = 0, int parts = 1) {
  if (o.type != LF_F32 && (reinterpret_cast<uintptr_t>(o.data) & 15) == 0 && o.stride % 8 == 0 && o.features % 8 == 0) {
    uint8_t* dst = static_cast<uint8_t*>(o.data) + (row0 * o.stride + f0) * 2;
    for (int c0 = 32 * part; c0 < valid; c0 += 32 * parts)
      store_chunk(d + uint32_t(c0), live, staging, o.type == LF_BF16, dst + c0 * o.stride * 2, o.stride * 2, valid - c0,
                  end - f0, lane);
  } else {
    for (int c0 = 16 * part; c0 < nt; c0 += 16 * parts) {
      uint32_t r[16];
      if (live) tc_ld16(d + uint32_t(c0), r);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (f0 + lane < end && c0 + j < valid)
          store_value(o, (row0 + c0 + j) * o.stride + f0 + lane, live ? __uint_as_float(r[j]) : 0.f);
    }
  }
}

// The same for a contraction split over the cluster's CTAs: the partial sums go to this CTA's
// `part` [columns][128 features], then every CTA adds a share of the columns over all CTAs in
// rank order.  `parts`: how often the caller came here before.  False after an expired wait.
template <typename F>
__device__ __forceinline__ bool store_split(const Output& o, uint32_t d, bool live, int f0, int end, int64_t row0, int nt,
                                            int valid, float* part, uint64_t* part_full, uint64_t* part_empty,
                                            int parts, int cluster, int rank, int quarter, int lane,
                                            volatile int* abort, F&& release) {
  if (!__all_sync(0xffffffffu, wait_cluster(part_empty, (uint32_t(parts) & 1u) ^ 1u, abort))) return false;
  float* mine = part + quarter * 32 + lane;
  for (int c0 = 0; c0 < nt; c0 += 16) {
    uint32_t r[16];
    if (live) tc_ld16(d + uint32_t(c0), r);
#pragma unroll
    for (int j = 0; j < 16; ++j) mine[(c0 + j) * 128] = live ? __uint_as_float(r[j]) : 0.f;
  }
  release();
  __syncwarp();
  if (lane < cluster) arrive_cluster(mapa(part_full, lane));
  if (!__all_sync(0xffffffffu, wait_cluster(part_full, uint32_t(parts) & 1u, abort))) return false;
  uint32_t peer[kMaxSplit];
#pragma unroll
  for (int q = 0; q < kMaxSplit; ++q)
    if (q < cluster) peer[q] = mapa(mine, q);
  for (int c0 = rank; c0 < valid; c0 += 4 * cluster) {  // four columns' loads in flight
    float sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = uint32_t(min(c0 + i * cluster, valid - 1)) * 512u;
      float v[kMaxSplit];
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        if (q < cluster) v[q] = lds_cluster(peer[q] + at);
      sum[i] = 0.f;
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        if (q < cluster) sum[i] += v[q];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + i * cluster;
      if (c < valid && f0 + lane < end) store_value(o, (row0 + c) * o.stride + f0 + lane, sum[i]);
    }
  }
  __syncwarp();
  if (lane < cluster) arrive_cluster(mapa(part_empty, lane));
  return true;
}

// How the narrow kernels cut the work: `height` features a tile (the MMA always takes 128 lanes;
// rows of A past the height are neither loaded nor stored) and the contraction over `split` CTAs.
struct Cut {
  int height, split;
};

// How many clusters of 1, 2, .. kMaxSplit CTAs the device holds at a time (148 SMs, one CTA each: 33 of
// 4, 15 of 8, as clusters stay inside a GPC), 0 where it cannot place one.  More in a persistent grid
// would run in a second wave.
struct Clusters {
  int at_once[kMaxSplit + 1];
};
inline int count_clusters(const void* kernel, int threads, int smem, Clusters* out) {
  for (int s = 1; s <= kMaxSplit; ++s) {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = s;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    config.gridDim = dim3(s);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess)
      return check_launch("cudaOccupancyMaxActiveClusters");
    out->at_once[s] = n > 0 ? n : 0;
  }
  return LF_OK;
}
// The same, counted once for a kernel, its threads and shared memory, and a device; from any thread.
template <typename P>
int clusters_of(void (*kernel)(P), int threads, int smem, Clusters* out) {
  struct Known {
    const void* kernel;
    int device, threads, smem;
    Clusters clusters;
  };
  constexpr int kMostKnown = 256;  // past these, counted in every call
  static std::mutex mutex;
  static Known known[kMostKnown];
  static int count = 0;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return check_launch("cudaGetDevice");
  const void* key = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(mutex);
  for (int i = 0; i < count; ++i)
    if (known[i].kernel == key && known[i].device == device && known[i].threads == threads && known[i].smem == smem) {
      *out = known[i].clusters;
      return LF_OK;
    }
  if (int rc = count_clusters(key, threads, smem, out)) return rc;
  if (count < kMostKnown) known[count++] = {key, device, threads, smem, *out};
  return LF_OK;
}

// The cut with the least time for `groups` groups of one row tile each and `steps` stages.  What
// costs is the bytes of the weights a CTA streams, height x stages of 128 bytes at some 44 GB/s:
// 2.9 ns each, the unit here.  Whole waves count (896 tiles of 128 over 148 CTAs are 7 waves for
// 6.05 waves' work; 1024 tiles of 112 are 6.9).  A tile costs 0.5 us more, and where a cluster adds
// up its parts 4 us that only other tiles' loads cover.  A CTA's steps are a multiple of `whole`.
// Splits over clusters that the device cannot place are left out.
inline Cut choose_cut(const Clusters& clusters, int64_t groups, int M, int steps, int whole, bool any_height) {
  Cut best{128, 1};
  double least = 1e30;
  for (int s = 1; s <= kMaxSplit && (s == 1 || steps >= 4 * s); ++s) {
    if (clusters.at_once[s] < 1) continue;
    for (int h = 128; h >= (any_height ? 64 : 128); h -= 8) {
      const int64_t tiles = groups * ceil_div(M, h), wave = clusters.at_once[s];
      const double waves = double((tiles + wave - 1) / wave), joined = s > 1 ? 1400 : 0;
      const double tile = double(h) * round_up(ceil_div(steps, s), whole) + 170;
      const double cost = waves * (tile > joined ? tile : joined) + joined;
      if (cost < 0.98 * least) {
        least = cost;
        best = {h, s};
      }
    }
  }
  return best;
}

// ------------------------------------------------------------------ launch
// CTAs of a persistent grid over at most `tiles` tiles, one cluster each at a time; 0, with the error
// set, where the device cannot place the cluster.
inline int grid_of(const Clusters& clusters, int64_t tiles, int cluster, const char* what) {
  const int at_once = clusters.at_once[cluster];
  if (at_once < 1) {
    last_error() = std::string(what) + ": the device cannot place a cluster of " + std::to_string(cluster) + " CTAs";
    return 0;
  }
  return int(tiles < at_once ? tiles : at_once) * cluster;
}

template <typename P>
int launch_clusters(void (*kernel)(P), int grid, int threads, int cluster, int smem, void* stream, const char* what,
                    const P& p) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 2;
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = static_cast<cudaStream_t>(stream);
  return launch_status(cudaLaunchKernelEx(&config, kernel, p), what);
}

}  // namespace grouped
}  // namespace lfb
