// Routing for mixture-of-experts layers and the weighted sum over a token's experts.
//
// Routing: with p = softmax(l) over E experts, each token takes the k largest logits (ties
// to the lowest index) and the weights w_j = scale . p_j, or scale . p_j / sum of the taken
// p (renormalised).  The taken (token, choice) slots are then sorted by expert, ties by
// slot, which gives the row tables that the expert products read.
//
// Combination: out[t] = sum_j w[t, j] . y[pos[t, j]], its gradient, and rows of no slot.
//
// All sums are FP32 in a fixed order; nothing depends on the order of atomics.
#include <float.h>

#include "launch.cuh"

namespace lfb {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kSortWarps = 8;         // of a block, that rank its slots
constexpr int kMaxRouteBlocks = 148;  // one wave; each block of the sort adds up the others' counts
constexpr int kMinBlockTokens = 64;  // two a warp; up to so many the whole call is one launch
constexpr int kBackThreads = 256;
constexpr int route_threads(int values) { return values > 8 ? kRouteThreads / 2 : kRouteThreads; }  // registers
constexpr int sort_bytes(int E) { return int(sizeof(int)) * E * (1 + kSortWarps); }

template <typename T>
__device__ __forceinline__ float load_value(const void* p, int64_t i);
template <>
__device__ __forceinline__ float load_value<f32_t>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float load_value<f16_t>(const void* p, int64_t i) {
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <>
__device__ __forceinline__ float load_value<bf16_t>(const void* p, int64_t i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_value(void* p, int64_t i, float v) {
  static_cast<typename T::storage*>(p)[i] = T::from_float(v);
}

// A logit as the routing sees it: NaN is never taken, +infinity is the largest finite value.
__device__ __forceinline__ float clean_logit(float v) {
  return v != v ? -INFINITY : fminf(v, FLT_MAX);
}

// Unsigned keys in the order of the floats (no NaN; -0 and +0 are one value).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kNoKey = 0x007fffffu;  // order_key(-infinity); 0 stands for a logit that was taken

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Lane holds the logits of experts lane, lane + 32, ...
template <typename T, int V>
__device__ __forceinline__ void load_logits(const void* logits, int64_t row, int E, int lane, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < E ? clean_logit(load_value<T>(logits, row + e)) : -INFINITY;
  }
}

// Stable sort of this block's slots by expert: base[e] (block b's first row of expert e) from
// the blocks' counts, then ranks inside the block from per-warp counts.
// kOwn: `counts` are this block's alone, in the same shared memory as the tables.
template <bool kOwn>
__device__ void scatter_slots(const int32_t* experts, const int32_t* counts, int blocks, int block, int64_t slot0,
                              int slots, int64_t all_slots, int E, int k, int32_t* offsets, int32_t* rows,
                              int32_t* positions, int* smem) {
  int* base = smem;                     // [E]: rows before expert e's, then before this block's of e
  int* wcount = base + E;               // [kSortWarps][E]
  int* found = wcount;                  // [parts][2][E] before that: all rows of e, those of earlier blocks
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x;
  __shared__ int warp_total[kRouteWarps];
  // Counts of the blocks, in up to four parts of them at a time.
  const int parts = kOwn ? 1 : max(1, min(kSortWarps / 2, threads / E));
  const int each = (blocks + parts - 1) / parts;
  for (int i = tid; i < parts * E; i += threads) {
    const int part = i / E, e = i - part * E;
    int total = 0, before = 0;
#pragma unroll 16
    for (int b = part * each; b < min(blocks, part * each + each); ++b) {
      const int c = kOwn ? counts[e] : __ldcg(counts + int64_t(b) * E + e);
      total += c;
      before += b < block ? c : 0;
    }
    found[(2 * part) * E + e] = total;
    found[(2 * part + 1) * E + e] = before;
  }
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += threads) {
    const int e = e0 + tid;
    int total = 0, before = 0;
    if (e < E)
      for (int part = 0; part < parts; ++part) {
        total += found[(2 * part) * E + e];
        before += found[(2 * part + 1) * E + e];
      }
    int scan = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += up;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int sums = lane < threads / 32 ? warp_total[lane] : 0;  // every warp scans the warps' totals
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sums, d);
      if (lane >= d) sums += up;
    }
    const int prefix = carry + (warp ? __shfl_sync(0xffffffffu, sums, warp - 1) : 0);
    carry += __shfl_sync(0xffffffffu, sums, 31);
    if (e < E) {
      base[e] = prefix + scan - total + before;
      if (block == 0) offsets[e] = prefix + scan - total;
    }
    __syncthreads();
  }
  if (block == 0 && tid == 0) offsets[E] = carry;
  // The first kSortWarps warps count their contiguous parts of the slots.
  const int part = (slots + kSortWarps - 1) / kSortWarps;
  const bool sorts = warp < kSortWarps;
  const int lo = sorts ? min(slots, warp * part) : 0, hi = sorts ? min(slots, lo + part) : 0;
  for (int i = tid; i < kSortWarps * E; i += threads) wcount[i] = 0;
  __syncthreads();
  for (int s = lo + lane; s < hi; s += 32) {
    const int e = experts[slot0 + s];
    if (e >= 0) atomicAdd(&wcount[warp * E + e], 1);
  }
  __syncthreads();
  for (int e = tid; e < E; e += threads) {
    int at = base[e];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = wcount[w * E + e];
      wcount[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int s0 = lo; s0 < hi; s0 += 32) {
    const int s = s0 + lane;
    const int e = s < hi ? experts[slot0 + s] : -1;
    const unsigned peers = __match_any_sync(0xffffffffu, e);
    int pos = -1;
    if (e >= 0) pos = wcount[warp * E + e] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && (peers >> lane) == 1u) wcount[warp * E + e] = pos + 1;  // the last of its peers
    __syncwarp();
    if (s < hi) {
      positions[slot0 + s] = pos;
      if (pos >= 0) rows[pos] = int32_t((slot0 + s) / k);
    }
  }
  // Rows of no slot.
  for (int64_t r = carry + int64_t(block) * threads + tid; r < all_slots; r += int64_t(blocks) * threads) rows[r] = -1;
}

// One warp a token: k times the largest remaining logit, as integer keys.  A lane keeps the best
// of its own V logits and looks through them again only after it lost it.  With one block the slots
// are sorted in the same launch, else the block leaves its counts for route_scatter_kernel.
// Bound by the latency of the k picks, so a block has a warp for every two of its 64 tokens.
// 8192 tokens, 256 experts, 8 taken: 20 us with the sort; one token of 64 experts: 4.
template <typename T, int V>
__global__ void __launch_bounds__(route_threads(V)) route_topk_kernel(
    const void* logits, int64_t stride, int num_tokens, int E, int k, int renormalize, float scale, int block_tokens,
    float* weights, int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* positions, int32_t* counts) {
  extern __shared__ int smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* hist = smem;
  for (int e = tid; e < E; e += blockDim.x) hist[e] = 0;
  pdl_wait();
  __syncthreads();
  // 64 bits: the last block's end passes 2^31 with near as many tokens.
  const int64_t t0 = int64_t(blockIdx.x) * block_tokens, t1 = min(int64_t(num_tokens), t0 + block_tokens);
  for (int64_t t = t0 + warp; t < t1; t += blockDim.x / 32) {
    float v[V];
    load_logits<T, V>(logits, t * stride, E, lane, v);
    uint32_t keys[V], best;
    int at;
#pragma unroll
    for (int i = 0; i < V; ++i) keys[i] = order_key(v[i]);
    auto look = [&]() {  // this lane's largest key, by halves: the lower index of two equal ones stays
      uint32_t m[V];
      int where[V];
#pragma unroll
      for (int i = 0; i < V; ++i) m[i] = keys[i], where[i] = i;
#pragma unroll
      for (int d = 1; d < V; d *= 2) {
#pragma unroll
        for (int i = 0; i + d < V; i += 2 * d) {
          const bool up = m[i + d] > m[i];
          m[i] = up ? m[i + d] : m[i];
          where[i] = up ? where[i + d] : where[i];
        }
      }
      best = m[0];
      at = where[0];
    };
    look();
    const uint32_t peak_key = __reduce_max_sync(0xffffffffu, best);
    const float peak = peak_key > kNoKey ? key_value(peak_key) : 0.f;
    uint32_t top = peak_key, my_key = 0;
    int my_expert = -1;
    for (int j = 0; j < k; ++j) {
      if (top <= kNoKey) break;
      const unsigned holders = __ballot_sync(0xffffffffu, best == top);
      int e = __shfl_sync(0xffffffffu, at * 32 + lane, __ffs(holders) - 1);
      if (holders & (holders - 1)) e = __reduce_min_sync(0xffffffffu, best == top ? at * 32 + lane : 0x7fffffff);
      if (lane == j) {
        my_expert = e;
        my_key = top;
      }
      if (lane == (e & 31)) {
#pragma unroll
        for (int i = 0; i < V; ++i) keys[i] = i == at ? 0 : keys[i];
        look();
      }
      __syncwarp();
      top = __reduce_max_sync(0xffffffffu, best);
    }
    const float mine = my_expert >= 0 ? expf(key_value(my_key) - peak) : 0.f;
    float sum = mine;
    if (!renormalize) {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += expf(v[i] - peak);
    }
    sum = warp_sum(sum);
    if (lane < k) {
      weights[t * k + lane] = my_expert >= 0 ? scale * (mine / sum) : 0.f;
      experts[t * k + lane] = my_expert;
      if (my_expert >= 0) atomicAdd(&hist[my_expert], 1);
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int e = tid; e < E; e += blockDim.x) counts[int64_t(blockIdx.x) * E + e] = hist[e];
    return;
  }
  scatter_slots<true>(experts, hist, 1, 0, 0, num_tokens * k, int64_t(num_tokens) * k, E, k, offsets, rows, positions,
                      smem);
}

__global__ void __launch_bounds__(kRouteThreads) route_scatter_kernel(const int32_t* experts, const int32_t* counts,
                                                                      int num_tokens, int E, int k, int block_tokens,
                                                                      int32_t* offsets, int32_t* rows,
                                                                      int32_t* positions) {
  extern __shared__ int smem[];
  pdl_wait();
  const int64_t t0 = int64_t(blockIdx.x) * block_tokens, t1 = min(int64_t(num_tokens), t0 + block_tokens);
  scatter_slots<false>(experts, counts, gridDim.x, blockIdx.x, t0 * k, int(t1 - t0) * k, int64_t(num_tokens) * k, E, k,
                       offsets, rows, positions, smem);
}

// dl_i = w_i (g_i - d) for the taken experts, with d = sum_j w_j g_j / scale, and for the
// others 0 (renormalised weights) or -scale . p_i . d.  One warp a token.
template <typename T, int V>
__global__ void __launch_bounds__(kBackThreads) route_backward_kernel(
    const void* logits, int64_t stride, const float* weights, const int32_t* experts, const float* grad,
    int64_t grad_stride, int num_tokens, int E, int k, int renormalize, float scale, void* grad_logits,
    int64_t out_stride) {
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * (kBackThreads / 32) + warp;
  if (t >= num_tokens) return;
  const int e = lane < k ? experts[t * k + lane] : -1;
  const bool live = e >= 0 && e < E;
  const float w = live ? weights[t * k + lane] : 0.f;
  const float g = live ? grad[t * grad_stride + lane] : 0.f;
  const float d = warp_sum(w * g) / scale;
  const bool any = __any_sync(0xffffffffu, live);
  const int64_t out = t * out_stride;
  if (renormalize || !any) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * 32 + lane < E) store_value<T>(grad_logits, out + i * 32 + lane, 0.f);
  } else {
    float v[V];
    load_logits<T, V>(logits, t * stride, E, lane, v);
    float peak = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) peak = fmaxf(peak, v[i]);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, m));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = expf(v[i] - peak);
      sum += v[i];
    }
    const float f = -scale * d / warp_sum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * 32 + lane < E) store_value<T>(grad_logits, out + i * 32 + lane, v[i] * f);
  }
  __syncwarp();  // the taken experts' entries are written after those of all
  if (live) store_value<T>(grad_logits, out + e, w * (g - d));
}

// ---------------------------------------------------------------- combination
// 16 bytes of T as FP32, and back.
template <typename T>
struct Vec;
template <typename T>
struct Vec16 {
  static constexpr int kWidth = 8;
  static __device__ __forceinline__ void load(const uint4& q, float* f) { unpack8<T>(q, f); }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 q;
    typename T::storage* h = reinterpret_cast<typename T::storage*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = T::from_float(f[i]);
    return q;
  }
};
template <>
struct Vec<bf16_t> : Vec16<bf16_t> {};
template <>
struct Vec<f16_t> : Vec16<f16_t> {};
template <>
struct Vec<f32_t> {
  static constexpr int kWidth = 4;
  static __device__ __forceinline__ void load(const uint4& q, float* f) {
    f[0] = __uint_as_float(q.x), f[1] = __uint_as_float(q.y), f[2] = __uint_as_float(q.z), f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// W values from column c: one 16-byte access, or element by element (unaligned rows, the end
// of a row; the values past it are zero).
template <typename T, bool kVector>
__device__ __forceinline__ void load_columns(const void* p, int64_t row, int c, int N, float* f) {
  constexpr int W = Vec<T>::kWidth;
  const typename T::storage* src = static_cast<const typename T::storage*>(p) + row + c;
  if (kVector) {
    Vec<T>::load(*reinterpret_cast<const uint4*>(src), f);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = c + i < N ? T::to_float(src[i]) : 0.f;
  }
}
template <typename T, bool kVector>
__device__ __forceinline__ void store_columns(void* p, int64_t row, int c, int N, const float* f) {
  constexpr int W = Vec<T>::kWidth;
  typename T::storage* dst = static_cast<typename T::storage*>(p) + row + c;
  if (kVector) {
    *reinterpret_cast<uint4*>(dst) = Vec<T>::pack(f);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (c + i < N) dst[i] = T::from_float(f[i]);
  }
}

// A thread sums one 16-byte column group over the token's k rows.  Bound by HBM: 8192 tokens x 2
// rows of 4096 BF16, 201 MB, in 35 us.
template <typename T, bool kVector>
__global__ void __launch_bounds__(128) combine_kernel(const void* y, int64_t y_stride, int64_t num_rows,
                                                      const float* weights, const int32_t* positions, int k, int N,
                                                      void* out, int64_t out_stride) {
  constexpr int W = Vec<T>::kWidth;
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int c = (blockIdx.y * 128 + threadIdx.x) * W;
  if (c >= N) return;
  float acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int pos = positions[t * k + j];
    if (pos < 0 || pos >= num_rows) continue;
    const float w = weights ? weights[t * k + j] : 1.f;
    float f[W];
    load_columns<T, kVector>(y, int64_t(pos) * y_stride, c, N, f);
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = fmaf(w, f[i], acc[i]);
  }
  store_columns<T, kVector>(out, t * out_stride, c, N, acc);
}

constexpr int kCombineWarps = 8;
constexpr int kTailBlocks = 64;

// One warp a slot: dy[pos] = w . g and dw = <g, y[pos]>.  The last blocks of the grid write
// zeros to the rows of no slot, which are the last ones: as many as slots without a position.
// Bound by HBM: 8192 tokens x 2 rows of 4096 BF16, 335 MB, in 49 us.  16-bit types take eight blocks
// an SM, so 32 registers: with 40, 2048 x 4 rows of 14336 FP16 took 115 us for 95.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kCombineWarps * 32, Vec<T>::kWidth == 8 ? 8 : 0) combine_backward_kernel(
    const void* grad, int64_t grad_stride, const void* y, int64_t y_stride, int64_t num_rows, const float* weights,
    const int32_t* positions, int64_t slots, int k, int N, void* grad_y, int64_t gy_stride, float* grad_weights,
    int slot_blocks) {
  constexpr int W = Vec<T>::kWidth;
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (int(blockIdx.x) >= slot_blocks) {
    __shared__ int part[kCombineWarps];
    int live = 0;
    for (int64_t s = threadIdx.x; s < slots; s += kCombineWarps * 32) live += positions[s] >= 0 ? 1 : 0;
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) part[warp] = live;
    __syncthreads();
    live = 0;
    for (int w = 0; w < kCombineWarps; ++w) live += part[w];
    float zero[W] = {};
    for (int64_t r = live + blockIdx.x - slot_blocks; r < num_rows; r += gridDim.x - slot_blocks)
      for (int c = threadIdx.x * W; c < N; c += kCombineWarps * 32 * W)
        store_columns<T, kVector>(grad_y, r * gy_stride, c, N, zero);
    return;
  }
  const int64_t s = int64_t(blockIdx.x) * kCombineWarps + warp;
  if (s >= slots) return;
  const int pos = positions[s];
  // Four sums a lane: chains of at most N / 128 + 1 additions, 7 more to join them and the lanes, so an
  // error of (N / 128 + 8) * 2^-24 of the sum of magnitudes.  (One sum: N / 32 additions.)
  float dot[4] = {};
  if (pos >= 0 && pos < num_rows) {
    const int64_t t = s / k;
    const float w = weights ? weights[s] : 1.f;
#pragma unroll 4
    for (int c = lane * W; c < N; c += 32 * W) {
      float g[W], v[W], d[W];
      load_columns<T, kVector>(grad, t * grad_stride, c, N, g);
      load_columns<T, kVector>(y, int64_t(pos) * y_stride, c, N, v);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        dot[i & 3] = fmaf(g[i], v[i], dot[i & 3]);
        d[i] = w * g[i];
      }
      store_columns<T, kVector>(grad_y, int64_t(pos) * gy_stride, c, N, d);
    }
  }
  const float sum = warp_sum((dot[0] + dot[1]) + (dot[2] + dot[3]));
  if (lane == 0 && grad_weights) grad_weights[s] = sum;
}

// ---------------------------------------------------------------- host
template <typename... Params, typename... Args>
int launch_pdl(void (*kernel)(Params...), dim3 grid, int threads, int smem, void* stream, const char* what,
               Args... args) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = static_cast<cudaStream_t>(stream);
  return launch_status(cudaLaunchKernelEx(&config, kernel, args...), what);
}

struct RoutePlan {
  int block_tokens, blocks;
};
RoutePlan route_plan(int64_t tokens) {
  int64_t per = (tokens + kMaxRouteBlocks - 1) / kMaxRouteBlocks;
  if (per < kMinBlockTokens) per = kMinBlockTokens;
  return {int(per), int((tokens + per - 1) / per)};
}

// tokens x k slots that int32 holds; the product is taken only where it fits 64 bits.
bool slots_ok(int64_t tokens, int k) {
  const int64_t limit = int64_t(1) << 31;
  return k >= 1 && k <= kMaxTopK && tokens >= 0 && tokens < limit && tokens * k < limit;
}

bool route_sizes_ok(int64_t tokens, int E, int k) {
  return E >= 1 && E <= kMaxExperts && k <= E && slots_ok(tokens, k);
}

// F<T, V> for the element type and the number of logits a lane holds.
template <typename T, typename F>
int with_width(int E, F&& f) {
  if (E <= 32) return f.template operator()<T, 1>();
  if (E <= 64) return f.template operator()<T, 2>();
  if (E <= 128) return f.template operator()<T, 4>();
  if (E <= 256) return f.template operator()<T, 8>();
  if (E <= 512) return f.template operator()<T, 16>();
  return f.template operator()<T, 32>();
}
template <typename F>
int with_type(int dtype, int E, F&& f) {
  if (dtype == LF_F32) return with_width<f32_t>(E, f);
  if (dtype == LF_F16) return with_width<f16_t>(E, f);
  return with_width<bf16_t>(E, f);
}

struct RouteCall {
  const void* logits;
  int64_t stride;
  int T, E, k, renormalize;
  float scale;
  float* weights;
  int32_t *experts, *offsets, *rows, *positions, *counts;
  void* stream;
  template <typename D, int V>
  int operator()() const {
    const RoutePlan plan = route_plan(T);
    const int threads = T > kSortWarps ? route_threads(V) : kSortWarps * 32;
    return launch_pdl(route_topk_kernel<D, V>, dim3(plan.blocks), threads, sort_bytes(E), stream, "route_experts", logits,
                      stride, T, E, k, renormalize, scale, plan.block_tokens, weights, experts, offsets, rows,
                      positions, counts);
  }
};

struct RouteBackwardCall {
  const void* logits;
  int64_t stride;
  const float* weights;
  const int32_t* experts;
  const float* grad;
  int64_t grad_stride;
  int T, E, k, renormalize;
  float scale;
  void* out;
  int64_t out_stride;
  void* stream;
  template <typename D, int V>
  int operator()() const {
    constexpr int kWarps = kBackThreads / 32;
    return launch_pdl(route_backward_kernel<D, V>, dim3(unsigned((int64_t(T) + kWarps - 1) / kWarps)), kBackThreads, 0,
                      stream, "route_experts_backward", logits, stride, weights, experts, grad, grad_stride, T, E, k,
                      renormalize, scale, out, out_stride);
  }
};

bool vector_rows(const void* p, int64_t stride, int N, int size) {
  return aligned16(p) && stride * size % 16 == 0 && int64_t(N) * size % 16 == 0;
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" int64_t lf_route_experts_workspace_ints(int64_t num_tokens, int32_t num_experts) {
  if (num_tokens < 0 || num_experts < 1 || num_experts > kMaxExperts) return -1;
  const int blocks = route_plan(num_tokens).blocks;
  return blocks > 1 ? int64_t(blocks) * num_experts : 0;
}

extern "C" int lf_route_experts(int32_t dtype, const void* logits, int64_t logits_stride, int64_t num_tokens,
                                int32_t num_experts, int32_t top_k, int32_t renormalize, float scale, float* weights,
                                int32_t* experts, int32_t* offsets, int32_t* rows, int32_t* positions,
                                int32_t* workspace, int64_t workspace_ints, void* stream) {
  if (!route_sizes_ok(num_tokens, num_experts, top_k))
    return fail(LF_E_INVALID, "route_experts: needs 1 <= top_k <= experts <= 1024, top_k <= 32 and slots that fit int32");
  if (dtype < LF_F32 || dtype > LF_BF16) return fail(LF_E_INVALID, "route_experts: unknown element type");
  if (!(scale > 0.f) || scale > FLT_MAX) return fail(LF_E_INVALID, "route_experts: scale must be positive and finite");
  if (logits_stride < num_experts) return fail(LF_E_INVALID, "route_experts: row stride below the number of experts");
  if (!offsets || (num_tokens && (!logits || !weights || !experts || !rows || !positions)))
    return fail(LF_E_INVALID, "route_experts: null buffer");
  if (num_tokens == 0) {
    if (cudaMemsetAsync(offsets, 0, sizeof(int32_t) * (size_t(num_experts) + 1), static_cast<cudaStream_t>(stream)) !=
        cudaSuccess)
      return check_launch("route_experts");
    return LF_OK;
  }
  const int64_t need = lf_route_experts_workspace_ints(num_tokens, num_experts);
  if (need && (!workspace || workspace_ints < need))
    return fail(LF_E_INVALID, "route_experts: workspace too small (see lf_route_experts_workspace_ints)");
  const RouteCall call{logits, logits_stride, int(num_tokens), num_experts, top_k,     renormalize ? 1 : 0, scale,
                       weights, experts,      offsets,         rows,        positions, workspace,           stream};
  if (int rc = with_type(dtype, num_experts, call)) return rc;
  const RoutePlan plan = route_plan(num_tokens);
  if (plan.blocks == 1) return LF_OK;
  return launch_pdl(route_scatter_kernel, dim3(plan.blocks), kRouteThreads, sort_bytes(num_experts), stream, "route_experts (sort)",
                    static_cast<const int32_t*>(experts), static_cast<const int32_t*>(workspace), int(num_tokens),
                    int(num_experts), int(top_k), plan.block_tokens, offsets, rows, positions);
}

extern "C" int lf_route_experts_backward(int32_t dtype, const void* logits, int64_t logits_stride,
                                         const float* weights, const int32_t* experts, const float* grad_weights,
                                         int64_t grad_stride, int64_t num_tokens, int32_t num_experts, int32_t top_k,
                                         int32_t renormalize, float scale, void* grad_logits, int64_t out_stride,
                                         void* stream) {
  if (!route_sizes_ok(num_tokens, num_experts, top_k))
    return fail(LF_E_INVALID, "route_experts_backward: needs 1 <= top_k <= experts <= 1024, top_k <= 32 and slots that fit int32");
  if (dtype < LF_F32 || dtype > LF_BF16) return fail(LF_E_INVALID, "route_experts_backward: unknown element type");
  if (!(scale > 0.f) || scale > FLT_MAX)
    return fail(LF_E_INVALID, "route_experts_backward: scale must be positive and finite");
  if (logits_stride < num_experts || out_stride < num_experts || grad_stride < top_k)
    return fail(LF_E_INVALID, "route_experts_backward: a row stride is below the row's length");
  if (num_tokens == 0) return LF_OK;
  if (!logits || !weights || !experts || !grad_weights || !grad_logits)
    return fail(LF_E_INVALID, "route_experts_backward: null buffer");
  return with_type(dtype, num_experts,
                   RouteBackwardCall{logits, logits_stride, weights, experts, grad_weights, grad_stride,
                                     int(num_tokens), num_experts, top_k, renormalize ? 1 : 0, scale, grad_logits,
                                     out_stride, stream});
}

namespace lfb {
namespace {
int combine_sizes(const char* what, int dtype, int64_t tokens, int k, int64_t rows, int N) {
  if (dtype < LF_F32 || dtype > LF_BF16) return fail(LF_E_INVALID, (std::string(what) + ": unknown element type").c_str());
  const int64_t limit = int64_t(1) << 31;  // the kernels' columns go up to 2048 past a row's last one
  if (!slots_ok(tokens, k) || rows < 0 || rows >= limit || N < 1 || N >= limit - 2048)
    return fail(LF_E_INVALID,
                (std::string(what) + ": needs 1 <= top_k <= 32 and slots, rows and columns that fit int32").c_str());
  return LF_OK;
}

template <typename T, bool kVector>
int launch_combine(const void* y, int64_t y_stride, int64_t rows, const float* weights, const int32_t* positions,
                   int64_t tokens, int k, int N, void* out, int64_t out_stride, void* stream) {
  using S = typename T::storage;
  constexpr int kColumns = 128 * Vec<T>::kWidth, kMost = 65535 * kColumns;  // of a block, and of a grid
  for (int64_t c = 0; c < N; c += kMost) {
    const int width = int(N - c < kMost ? N - c : kMost);
    if (int rc = launch_pdl(combine_kernel<T, kVector>, dim3(unsigned(tokens), (width + kColumns - 1) / kColumns), 128, 0,
                            stream, "combine_experts", static_cast<const void*>(static_cast<const S*>(y) + c), y_stride,
                            rows, weights, positions, k, width, static_cast<void*>(static_cast<S*>(out) + c), out_stride))
      return rc;
  }
  return LF_OK;
}

template <typename T, bool kVector>
int launch_combine_backward(const void* grad, int64_t grad_stride, const void* y, int64_t y_stride, int64_t rows,
                            const float* weights, const int32_t* positions, int64_t slots, int k, int N, void* grad_y,
                            int64_t gy_stride, float* grad_weights, void* stream) {
  const int blocks = int((slots + kCombineWarps - 1) / kCombineWarps);
  return launch_pdl(combine_backward_kernel<T, kVector>, dim3(blocks + kTailBlocks), kCombineWarps * 32, 0, stream,
                    "combine_experts_backward", grad, grad_stride, y, y_stride, rows, weights, positions, slots, k, N,
                    grad_y, gy_stride, grad_weights, blocks);
}
}  // namespace
}  // namespace lfb

extern "C" int lf_combine_experts(int32_t dtype, const void* y, int64_t y_stride, int64_t num_rows,
                                  const float* weights, const int32_t* positions, int64_t num_tokens, int32_t top_k,
                                  int32_t width, void* out, int64_t out_stride, void* stream) {
  if (int rc = combine_sizes("combine_experts", dtype, num_tokens, top_k, num_rows, width)) return rc;
  if (y_stride < width || out_stride < width)
    return fail(LF_E_INVALID, "combine_experts: a row stride is below the width");
  if (num_tokens == 0) return LF_OK;
  if ((num_rows && !y) || !positions || !out) return fail(LF_E_INVALID, "combine_experts: null buffer");
  const int size = dtype == LF_F32 ? 4 : 2;
  const bool vec = vector_rows(y, y_stride, width, size) && vector_rows(out, out_stride, width, size);
#define LFB_COMBINE(T)                                                                                          \
  return vec ? launch_combine<T, true>(y, y_stride, num_rows, weights, positions, num_tokens, top_k, width, out, \
                                       out_stride, stream)                                                      \
             : launch_combine<T, false>(y, y_stride, num_rows, weights, positions, num_tokens, top_k, width, out, \
                                        out_stride, stream)
  if (dtype == LF_F32) LFB_COMBINE(f32_t);
  if (dtype == LF_F16) LFB_COMBINE(f16_t);
  LFB_COMBINE(bf16_t);
#undef LFB_COMBINE
}

extern "C" int lf_combine_experts_backward(int32_t dtype, const void* grad, int64_t grad_stride, const void* y,
                                           int64_t y_stride, int64_t num_rows, const float* weights,
                                           const int32_t* positions, int64_t num_tokens, int32_t top_k, int32_t width,
                                           void* grad_y, int64_t grad_y_stride, float* grad_weights, void* stream) {
  if (int rc = combine_sizes("combine_experts_backward", dtype, num_tokens, top_k, num_rows, width)) return rc;
  if (y_stride < width || grad_stride < width || grad_y_stride < width)
    return fail(LF_E_INVALID, "combine_experts_backward: a row stride is below the width");
  if (num_tokens == 0 && num_rows == 0) return LF_OK;
  if ((num_tokens && (!grad || !positions)) || (num_rows && (!y || !grad_y)))
    return fail(LF_E_INVALID, "combine_experts_backward: null buffer");
  const int size = dtype == LF_F32 ? 4 : 2;
  const bool vec = vector_rows(y, y_stride, width, size) && vector_rows(grad, grad_stride, width, size) &&
                   vector_rows(grad_y, grad_y_stride, width, size);
  const int64_t slots = num_tokens * top_k;
#define LFB_COMBINE(T)                                                                                            \
  return vec ? launch_combine_backward<T, true>(grad, grad_stride, y, y_stride, num_rows, weights, positions,      \
                                                slots, top_k, width, grad_y, grad_y_stride, grad_weights, stream)  \
             : launch_combine_backward<T, false>(grad, grad_stride, y, y_stride, num_rows, weights, positions,     \
                                                 slots, top_k, width, grad_y, grad_y_stride, grad_weights, stream)
  if (dtype == LF_F32) LFB_COMBINE(f32_t);
  if (dtype == LF_F16) LFB_COMBINE(f16_t);
  LFB_COMBINE(bf16_t);
#undef LFB_COMBINE
}
