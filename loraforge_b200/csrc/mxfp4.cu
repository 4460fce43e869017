// MXFP4 quantisation: blocks of 32 values along a row share a power of two, each value is a
// 4-bit E2M1 number (sign, magnitudes 0 0.5 1 1.5 2 3 4 6).
//
// For a block of largest magnitude m the scale is 2^e, e = floor(log2 m) - 2 (2 is E2M1's
// largest exponent), not below 2^-127, held as the byte e + 127; the codes are x / 2^e rounded
// to nearest, ties to even, magnitudes over 6 to 6.  e comes from m's exponent bits and the
// division is by a power of two, so nothing is rounded but the code itself.  A block with an
// infinity or a NaN gets scale byte 255 (NaN) and codes 0.
//
// Both kernels are bound by HBM: 4.25 bits a value on one side, 16 or 32 on the other.  In the
// quantiser a thread takes 16 values, so two neighbouring lanes share a block: with 8 values a
// thread the address arithmetic, the shuffles and the scale's stores of every 8 values made it
// issue-bound (28672 x 4096 BF16: 82 us, now 44.5; back to BF16 46.9: 297 MB at 6.3-6.7 TB/s).
// Magnitudes of 16-bit types are compared in pairs.
#include "launch.cuh"

namespace lfb {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;  // dequantiser: groups of 8 values in flight a thread
constexpr int kUnits = 2;      // quantiser: units of 16 values in flight a thread

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Eight values as E2M1 codes, the first in the lowest nibble (nearest even, saturating).
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t codes;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(codes)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return codes;
}

// 16 values of T in 16-byte words, their FP32 values, and the bits of the largest magnitude as
// FP32, where an infinity or a NaN ends at 0x7f800000 or above.
template <typename T>
struct Unit {  // 16-bit types
  static constexpr int kWords = 2;
  static __device__ __forceinline__ void values(const uint4 (&q)[2], float* f) {
    unpack8<T>(q[0], f);
    unpack8<T>(q[1], f + 8);
  }
  static __device__ __forceinline__ uint32_t peak(const uint4 (&q)[2]) {
    // Magnitudes order like their bits, so two halves compare at once.
    const uint32_t w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    const uint32_t top = max(m & 0xffffu, m >> 16);
    typename T::storage h;
    *reinterpret_cast<uint16_t*>(&h) = uint16_t(top);
    return __float_as_uint(T::to_float(h)) & 0x7fffffffu;
  }
};
template <>
struct Unit<f32_t> {
  static constexpr int kWords = 4;
  static __device__ __forceinline__ void values(const uint4 (&q)[4], float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[4 * i] = __uint_as_float(q[i].x), f[4 * i + 1] = __uint_as_float(q[i].y);
      f[4 * i + 2] = __uint_as_float(q[i].z), f[4 * i + 3] = __uint_as_float(q[i].w);
    }
  }
  static __device__ __forceinline__ uint32_t peak(const uint4 (&q)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = max(m, max(max(q[i].x & 0x7fffffffu, q[i].y & 0x7fffffffu), max(q[i].z & 0x7fffffffu, q[i].w & 0x7fffffffu)));
    return m;
  }
};

// units: units of 16 values in all, per_row of them a row; a row of x starts at row * stride.
// Rows without gaps are one long row.  units is even, so both lanes of a block take part.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const typename T::storage* x, int64_t stride,
                                                            int64_t per_row, int64_t units, uint2* codes,
                                                            uint8_t* scales) {
  using U = Unit<T>;
  pdl_wait();
  const int64_t first = int64_t(blockIdx.x) * (kThreads * kUnits);
  const int live = int(min(units - first, int64_t(kThreads * kUnits)));  // units of this block
  uint4 q[kUnits][U::kWords];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int i = u * kThreads + threadIdx.x;
    if (i >= live) continue;
    const int64_t unit = first + i;
    const int64_t row = per_row == units ? 0 : unit / per_row;
    const typename T::storage* src = x + row * stride + (unit - row * per_row) * 16;
    if (kVector) {
#pragma unroll
      for (int w = 0; w < U::kWords; ++w) q[u][w] = reinterpret_cast<const uint4*>(src)[w];
    } else {
      typename T::storage* dst = reinterpret_cast<typename T::storage*>(q[u]);
#pragma unroll
      for (int j = 0; j < 16; ++j) dst[j] = src[j];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int i = u * kThreads + threadIdx.x;
    uint32_t peak = i < live ? U::peak(q[u]) : 0;
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    if (i >= live) continue;
    const bool finite = peak < 0x7f800000u;
    const int scale = finite ? max(int(peak >> 23) - 2, 0) : 255;
    const float inverse = __uint_as_float(uint32_t(254 - scale) << 23);  // 2^(127 - scale), exact
    float f[16];
    U::values(q[u], f);
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] *= inverse;
    const uint2 c = make_uint2(e2m1x8(f), e2m1x8(f + 8));
    (codes + first)[i] = finite ? c : make_uint2(0, 0);
    if ((i & 1) == 0) (scales + first / 2)[i >> 1] = uint8_t(scale);
  }
}

// Two E2M1 codes of a byte as FP32 (exact).
__device__ __forceinline__ float2 e2m1x2_value(uint32_t byte) {
  uint32_t h;
  asm("{\n .reg .b8 b;\n cvt.u8.u32 b, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint32_t* codes, const uint8_t* scales,
                                                              int64_t groups, typename T::storage* out) {
  pdl_wait();
  const int64_t first = int64_t(blockIdx.x) * (kThreads * kPerThread) + threadIdx.x;
  uint32_t c[kPerThread], s[kPerThread];
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t g = first + u * kThreads;
    if (g >= groups) continue;
    c[u] = codes[g];
    s[u] = scales[g >> 2];
  }
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t g = first + u * kThreads;
    if (g >= groups) continue;
    const float scale = __uint_as_float(s[u] == 255 ? 0x7fffffffu : s[u] == 0 ? 0x00400000u : s[u] << 23);
    alignas(16) typename T::storage o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e2m1x2_value(c[u] >> (8 * i) & 0xffu);
      o[2 * i] = T::from_float(f.x * scale);
      o[2 * i + 1] = T::from_float(f.y * scale);
    }
    constexpr int kWords = int(sizeof(typename T::storage)) * 8 / 16;
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      reinterpret_cast<uint4*>(out + g * 8)[i] = reinterpret_cast<const uint4*>(o)[i];
  }
}

template <typename... Params, typename... Args>
int launch_flat(void (*kernel)(Params...), int64_t blocks, void* stream, const char* what, Args... args) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  config.gridDim = dim3(unsigned(blocks));
  config.blockDim = dim3(kThreads);
  config.stream = static_cast<cudaStream_t>(stream);
  return launch_status(cudaLaunchKernelEx(&config, kernel, args...), what);
}

template <typename T>
int launch_quantize(const void* x, int64_t stride, int64_t rows, int64_t width, uint8_t* codes, uint8_t* scales,
                    void* stream) {
  using S = typename T::storage;
  const bool flat = stride == width || rows == 1;
  const int64_t units = rows * (width / 16), per_row = flat ? units : width / 16;
  const bool vec = aligned16(x) && (rows == 1 || stride * int64_t(sizeof(S)) % 16 == 0);
  return launch_flat(vec ? quantize_kernel<T, true> : quantize_kernel<T, false>,
                     (units + kThreads * kUnits - 1) / (kThreads * kUnits), stream, "mxfp4_quantize",
                     static_cast<const S*>(x), stride, per_row, units, reinterpret_cast<uint2*>(codes), scales);
}

template <typename T>
int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t groups, void* out, void* stream) {
  return launch_flat(dequantize_kernel<T>, (groups + kThreads * kPerThread - 1) / (kThreads * kPerThread), stream, "mxfp4_dequantize",
                     reinterpret_cast<const uint32_t*>(codes), scales, groups,
                     static_cast<typename T::storage*>(out));
}

int check_mx(const char* what, int dtype, int64_t rows, int64_t width) {
  if (dtype < LF_F32 || dtype > LF_BF16) return fail(LF_E_INVALID, (std::string(what) + ": unknown element type").c_str());
  if (rows < 0 || width < 32 || width % 32 || width >= (int64_t(1) << 31) || rows > (int64_t(1) << 40) / width)
    return fail(LF_E_INVALID, (std::string(what) + ": needs a width that is a multiple of 32 and at most 2^40 values").c_str());
  return LF_OK;
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" int lf_mxfp4_quantize(int32_t dtype, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                                 uint8_t* codes, uint8_t* scales, void* stream) {
  if (int rc = check_mx("mxfp4_quantize", dtype, rows, width)) return rc;
  if (x_stride < width) return fail(LF_E_INVALID, "mxfp4_quantize: row stride below the width");
  if (rows == 0) return LF_OK;
  if (!x || !codes || !scales || !aligned16(codes))
    return fail(LF_E_INVALID, "mxfp4_quantize: null buffer or codes not 16-byte aligned");
  if (dtype == LF_F32) return launch_quantize<f32_t>(x, x_stride, rows, width, codes, scales, stream);
  if (dtype == LF_F16) return launch_quantize<f16_t>(x, x_stride, rows, width, codes, scales, stream);
  return launch_quantize<bf16_t>(x, x_stride, rows, width, codes, scales, stream);
}

extern "C" int lf_mxfp4_dequantize(int32_t dtype, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                   int64_t width, void* out, void* stream) {
  if (int rc = check_mx("mxfp4_dequantize", dtype, rows, width)) return rc;
  if (rows == 0) return LF_OK;
  if (!codes || !scales || !out || !aligned16(codes) || !aligned16(out))
    return fail(LF_E_INVALID, "mxfp4_dequantize: null buffer, or codes or output not 16-byte aligned");
  const int64_t groups = rows * (width / 8);
  if (dtype == LF_F32) return launch_dequantize<f32_t>(codes, scales, groups, out, stream);
  if (dtype == LF_F16) return launch_dequantize<f16_t>(codes, scales, groups, out, stream);
  return launch_dequantize<bf16_t>(codes, scales, groups, out, stream);
}
