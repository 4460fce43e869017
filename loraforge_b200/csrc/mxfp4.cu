// MXFP4 quantisation: blocks of 32 values along a row share a power of two, each value is a
// 4-bit E2M1 number (sign, magnitudes 0 0.5 1 1.5 2 3 4 6).
//
// For a block of largest magnitude m the scale is 2^e, e = floor(log2 m) - 2 (2 is E2M1's
// largest exponent), not below 2^-127, held as the byte e + 127; the codes are x / 2^e rounded
// to nearest, ties to even, magnitudes over 6 to 6.  e comes from m's exponent bits and the
// division is by a power of two, so nothing is rounded but the code itself.  A block with an
// infinity or a NaN gets scale byte 255 (NaN) and codes 0.
//
// Both kernels are bound by HBM: 4.25 bits a value on one side, 16 or 32 on the other.  A
// thread takes 8 values (one or two 16-byte loads, 4 bytes of codes), so that four
// neighbouring lanes share a block and every access of a warp is contiguous.
#include "launch.cuh"

namespace lfb {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;  // groups of 8 values in flight a thread

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename T, bool kVector>
__device__ __forceinline__ void load8(const typename T::storage* p, float* f) {
  if (!kVector) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = T::to_float(p[i]);
  } else if constexpr (sizeof(typename T::storage) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
  }
}

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

// groups: groups of 8 values in all, per_row of them a row; a row of x starts at row * stride.
// Rows without gaps are one long row.  Every lane of a block's four takes part together:
// groups is a multiple of 4.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const typename T::storage* x, int64_t stride,
                                                            int64_t per_row, int64_t groups, uint32_t* codes,
                                                            uint8_t* scales) {
  pdl_wait();
  const int64_t first = int64_t(blockIdx.x) * (kThreads * kPerThread) + threadIdx.x;
  float v[kPerThread][8];
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t g = first + u * kThreads;
    if (g >= groups) continue;
    const int64_t row = g < per_row ? 0 : g / per_row;
    load8<T, kVector>(x + row * stride + (g - row * per_row) * 8, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t g = first + u * kThreads;
    uint32_t peak = 0;  // the largest magnitude's bits order like the magnitudes
    if (g < groups) {
#pragma unroll
      for (int i = 0; i < 8; ++i) peak = max(peak, __float_as_uint(v[u][i]) & 0x7fffffffu);
    }
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
    if (g >= groups) continue;
    const bool finite = peak < 0x7f800000u;
    const int scale = finite ? max(int(peak >> 23) - 2, 0) : 255;
    const float inverse = __uint_as_float(uint32_t(254 - scale) << 23);  // 2^(127 - scale), exact
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = finite ? v[u][i] * inverse : 0.f;
    codes[g] = e2m1x8(w);
    if ((g & 3) == 0) scales[g >> 2] = uint8_t(scale);
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
int launch_flat(void (*kernel)(Params...), int64_t groups, void* stream, const char* what, Args... args) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  config.gridDim = dim3(unsigned((groups + kThreads * kPerThread - 1) / (kThreads * kPerThread)));
  config.blockDim = dim3(kThreads);
  config.stream = static_cast<cudaStream_t>(stream);
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args...);
  if (err != cudaSuccess) {
    last_error() = std::string(what) + ": " + cudaGetErrorString(err);
    return LF_E_CUDA;
  }
  return LF_OK;
}

template <typename T>
int launch_quantize(const void* x, int64_t stride, int64_t rows, int64_t width, uint8_t* codes, uint8_t* scales,
                    void* stream) {
  using S = typename T::storage;
  const bool flat = stride == width || rows == 1;
  const int64_t groups = rows * (width / 8), per_row = flat ? groups : width / 8;
  const bool vec = aligned16(x) && (rows == 1 || stride * int64_t(sizeof(S)) % 16 == 0);
  return launch_flat(vec ? quantize_kernel<T, true> : quantize_kernel<T, false>, groups, stream, "mxfp4_quantize",
                     static_cast<const S*>(x), stride, per_row, groups, reinterpret_cast<uint32_t*>(codes), scales);
}

template <typename T>
int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t groups, void* out, void* stream) {
  return launch_flat(dequantize_kernel<T>, groups, stream, "mxfp4_dequantize",
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
