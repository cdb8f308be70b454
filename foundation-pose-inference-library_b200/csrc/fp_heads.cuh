// Rows of heads, packed sequences and pages of cached rows: what the kernels
// behind fpk_qk_norm_rotary, fpk_cache_write / _read, fpk_attention_packed and
// fpk_attention_paged share. Device addressing, 16-bit and e4m3 conversions,
// and the host's checks of the descriptors (include/fpk.h).
//
// These kernels begin while the one before may still be writing what they will
// read (fp_launch.hpp), so they read with plain loads behind the wait: a load
// through the read-only path asks for memory that no one writes while the kernel
// lives.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "fpk.h"

namespace fpb {

int fail(const std::string& msg);
int checkLaunch(const char* what);

namespace heads {

// Address of 16-byte group g of head h in row r.
__device__ __forceinline__ unsigned char* record(const fpk_heads_t& v, int h, long long r, int g) {
  return static_cast<unsigned char*>(v.data) + h * v.head_stride + r * v.row_stride + g * v.plane_stride;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// Two e4m3 values as fp16 pairs (exact).
__device__ __forceinline__ uint32_t e4m3x2ToHalf2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

template <typename T>
__device__ __forceinline__ float largest() {
  return std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
}

// Whether a record holds NaN: 0x7f without its sign is the one code that 1 carries into bit 7.
__device__ __forceinline__ bool hasNan(const uint4& c) {
  const uint32_t m = 0x7f7f7f7fu, one = 0x01010101u;
  return ((((c.x & m) + one) | ((c.y & m) + one) | ((c.z & m) + one) | ((c.w & m) + one)) & 0x80808080u) != 0;
}

// The four e4m3 codes of a word times a row's scale, as two pairs of T, for
// scales from `low` to `high` (products within T's range) and words without
// NaN; dequantise16 below takes the others. One rounding at most.
template <typename T>
struct FastScale;
template <>
struct FastScale<__half> {
  static constexpr float low = 5.9604644775390625e-8f, high = 128.0f;  // 2^-24: what fp16 holds; 448 * 2^7 < 65504
  uint32_t factor;
  __device__ __forceinline__ explicit FastScale(float scale) {
    const __half2 h = __float2half2_rn(scale);
    factor = *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ uint32_t pair(uint32_t two) const {
    const uint32_t h = e4m3x2ToHalf2(two);
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&factor));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ uint2 operator()(uint32_t four) const { return make_uint2(pair(four), pair(four >> 16)); }
};
template <>
struct FastScale<__nv_bfloat16> {
  static constexpr float low = 7.888609052210118e-31f, high = 128.0f;  // 2^-100, 2^7: scale * 2^120 is a normal number
  uint32_t factor;
  __device__ __forceinline__ explicit FastScale(float scale) { factor = (__float_as_uint(scale * 1.329227995784916e36f) >> 16) * 0x10001u; }
  // Sign, exponent and mantissa moved to bf16's places are the value times
  // 2^-120 (subnormal numbers too); the factor holds the 2^120.
  __device__ __forceinline__ uint32_t pair(uint32_t codes_high) const {
    const uint32_t b = ((codes_high >> 4) & 0x07f007f0u) | (codes_high & 0x80008000u);
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&factor));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ uint2 operator()(uint32_t four) const {
    return make_uint2(pair(__byte_perm(four, 0, 0x1404)), pair(__byte_perm(four, 0, 0x3424)));
  }
};

// One 16-byte e4m3 record as two groups of 8 elements of T.
template <typename T>
__device__ __forceinline__ void dequantise16(const uint4& codes, float scale, uint4 (&out)[2]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t h = e4m3x2ToHalf2(w[half * 2 + (i >> 1)] >> ((i & 1) * 16));
      const float2 f = unpack2<__half>(h);
      x[2 * i] = f.x * scale;
      x[2 * i + 1] = f.y * scale;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // NaN passes (both comparisons are false).
      x[i] = x[i] > largest<T>() ? largest<T>() : (x[i] < -largest<T>() ? -largest<T>() : x[i]);
    }
    out[half] = pack8<T>(x);
  }
}

__device__ __forceinline__ void reportIndex(int* error_flag, int code) {
  if (error_flag != nullptr) atomicCAS(error_flag, 0, code);
}

// ---- host checks ----

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Arrays of int32 or float (NULL passes): a misaligned one would fault in the kernel.
inline bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// nullptr if the heads can be addressed, else what is wrong with them.
inline const char* headsProblem(const fpk_heads_t& v) {
  if (v.data == nullptr) return "null pointer";
  if (!aligned16(v.data) || v.head_stride % 16 || v.row_stride % 16 || v.plane_stride % 16) {
    return "data and strides must be multiples of 16 bytes";
  }
  return nullptr;
}

// Most rows of a call, and most rows times heads or keys of a sequence: kernels round
// them up to blocks in 32 bits.
constexpr long long kMost = (1LL << 31) - 1024;

inline bool is16Bit(int dtype) { return dtype == FPK_DTYPE_F16 || dtype == FPK_DTYPE_BF16; }

inline std::string cacheProblem(const fpk_kv_cache_t& c, int dtype) {
  if (c.k == nullptr || c.v == nullptr) return "the cache is null";
  if (!aligned16(c.k) || !aligned16(c.v)) return "the cache must be 16-byte aligned";
  if (c.dtype != FPK_DTYPE_E4M3 && c.dtype != dtype) return "a 16-bit cache must have the rows' type";
  if (c.dtype == FPK_DTYPE_E4M3 && (c.k_scale == nullptr || c.v_scale == nullptr)) return "an e4m3 cache needs k_scale and v_scale";
  if (!aligned4(c.k_scale) || !aligned4(c.v_scale)) return "k_scale and v_scale must be 4-byte aligned";
  if (c.head_dim != 64 && c.head_dim != 128) return "head_dim must be 64 or 128";
  if (c.page_rows < 16 || c.page_rows > 1024 || (c.page_rows & (c.page_rows - 1)) != 0) {
    return "page_rows must be a power of two from 16 to 1024";
  }
  if (c.n_pages <= 0 || c.kv_heads <= 0) return "n_pages and kv_heads must be positive";
  if (static_cast<long long>(c.n_pages) * c.page_rows >= (1LL << 31)) return "n_pages * page_rows must be below 2^31";
  return std::string();
}

// The launch goes to the current device: memory of another one, or of the host, is
// refused here instead of faulting there. Of all pointers of a call (NULL passes),
// some 30 ns each: the first, its largest array, must be device memory; page-locked
// host memory, which kernels reach, may hold the others.
inline std::string deviceProblem(std::initializer_list<const void*> pointers) {
  using Get = CUresult (*)(void*, CUpointer_attribute, CUdeviceptr);
  static const Get get = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r{};
    const bool ok = cudaGetDriverEntryPoint("cuPointerGetAttribute", &f, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<Get>(f) : nullptr;
  }();
  if (get == nullptr) return "cuPointerGetAttribute is not available";
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return std::string("current device: ") + cudaGetErrorString(e);
  unsigned type = 0;
  if (get(&type, CU_POINTER_ATTRIBUTE_MEMORY_TYPE, reinterpret_cast<CUdeviceptr>(*pointers.begin())) != CUDA_SUCCESS ||
      type == CU_MEMORYTYPE_HOST) {
    return "data is not in device memory";
  }
  for (const void* p : pointers) {
    if (p == nullptr) continue;
    int of = -1;
    if (get(&of, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, reinterpret_cast<CUdeviceptr>(p)) != CUDA_SUCCESS) return "data is not in device memory";
    if (of == dev) continue;
    cudaPointerAttributes at{};  // managed and host memory may belong to any
    if (cudaPointerGetAttributes(&at, p) == cudaSuccess && at.type == cudaMemoryTypeDevice) {
      return "data is on device " + std::to_string(of) + ", the current device is " + std::to_string(dev);
    }
  }
  return std::string();
}

}  // namespace heads
}  // namespace fpb
