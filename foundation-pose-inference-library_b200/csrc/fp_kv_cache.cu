// Rows of keys and values into a paged cache and back (fpk_cache_write,
// fpk_cache_read, include/fpk.h).
//
// A cache page holds, per head, planes of 16-byte records (8 channels of a
// 16-bit cache, 16 of an e4m3 cache) over its rows: the tile that the attention
// kernels read without reordering it. e4m3 rows carry one power-of-two scale:
//   e = min{ e >= -100 : max|x| <= 448 * 2^e },  code = e4m3(x * 2^-e)
// A power of two costs e4m3, a floating format, no precision within its range,
// and makes code * scale exact in bf16, so that attention over the cache and
// reading it back use the same values.
//
// Both directions move each byte once and are bound by memory. Lanes take the
// groups of a row where those lie side by side in the dense rows (row-major),
// and 32 rows where the rows do (planar); the cache side is reached in 16-byte
// records either way, because slots are arbitrary.
#include <cfloat>
#include <cstdint>
#include <string>

#include "fp_heads.cuh"
#include "fp_launch.hpp"
#include "fp_profile.hpp"
#include "fp_tc.cuh"

namespace fpb {
namespace kvcache {

using namespace heads;

struct Args {
  unsigned char* cache[2];  // keys, values
  float* scale[2];
  fpk_heads_t dense[2];
  int rows, kv_heads, page_rows, page_shift;
  uint32_t total;  // slots of the cache
  const int32_t* slots;
  int* error_flag;
};

// max|x| over finite elements.
__device__ __forceinline__ float finiteMax(const float (&x)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = fabsf(x[i]);
    m = fmaxf(m, f <= FLT_MAX ? f : 0.0f);  // false for infinity and NaN
  }
  return m;
}

// Exponent of the scale. m = (1 + mant * 2^-23) * 2^(E - 127), 448 = 1.75 * 2^8.
__device__ __forceinline__ int scaleExponent(float m) {
  const int bits = __float_as_int(m);
  if (bits == 0) return 0;
  return max((bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), -100);
}

__device__ __forceinline__ float powerOfTwo(int e) { return __int_as_float((e + 127) << 23); }

// 8 elements as e4m3 codes; an infinity becomes NaN (e4m3 has none).
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float inv_scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = make_float2(x[2 * i] * inv_scale, x[2 * i + 1] * inv_scale);
    if (!(fabsf(f.x) <= FLT_MAX)) f.x = __int_as_float(0x7fffffff);
    if (!(fabsf(f.y) <= FLT_MAX)) f.y = __int_as_float(0x7fffffff);
    w[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Address of record `plane` of (slot, head).
template <int kPlanes>
__device__ __forceinline__ unsigned char* cacheRecord(const Args& a, int side, int slot, int head, int plane) {
  const int page = slot >> a.page_shift;
  const int r = slot & (a.page_rows - 1);
  const long long n = (static_cast<long long>(page) * a.kv_heads + head) * kPlanes + plane;
  return a.cache[side] + ((n << a.page_shift) + r) * 16;
}

__device__ __forceinline__ float* cacheScale(const Args& a, int side, int slot, int head) {
  const int page = slot >> a.page_shift;
  const int r = slot & (a.page_rows - 1);
  return a.scale[side] + (((static_cast<long long>(page) * a.kv_heads + head) << a.page_shift) + r);
}

// The row's slot, or -1 where it is left out.
__device__ __forceinline__ int slotOf(const Args& a, int row) {
  const int slot = __ldg(a.slots + row);
  if (slot < 0) return -1;
  if (static_cast<uint32_t>(slot) >= a.total) {
    reportIndex(a.error_flag, FPK_ERROR_SLOT);
    return -1;
  }
  return slot;
}

constexpr int kThreads = 256;

// Row-major rows: kGroups lanes per (row, keys or values, head).
template <typename T, int kGroups, bool kE4m3>
__global__ void __launch_bounds__(kThreads) writeRowsKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  constexpr int kPerBlock = kThreads / kGroups;
  const int g = threadIdx.x % kGroups;
  const long long item = static_cast<long long>(blockIdx.x) * kPerBlock + threadIdx.x / kGroups;
  const int per_row = 2 * a.kv_heads;
  const long long row_l = item / per_row;
  const bool inside = row_l < a.rows;
  const int row = inside ? static_cast<int>(row_l) : 0;
  const int rest = static_cast<int>(item - row_l * per_row);
  const int side = rest >= a.kv_heads ? 1 : 0;
  const int head = rest - side * a.kv_heads;
  const int slot = inside ? slotOf(a, row) : -1;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (slot >= 0) raw = *reinterpret_cast<const uint4*>(record(a.dense[side], head, row, g));
  if constexpr (!kE4m3) {
    if (slot >= 0) *reinterpret_cast<uint4*>(cacheRecord<kGroups>(a, side, slot, head, g)) = raw;
  } else {
    float x[8];
    unpack8<T>(raw, x);
    float m = finiteMax(x, 0.0f);
#pragma unroll
    for (int o = kGroups / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int e = scaleExponent(m);
    const uint2 codes = quantise8(x, powerOfTwo(-e));
    const uint32_t hx = __shfl_down_sync(0xffffffffu, codes.x, 1);
    const uint32_t hy = __shfl_down_sync(0xffffffffu, codes.y, 1);
    if (slot >= 0) {
      if (g % 2 == 0) {
        *reinterpret_cast<uint4*>(cacheRecord<kGroups / 2>(a, side, slot, head, g / 2)) = make_uint4(codes.x, codes.y, hx, hy);
      }
      if (g == 0) *cacheScale(a, side, slot, head) = powerOfTwo(e);
    }
  }
}

// Planar rows: a thread per (row, keys or values, head); a warp covers 32 rows.
template <typename T, int kGroups, bool kE4m3>
__global__ void __launch_bounds__(kThreads) writePlanarKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  const int row = blockIdx.x * 32 + (threadIdx.x & 31);
  const int rest = blockIdx.y * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.rows || rest >= 2 * a.kv_heads) return;
  const int side = rest >= a.kv_heads ? 1 : 0;
  const int head = rest - side * a.kv_heads;
  const int slot = slotOf(a, row);
  if (slot < 0) return;
  const unsigned char* src = record(a.dense[side], head, row, 0);
  const long long step = a.dense[side].plane_stride;
  uint4 raw[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) raw[g] = *reinterpret_cast<const uint4*>(src + g * step);
  if constexpr (!kE4m3) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) *reinterpret_cast<uint4*>(cacheRecord<kGroups>(a, side, slot, head, g)) = raw[g];
  } else {
    float m = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float x[8];
      unpack8<T>(raw[g], x);
      m = finiteMax(x, m);
    }
    const int e = scaleExponent(m);
    const float inv = powerOfTwo(-e);
#pragma unroll
    for (int g = 0; g < kGroups; g += 2) {
      float x[8], y[8];
      unpack8<T>(raw[g], x);
      unpack8<T>(raw[g + 1], y);
      const uint2 lo = quantise8(x, inv), hi = quantise8(y, inv);
      *reinterpret_cast<uint4*>(cacheRecord<kGroups / 2>(a, side, slot, head, g / 2)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    *cacheScale(a, side, slot, head) = powerOfTwo(e);
  }
}

// kPlanes lanes per (row, keys or values, head), one cache record each.
template <typename T, int kPlanes, bool kE4m3>
__global__ void __launch_bounds__(kThreads) readRowsKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  constexpr int kPerBlock = kThreads / kPlanes;
  const int p = threadIdx.x % kPlanes;
  const long long item = static_cast<long long>(blockIdx.x) * kPerBlock + threadIdx.x / kPlanes;
  const int per_row = 2 * a.kv_heads;
  const long long row_l = item / per_row;
  if (row_l >= a.rows) return;
  const int row = static_cast<int>(row_l);
  const int rest = static_cast<int>(item - row_l * per_row);
  const int side = rest >= a.kv_heads ? 1 : 0;
  const int head = rest - side * a.kv_heads;
  const int slot = slotOf(a, row);
  if (slot < 0) return;
  const uint4 raw = *reinterpret_cast<const uint4*>(cacheRecord<kPlanes>(a, side, slot, head, p));
  if constexpr (!kE4m3) {
    *reinterpret_cast<uint4*>(record(a.dense[side], head, row, p)) = raw;
  } else {
    uint4 out[2];
    dequantise16<T>(raw, *cacheScale(a, side, slot, head), out);
    *reinterpret_cast<uint4*>(record(a.dense[side], head, row, 2 * p)) = out[0];
    *reinterpret_cast<uint4*>(record(a.dense[side], head, row, 2 * p + 1)) = out[1];
  }
}

template <typename T, int kPlanes, bool kE4m3>
__global__ void __launch_bounds__(kThreads) readPlanarKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  const int row = blockIdx.x * 32 + (threadIdx.x & 31);
  const int rest = blockIdx.y * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.rows || rest >= 2 * a.kv_heads) return;
  const int side = rest >= a.kv_heads ? 1 : 0;
  const int head = rest - side * a.kv_heads;
  const int slot = slotOf(a, row);
  if (slot < 0) return;
  unsigned char* dst = record(a.dense[side], head, row, 0);
  const long long step = a.dense[side].plane_stride;
  uint4 raw[kPlanes];
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) raw[p] = *reinterpret_cast<const uint4*>(cacheRecord<kPlanes>(a, side, slot, head, p));
  if constexpr (!kE4m3) {
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) *reinterpret_cast<uint4*>(dst + p * step) = raw[p];
  } else {
    const float scale = *cacheScale(a, side, slot, head);
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
      uint4 out[2];
      dequantise16<T>(raw[p], scale, out);
      *reinterpret_cast<uint4*>(dst + (2 * p) * step) = out[0];
      *reinterpret_cast<uint4*>(dst + (2 * p + 1) * step) = out[1];
    }
  }
}

template <typename T, int kGroups, bool kE4m3>
cudaError_t launch(const Args& a, bool write, cudaStream_t s) {
  constexpr int kPlanes = kE4m3 ? kGroups / 2 : kGroups;
  prof::countLaunch(prof::kOther);
  if (a.dense[0].row_stride == 16 && a.dense[1].row_stride == 16) {
    const dim3 grid((a.rows + 31) / 32, (2 * a.kv_heads + kThreads / 32 - 1) / (kThreads / 32));
    return write ? launchPdl(writePlanarKernel<T, kGroups, kE4m3>, grid, dim3(kThreads), 0, s, a)
                 : launchPdl(readPlanarKernel<T, kPlanes, kE4m3>, grid, dim3(kThreads), 0, s, a);
  }
  const long long items = static_cast<long long>(a.rows) * 2 * a.kv_heads;
  const int per_block = kThreads / (write ? kGroups : kPlanes);
  const long long blocks = (items + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return write ? launchPdl(writeRowsKernel<T, kGroups, kE4m3>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, a)
               : launchPdl(readRowsKernel<T, kPlanes, kE4m3>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, a);
}

template <typename T>
cudaError_t launchType(const Args& a, int head_dim, bool e4m3, bool write, cudaStream_t s) {
  if (head_dim == 64) return e4m3 ? launch<T, 8, true>(a, write, s) : launch<T, 8, false>(a, write, s);
  return e4m3 ? launch<T, 16, true>(a, write, s) : launch<T, 16, false>(a, write, s);
}

int copy(const char* name, const fpk_cache_copy_desc_t* d, bool write, void* stream) {
  if (d == nullptr) return fail(std::string(name) + ": null descriptor");
  if (!is16Bit(d->dtype)) return fail(std::string(name) + ": dtype must be f16 or bf16");
  const std::string p = cacheProblem(d->cache, d->dtype);
  if (!p.empty()) return fail(std::string(name) + ": " + p);
  if (d->rows < 0 || d->cache.kv_heads > 65535) return fail(std::string(name) + ": bad sizes");
  if (d->rows == 0) return 0;
  for (const fpk_heads_t* v : {&d->k, &d->v}) {
    if (const char* q = headsProblem(*v)) return fail(std::string(name) + ": " + q);
  }
  if (d->slots == nullptr) return fail(std::string(name) + ": slots are required");
  const std::string where = deviceProblem(d->cache.k);
  if (!where.empty()) return fail(std::string(name) + ": " + where);
  Args a{};
  a.cache[0] = static_cast<unsigned char*>(d->cache.k);
  a.cache[1] = static_cast<unsigned char*>(d->cache.v);
  a.scale[0] = d->cache.k_scale;
  a.scale[1] = d->cache.v_scale;
  a.dense[0] = d->k;
  a.dense[1] = d->v;
  a.rows = d->rows;
  a.kv_heads = d->cache.kv_heads;
  a.page_rows = d->cache.page_rows;
  while ((1 << a.page_shift) < a.page_rows) ++a.page_shift;
  a.total = static_cast<uint32_t>(d->cache.n_pages) * static_cast<uint32_t>(d->cache.page_rows);
  a.slots = d->slots;
  a.error_flag = d->error_flag;
  const bool e4m3 = d->cache.dtype == FPK_DTYPE_E4M3;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == FPK_DTYPE_BF16 ? launchType<__nv_bfloat16>(a, d->cache.head_dim, e4m3, write, s)
                                                   : launchType<__half>(a, d->cache.head_dim, e4m3, write, s);
  if (e != cudaSuccess) return fail(std::string(name) + ": " + cudaGetErrorString(e));
  return 0;
}

}  // namespace kvcache
}  // namespace fpb

extern "C" int fpk_cache_write(const fpk_cache_copy_desc_t* desc, void* stream) {
  return fpb::kvcache::copy("fpk_cache_write", desc, true, stream);
}

extern "C" int fpk_cache_read(const fpk_cache_copy_desc_t* desc, void* stream) {
  return fpb::kvcache::copy("fpk_cache_read", desc, false, stream);
}
