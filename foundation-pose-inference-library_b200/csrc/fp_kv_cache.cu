// Rows of keys and values into a paged cache and back (fpk_cache_write,
// fpk_cache_read, include/fpk.h).
//
// A cache page holds, per head, planes of 16-byte records (8 channels of a
// 16-bit cache, 16 of an e4m3 cache) over its rows: a 16-bit tile is what the
// attention kernels read without reordering it. e4m3 rows carry one power-of-two scale:
//   e = min{ e >= -100 : max|x| <= 448 * 2^e },  code = e4m3(x * 2^-e)
// A power of two costs e4m3, a floating format, no precision within its range,
// and makes code * scale exact in bf16, so that attention over the cache and
// reading it back use the same values.
//
// Both directions move each byte once and are bound by memory. Lanes take the
// groups of a row where those lie side by side in the dense rows (row-major),
// and 32 rows where the rows do (planar); the cache side is reached in 16-byte
// records either way, because slots are arbitrary.
//
// Measured (8 heads of 128, bf16 rows, pages of 64; us): e4m3 cache, 16,384 rows
// written to random slots 71, to slots in order 28; 20,011 read back from random
// slots 35, in order 28 (floors 15.5 and 19). 16-bit cache 139, 41, 70 and 31 (floors
// 20.5 and 25). A random slot touches half of each 32-byte sector, and those touches,
// not bytes, are what the L2 is busy with; in order too a row's records are stored
// and read by themselves, page_rows x 16 bytes apart.
#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <string>
#include <type_traits>

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

// max|x| of a 16-byte group of T, NaN left out.
template <typename T>
__device__ __forceinline__ float groupMax(const uint4& w) {
  using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
  auto abs2 = [](const uint32_t& u) { return __habs2(*reinterpret_cast<const T2*>(&u)); };
  const T2 m = __hmax2(__hmax2(abs2(w.x), abs2(w.y)), __hmax2(abs2(w.z), abs2(w.w)));
  const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&m));
  return fmaxf(f.x, f.y);
}

// The same over finite elements only, for rows that hold an infinity.
template <typename T>
__device__ __noinline__ float groupFiniteMax(uint4 w) {
  float x[8], m = 0.0f;
  unpack8<T>(w, x);
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

// 8 elements as e4m3 codes, rounded to nearest even. NaN stays NaN; an infinity
// becomes NaN (e4m3 has none), which `finite` says need not be looked for.
template <typename T>
__device__ __forceinline__ uint2 quantise8(const uint4& raw, float inv_scale, bool finite) {
  float x[8];
  unpack8<T>(raw, x);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = make_float2(x[2 * i] * inv_scale, x[2 * i + 1] * inv_scale);
    if (!finite) {
      if (!(fabsf(f.x) <= FLT_MAX)) f.x = __int_as_float(0x7fffffff);
      if (!(fabsf(f.y) <= FLT_MAX)) f.y = __int_as_float(0x7fffffff);
    }
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
  const int slot = a.slots[row];
  if (slot < 0) return -1;
  if (static_cast<uint32_t>(slot) >= a.total) {
    reportIndex(a.error_flag, FPK_ERROR_SLOT);
    return -1;
  }
  return slot;
}

// Dense rows that are written pass once and give way in L2 to the cache's
// lines, whose other records other rows will ask for.
__device__ __forceinline__ uint64_t passingPolicy() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void storePassing(void* p, const uint4& v, uint64_t policy) {
  asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1,%2,%3,%4}, %5;" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "l"(policy) : "memory");
}

constexpr int kThreads = 256;

// Row-major rows: kLanes lanes per (row, keys or values, head). A thread keeps
// its (side, head, group) and takes kUnroll rows, whose loads are in flight
// together: slots and elements do not wait for each other.
struct Lane {
  int row, step;  // first row, distance to the next
  int side, head, group;
  bool active;
};

// Rows of a thread. Writing, and reading 16-bit rows, gain from loads in flight
// (sequential slots of 16-bit rows: 30 us read with 4, 42 with 1, for 20,011
// rows of 8 heads); reading e4m3 gains from more warps (36 us with 1, 46 with 4).
constexpr int kWriteRows = 4;
template <bool kE4m3>
constexpr int kReadRows = kE4m3 ? 1 : 4;

// Block of kThreads: as many rows side by side as fit; blockIdx.y walks the
// lanes of a row wider than a block.
template <int kLanes, int kUnroll>
__device__ __forceinline__ Lane laneOf(const Args& a) {
  const int width = 2 * a.kv_heads * kLanes;
  const int side_by_side = max(kThreads / width, 1);
  const int x = threadIdx.x + blockIdx.y * kThreads;
  Lane n;
  const int sub = width > kThreads ? 0 : x / width;
  const int rest = x - sub * width;
  n.row = blockIdx.x * side_by_side * kUnroll + sub;
  n.step = side_by_side;
  n.active = sub < side_by_side && rest < width;
  const int item = n.active ? rest / kLanes : 0;
  n.group = rest % kLanes;
  n.side = item >= a.kv_heads ? 1 : 0;
  n.head = item - n.side * a.kv_heads;
  return n;
}

inline dim3 laneGrid(const Args& a, int lanes, int unroll) {
  const int width = 2 * a.kv_heads * lanes;
  const int rows = std::max(kThreads / width, 1) * unroll;
  return dim3((a.rows + rows - 1) / rows, width > kThreads ? (width + kThreads - 1) / kThreads : 1);
}

template <typename T, int kGroups, bool kE4m3>
__global__ void __launch_bounds__(kThreads) writeRowsKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  constexpr int kUnroll = kWriteRows;
  const Lane n = laneOf<kGroups, kUnroll>(a);
  int slot[kUnroll];
  uint4 raw[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int row = n.row + i * n.step;
    const bool in = n.active && row < a.rows;
    slot[i] = in ? slotOf(a, row) : -1;
    raw[i] = in ? *reinterpret_cast<const uint4*>(record(a.dense[n.side], n.head, row, n.group)) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if constexpr (!kE4m3) {
      if (slot[i] >= 0) *reinterpret_cast<uint4*>(cacheRecord<kGroups>(a, n.side, slot[i], n.head, n.group)) = raw[i];
    } else {
      float m = groupMax<T>(raw[i]);
#pragma unroll
      for (int o = kGroups / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool finite = __all_sync(0xffffffffu, m <= FLT_MAX);
      if (!finite) {
        m = groupFiniteMax<T>(raw[i]);
#pragma unroll
        for (int o = kGroups / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      const int e = scaleExponent(m);
      const uint2 codes = quantise8<T>(raw[i], powerOfTwo(-e), finite);
      const uint32_t hx = __shfl_down_sync(0xffffffffu, codes.x, 1);
      const uint32_t hy = __shfl_down_sync(0xffffffffu, codes.y, 1);
      if (slot[i] >= 0) {
        if (n.group % 2 == 0) {
          *reinterpret_cast<uint4*>(cacheRecord<kGroups / 2>(a, n.side, slot[i], n.head, n.group / 2)) = make_uint4(codes.x, codes.y, hx, hy);
        }
        if (n.group == 0) *cacheScale(a, n.side, slot[i], n.head) = powerOfTwo(e);
      }
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
  // e4m3 reads its row twice, the second time from L1: held in registers it
  // would leave room for few warps.
  unsigned char* dst = cacheRecord<kE4m3 ? kGroups / 2 : kGroups>(a, side, slot, head, 0);
  const int dst_step = a.page_rows * 16;
  int e = 0;
  bool finite = true;
  if constexpr (kE4m3) {
    float m = 0.0f;
#pragma unroll 8
    for (int g = 0; g < kGroups; ++g) m = fmaxf(m, groupMax<T>(*reinterpret_cast<const uint4*>(src + g * step)));
    finite = m <= FLT_MAX;
    if (!finite) {
      m = 0.0f;
      for (int g = 0; g < kGroups; ++g) m = fmaxf(m, groupFiniteMax<T>(*reinterpret_cast<const uint4*>(src + g * step)));
    }
    e = scaleExponent(m);
    *cacheScale(a, side, slot, head) = powerOfTwo(e);
  }
#pragma unroll 1
  for (int g0 = 0; g0 < kGroups; g0 += 4) {
    uint4 raw[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) raw[g] = *reinterpret_cast<const uint4*>(src + (g0 + g) * step);
    if constexpr (!kE4m3) {
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(dst + (g0 + g) * dst_step) = raw[g];
    } else {
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        const uint2 lo = quantise8<T>(raw[g], powerOfTwo(-e), finite), hi = quantise8<T>(raw[g + 1], powerOfTwo(-e), finite);
        *reinterpret_cast<uint4*>(dst + (g0 + g) / 2 * dst_step) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  }
}

template <typename T>
__device__ __noinline__ void dequantiseAny(uint4 codes, float scale, uint4* out) {
  uint4 o[2];
  dequantise16<T>(codes, scale, o);
  out[0] = o[0];
  out[1] = o[1];
}

// 16 codes as two groups of T.
template <typename T>
__device__ __forceinline__ void dequantise(const uint4& codes, float scale, uint4 (&out)[2]) {
  if (scale >= FastScale<T>::low && scale <= FastScale<T>::high && !hasNan(codes)) {
    const FastScale<T> fast(scale);
    const uint2 x = fast(codes.x), y = fast(codes.y), z = fast(codes.z), w = fast(codes.w);
    out[0] = make_uint4(x.x, x.y, y.x, y.y);
    out[1] = make_uint4(z.x, z.y, w.x, w.y);
  } else {
    dequantiseAny<T>(codes, scale, out);
  }
}

// kPlanes lanes per (row, keys or values, head), one cache record each.
template <typename T, int kPlanes, bool kE4m3>
__global__ void __launch_bounds__(kThreads) readRowsKernel(const Args a) {
  tc::pdlTrigger();
  tc::pdlWait();
  constexpr int kUnroll = kReadRows<kE4m3>;
  const Lane n = laneOf<kPlanes, kUnroll>(a);
  const uint64_t policy = passingPolicy();
  int slot[kUnroll];
  uint4 raw[kUnroll];
  float scale[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int row = n.row + i * n.step;
    slot[i] = n.active && row < a.rows ? slotOf(a, row) : -1;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (slot[i] >= 0) {
      raw[i] = *reinterpret_cast<const uint4*>(cacheRecord<kPlanes>(a, n.side, slot[i], n.head, n.group));
      if constexpr (kE4m3) scale[i] = *cacheScale(a, n.side, slot[i], n.head);
    }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (slot[i] < 0) continue;
    const int row = n.row + i * n.step;
    if constexpr (!kE4m3) {
      storePassing(record(a.dense[n.side], n.head, row, n.group), raw[i], policy);
    } else {
      uint4 out[2];
      dequantise<T>(raw[i], scale[i], out);
      storePassing(record(a.dense[n.side], n.head, row, 2 * n.group), out[0], policy);
      storePassing(record(a.dense[n.side], n.head, row, 2 * n.group + 1), out[1], policy);
    }
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
  const unsigned char* src = cacheRecord<kPlanes>(a, side, slot, head, 0);
  const int src_step = a.page_rows * 16;
  float scale = 0.0f;
  if constexpr (kE4m3) scale = *cacheScale(a, side, slot, head);
#pragma unroll 1
  for (int p0 = 0; p0 < kPlanes; p0 += 4) {
    uint4 raw[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) raw[p] = *reinterpret_cast<const uint4*>(src + (p0 + p) * src_step);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if constexpr (!kE4m3) {
        *reinterpret_cast<uint4*>(dst + (p0 + p) * step) = raw[p];
      } else {
        uint4 out[2];
        dequantise<T>(raw[p], scale, out);
        *reinterpret_cast<uint4*>(dst + 2 * (p0 + p) * step) = out[0];
        *reinterpret_cast<uint4*>(dst + (2 * (p0 + p) + 1) * step) = out[1];
      }
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
  return write ? launchPdl(writeRowsKernel<T, kGroups, kE4m3>, laneGrid(a, kGroups, kWriteRows), dim3(kThreads), 0, s, a)
               : launchPdl(readRowsKernel<T, kPlanes, kE4m3>, laneGrid(a, kPlanes, kReadRows<kE4m3>), dim3(kThreads), 0, s, a);
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
  if (d->rows < 0 || d->cache.kv_heads > 4096) return fail(std::string(name) + ": bad sizes");
  if (d->rows > kMost) return fail(std::string(name) + ": rows must be at most 2^31 - 1024");
  if (d->rows == 0) return 0;
  for (const fpk_heads_t* v : {&d->k, &d->v}) {
    if (const char* q = headsProblem(*v)) return fail(std::string(name) + ": " + q);
  }
  if (d->slots == nullptr) return fail(std::string(name) + ": slots are required");
  if (!aligned4(d->slots) || !aligned4(d->error_flag)) return fail(std::string(name) + ": slots and error_flag must be 4-byte aligned");
  const bool e4m3 = d->cache.dtype == FPK_DTYPE_E4M3;
  const std::string where = deviceProblem({d->cache.k, d->cache.v, d->k.data, d->v.data, d->slots, d->error_flag,
                                           e4m3 ? d->cache.k_scale : nullptr, e4m3 ? d->cache.v_scale : nullptr});
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
