// RMS norm of query and key heads and rotary positions in one pass
// (fpk_qk_norm_rotary, include/fpk.h).
//
//   r = rsqrt(mean(x^2) + eps),  x' = x r w,  (a, b) -> (a c - b s, b c + a s)
//   c, s = rotary_scale * cos, sin(position * inv_freq[i])
//
// Every element is read once and written once (4 bytes for some ten
// operations), so the pass is bound by memory. Two mappings of lanes, by the
// layout, because a warp must touch whole 128-byte lines:
//   rows    16-byte groups of a head lie side by side (row-major): lanes take
//           two groups each, a warp takes one token and walks its heads with
//           the token's angles in registers; the norm is a sum over the head's
//           lanes.
//   planar  rows of a group lie side by side (row_stride 16): lanes take 32
//           rows, a thread owns its row's whole head and reads it twice (the
//           second time from L1) instead of holding it; the angles of the 32
//           rows are a table in shared memory that the block's heads share.
// Measured: 16,384 tokens of 40 heads of 128, bf16, normalised, rows: 63 us = 5.3
// TB/s, 81 % of the copy rate (sharing the angles between a warp's heads changes
// nothing: it waits for memory); 5,003 rows of 8 heads, planar, 9.1 us (its 157 CTAs
// form the angles before the first load, and a thread has four loads in flight).
#include <cmath>
#include <cstdint>
#include <string>

#include "fp_heads.cuh"
#include "fp_launch.hpp"
#include "fp_profile.hpp"
#include "fp_tc.cuh"

namespace fpb {
namespace rotary {

using namespace heads;

struct Args {
  fpk_heads_t q, k, q_out, k_out;
  int rows, q_heads, kv_heads, groups, rotary_dim, interleaved;
  const float* q_weight;
  const float* k_weight;
  float eps, inv_dim;
  const int32_t* positions;
  const float* inv_freq;
  float scale;
};

// cos and sin of position * inv_freq. The product and its reduction to one turn
// are in double (fp32 would lose the angle itself: at position 10^6 its last
// bit is 0.06 rad); the remainder, at most half a turn, keeps fp32 accuracy.
__device__ __forceinline__ float2 turn(int position, float inv_freq, float scale) {
  const double t = static_cast<double>(position) * static_cast<double>(inv_freq) * 0.15915494309189533577;
  const float f = static_cast<float>(t - rint(t));
  float s, c;
  sincospif(2.0f * f, &s, &c);
  return make_float2(c * scale, s * scale);
}

constexpr int kRowsWarps = 4;
// Heads in flight per lane group: 16,384 tokens of 40 heads take 63 us with 2, 68
// with 4 (fewer warps fit), 66 with 2 that are loaded ahead of the angles.
constexpr int kBatch = 2;

// A lane holds two groups of a head: the two that a pair of channels lies in
// (half layout), so that nothing is exchanged, or two neighbours.
template <typename T>
__global__ void __launch_bounds__(kRowsWarps * 32) rotaryRowsKernel(const Args a, int lanes) {
  tc::pdlTrigger();
  tc::pdlWait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int slots = 32 / lanes;  // heads that a warp holds side by side
  const int slot = lane / lanes;
  const int k = lane - slot * lanes;  // pair of groups
  const int half_groups = a.rotary_dim >> 4;  // groups of half the rotated part
  const bool rotated = k < half_groups;
  const bool halves = !a.interleaved && rotated;
  const int ga = halves ? k : 2 * k;
  const int gb = halves ? k + half_groups : 2 * k + 1;
  const bool has_a = ga < a.groups, has_b = gb < a.groups;

  // cos and sin of channel i of the pair's groups (half layout: the same in
  // both), or of the four pairs of each.
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (rotated) {
    const int position = a.positions[row];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 cs = turn(position, a.inv_freq[k * 8 + i], a.scale);
      c[i] = cs.x;
      s[i] = cs.y;
    }
  }

  for (int part = 0; part < 2; ++part) {
    const fpk_heads_t& in = part == 0 ? a.q : a.k;
    const fpk_heads_t& out = part == 0 ? a.q_out : a.k_out;
    const int n_heads = part == 0 ? a.q_heads : a.kv_heads;
    const float* weight = part == 0 ? a.q_weight : a.k_weight;
    const bool norm = weight != nullptr;
    float wa[8], wb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa[i] = norm && has_a && n_heads > 0 ? weight[ga * 8 + i] : 1.0f;
      wb[i] = norm && has_b && n_heads > 0 ? weight[gb * 8 + i] : 1.0f;
    }
    const int stride = gridDim.y * slots;
    // Uniform trip count: every lane takes part in the shuffles.
    for (int h0 = blockIdx.y * slots; h0 < n_heads; h0 += stride * kBatch) {
      uint4 raw[kBatch][2];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + b * stride + slot;
        raw[b][0] = raw[b][1] = make_uint4(0, 0, 0, 0);
        if (has_a && h < n_heads) raw[b][0] = *reinterpret_cast<const uint4*>(record(in, h, row, ga));
        if (has_b && h < n_heads) raw[b][1] = *reinterpret_cast<const uint4*>(record(in, h, row, gb));
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (h0 + b * stride >= n_heads) break;  // warp-uniform
        const int h = h0 + b * stride + slot;
        float x[8], y[8];
        unpack8<T>(raw[b][0], x);
        unpack8<T>(raw[b][1], y);
        float r = 1.0f;
        if (norm) {
          float sum = 0.0f, more = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum = fmaf(x[i], x[i], sum);
            more = fmaf(y[i], y[i], more);
          }
          sum += more;
          for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
        }
        if (!rotated) {  // its own branch: an infinity must not meet 0 sin
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= wa[i] * r;
            y[i] *= wb[i] * r;
          }
        } else if (halves) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float u = x[i] * wa[i], v = y[i] * wb[i];
            x[i] = (u * c[i] - v * s[i]) * r;
            y[i] = (v * c[i] + u * s[i]) * r;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float u = x[2 * i] * wa[2 * i], v = x[2 * i + 1] * wa[2 * i + 1];
            x[2 * i] = (u * c[i] - v * s[i]) * r;
            x[2 * i + 1] = (v * c[i] + u * s[i]) * r;
            const float p = y[2 * i] * wb[2 * i], q = y[2 * i + 1] * wb[2 * i + 1];
            y[2 * i] = (p * c[4 + i] - q * s[4 + i]) * r;
            y[2 * i + 1] = (q * c[4 + i] + p * s[4 + i]) * r;
          }
        }
        if (has_a && h < n_heads) *reinterpret_cast<uint4*>(record(out, h, row, ga)) = pack8<T>(x);
        if (has_b && h < n_heads) *reinterpret_cast<uint4*>(record(out, h, row, gb)) = pack8<T>(y);
      }
    }
  }
}

constexpr int kPlanarWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kPlanarWarps * 32) rotaryPlanarKernel(const Args a) {
  extern __shared__ float2 table[];  // [rotary_dim / 2][32 rows]
  tc::pdlTrigger();
  tc::pdlWait();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const bool valid = row < a.rows;
  const int half = a.rotary_dim >> 1;
  if (half > 0) {
    const int position = valid ? a.positions[row] : 0;
    for (int i = warp; i < half; i += kPlanarWarps) table[i * 32 + lane] = turn(position, a.inv_freq[i], a.scale);
  }
  __syncthreads();
  if (!valid) return;

  const int n_heads = a.q_heads + a.kv_heads;
  for (int n = blockIdx.y * kPlanarWarps + warp; n < n_heads; n += gridDim.y * kPlanarWarps) {
    const bool is_q = n < a.q_heads;
    const fpk_heads_t& in = is_q ? a.q : a.k;
    const fpk_heads_t& out = is_q ? a.q_out : a.k_out;
    const float* weight = is_q ? a.q_weight : a.k_weight;
    const int h = is_q ? n : n - a.q_heads;
    const unsigned char* src = record(in, h, row, 0);
    unsigned char* dst = record(out, h, row, 0);
    float r = 1.0f;
    if (weight != nullptr) {
      float sum = 0.0f;
#pragma unroll 8
      for (int g = 0; g < a.groups; ++g) {
        float x[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(src + g * in.plane_stride), x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
      }
      r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
    }
    auto load = [&](int g, float (&x)[8]) {
      unpack8<T>(*reinterpret_cast<const uint4*>(src + g * in.plane_stride), x);
      if (weight != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * weight[g * 8 + i];
      }
    };
    auto store = [&](int g, const float (&y)[8]) { *reinterpret_cast<uint4*>(dst + g * out.plane_stride) = pack8<T>(y); };
    const int rotated_groups = a.rotary_dim >> 3;
    if (a.interleaved) {
#pragma unroll 4
      for (int g = 0; g < rotated_groups; ++g) {
        float x[8];
        load(g, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 cs = table[(g * 4 + i) * 32 + lane];
          const float u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = u * cs.x - v * cs.y;
          x[2 * i + 1] = v * cs.x + u * cs.y;
        }
        store(g, x);
      }
    } else {
      const int hg = rotated_groups >> 1;
#pragma unroll 2
      for (int g = 0; g < hg; ++g) {
        float x[8], y[8];
        load(g, x);
        load(g + hg, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 cs = table[(g * 8 + i) * 32 + lane];
          const float u = x[i], v = y[i];
          x[i] = u * cs.x - v * cs.y;
          y[i] = v * cs.x + u * cs.y;
        }
        store(g, x);
        store(g + hg, y);
      }
    }
    if (weight != nullptr || src != dst) {
#pragma unroll 4
      for (int g = rotated_groups; g < a.groups; ++g) {
        float x[8];
        load(g, x);
        store(g, x);
      }
    }
  }
}

template <typename T>
cudaError_t launch(const Args& a, cudaStream_t s) {
  const int n_heads = a.q_heads + a.kv_heads;
  auto planar = [](const fpk_heads_t& v) { return v.row_stride == 16; };
  const bool q_planar = a.q_heads == 0 || (planar(a.q) && planar(a.q_out));
  const bool k_planar = a.kv_heads == 0 || (planar(a.k) && planar(a.k_out));
  prof::countLaunch(prof::kOther);
  if (q_planar && k_planar) {
    const int blocks = (a.rows + 31) / 32;
    const int most = (n_heads + kPlanarWarps - 1) / kPlanarWarps;
    return launchPdl(rotaryPlanarKernel<T>, dim3(blocks, most), dim3(kPlanarWarps * 32), static_cast<size_t>(a.rotary_dim) * 128, s, a);
  }
  int lanes = 1;
  while (2 * lanes < a.groups) lanes *= 2;
  const int blocks = (a.rows + kRowsWarps - 1) / kRowsWarps;
  // Few rows: the heads are split over blocks too, so that the GPU fills.
  const int per_warp = (32 / lanes) * kBatch;
  const int most = (n_heads + per_warp - 1) / per_warp;
  int split = 1;
  while (split < most && blocks * split < 592) ++split;
  return launchPdl(rotaryRowsKernel<T>, dim3(blocks, split), dim3(kRowsWarps * 32), 0, s, a, lanes);
}

}  // namespace rotary
}  // namespace fpb

extern "C" int fpk_qk_norm_rotary(const fpk_qk_rotary_desc_t* d, void* stream) {
  using namespace fpb;
  if (d == nullptr) return fail("fpk_qk_norm_rotary: null descriptor");
  if (!heads::is16Bit(d->dtype)) return fail("fpk_qk_norm_rotary: dtype must be f16 or bf16");
  if (d->rows < 0 || d->q_heads < 0 || d->kv_heads < 0 || d->head_dim <= 0 || d->head_dim > 256 || d->head_dim % 8) {
    return fail("fpk_qk_norm_rotary: bad sizes (head_dim is a multiple of 8 up to 256)");
  }
  if (static_cast<long long>(d->q_heads) + d->kv_heads > 65535) return fail("fpk_qk_norm_rotary: bad sizes (at most 65535 heads)");
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 16) {
    return fail("fpk_qk_norm_rotary: rotary_dim must be a multiple of 16 up to head_dim");
  }
  if (d->rows > heads::kMost) return fail("fpk_qk_norm_rotary: rows must be at most 2^31 - 1024");
  if (d->rows == 0 || d->q_heads + d->kv_heads == 0) return 0;
  for (int i = 0; i < 4; ++i) {
    const bool is_q = i % 2 == 0;
    if ((is_q ? d->q_heads : d->kv_heads) == 0) continue;
    const fpk_heads_t& v = i == 0 ? d->q : i == 1 ? d->k : i == 2 ? d->q_out : d->k_out;
    if (const char* p = heads::headsProblem(v)) return fail(std::string("fpk_qk_norm_rotary: ") + p);
  }
  if (d->rotary_dim > 0 && (d->positions == nullptr || d->inv_freq == nullptr)) {
    return fail("fpk_qk_norm_rotary: positions and inv_freq are required");
  }
  if (!heads::aligned4(d->positions) || !heads::aligned4(d->inv_freq) || !heads::aligned4(d->q_weight) || !heads::aligned4(d->k_weight)) {
    return fail("fpk_qk_norm_rotary: positions, inv_freq and weights must be 4-byte aligned");
  }
  if ((d->q_weight != nullptr || d->k_weight != nullptr) && !(d->eps >= 0.0f)) return fail("fpk_qk_norm_rotary: eps must not be negative");
  const bool q = d->q_heads > 0, k = d->kv_heads > 0, turn = d->rotary_dim > 0;
  const std::string where = heads::deviceProblem({q ? d->q.data : d->k.data, q ? d->q_out.data : nullptr, k ? d->k.data : nullptr,
                                                  k ? d->k_out.data : nullptr, q ? d->q_weight : nullptr, k ? d->k_weight : nullptr,
                                                  turn ? d->positions : nullptr, turn ? d->inv_freq : nullptr});
  if (!where.empty()) return fail("fpk_qk_norm_rotary: " + where);
  rotary::Args a{};
  a.q = d->q;
  a.k = d->k;
  a.q_out = d->q_out;
  a.k_out = d->k_out;
  a.rows = d->rows;
  a.q_heads = d->q_heads;
  a.kv_heads = d->kv_heads;
  a.groups = d->head_dim / 8;
  a.rotary_dim = d->rotary_dim;
  a.interleaved = d->interleaved != 0;
  a.q_weight = d->q_weight;
  a.k_weight = d->k_weight;
  a.eps = d->eps;
  a.inv_dim = 1.0f / static_cast<float>(d->head_dim);
  a.positions = d->positions;
  a.inv_freq = d->inv_freq;
  a.scale = d->rotary_scale;
  const cudaError_t e = d->dtype == FPK_DTYPE_BF16 ? rotary::launch<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream))
                                                   : rotary::launch<__half>(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(std::string("fpk_qk_norm_rotary: ") + cudaGetErrorString(e));
  return 0;
}
