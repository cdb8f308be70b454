// Attention of few query rows over many keys (decoding): fpk_attention_paged
// and fpk_attention_packed where a sequence has at most 16 query rows (tokens x
// query heads to a key head), or there is little work in all.
//
// Bound by the keys' and values' bytes, each read once from HBM, so everything
// serves the stream of loads:
// * Each warp streams steps of 16 keys through its own ring in shared memory
//   (cp.async; no barrier between warps), deep enough that some 100 KB an SM are
//   under way. From there 16-byte records become matrix fragments (mma m16n8k16)
//   as they are, keys and values always the operand of 16 rows, so that 8 query
//   rows fill a product: S^T = K Q^T with 16 keys, O^T = V^T P^T with 16 channels.
//   A contraction does not care for the order of its index: scores contract the 8
//   channels of a record in two products, and score row g of 8-key block j stands
//   for key 8j + 4(g%2) + g/2, so that, once P is transposed (movmatrix), a
//   thread's probabilities belong to keys t, 4+t, 8+t, 12+t (t = lane%4) and its
//   four value records, one of each key and of plane lane/4, need only a byte
//   permute to become fragments. The planes of a step are padded so that both
//   readings are free of bank conflicts.
// * e4m3 records become fp16 (exact) in registers. The key's scale multiplies
//   its scores; the value's scale v joins the exponent: P' = 2^(s + log2 v - m),
//   O = sum P' code, l = sum P'/v, so P' is at most 2^15 whatever the scales are.
//   A product with V keeps P' to 2^-25, so a key counts against the largest weight
//   times value, not the largest weight. A row of zeros would set m by a scale
//   that stands for nothing, and the others' P' would fall out of fp16: it counts
//   as 2^-48 there, and its weight in l alone. Queries become fp16 with a power of
//   two taken out of each row, exact down to 2^-14 of its maximum.
// * Softmax in one pass, statistics and sums in fp32. A row's reference m moves
//   only when a score exceeds it by 2^15, a warp vote, so most steps need no
//   shuffle.
// * The key axis is split evenly: all (sequence, row tile, key head) units of 64
//   keys form one line that the CTAs share out, each finding its part from the
//   lengths on the device. A tile that crosses CTAs leaves fp32 partials that a
//   second launch joins in order (deterministic, no atomics).
// * Under a causal mask 0 * v of a key that a row does not see is NaN where v is an
//   infinity or NaN. A tile with NaN in its output and with such keys is done again,
//   token by token.
// * Short sequences instead take a cluster of CTAs for each tile, which share its
//   keys out evenly and join over distributed shared memory: no second launch.
//
// Measured (32 query heads over 8 key heads of 128, bf16): one token of each of 8
// sequences of 8,000 to 131,072 keys 154 us over e4m3 (941 MB, 6.1 TB/s, 93 % of
// the copy rate; 169 under the power cap) and 280 us over 16 bits (1.82 GB, the
// copy rate); of each of 4 sequences of 40 to 1,000 keys 8.8 us, launch and latency.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "fp_attention_seq.cuh"
#include "fp_launch.hpp"
#include "fp_profile.hpp"
#include "fp_tc.cuh"

namespace fpb {
namespace seqattn {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnitKeys = 64;     // one unit of the split: 16 keys of each warp
// Shares of 128 keys or more. One token over 6,000 keys: 16.9 us with 64, 14.4
// with 128, 15.0 with 256, 17.2 with 512.
constexpr int kMinUnits = 2;
// A row's reference lies 2^7 below the maximum it was set by and stays until a
// score is 2^15 above it: probabilities up to 2^15 use fp16's range on both sides
// of 1, so that weights down to 2^-32 of the largest reach a product (2^-25 with
// the maximum itself as the reference).
constexpr float kHeadLog2 = 7.0f;
constexpr float kGrowLog2 = 15.0f;
// e4m3: a row of zeros moves the reference only when its score is this far above.
constexpr float kZerosLog2 = 48.0f;
constexpr int kClusterKeys = 512;  // a cluster's most keys to a CTA

// A pass over a tile: its rows lo .. hi - 1 (all, or those of one token, see `nan`).
struct Pass {
  int again;  // first row of the pass in a tile that is done again, else -1
  int lo, hi;
  int hides;  // a row of the pass does not see some keys of it
  int nan;    // and the output holds NaN
};

// The tile that a CTA's range begins inside, for the joining launch.
struct Split {
  long long first_unit, last_unit;  // of the tile; first_unit < 0: nothing to join here
  int seq, tile, head, rows;        // rows: valid query rows of the tile
};

constexpr size_t partialFloats(int d) { return static_cast<size_t>(kStreamRows) * d + 2 * kStreamRows; }

// Quotient of non-negative numbers. Those past 32 bits are rare, and their
// division is long: it stays out of the code that every launch fetches.
__device__ __noinline__ long long divideLong(long long x, long long y) { return x / y; }
__device__ __forceinline__ long long divide(long long x, long long y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return divideLong(x, y);
}

// The first `rest` CTAs take size + 1 units, the others size.
struct Share {
  long long size, rest;
};

__device__ __forceinline__ long long shareBegin(const Share& s, long long c) { return c * s.size + min(c, s.rest); }
__device__ __forceinline__ long long shareOwner(const Share& s, long long u) {
  const long long large = s.rest * (s.size + 1);
  return u < large ? divide(u, s.size + 1) : s.rest + divide(u - large, s.size);
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void copyAsync16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copyAsync4(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 loadShared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 loadShared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ float loadShared4(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// An 8 x 8 matrix of 16-bit elements, two of row lane/4 to a lane, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// From another CTA of the cluster.
__device__ __forceinline__ float4 loadCluster16(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ float loadCluster4(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// The four e4m3 codes of a word as two fp16 pairs.
__device__ __forceinline__ uint2 halves(uint32_t four) {
  uint2 r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(r.x), "=r"(r.y) : "r"(four));
  return r;
}

// A row's output. One that saw no key gets zeros, whatever the values held that
// its tile's other rows saw.
__device__ __forceinline__ float normalised(float o, float l) { return l == 0.0f ? 0.0f : o * (1.0f / l); }

// Shapes of one 16-key step in a warp's ring.
template <int D, bool kE4m3>
struct Step {
  static constexpr int kPlanes = kE4m3 ? D / 16 : D / 8;
  static constexpr int kKRecords = kPlanes / 4;               // K records of a thread per 8 keys
  static constexpr int kVCh = kE4m3 && D == 128 ? 16 : 8;     // channels of a thread's V record
  static constexpr int kVRecords = D / (8 * kVCh);            // V records of a thread per key
  static constexpr int kKPlane = 16 * 16 + 16, kVPlane = 16 * 16 + 64;
  static constexpr int kV = kPlanes * kKPlane;                // byte of V
  static constexpr int kScales = kV + kPlanes * kVPlane;      // byte of the scales, keys' then values'
  static constexpr int kBytes = kScales + (kE4m3 ? 128 : 0);
  // Three CTAs to an SM share its 227 KB.
  static constexpr int kDepth = 75776 / (kWarps * kBytes) < 5 ? 75776 / (kWarps * kBytes) : 5;
  static constexpr int kRing = kWarps * kDepth * kBytes;
  static_assert(kDepth >= 2 && kRing >= (kWarps * kStreamRows * (D + 4) + kStreamRows * D) * 4, "the outputs' exchange lies over the ring");
};

}  // namespace

template <typename T, int D, KvKind kKind, int R, bool kCluster>
__global__ void __launch_bounds__(kThreads, 3) attentionStreamKernel(const Args a, int cluster) {
  constexpr bool kE4m3 = kKind == kPagedE4m3;
  constexpr int kCols = R / 8;  // blocks of 8 query rows
  using S = Step<D, kE4m3>;
  using M = std::conditional_t<kE4m3, __half, T>;  // type of the products
  // On a line of shared memory: 96 bytes past one, one token over 8 x 131,072 e4m3
  // keys takes 169 us, on one 154.
  extern __shared__ __align__(128) unsigned char ring_raw[];
  auto o_s = reinterpret_cast<float(*)[kStreamRows][D + 4]>(ring_raw);  // [kWarps], once the ring is empty
  __shared__ float ml_s[kWarps][2][kStreamRows];
  __shared__ long long scan_s[kWarps + 1];
  __shared__ long long found_s[2];
  __shared__ int owner_s;                     // clusters: the sequence, the last that has this tile
  __shared__ float joined_s[2][kStreamRows];  // clusters: this CTA's m and l
  __shared__ Pass pass_s;

  tc::pdlTrigger();
  tc::pdlWait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  if (tid == 0) pass_s.again = -1;

  Split* splits = reinterpret_cast<Split*>(a.workspace);
  float* partials = reinterpret_cast<float*>(a.workspace + sizeof(Split) * kStreamCtas);
  Split* split = splits + blockIdx.x;
  Share share{};
  long long begin = 0, end = 1, seq_first = 0, seq_units = 1;
  int seq = 0, rank = 0, cluster_tile = 0, cluster_head = 0;
  Sequence q{};
  // ---- this CTA's part of the line ----
  auto unitsOf = [&](int s, Sequence* out) -> long long {
    const Sequence q = sequence<kKind>(a, s);
    if (out != nullptr) *out = q;
    const long long tiles = (q.nq * a.group + R - 1) / R;
    return tiles * a.kv_heads * max((q.nk + kUnitKeys - 1) / kUnitKeys, 1);  // no keys: still zeros to write
  };
  if constexpr (kCluster) {
    // Tiles of sequence s have the numbers q0 * group / R + s + 0, 1, ...: apart
    // from those of the next, whatever the lengths are. Starts that overlap (an
    // error) give all CTAs of a cluster the same one: the last.
    rank = static_cast<int>(tc::clusterCtaRank());
    const int x = static_cast<int>(blockIdx.x) / cluster;
    const int number = x / a.kv_heads;
    cluster_head = x - number * a.kv_heads;
    if (tid == 0) owner_s = -1;
    __syncthreads();
    if (tid < a.n_seq) {  // at most kThreads sequences: clusterOf()
      const Sequence c = sequence<kKind>(a, tid);
      const int tile = number - c.q0 * a.group / R - tid;
      if (tile >= 0 && tile < (c.nq * a.group + R - 1) / R) atomicMax(&owner_s, tid);
    }
    __syncthreads();
    if (owner_s < 0) return;  // a number without a tile: the whole cluster leaves
    seq = owner_s;
    q = sequence<kKind>(a, seq);
    cluster_tile = number - q.q0 * a.group / R - seq;
  } else {
    // Units of kThreads sequences and their sums up to each thread's.
    long long mine = 0, at = 0, total = 0;
    auto scan = [&](int s0) -> long long {
      mine = s0 + tid < a.n_seq ? unitsOf(s0 + tid, nullptr) : 0;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      __syncthreads();
      if (lane == 31) scan_s[warp] = upto;
      __syncthreads();
      long long all = 0;
      at = upto - mine;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += scan_s[w];
        all += scan_s[w];
      }
      return all;
    };
    for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) total += scan(s0);
    const long long ctas = min(static_cast<long long>(gridDim.x), (total + kMinUnits - 1) / kMinUnits);
    if (static_cast<long long>(blockIdx.x) >= ctas) {
      if (tid == 0) split->first_unit = -1;
      return;
    }
    share.size = divide(total, ctas);
    share.rest = total - share.size * ctas;
    begin = shareBegin(share, blockIdx.x);
    end = shareBegin(share, blockIdx.x + 1LL);
    // The sequence that holds unit `begin`.
    long long before = 0;
    for (int s0 = 0; s0 < a.n_seq && before <= begin; s0 += kThreads) {
      const long long all = a.n_seq > kThreads ? scan(s0) : total;  // one pass: still at hand
      if (begin >= before + at && begin < before + at + mine) {
        found_s[0] = s0 + tid;
        found_s[1] = before + at;
      }
      before += all;
    }
    __syncthreads();
    seq = static_cast<int>(found_s[0]);
    seq_first = found_s[1];
    seq_units = unitsOf(seq, &q);
  }

  const int q_heads_per = a.group;
  bool first_piece = true;
  for (long long u = begin; u < end;) {
    int blocks, tile, head, b0, b1;
    long long tile_first = 0;
    if constexpr (kCluster) {
      blocks = max((q.nk + kUnitKeys - 1) / kUnitKeys, 1);
      tile = cluster_tile;
      head = cluster_head;
      b0 = blocks * rank / cluster;
      b1 = blocks * (rank + 1) / cluster;
    } else {
      while (u >= seq_first + seq_units) {  // the next sequence with rows
        seq_first += seq_units;
        seq_units = unitsOf(++seq, &q);
      }
      blocks = max((q.nk + kUnitKeys - 1) / kUnitKeys, 1);
      const long long tile_head = divide(u - seq_first, blocks);
      tile = static_cast<int>(divide(tile_head, a.kv_heads));
      head = static_cast<int>(tile_head - static_cast<long long>(tile) * a.kv_heads);
      tile_first = seq_first + tile_head * blocks;
      b0 = static_cast<int>(u - tile_first);
      b1 = static_cast<int>(min(static_cast<long long>(blocks), end - tile_first));
    }
    const int rows = min(R, q.nq * a.group - tile * R);
    // Rows of this pass: the tile's, or those of a token.
    const int lo = max(pass_s.again, 0);
    const int hi = pass_s.again < 0 ? rows : min(rows, ((tile * R + lo) / q_heads_per + 1) * q_heads_per - tile * R);

    // This thread's score columns are rows 8 n + 2t and 8 n + 2t + 1 of the tile.
    int vis[kCols][2];
    int min_vis = q.nk;
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = 8 * n + 2 * t + i;  // tile * R + rr is below 2^31: checked by the host
        vis[n][i] = rr >= lo && rr < hi ? visible(a, q, (tile * R + rr) / q_heads_per) : q.nk;
        min_vis = min(min_vis, vis[n][i]);
      }
    }
    const int last_vis = visible(a, q, (tile * R + hi - 1) / q_heads_per);
    min_vis = min(min_vis, __shfl_xor_sync(0xffffffffu, min_vis, 1));
    min_vis = min(min_vis, __shfl_xor_sync(0xffffffffu, min_vis, 2));
    if (tid == 0) {
      pass_s.lo = lo;
      pass_s.hi = hi;
      pass_s.hides = min_vis < last_vis;
      pass_s.nan = 0;
    }

    // Steps of 16 keys, one warp after the other, up to the last visible key.
    const int step_end = min(b1 * (kUnitKeys / 16), (last_vis + 15) >> 4);
    const int step_first = b0 * (kUnitKeys / 16) + warp;
    const uint32_t ring = tc::smemU32(ring_raw) + warp * S::kDepth * S::kBytes;
    // This lane copies row lane%16 of planes lane/16, 2 + lane/16, ...
    const int copy_row = lane & 15, copy_plane = lane >> 4;
    const int row_key = 4 * (g & 1) + (g >> 1);
    uint32_t bad_steps = 0;  // by ring place: the step's page does not exist
    int page_next = 0;
    auto pageAt = [&](int step) -> int {
      if constexpr (kKind == kPacked16) return 0;
      return step < step_end ? pageOf(a, seq, step * 16) : 0;
    };
    auto copyStep = [&](int step, int place) {
      if (step < step_end) {
        const int key0 = step * 16;
        bool in = key0 + copy_row < last_vis;
        const uint32_t to = ring + place * S::kBytes;
        long long row = 0, page_at = 0;
        if constexpr (kKind == kPacked16) {
          row = static_cast<long long>(q.k0) + key0 + copy_row;
        } else {
          int page = page_next;
          page_next = pageAt(step + kWarps);
          bad_steps &= ~(1u << place);
          if (page < 0) {
            reportIndex(a.error_flag, FPK_ERROR_PAGE);
            bad_steps |= 1u << place;
            page = 0;
            in = false;
          }
          row = (key0 + copy_row) & ((1 << a.page_shift) - 1);
          page_at = page * a.page_stride;
          if constexpr (kE4m3) {
            const float* scale = (copy_plane == 0 ? a.k_scale : a.v_scale) + (((static_cast<long long>(page) * a.kv_heads + head) << a.page_shift) + row);
            copyAsync4(to + S::kScales + lane * 4, scale, in);
          }
        }
        if (!in) row = 0, page_at = 0;  // an address that exists; nothing is read
        if constexpr (kKind == kPacked16) {
          if (!in) row = q.k0;
        }
        const unsigned char* ks = record(a.k, head, row, copy_plane) + page_at;
        const unsigned char* vs = record(a.v, head, row, copy_plane) + page_at;
        const uint32_t kd = to + copy_plane * S::kKPlane + copy_row * 16, vd = to + S::kV + copy_plane * S::kVPlane + copy_row * 16;
#pragma unroll
        for (int p = 0; p < S::kPlanes / 2; ++p) {
          copyAsync16(kd + p * 2 * S::kKPlane, ks, in);
          copyAsync16(vd + p * 2 * S::kVPlane, vs, in);
          ks += 2 * a.k.plane_stride;
          vs += 2 * a.v.plane_stride;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    page_next = pageAt(step_first);
#pragma unroll
    for (int i = 0; i < S::kDepth - 1; ++i) copyStep(step_first + i * kWarps, i);
    // Query fragments: of row g of each block the channels that this thread's K records hold.
    uint32_t qf[kCols][D / 16][2];
    float row_scale[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int r = tile * R + 8 * c + g;
      const int token = r / q_heads_per;
      const unsigned char* qp = 8 * c + g < rows ? record(a.q, head * q_heads_per + r - token * q_heads_per, q.q0 + token, 0) : nullptr;
      uint4 raw[D / 32];
#pragma unroll
      for (int n = 0; n < D / 32; ++n) {
        const int plane = kE4m3 ? 2 * (4 * (n / 2) + t) + n % 2 : 4 * n + t;
        raw[n] = qp != nullptr ? *reinterpret_cast<const uint4*>(qp + plane * a.q.plane_stride) : make_uint4(0, 0, 0, 0);
      }
      if constexpr (kE4m3) {
        float m = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
          float x[8];
          unpack8<T>(raw[n], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // 2^(exponent of m), kept where its inverse is a normal number.
        const int e = min(max((__float_as_int(m) >> 23) & 0xff, 1), 253) - 127;
        const float mine = m > 0.0f ? __int_as_float((e + 127) << 23) : 1.0f;
        const float inv = m > 0.0f ? __int_as_float((127 - e) << 23) : 1.0f;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
          float x[8];
          unpack8<T>(raw[n], x);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= inv;
          raw[n] = pack8<__half>(x);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) row_scale[c][i] = __shfl_sync(0xffffffffu, mine, (2 * t + i) * 4) * a.scale_log2;
      }
#pragma unroll
      for (int n = 0; n < D / 32; ++n) {
        qf[c][2 * n][0] = raw[n].x, qf[c][2 * n][1] = raw[n].y;
        qf[c][2 * n + 1][0] = raw[n].z, qf[c][2 * n + 1][1] = raw[n].w;
      }
    }

    float o[kCols][S::kVRecords][S::kVCh / 2][4];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
#pragma unroll
      for (int i = 0; i < S::kVRecords; ++i) {
#pragma unroll
        for (int e = 0; e < S::kVCh / 2; ++e) o[c][i][e][0] = o[c][i][e][1] = o[c][i][e][2] = o[c][i][e][3] = 0.0f;
      }
    }
    float m[kCols][2], l[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c) m[c][0] = m[c][1] = -INFINITY, l[c][0] = l[c][1] = 0.0f;

    int place = 0;
    for (int step = step_first; step < step_end; step += kWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kDepth - 2) : "memory");
      __syncwarp();
      const uint32_t from = ring + place * S::kBytes;
      const int key0 = step * 16;
      const int lim = (bad_steps >> place) & 1u ? 0 : min(16, last_vis - key0);
      // Keys row_key and 8 + row_key of the step: rows g and g + 8 of its scores.
      float ks[2] = {}, vs[2] = {};
      if constexpr (kE4m3) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ks[j] = loadShared4(from + S::kScales + (8 * j + row_key) * 4);
          vs[j] = loadShared4(from + S::kScales + 64 + (8 * j + row_key) * 4);
        }
      }
      float sc[kCols][4] = {}, sc1[kCols][4] = {};  // two chains, of half the latency each
      const uint32_t k_at = from + t * S::kKPlane + row_key * 16;
#pragma unroll
      for (int n = 0; n < S::kKRecords; ++n) {
        const uint4 k0 = loadShared16(k_at + 4 * n * S::kKPlane), k1 = loadShared16(k_at + 4 * n * S::kKPlane + 128);
        if constexpr (kE4m3) {
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint2 h0 = halves(w0[e]), h1 = halves(w1[e]);
            const uint32_t f[4] = {h0.x, h1.x, h0.y, h1.y};
#pragma unroll
            for (int c = 0; c < kCols; ++c) mma<M>(e & 1 ? sc1[c] : sc[c], f, qf[c][4 * n + e][0], qf[c][4 * n + e][1]);
          }
        } else {
          const uint32_t f0[4] = {k0.x, k1.x, k0.y, k1.y}, f1[4] = {k0.z, k1.z, k0.w, k1.w};
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            mma<M>(sc[c], f0, qf[c][2 * n][0], qf[c][2 * n][1]);
            mma<M>(sc1[c], f1, qf[c][2 * n + 1][0], qf[c][2 * n + 1][1]);
          }
        }
      }
      float x[kCols][2][2];  // [block][key j][row i], log2 domain
      float inv_v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int ve = (__float_as_int(vs[j]) >> 23) - 127;
        inv_v[j] = __int_as_float((127 - ve) << 23);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float s = sc[c][2 * j + i] + sc1[c][2 * j + i];
            x[c][j][i] = kE4m3 ? fmaf(s * row_scale[c][i], ks[j], static_cast<float>(ve)) : s * a.scale_log2;
          }
        }
      }
      if (key0 + lim > min_vis || lim < 16) {  // the causal edge, the last keys, a bad page
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = 8 * j + row_key;
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (key >= lim || key0 + key >= vis[c][i]) x[c][j][i] = -INFINITY;
            }
          }
        }
      }
      bool grow = false;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
#pragma unroll
        for (int i = 0; i < 2; ++i) grow |= fmaxf(x[c][0][i], x[c][1][i]) > m[c][i] + kGrowLog2;
      }
      if (__any_sync(0xffffffffu, grow)) {
        // Keys whose values are all zeros (their scale says nothing): no word of
        // theirs has a bit beside the signs. The four lanes of a score row share the planes.
        bool zeros[2] = {false, false};
        if constexpr (kE4m3) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t any = 0;
#pragma unroll
            for (int p = 0; p < S::kPlanes; p += 4) {
              const uint4 w = loadShared16(from + S::kV + (p + t) * S::kVPlane + (8 * j + row_key) * 16);
              any |= w.x | w.y | w.z | w.w;
            }
            any |= __shfl_xor_sync(0xffffffffu, any, 1);
            any |= __shfl_xor_sync(0xffffffffu, any, 2);
            zeros[j] = (any & 0x7f7f7f7fu) == 0;
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              const float ve = static_cast<float>((__float_as_int(vs[j]) >> 23) - 127);
              if (zeros[j]) x[c][j][0] -= ve + kZerosLog2, x[c][j][1] -= ve + kZerosLog2;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float m_new = fmaxf(m[c][i], fmaxf(x[c][0][i], x[c][1][i]) - kHeadLog2);
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, z));
            const float f = m[c][i] == m_new ? 1.0f : exp2Approx(m[c][i] - m_new);  // -inf stays: nothing to scale
            m[c][i] = m_new;
            l[c][i] *= f;
#pragma unroll
            for (int r = 0; r < S::kVRecords; ++r) {
#pragma unroll
              for (int e = 0; e < S::kVCh / 2; ++e) {
                o[c][r][e][i] *= f;
                o[c][r][e][2 + i] *= f;
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (kE4m3 && zeros[j] && x[c][j][i] != -INFINITY) {  // the weight alone, which may be past fp16
                l[c][i] += exp2Approx(x[c][j][i] + kZerosLog2 - m_new);
                x[c][j][i] = -INFINITY;
              }
            }
          }
        }
      }
      uint32_t p[kCols][2];
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        float neg[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) neg[i] = m[c][i] == -INFINITY ? 0.0f : -m[c][i];  // a row that has seen no key yet
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e0 = exp2Approx(x[c][j][0] + neg[0]), e1 = exp2Approx(x[c][j][1] + neg[1]);
          l[c][0] = kE4m3 ? fmaf(e0, inv_v[j], l[c][0]) : l[c][0] + e0;
          l[c][1] = kE4m3 ? fmaf(e1, inv_v[j], l[c][1]) : l[c][1] + e1;
          p[c][j] = transpose8x8(pack2<M>(e0, e1));  // from keys x rows to rows x keys
        }
      }
      // O^T += V^T P^T. Byte permutes bring two keys of one channel together.
#pragma unroll
      for (int i = 0; i < S::kVRecords; ++i) {
        if constexpr (kE4m3) {
          uint32_t v[4][S::kVCh / 4];
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if constexpr (S::kVCh == 16) {
              const uint4 w = loadShared16(from + S::kV + g * S::kVPlane + (4 * kk + t) * 16);
              v[kk][0] = w.x, v[kk][1] = w.y, v[kk][2] = w.z, v[kk][3] = w.w;
            } else {
              const uint2 w = loadShared8(from + S::kV + (g >> 1) * S::kVPlane + (4 * kk + t) * 16 + (g & 1) * 8);
              v[kk][0] = w.x, v[kk][1] = w.y;
            }
          }
#pragma unroll
          for (int e = 0; e < S::kVCh; e += 4) {
            // Codes of keys 0, 1 (2, 3) side by side, then two channels to a word.
            const uint2 a0 = halves(__byte_perm(v[0][e / 4], v[1][e / 4], 0x5140)), a1 = halves(__byte_perm(v[0][e / 4], v[1][e / 4], 0x7362));
            const uint2 c0 = halves(__byte_perm(v[2][e / 4], v[3][e / 4], 0x5140)), c1 = halves(__byte_perm(v[2][e / 4], v[3][e / 4], 0x7362));
            const uint32_t f0[4] = {a0.x, a0.y, c0.x, c0.y}, f1[4] = {a1.x, a1.y, c1.x, c1.y};
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              mma<M>(o[c][i][e / 2], f0, p[c][0], p[c][1]);
              mma<M>(o[c][i][e / 2 + 1], f1, p[c][0], p[c][1]);
            }
          }
        } else {
          uint32_t v[4][4];
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint4 w = loadShared16(from + S::kV + (8 * i + g) * S::kVPlane + (4 * kk + t) * 16);
            v[kk][0] = w.x, v[kk][1] = w.y, v[kk][2] = w.z, v[kk][3] = w.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t f[4] = {__byte_perm(v[0][e], v[1][e], 0x5410), __byte_perm(v[0][e], v[1][e], 0x7632),
                                   __byte_perm(v[2][e], v[3][e], 0x5410), __byte_perm(v[2][e], v[3][e], 0x7632)};
#pragma unroll
            for (int c = 0; c < kCols; ++c) mma<M>(o[c][i][e], f, p[c][0], p[c][1]);
          }
        }
      }
      __syncwarp();
      const int refill = place == 0 ? S::kDepth - 1 : place - 1;  // the place read a step before
      copyStep(step + (S::kDepth - 1) * kWarps, refill);
      place = place + 1 == S::kDepth ? 0 : place + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring is free for the exchange

    // ---- join the warps ----
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = 8 * c + 2 * t + i;
#pragma unroll
        for (int z = 4; z < 32; z <<= 1) l[c][i] += __shfl_xor_sync(0xffffffffu, l[c][i], z);
        if (g == 0) {
          ml_s[warp][0][rr] = m[c][i];
          ml_s[warp][1][rr] = l[c][i];
        }
#pragma unroll
        for (int r = 0; r < S::kVRecords; ++r) {
#pragma unroll
          for (int e = 0; e < S::kVCh / 2; ++e) {
            *reinterpret_cast<float2*>(&o_s[warp][rr][(8 * r + g) * S::kVCh + 2 * e]) = make_float2(o[c][r][e][i], o[c][r][e][2 + i]);
          }
        }
      }
    }
    __syncthreads();
    const bool whole = kCluster ? cluster == 1 : b0 == 0 && b1 == blocks;
    // A partial: in this CTA's shared memory behind the exchange, or in the workspace.
    float* part;
    if constexpr (kCluster) {
      part = reinterpret_cast<float*>(ring_raw) + kWarps * kStreamRows * (D + 4);
    } else {
      part = partials + (2 * static_cast<size_t>(blockIdx.x) + (first_piece && b0 > 0 ? 0 : 1)) * partialFloats(D);
    }
    for (int i = tid; i < R * (D / 8); i += kThreads) {
      const int rr = i / (D / 8), grp = i % (D / 8);
      if (rr < pass_s.lo || rr >= pass_s.hi) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml_s[w][0][rr]);
      float ll = 0.0f, acc[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ml_s[w][0][rr];
        const float f = mw == mm ? 1.0f : exp2Approx(mw - mm);
        ll = fmaf(ml_s[w][1][rr], f, ll);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(o_s[w][rr][grp * 8 + e], f, acc[e]);
      }
      if (pass_s.hides) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (acc[e] != acc[e]) pass_s.nan = 1;
        }
      }
      if (whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = normalised(acc[e], ll);
        const int r = tile * R + rr;  // below 2^31: checked by the host
        const int token = r / q_heads_per;
        const int h = head * q_heads_per + r - token * q_heads_per;
        *reinterpret_cast<uint4*>(record(a.out, h, q.q0 + token, grp)) = pack8<T>(acc);
      } else {
        float4* dst = reinterpret_cast<float4*>(part + rr * D + grp * 8);
        dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (grp == 0) {
          (kCluster ? joined_s[0] : part + kStreamRows * D)[rr] = mm;
          (kCluster ? joined_s[1] : part + kStreamRows * D + kStreamRows)[rr] = ll;
        }
      }
    }
    bool nan = false;
    if constexpr (kCluster) {
      if (cluster > 1) {
        __syncwarp();  // the barrier is one of whole warps, and lanes leave the loop apart
        tc::clusterSync();
        const uint32_t part_at = tc::smemU32(part), ml_at = tc::smemU32(&joined_s[0][0]);
        for (int i = rank * kThreads + tid; i < rows * (D / 8); i += cluster * kThreads) {
          const int rr = i / (D / 8), grp = i % (D / 8);
          if (rr < pass_s.lo || rr >= pass_s.hi) continue;
          float m_all = -INFINITY, l_all = 0.0f, x[8] = {};
          for (int c = 0; c < cluster; ++c) m_all = fmaxf(m_all, loadCluster4(tc::mapaShared(ml_at + rr * 4, c)));
          for (int c = 0; c < cluster; ++c) {
            const float mc = loadCluster4(tc::mapaShared(ml_at + rr * 4, c));
            const float f = mc == m_all ? 1.0f : exp2Approx(mc - m_all);
            l_all = fmaf(loadCluster4(tc::mapaShared(ml_at + (kStreamRows + rr) * 4, c)), f, l_all);
            const uint32_t at = tc::mapaShared(part_at + (rr * D + grp * 8) * 4, c);
            const float4 y = loadCluster16(at), z = loadCluster16(at + 16);
            const float v[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaf(v[e], f, x[e]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = normalised(x[e], l_all);
          const int r = tile * R + rr;
          const int token = r / q_heads_per;
          *reinterpret_cast<uint4*>(record(a.out, head * q_heads_per + r - token * q_heads_per, q.q0 + token, grp)) = pack8<T>(x);
        }
        if (pass_s.hides) {
          for (int c = 0; c < cluster; ++c) nan |= __float_as_int(loadCluster4(tc::mapaShared(tc::smemU32(&pass_s.nan), c))) != 0;
        }
        __syncwarp();
        tc::clusterSync();  // no CTA leaves while another reads its memory
      }
    }
    if (pass_s.hides && (!kCluster || cluster == 1)) {
      __syncthreads();
      nan = pass_s.nan != 0;
    }
    // Where a row does not see a key, an infinity or NaN among its values makes
    // 0 * v NaN: the tile is done again token by token, whose rows see the same keys
    // and the others are not read.
    if (pass_s.again >= 0 || nan) {
      const int next = pass_s.again < 0 ? 0 : pass_s.hi < min(R, q.nq * a.group - tile * R) ? pass_s.hi : -1;
      __syncthreads();
      if (tid == 0) pass_s.again = next;
      __syncthreads();
      if (next >= 0) continue;
    }
    if constexpr (kCluster) return;
    if (first_piece && tid == 0) {
      if (b0 > 0) {
        split->first_unit = tile_first;
        split->last_unit = tile_first + blocks - 1;
        split->seq = seq;
        split->tile = tile;
        split->head = head;
        split->rows = rows;
      } else {
        split->first_unit = -1;
      }
      // The joining launch needs the shares too.
      if (blockIdx.x == 0) *reinterpret_cast<Share*>(partials + 2 * static_cast<size_t>(kStreamCtas) * partialFloats(D)) = share;
    }
    first_piece = false;
    u = tile_first + b1;
    __syncthreads();
  }
}

constexpr int kJoinWarps = 16;

// Joins the partials of a tile that several CTAs worked on: CTA c looks after
// the tile in which share c begins, if it is the first share to begin there.
template <typename T, int D, KvKind kKind, int R>
__global__ void __launch_bounds__(kJoinWarps * 32) joinStreamKernel(const Args a) {
  __shared__ float acc_s[kJoinWarps][D];
  __shared__ float ml_s[kJoinWarps][2];
  tc::pdlTrigger();
  tc::pdlWait();
  const float* partials = reinterpret_cast<const float*>(a.workspace + sizeof(Split) * kStreamCtas);
  const Split split = reinterpret_cast<const Split*>(a.workspace)[blockIdx.x];
  if (split.first_unit < 0) return;
  const Share share = *reinterpret_cast<const Share*>(partials + 2 * static_cast<size_t>(kStreamCtas) * partialFloats(D));
  const long long c0 = shareOwner(share, split.first_unit);
  if (c0 != static_cast<long long>(blockIdx.x) - 1) return;
  const int n = static_cast<int>(shareOwner(share, split.last_unit) - c0) + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Warps of one row: kJoinWarps over the rows, rounded down to a power of two.
  int per_row = 1;
  while (per_row * 2 * split.rows <= kJoinWarps) per_row *= 2;
  const int row = warp / per_row, sub = warp - row * per_row;
  constexpr int kPer = D / 32;  // channels of a lane
  float acc[kPer] = {}, m = -INFINITY, l = 0.0f;
  if (row < split.rows) {
    // Piece i of the tile is CTA c0 + i's: its last piece (1) for i = 0, its
    // first (0) after. Four are read at a time.
    for (int i0 = sub; i0 < n; i0 += 4 * per_row) {
      float pm[4], pl[4], po[4][kPer];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = i0 + x * per_row;
        const bool in = i < n;
        const float* p = partials + (2 * static_cast<size_t>(c0 + (in ? i : i0)) + ((in ? i : i0) == 0 ? 1 : 0)) * partialFloats(D);
        pm[x] = in ? p[kStreamRows * D + row] : -INFINITY;
        pl[x] = in ? p[kStreamRows * D + kStreamRows + row] : 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) po[x][e] = in ? p[row * D + e * 32 + lane] : 0.0f;
      }
      const float top = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
      const float keep = m == top ? 1.0f : exp2Approx(m - top);
      m = top;
      l *= keep;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] *= keep;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float f = pm[x] == m ? 1.0f : exp2Approx(pm[x] - m);
        l = fmaf(pl[x], f, l);
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(po[x][e], f, acc[e]);
      }
    }
    if (lane == 0) {
      ml_s[warp][0] = m;
      ml_s[warp][1] = l;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc_s[warp][e * 32 + lane] = acc[e];
  }
  __syncthreads();
  const Sequence q = sequence<kKind>(a, split.seq);
  for (int i = threadIdx.x; i < split.rows * (D / 8); i += kJoinWarps * 32) {
    const int rr = i / (D / 8), grp = i % (D / 8);
    float mm = -INFINITY;
    for (int w = 0; w < per_row; ++w) mm = fmaxf(mm, ml_s[rr * per_row + w][0]);
    float ll = 0.0f, x[8] = {};
    for (int w = 0; w < per_row; ++w) {
      const float mw = ml_s[rr * per_row + w][0];
      const float f = mw == mm ? 1.0f : exp2Approx(mw - mm);
      ll = fmaf(ml_s[rr * per_row + w][1], f, ll);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmaf(acc_s[rr * per_row + w][grp * 8 + e], f, x[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = normalised(x[e], ll);
    const int r = split.tile * R + rr;
    const int token = r / a.group;
    const int h = split.head * a.group + r - token * a.group;
    *reinterpret_cast<uint4*>(record(a.out, h, q.q0 + token, grp)) = pack8<T>(x);
  }
}

long long streamWorkspaceBytes(int head_dim) {
  return static_cast<long long>(sizeof(Split) * kStreamCtas + 2 * kStreamCtas * partialFloats(head_dim) * sizeof(float) + sizeof(Share));
}

namespace {

// CTAs to a tile where sequences are at most max_keys long, 0: even shares of
// the line instead, joined by a second launch. A cluster grows while all CTAs run
// at once (8 hypothesis groups of 3 to 252 rows: 10.6 us with 2 CTAs to a tile,
// 16.8 with 4 in two waves) and have two units or more, but up to 256 keys stay one CTA's (4 x 256
// keys 7.0 us, with two CTAs 7.6), and is taken where none of its CTAs gets more
// than kClusterKeys keys. Measured with 8 key heads, clusters against shares (us):
// 4 x 64 keys 4.4 / 14.2, 4 x 1000 (128 keys to a CTA) 9.7 / 12.7, 4 x 2000 (256)
// 12.7 / 14.8, 32 x 500 (512) 15.3 / 20.9, 1 x 4000 (512) 13.2 / 13.2, 16 x 2000
// (1024) 29.2 / 20.0, 8 x 4000 (1024) 28.4 / 18.9.
long long numbersOf(const Args& a, int rows) { return (static_cast<long long>(a.q_rows) * a.group / rows + a.n_seq) * a.kv_heads; }

int clusterOf(const Args& a, long long tiles, int max_keys, int resident) {
  if (a.n_seq > kThreads) return 0;  // each thread looks at one sequence
  if (tiles > 0x7fffffffLL / 8) return 0;
  int n = 1;
  while (n < 8 && max_keys > 4 * kUnitKeys && 2 * n * tiles <= resident && 2 * n * 2 * kUnitKeys <= max_keys) n *= 2;
  return max_keys <= n * kClusterKeys ? n : 0;
}

template <typename T, int D, KvKind kKind, int R>
cudaError_t launchOne(const Args& a, int max_keys, cudaStream_t s) {
  constexpr int kRing = Step<D, kKind == kPagedE4m3>::kRing;
  static DeviceOnce smem_attr;
  const cudaError_t ae = smem_attr.run([] {
    const cudaError_t e = cudaFuncSetAttribute(attentionStreamKernel<T, D, kKind, R, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(attentionStreamKernel<T, D, kKind, R, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
  });
  if (ae != cudaSuccess) return ae;
  // As many CTAs as stay resident, so that equal shares end together.
  static DeviceValue resident;
  const int ctas = resident.get([](int dev) {
    int sms = 148, per = 1;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, attentionStreamKernel<T, D, kKind, R, false>, kThreads, kRing);
    return std::min(kStreamCtas, sms * std::max(per, 1));
  });
  const long long tiles = numbersOf(a, R);
  if (const int cluster = clusterOf(a, tiles, max_keys, ctas); cluster > 0) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kRing;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    prof::countLaunch(prof::kAttention);
    return cudaLaunchKernelEx(&cfg, attentionStreamKernel<T, D, kKind, R, true>, a, cluster);
  }
  prof::countLaunch(prof::kAttention, 2);
  cudaError_t e = launchPdl(attentionStreamKernel<T, D, kKind, R, false>, dim3(ctas), dim3(kThreads), kRing, s, a, 0);
  if (e != cudaSuccess) return e;
  return launchPdl(joinStreamKernel<T, D, kKind, R>, dim3(ctas), dim3(kJoinWarps * 32), 0, s, a);
}

// Rows of a tile: 8 where sequences have at most 8 on average, else 16. One row
// over 8 x 131,072 e4m3 keys (4 rows a tile): 151 us, with tiles of 16 172; 16 rows:
// 178 in one tile of 16.
template <typename T, int D, KvKind kKind>
cudaError_t launchRows(const Args& a, int max_keys, cudaStream_t s) {
  const bool few = static_cast<long long>(a.q_rows) * a.group <= 8LL * a.n_seq;
  return few ? launchOne<T, D, kKind, 8>(a, max_keys, s) : launchOne<T, D, kKind, 16>(a, max_keys, s);
}

template <typename T, int D>
cudaError_t launchKind(const Args& a, KvKind kind, int max_keys, cudaStream_t s) {
  switch (kind) {
    case kPacked16: return launchRows<T, D, kPacked16>(a, max_keys, s);
    case kPaged16: return launchRows<T, D, kPaged16>(a, max_keys, s);
    default: return launchRows<T, D, kPagedE4m3>(a, max_keys, s);
  }
}

}  // namespace

cudaError_t launchStream(const Args& a, KvKind kind, int head_dim, int dtype, cudaStream_t s) {
  const long long most = kind == kPacked16 ? a.kv_rows : static_cast<long long>(a.table_pages) << a.page_shift;
  const int max_keys = static_cast<int>(std::min(most, 0x7fffffffLL));
  if (dtype == FPK_DTYPE_BF16) {
    return head_dim == 64 ? launchKind<__nv_bfloat16, 64>(a, kind, max_keys, s) : launchKind<__nv_bfloat16, 128>(a, kind, max_keys, s);
  }
  return head_dim == 64 ? launchKind<__half, 64>(a, kind, max_keys, s) : launchKind<__half, 128>(a, kind, max_keys, s);
}

}  // namespace seqattn
}  // namespace fpb
