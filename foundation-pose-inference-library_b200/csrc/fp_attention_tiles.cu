// Attention of many query rows (prompts, chunks over a cache) on tcgen05 tensor
// cores: fpk_attention_packed and fpk_attention_paged where a sequence has more
// than 16 query rows (tokens x query heads to a key head) and there is enough work.
//
// Bound by the tensor cores (4 d FLOP for each query row and key) and, as
// closely, by the exponential unit: for d = 128 a 128 x 128 block of scores
// takes 1,024 cycles of MMA and 16,384 / 16 = 1,024 cycles of ex2.
//
// One persistent CTA per SM, 512 threads. Its tile is 256 query rows of one
// (sequence, key head), two halves of 128 rows: while the softmax of one half
// runs, the tensor core works for the other.
//   warps 0-3, 4-7  softmax of half 0 and 1, one query row per thread: the
//                   row's 128 scores from TMEM, 64 at a time: running maximum
//                   and sum in fp32, P = 2^(s - m) rounded to the element type
//                   over the scores' own TMEM columns. m lies 2^7 below a row's
//                   maximum; O is rescaled only when that grows by more than 2^8.
//                   After the last, O / l.
//   warps 8-11      loads of Q, K and V rows, K and V in four stages of 128 rows.
//                   Two layouts in shared memory, each the one that its source
//                   fills line by line (the other way round the copies take
//                   eight times the shared-memory cycles and hold up the
//                   softmax): planar sources and pages as [group of 8
//                   channels][row][16 B], K and V by bulk copies of whole
//                   groups; row-major sources as rows of 64 channels with the
//                   128-byte swizzle, by cp.async, which takes any strides. e4m3
//                   rows pass through registers, where they become the element
//                   type (exact in bf16). Values of keys that nobody sees are
//                   zeroed; their scores are masked.
//   warps 12, 15    MMA issue for half 0 and 1: S = Q K^T, then for each block
//                   O += P V (its first 64 keys as soon as they are there) and
//                   the next block's scores, across tiles too. One warp for
//                   both would be bound by its own instructions.
//   warp 13         the walk: the next pieces of work for the others.
//   warp 14         the proxy fence between a load's arrival and the MMAs that
//                   read it, which would cost the issuing warp 300-600 cycles.
//
// Under a causal mask 0 * v of a key that a row does not see is NaN where v is an
// infinity or NaN. An item with NaN in such a row is walked a second time, when
// warp 14 takes these values out and the softmax warps add them to the rows that
// see them (looked for in every item they cost prompts 1 to 8 %).
// TMEM: S_0 S_1 (128 columns each) O_0 O_1 (d each), one CTA per SM.
//
// The work of all tiles is laid on one line (a tile's length: the keys that it
// sees) and cut into one share per CTA, so that causal and ragged batches and
// few long rows all end together. A tile cut inside leaves fp32 partials that a
// second launch joins in order; where tiles are short against a share, cuts
// move to tile ends and nothing is joined. All mbarrier waits are bounded.
//
// Measured: 4 causal prompts of 700 to 8,192 tokens, 16 heads over 2 of 128, bf16,
// 542 us = 958 TFLOP/s, without a mask 1,028; 252 sequences of 400, 4 heads of 128,
// fp16, 153 us = 540 TFLOP/s (a fifth of the rows of its tiles are empty). A block
// of 128 keys takes some 3,900 cycles for the 256 rows, of 2,048 that either the
// tensor core or the exponentials need: each half waits for its scores (1,200), then
// for its own 2 x 64 exponentials (2,400, the other half's among them). Tried and not
// kept: the halves in turns (with a separate pass for the maximum), a quarter of the
// exponentials as polynomials (slower by 3 to 8 %), both halves of a block unrolled
// with loads ahead (no gain, crops 8 % slower),
// two threads to a row in 16 warps of 80 registers (13 to 30 % slower), scores of 64
// keys two parts ahead in either half of their columns (prompts the same, crops
// 164: a product with 64 keys takes 53 cycles for half of the 64 that 128 take).
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

using namespace tc;

constexpr int kHalf = 128;       // rows of a half tile = TMEM lanes
constexpr int kKeys = 128;       // keys of a block
constexpr int kStages = 4;       // K 0, V 0, K 1, V 1
constexpr int kItems = 4;        // work items in flight between the roles
constexpr int kLoadWarps = 4;
constexpr int kThreads = 512;
constexpr uint32_t kChunk = kKeys * 128;      // 128 rows of 64 channels
constexpr uint32_t kPlane = kKeys * 16;       // 128 rows of 8 channels
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;
// A row's reference lies 2^7 below the maximum it was set by and stays until a
// score is 2^15 above it: fp16 probabilities down to 2^-32 of the largest reach
// the products.
constexpr float kHeadLog2 = 7.0f;
constexpr float kGrowLog2 = 15.0f;
// A tile's work beside its keys, in keys (of 192 to 384 none is better).
constexpr int kTileCost = 384;
// Least share, in keys. One prompt of 100 rows: 13.6 us with 256, 17.6 with 512.
constexpr int kMinShare = 256;
// Smallest piece of a page, in rows, for bulk copies: their issue takes some 70
// cycles each whatever the size. Four chunks over 12,000 keys, bulk against 16
// bytes at a time (us): pages of 16 rows 259 / 196, of 32 193 / 216, of 64 205 /
// 217, of 128 191 / 214.
constexpr int kBulkRows = 32;
// A tile shorter than 1/8 share is not cut. Crops (short tiles) 150 us, 155 if
// all are cut; at 1/2 chunks over pages lose 10 % to uneven shares.
constexpr int kSnap = 8;

struct Item {
  int halves;                  // halves with rows; 0: no more work, -1: none in this item
  int seq, head, tile;
  int q0, nq, k0, nk;
  int jb, je;                  // key blocks of this piece
  int lim;                     // keys that the tile sees
  int part;                    // -1: the whole tile; else the partial's index
};

// What the joining launch needs of a CTA: the tile that its share begins inside.
struct Cut {
  long long tile_at;           // the tile's place on the line, -1: nothing cut
  int jb, blocks;
  int seq, head, tile;
  int failed;                  // a wait of this CTA ran out: its pieces may be missing
};

struct Smem {
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t q_ready[2], kv_ready[kStages];  // full, and fenced for the tensor core
  uint64_t s_full[2], p_half[2], p_full[2], pv_half[2], pv_done[2], o_free[2];  // half: of a block's first 64 keys
  uint64_t drained[2];
  Item items[kItems];
  int again[kItems];   // the item is done a second time: hidden values are taken out
  int redo[kItems];    // it has to be
  int hidden[kItems];  // its hidden values are in the table
  long long scan[kThreads / 32 + 1];
  long long found[2];
  uint32_t tmem;
  int stop;                    // a wait ran out: every role leaves
};

template <int D>
struct Geo {
  static constexpr int kPlanes = D / 8;
  static constexpr uint32_t kTileBytes = D / 64 * kChunk;  // 128 rows
  static constexpr size_t kSmem = 1024 + (2 + kStages) * static_cast<size_t>(kTileBytes) + 1024;
};
static_assert(sizeof(Smem) <= 1024, "barrier block");

// fp32 partial of a piece: [D/4][256 rows][4], m [256], l [256].
constexpr size_t partialFloats(int d) { return static_cast<size_t>(kTileRows) * d + 2 * kTileRows; }

// ---- the line of work ----

// Tile i of a sequence and head is long w(i): the keys that its last full token
// row sees (causal: growing by the tokens of a tile) and kTileCost for what a
// tile costs beside its keys, in closed form.
struct Line {
  int tiles;
  int first, step;  // w(i) = kTileCost + clamp(first + i * step, 0, nk)
  int nk;
  int k0, k1;       // the clamp is 0 below tile k0, nk from tile k1 on
};

__device__ __forceinline__ Line lineOf(const Args& a, const Sequence& q) {
  Line n;
  n.tiles = (q.nq * a.group + kTileRows - 1) / kTileRows;  // below 2^31: checked by the host
  n.nk = q.nk;
  n.step = a.causal ? max(kTileRows / a.group, 1) : 0;
  n.first = a.causal ? q.nk - q.nq + n.step : q.nk;
  n.k0 = n.first >= 0 ? 0 : (-n.first + n.step - 1) / n.step;
  n.k1 = n.first >= n.nk ? 0 : (n.nk - n.first + n.step - 1) / n.step;
  return n;
}

__device__ __forceinline__ int tileLength(const Line& n, int i) {
  return kTileCost + (i < n.k0 ? 0 : i >= n.k1 ? n.nk : n.first + i * n.step);
}

// Sum of tileLength over tiles 0 .. i-1.
__device__ __forceinline__ long long lengthBefore(const Line& n, int i) {
  const long long lo = min(n.k0, i), hi = min(max(n.k1, n.k0), i);
  const long long ramp = hi - lo;
  return static_cast<long long>(i) * kTileCost + ramp * n.first + n.step * ((lo + hi - 1) * ramp / 2) + (i - hi) * n.nk;
}

// The tile that holds place x of a head's line.
__device__ __forceinline__ int tileAt(const Line& n, long long x) {
  int lo = 0, hi = n.tiles - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (lengthBefore(n, mid) <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int blocksOf(int lim) { return max((lim + kKeys - 1) / kKeys, 1); }

// Keys that a tile sees: those of its last row.
__device__ __forceinline__ int tileLimit(const Args& a, const Sequence& q, int tile) {
  return visible(a, q, (min(q.nq * a.group, (tile + 1) * kTileRows) - 1) / a.group);
}

// Key block at which place y of a tile of length w cuts it. The two CTAs on
// either side of a cut compute it alike, and it grows with y: fp32 will do.
__device__ __forceinline__ int cutBlock(int y, int w, int blocks, int snap) {
  if (w <= snap) return y < w - y ? 0 : blocks;
  return min(static_cast<int>(__fdividef(static_cast<float>(y), static_cast<float>(w)) * static_cast<float>(blocks)), blocks);
}

// ---- waits ----

__device__ __noinline__ bool waitSlow(uint64_t* bar, uint32_t parity, volatile int* stop, int* err, int code) {
  const long long start = clock64();
  for (uint32_t i = 0;; ++i) {
    if (mbarTryWait(bar, parity)) return true;
    if ((i & 255u) == 255u) {
      if (*stop != 0) return false;
      if (clock64() - start > kTimeoutCycles) {
        *stop = 1;
        reportIndex(err, code);
        return false;
      }
    }
  }
}

// By a whole (converged) warp. The vote also tells the compiler that the warp
// stays together, which keeps the MMA issue on the uniform datapath.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Smem& sm, int* err, int code) {
  if (__all_sync(0xffffffffu, mbarTryWait(bar, parity))) return true;
  return __all_sync(0xffffffffu, waitSlow(bar, parity, &sm.stop, err, code));
}

__host__ __device__ constexpr uint32_t idesc(uint32_t fmt, int n, bool b_mn_major) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kHalf >> 4) << 24);
}

// One lane of a converged warp, always the same.
__device__ __forceinline__ bool electOne() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r != 0;
}

// MMAs and commits of one thread, in a branch of their own: guarded one by one
// they take twice the instructions.
template <int kAdd>
__device__ __forceinline__ void mmaScores(uint32_t d, uint64_t q, uint64_t k, uint32_t id) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(q),
               "l"(k), "r"(id), "n"(kAdd)
               : "memory");
}
__device__ __forceinline__ void mmaValues(uint32_t d, uint32_t p, uint64_t v, uint32_t id, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(p),
               "l"(v), "r"(id), "r"(add)
               : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smemU32(bar)) : "memory");
}

// Operand descriptors and the distance of K steps (16 channels or keys) in
// them. Either layout holds 64 channels of 128 rows in 16 KB.
//   Q, K (K-major)   planar: groups of 8 rows 128 B apart, groups of channels
//                    2 KB, a step 4 KB; swizzled: rows of 128 B, a step 32 B.
//   V (MN-major)     planar: groups of 8 keys 128 B apart, of channels 2 KB, a
//                    step 256 B; swizzled: groups of 8 keys 1 KB apart, a step
//                    2 KB, 64 channels to a chunk.
struct Operand {
  uint64_t desc;
  uint32_t step;
};
__device__ __forceinline__ Operand keyOperand(uint32_t addr, bool planar) {
  return planar ? Operand{smemDesc(addr, kPlane, 128, kLayoutNone), 2 * kPlane >> 4} : Operand{smemDesc(addr, 16, 1024, kLayoutSw128), 32 >> 4};
}
__device__ __forceinline__ Operand valueOperand(uint32_t addr, bool planar) {
  return planar ? Operand{smemDesc(addr, 128, kPlane, kLayoutNone), 256 >> 4} : Operand{smemDesc(addr, kChunk, 1024, kLayoutSw128), 2048 >> 4};
}

template <int D>
__device__ __forceinline__ void issueScores(uint32_t d, const Operand& q, uint64_t k, uint32_t k_step, uint32_t id) {
  mmaScores<0>(d, q.desc, k, id);
#pragma unroll
  for (int ks = 1; ks < D / 16; ++ks) {
    const uint32_t chunk = (ks / 4) * (kChunk >> 4);
    mmaScores<1>(d, q.desc + (chunk + (ks % 4) * q.step), k + (chunk + (ks % 4) * k_step), id);
  }
}

// Steps kFirst .. kFirst + 3 of a block's 8, as far as it has keys.
template <int kFirst>
__device__ __forceinline__ void issueValues(uint32_t d, uint32_t p, uint64_t v, uint32_t v_step, uint32_t id, int steps, bool add) {
#pragma unroll
  for (int ks = kFirst; ks < kFirst + 4; ++ks) {
    if (ks < steps) mmaValues(d, p + ks * 8, v + ks * v_step, id, ks > kFirst || add ? 1u : 0u);
  }
}

__device__ __forceinline__ float exp2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float max3Nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// Masks 64 scores: those from lim on, and groups of 16 whose bit in bad is set.
__device__ __noinline__ uint2 keepMask(int lim, uint32_t bad) {
  uint32_t keep[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int in = min(max(lim - 32 * c, 0), 32);
    keep[c] = in == 32 ? 0xffffffffu : (1u << in) - 1u;
    if ((bad >> (2 * c)) & 1u) keep[c] &= 0xffff0000u;
    if ((bad >> (2 * c + 1)) & 1u) keep[c] &= 0x0000ffffu;
  }
  return make_uint2(keep[0], keep[1]);
}
__device__ __forceinline__ void hide(uint32_t (&s)[64], int lim, uint32_t bad) {
  const uint2 keep = keepMask(lim, bad);
#pragma unroll
  for (int e = 0; e < 64; ++e) {
    if ((((e < 32 ? keep.x : keep.y) >> (e & 31)) & 1u) == 0) s[e] = __float_as_uint(-INFINITY);
  }
}

__device__ __forceinline__ void copyAsync16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// `bytes` of a bulk copy, and one arrival of this thread that waits for them.
__device__ __forceinline__ void copyBulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  mbarExpectTx(bar, bytes);
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(smemU32(bar))
               : "memory");
}
// One arrival of this thread on `bar` once its earlier copyAsync16 have landed.
__device__ __forceinline__ void copyArrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smemU32(bar)) : "memory");
}
__device__ __forceinline__ void copyDrain() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint4 loadShared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void storeShared16(uint32_t dst, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ---- hidden values that are not finite, in items that are done again ----
//
// Such an element becomes 0, and the lowest key that held one is noted by channel.
// As a row sees the keys below its limit, it sees one exactly if its limit is above
// that key, and gets it at the end.

// Whether a record of T holds an infinity or NaN: 1 carries the exponent's ones into bit 15.
template <typename T>
__device__ __forceinline__ bool hasNotFinite(const uint4& w) {
  const uint32_t m = 0x7fff7fffu, one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((((w.x & m) + one) | ((w.y & m) + one) | ((w.z & m) + one) | ((w.w & m) + one)) & 0x80008000u) != 0;
}

constexpr int kNoKey = 0x7fffffff;

// Record of `key` with such elements as zeros. first[c] is the lowest key with
// +infinity or NaN in channel c of the record, first[negative + c] with -infinity or NaN.
template <typename T>
__device__ __noinline__ uint4 hideNotFinite(uint4 w, int key, int* first, int negative) {
  const uint32_t exponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t h = (u[e / 2] >> (16 * (e & 1))) & 0xffffu;
    if ((h & exponent) != exponent) continue;
    const bool nan = (h & 0x7fffu) != exponent, minus = (h & 0x8000u) != 0;
    if (nan || !minus) atomicMin(first + e, key);
    if (nan || minus) atomicMin(first + negative + e, key);
    u[e / 2] &= ~(0xffffu << (16 * (e & 1)));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// What a row that sees the keys below `visible` adds to a channel's sum.
__device__ __forceinline__ float seenNotFinite(int first_plus, int first_minus, int visible) {
  if (first_plus < visible) return first_minus < visible ? __int_as_float(0x7fffffff) : __int_as_float(0x7f800000);
  return first_minus < visible ? __int_as_float(static_cast<int>(0xff800000u)) : 0.0f;
}

// Record of row r and plane p of a tile. 32 rows of a plane give neither layout a bank conflict.
__device__ __forceinline__ uint32_t recordAt(uint32_t tile, bool planar, int r, int p) {
  return tile + (planar ? p * kPlane + r * 16 : (p >> 3) * kChunk + r * 128 + (((p ^ r) & 7) << 4));
}

// Whether keys edge .. lim - 1 of a V tile have any. This and the next two by a whole warp.
template <typename T, int D>
__device__ __noinline__ bool hasHidden(uint32_t tile, bool planar, int key0, int edge, int lim) {
  const int lane = threadIdx.x & 31, rows = min(lim - key0, kKeys);
  bool found = false;
#pragma unroll 1
  for (int r = max(edge - key0, 0) + lane; r < rows; r += 32) {
    for (int p = 0; p < D / 8; ++p) found |= hasNotFinite<T>(loadShared16(recordAt(tile, planar, r, p)));
  }
  return __any_sync(0xffffffffu, found);
}

// Takes them out and notes them in a table of 2 x D, which `begun` says holds some already.
template <typename T, int D>
__device__ __noinline__ void hideValues(uint32_t tile, bool planar, int key0, int edge, int lim, int* table, bool begun) {
  const int lane = threadIdx.x & 31, rows = min(lim - key0, kKeys);
  if (!begun) {
    for (int c = lane; c < 2 * D; c += 32) table[c] = kNoKey;
    __syncwarp();
  }
#pragma unroll 1
  for (int r = max(edge - key0, 0) + lane; r < rows; r += 32) {
#pragma unroll 1
    for (int p = 0; p < D / 8; ++p) {
      const uint4 v = loadShared16(recordAt(tile, planar, r, p));
      if (hasNotFinite<T>(v)) storeShared16(recordAt(tile, planar, r, p), hideNotFinite<T>(v, key0 + r, table + 8 * p, D));
    }
  }
  __syncwarp();
}

// Adds to a row's O what those that it sees make of it.
template <int D>
__device__ __noinline__ void addHidden(uint32_t o, const volatile int* table, int visible) {
#pragma unroll 1
  for (int c = 0; c < D; c += 16) {
    uint32_t x[16];
    FPB_TMEM_LD16(o + c, x);
    tmemWaitLd();
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) + seenNotFinite(table[c + e], table[D + c + e], visible));
    FPB_TMEM_ST16(o + c, x);
  }
  tmemStoreWait();
}

// An e4m3 record with NaN or an unusual scale, into two groups of a planar tile.
template <typename T>
__device__ __noinline__ void storeRecord(uint32_t dst, uint4 codes, float scale) {
  uint4 out[2];
  dequantise16<T>(codes, scale, out);
  storeShared16(dst, out[0]);
  storeShared16(dst + kPlane, out[1]);
}

}  // namespace

template <typename T, int D, KvKind kKind>
__global__ void __launch_bounds__(kThreads, 1) attentionTilesKernel(const Args a) {
  using G = Geo<D>;
  constexpr int kPlanes = G::kPlanes;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Smem& sm = *reinterpret_cast<Smem*>(base);
  const uint32_t q_s = smemU32(base + 1024);
  const uint32_t kv_s = q_s + 2 * G::kTileBytes;

  tc::pdlTrigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kItems; ++i) {
      mbarInit(&sm.item_full[i], 1);
      mbarInit(&sm.item_empty[i], 8 + 3 + kLoadWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbarInit(&sm.q_full[i], kLoadWarps * 32);
      mbarInit(&sm.q_empty[i], 1);
      mbarInit(&sm.q_ready[i], 1);
      mbarInit(&sm.s_full[i], 1);
      mbarInit(&sm.p_half[i], 4);
      mbarInit(&sm.p_full[i], 4);
      mbarInit(&sm.pv_half[i], 1);
      mbarInit(&sm.pv_done[i], 1);
      mbarInit(&sm.o_free[i], 4);
      mbarInit(&sm.drained[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbarInit(&sm.kv_full[i], kLoadWarps * 32);
      mbarInit(&sm.kv_empty[i], 2);
      mbarInit(&sm.kv_ready[i], 1);
    }
    sm.stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemU32(&sm.tmem)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc::pdlWait();

  // ---- this CTA's share of the line ----
  Cut* cuts = reinterpret_cast<Cut*>(a.workspace);
  float* partials = reinterpret_cast<float*>(a.workspace + sizeof(Cut) * kTileCtas);
  // Hidden values of items done again. Not in shared memory, where 1 KB more costs L1.
  int* table = reinterpret_cast<int*>(partials + 2 * kTileCtas * partialFloats(D)) + blockIdx.x * 2 * D;
  auto lengthOf = [&](int s) -> long long {
    if (s >= a.n_seq) return 0;
    const Line n = lineOf(a, sequence<kKind>(a, s));
    return lengthBefore(n, n.tiles) * a.kv_heads;
  };
  // Lengths of kThreads sequences and their sums up to each thread's.
  long long mine = 0, at = 0, total = 0;
  auto scan = [&](int s0) -> long long {
    mine = lengthOf(s0 + tid);
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) sm.scan[warp] = upto;
    __syncthreads();
    long long all = 0;
    at = upto - mine;
#pragma unroll 1
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += sm.scan[w];
      all += sm.scan[w];
    }
    return all;
  };
  for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) total += scan(s0);
  // Shares of kMinShare keys or more: none is empty, and a tile's cuts differ.
  const long long n_cta = max(1LL, min(static_cast<long long>(gridDim.x), total / kMinShare));
  const long long share = total / n_cta, rest = total - share * n_cta;
  auto shareBegin = [&](long long c) { return c >= n_cta ? total : c * share + min(c, rest); };
  const long long begin = shareBegin(blockIdx.x), end = shareBegin(blockIdx.x + 1LL);
  if (begin < end) {
    long long before = 0;
    for (int s0 = 0; s0 < a.n_seq && before <= begin; s0 += kThreads) {
      const long long all = a.n_seq > kThreads ? scan(s0) : total;  // one pass: still at hand
      if (begin >= before + at && begin < before + at + mine) {
        sm.found[0] = s0 + tid;
        sm.found[1] = before + at;
      }
      before += all;
    }
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  int* err = a.error_flag;
  // Layouts in shared memory.
  const bool q_planar = a.q.row_stride == 16;
  const bool k_planar = kKind != kPacked16 || a.k.row_stride == 16, v_planar = kKind != kPacked16 || a.v.row_stride == 16;

  if (warp >= 12) {
    if (warp == 12 || warp == 15) {
      // ---------------- MMA issue, a warp to each half ----------------
      auto uniform = [](int x) { return __reduce_max_sync(0xffffffffu, x); };  // the same in every lane, and known to be
      const int t = uniform(warp == 12 ? 0 : 1);
      const uint32_t idesc_o = idesc(kFmt, D, true);
      const Operand q_op = keyOperand(q_s + t * G::kTileBytes, q_planar), k_op = keyOperand(kv_s, k_planar), v_op = valueOperand(kv_s, v_planar);
      const uint32_t s_at = uniform(tmem) + t * kKeys, o_at = uniform(tmem) + kOCol + t * D;
      struct Cursor {
        int item, halves, jb, je, lim;  // the piece of work
        int j, block;                   // its next key block, that block's number in all
      };
      bool ok = true;
      auto release = [&](const Cursor& c) {
        __syncwarp();
        if (lane == 0) mbarArrive(&sm.item_empty[c.item % kItems]);
      };
      int tiles = 0, outputs = 0, done = 0;  // of this half: tiles begun, outputs begun, blocks done
      // Scores run one block ahead of the products with V, across pieces too.
      Cursor sc{}, pv{};
      bool ahead = false, fetch = true;
      for (;;) {
        if (fetch) {
          fetch = false;
          const int slot = sc.item % kItems;
          ok = wait(&sm.item_full[slot], (sc.item / kItems) & 1, sm, err, 55);
          if (!ok) break;
          const Item& it = sm.items[slot];
          sc.halves = uniform(it.halves);
          sc.jb = sc.j = uniform(it.jb);
          sc.je = uniform(it.je);
          sc.lim = uniform(it.lim);
          if (!ahead) pv = sc;
        }
        const bool scores = t < sc.halves;
        const int k_stage = (sc.block & 1) * 2, v_stage = (pv.block & 1) * 2 + 1;
        // All that the next scores need is waited for before P: their MMAs then
        // follow the products' at once (some 450 cycles of a block's 4,100).
        // The tensor core takes them in this order, so the scores may overwrite P.
        if (scores) {
          if (sc.j == sc.jb) {
            ok = wait(&sm.q_ready[t], tiles & 1, sm, err, 56);
            ++tiles;
          }
          if (ok) ok = wait(&sm.kv_ready[k_stage], (sc.block >> 1) & 1, sm, err, 57);
          if (!ok) break;
        }
        const int keys = min(kKeys, max(sc.lim - sc.j * kKeys, 1));
        const int steps = (min(kKeys, max(pv.lim - pv.j * kKeys, 1)) + 15) >> 4;
        const uint64_t v = v_op.desc + v_stage * (G::kTileBytes >> 4);
        if (ahead) {
          ok = wait(&sm.kv_ready[v_stage], (pv.block >> 1) & 1, sm, err, 57);
          if (ok && pv.j == pv.jb) {
            if (outputs > 0) ok = wait(&sm.o_free[t], (outputs - 1) & 1, sm, err, 59);
            ++outputs;
          }
          if (ok) ok = wait(&sm.p_half[t], done & 1, sm, err, 58);
          if (!ok) break;
          tcFenceAfter();
          if (electOne()) {
            issueValues<0>(o_at, s_at, v, v_op.step, idesc_o, steps, pv.j > pv.jb);
            commit(&sm.pv_half[t]);
          }
          __syncwarp();
          ok = wait(&sm.p_full[t], done & 1, sm, err, 58);
          if (!ok) break;
        }
        if (ahead || scores) {
          tcFenceAfter();
          if (electOne()) {
            if (ahead) {
              issueValues<4>(o_at, s_at, v, v_op.step, idesc_o, steps, true);
              commit(&sm.pv_done[t]);
              commit(&sm.kv_empty[v_stage]);
            }
            if (scores) {
              issueScores<D>(s_at, q_op, k_op.desc + k_stage * (G::kTileBytes >> 4), k_op.step, idesc(kFmt, (keys + 15) & ~15, false));
              commit(&sm.s_full[t]);
              commit(&sm.kv_empty[k_stage]);
              if (sc.j + 1 == sc.je) commit(&sm.q_empty[t]);
            }
          }
          __syncwarp();
          if (ahead) {
            ++done;
            ++pv.block;
            if (++pv.j == pv.je) {
              release(pv);
              pv = sc;  // the next piece, already fetched and not begun
            }
          }
          if (scores) {
            ++sc.block;
            if (++sc.j == sc.je) {
              ++sc.item;
              fetch = true;
            }
          }
          ahead = scores;
        } else if (sc.halves < 0) {
          release(sc);
          ++sc.item;
          fetch = true;
        } else if (sc.halves > 0) {  // no rows here: the keys are the other half's
          for (; sc.j < sc.je && ok; ++sc.j, ++sc.block) {
            for (int side = 0; side < 2 && ok; ++side) {
              const int stage = (sc.block & 1) * 2 + side;
              ok = wait(&sm.kv_ready[stage], (sc.block >> 1) & 1, sm, err, 57);
              __syncwarp();
              if (ok && lane == 0) mbarArrive(&sm.kv_empty[stage]);
            }
          }
          if (!ok) break;
          release(sc);
          ++sc.item;
          fetch = true;
        } else {
          break;
        }
      }
      // Everything issued has completed before TMEM and shared memory go.
      __syncwarp();
      if (electOne()) commit(&sm.drained[t]);
      __syncwarp();
      if (lane == 0) drainBar(&sm.drained[t], 0);
      __syncwarp();
    } else if (warp == 13) {
      // ---------------- the walk ----------------
      int seq = static_cast<int>(sm.found[0]), head = 0, tile = 0;
      long long at = end;  // of the tile; a CTA without a share is at its end already
      Sequence q{};
      Line line{};
      if (begin < end) {
        q = sequence<kKind>(a, seq);
        line = lineOf(a, q);
        const long long head_length = lengthBefore(line, line.tiles);
        at = sm.found[1];
        while (begin - at >= head_length) {
          at += head_length;
          ++head;
        }
        tile = tileAt(line, begin - at);
        at += lengthBefore(line, tile);
      } else if (lane == 0) {
        cuts[blockIdx.x].tile_at = -1;
        cuts[blockIdx.x].failed = 0;
      }
      const int snap = static_cast<int>(min(share / kSnap, 0x7fffffffLL));
      bool first = true;
      auto nextItem = [&](Item& it) {
        it.halves = 0;
        while (it.halves == 0) {
          if (!first) {
            at += tileLength(line, tile);
            ++tile;
          }
          if (at >= end) return;
          if (tile >= line.tiles) {
            tile = 0;
            if (++head >= a.kv_heads) {
              head = 0;
              do {  // at < end: a sequence with rows follows
                q = sequence<kKind>(a, ++seq);
                line = lineOf(a, q);
              } while (line.tiles == 0);
            }
          }
          const int length = tileLength(line, tile);
          it.lim = tileLimit(a, q, tile);
          const int blocks = blocksOf(it.lim);
          it.jb = begin <= at ? 0 : cutBlock(static_cast<int>(begin - at), length, blocks, snap);
          it.je = end >= at + length ? blocks : cutBlock(static_cast<int>(end - at), length, blocks, snap);
          if (first && lane == 0) {
            Cut cut{};
            cut.tile_at = it.jb > 0 && it.jb < blocks ? at : -1;
            cut.jb = it.jb;
            cut.blocks = blocks;
            cut.seq = seq;
            cut.head = head;
            cut.tile = tile;
            cuts[blockIdx.x] = cut;
          }
          first = false;
          if (it.jb >= it.je) continue;
          it.seq = seq;
          it.head = head;
          it.tile = tile;
          it.q0 = q.q0;
          it.nq = q.nq;
          it.k0 = q.k0;
          it.nk = q.nk;
          it.halves = q.nq * a.group - tile * kTileRows > kHalf ? 2 : 1;
          it.part = it.jb == 0 && it.je == blocks ? -1 : 2 * static_cast<int>(blockIdx.x) + (it.jb > 0 ? 0 : 1);
        }
      };
      // Items published and looked at once they are done: a causal item that asks
      // for it is done a second time. So the walk waits for the last ones; an empty
      // item lets the MMA warps finish them, who look one item ahead.
      int i = 0, looked = 0, empty = -1;
      bool more = true;
      for (;;) {
        Item it{};
        bool again = false;
        if (i - looked == kItems || looked < empty) {
          const int slot = looked % kItems;
          if (!wait(&sm.item_empty[slot], (looked / kItems) & 1, sm, err, 51)) break;
          ++looked;
          if (*const_cast<volatile int*>(&sm.redo[slot]) == 0) continue;
          it = sm.items[slot];
          again = true;
        } else if (more) {
          nextItem(it);
          more = it.halves > 0;
          if (!more && a.causal && i > 0) {
            it.halves = -1;
            empty = i;
          }
        }
        const int slot = i % kItems;
        __syncwarp();
        if (lane == 0) {
          sm.items[slot] = it;
          sm.again[slot] = again;
          sm.redo[slot] = 0;
          sm.hidden[slot] = 0;
          mbarArrive(&sm.item_full[slot]);
        }
        __syncwarp();
        if (it.halves == 0) break;
        ++i;
      }
    } else if (warp == 14) {
      // ---------------- fences ----------------
      // What has landed becomes visible to the tensor core, in the order of the loads.
      bool ok = true;
      int n = 0, used0 = 0, used1 = 0;  // key blocks, loads of Q's halves
      int table_item = -1;              // the last item that noted hidden values
      for (int i = 0; ok; ++i) {
        const int slot = i % kItems;
        ok = wait(&sm.item_full[slot], (i / kItems) & 1, sm, err, 52);
        if (!ok) break;
        const int halves = sm.items[slot].halves, blocks = sm.items[slot].je - sm.items[slot].jb;
        const bool again = halves > 0 && sm.again[slot] != 0;
        // In an item that is done again: values of the keys from `edge` on, which some
        // row of the tile does not see, are looked through.
        bool hidden = false;
        int edge = 0, lim = 0, key0 = 0;
        if (again) {
          const Item& it = sm.items[slot];
          edge = visible(a, Sequence{it.q0, it.nq, it.k0, it.nk}, it.tile * kTileRows / a.group);
          lim = it.lim;
          key0 = it.jb * kKeys;
        }
        __syncwarp();
        if (lane == 0) mbarArrive(&sm.item_empty[slot]);
        if (halves == 0) break;
        if (halves < 0) continue;
        // K, Q's halves, V, then K and V of each block.
        auto pass = [&](int x, auto&& look) {
          const bool is_q = x >= 1 && x <= halves;
          const int t = x - 1, y = is_q ? 0 : x > halves ? x - halves : x;  // y: 2 * block + side
          const int m = n + (y >> 1), stage = (m & 1) * 2 + (y & 1);
          ok = wait(is_q ? &sm.q_full[t] : &sm.kv_full[stage], (is_q ? (t == 0 ? used0 : used1) : m >> 1) & 1, sm, err, 60);
          if (ok && !is_q && (y & 1) == 1) look(y >> 1, kv_s + stage * G::kTileBytes);
          fenceProxyAsyncSmem();
          __syncwarp();
          if (ok && lane == 0) mbarArrive(is_q ? &sm.q_ready[t] : &sm.kv_ready[stage]);
        };
        if (!again) {
          for (int x = 0; x < 2 * blocks + halves && ok; ++x) pass(x, [](int, uint32_t) {});
        } else {
#pragma unroll 1
          for (int x = 0; x < 2 * blocks + halves && ok; ++x) {
            pass(x, [&](int block, uint32_t tile) {
              const int key = key0 + block * kKeys;
              if (!hasHidden<T, D>(tile, v_planar, key, edge, lim)) return;
              // The table is free once the softmax has let go of the item that used
              // it last, an earlier one, which waits for nothing of this one.
              if (!hidden && table_item >= 0 && i - table_item < kItems) {
                ok = wait(&sm.item_empty[table_item % kItems], (table_item / kItems) & 1, sm, err, 60);
              }
              if (ok) hideValues<T, D>(tile, v_planar, key, edge, lim, table, hidden);
              if (lane == 0) sm.hidden[slot] = 1;
              hidden = true;
              table_item = i;
            });
          }
        }
        n += blocks;
        ++used0;
        if (halves > 1) ++used1;
      }
    }
  } else if (warp >= 8) {
    // ---------------- loads ----------------
    constexpr int kWarpPlanes = kPlanes / kLoadWarps;  // planes of a warp where lanes take rows
    constexpr int kRowsAtOnce = 32 / kPlanes;          // rows of a warp's copy where lanes take planes
    constexpr int kRowStep = kLoadWarps * kRowsAtOnce;
    const int w = warp - 8;
    const int p_lane = lane % kPlanes;
    const int r_lane = w * kRowsAtOnce + lane / kPlanes;
    static_assert(kRowStep % 8 == 0, "a lane's rows have one place in the swizzle");
    // A lane's place in the swizzled layout: chunk p/8, row r, 16-byte column p%8 ^ r%8.
    const uint32_t put_rows = (p_lane >> 3) * kChunk + r_lane * 128 + (((p_lane & 7) ^ (r_lane & 7)) << 4);
    const int thread = w * 32 + lane;
    bool ok = true;
    int n = 0;             // key blocks so far
    int used[2] = {0, 0};  // times that Q's halves were loaded
    uint32_t in_flight = 0;  // by stage: this thread's last bulk copy, and the parity of its phase
    for (int i = 0; ok; ++i) {
      const int slot = i % kItems;
      ok = wait(&sm.item_full[slot], (i / kItems) & 1, sm, err, 52);
      if (!ok) break;
      const Item it = sm.items[slot];
      __syncwarp();
      if (lane == 0) mbarArrive(&sm.item_empty[slot]);
      if (it.halves == 0) break;
      if (it.halves < 0) continue;

      // Pages of a block: lane x holds that of its rows 16 x .. 16 x + 15.
      auto pagesOf = [&](int j) -> int {
        if constexpr (kKind == kPacked16) return 0;
        const int key = j * kKeys + lane * 16;
        return lane < kKeys / 16 && key < it.lim ? pageOf(a, it.seq, key) : 0;
      };
      int page_next = pagesOf(it.jb);

      // Q: rows r = token * group + g, counted from the tile's first token.
      const int row0 = it.tile * kTileRows;
      const int token0 = row0 / a.group;
      const int rest0 = row0 - token0 * a.group;
      const int rows = min(kTileRows, it.nq * a.group - row0);
      auto rowOf = [&](int rr, int p) -> const unsigned char* {
        const int x = rest0 + rr;  // below 256 + 128: the reciprocal's quotient is exact
        const int tok = (x * a.group_inv) >> 16;
        return record(a.q, it.head * a.group + x - tok * a.group, static_cast<long long>(it.q0) + token0 + tok, p);
      };
      auto loadQ = [&]() {
        for (int t = 0; t < it.halves && ok; ++t) {
          if (used[t] > 0) ok = wait(&sm.q_empty[t], (used[t] - 1) & 1, sm, err, 53);
          if (!ok) break;
          ++used[t];
          const uint32_t dst = q_s + t * G::kTileBytes;
          if (a.q.row_stride == 16) {
#pragma unroll 1
            for (int rr = 0; rr < kHalf; rr += 32) {
              const bool in = t * kHalf + rr + lane < rows;
              const unsigned char* src = rowOf(in ? t * kHalf + rr + lane : 0, w * kWarpPlanes);
#pragma unroll
              for (int p = 0; p < kWarpPlanes; ++p) {
                copyAsync16(dst + (w * kWarpPlanes + p) * kPlane + (rr + lane) * 16, src, in);
                src += a.q.plane_stride;
              }
            }
          } else {
#pragma unroll 1
            for (int rr = r_lane; rr < kHalf; rr += kRowStep) {
              const bool in = t * kHalf + rr < rows;
              copyAsync16(dst + put_rows + (rr - r_lane) * 128, rowOf(in ? t * kHalf + rr : 0, p_lane), in);
            }
          }
          copyArrive(&sm.q_full[t]);
        }
      };

      // e4m3: this thread's row of a tile, records and scale.
      uint4 next_codes[kPlanes / 2];
      float next_scale = 0.0f;
      bool next_in = false;
      auto fetch = [&](int j, int side, int page) {
        const fpk_heads_t& v = side == 0 ? a.k : a.v;
        const int r = (j * kKeys + thread) & ((1 << a.page_shift) - 1);
        next_in = j * kKeys + thread < it.lim && page >= 0;
        const unsigned char* src = static_cast<const unsigned char*>(v.data) + (next_in ? it.head * v.head_stride + page * a.page_stride + r * 16LL : 0);
#pragma unroll
        for (int p = 0; p < kPlanes / 2; ++p) {
          next_codes[p] = next_in ? *reinterpret_cast<const uint4*>(src + p * v.plane_stride) : make_uint4(0, 0, 0, 0);
        }
        const float* scales = side == 0 ? a.k_scale : a.v_scale;
        next_scale = next_in ? scales[((static_cast<long long>(page) * a.kv_heads + it.head) << a.page_shift) + r] : 0.0f;
      };
      if constexpr (kKind == kPagedE4m3) fetch(it.jb, 0, __shfl_sync(0xffffffffu, page_next, thread >> 4));

      for (int j = it.jb; j < it.je && ok; ++j, ++n) {
        const int page = page_next;
        if (j + 1 < it.je) page_next = pagesOf(j + 1);
        if (kKind != kPacked16 && page < 0) reportIndex(err, FPK_ERROR_PAGE);
        const int lim = it.lim - j * kKeys;  // rows of the block that somebody sees
        // Paged: rows of a page in the block, and the page of this thread's copy
        // (group `plane` of piece `piece`) and of its row.
        const int piece_rows = kKind == kPacked16 ? kKeys : min(1 << a.page_shift, kKeys);
        const int copy = lane * kLoadWarps + w;  // copies go round the warps, which issue them one by one
        const int plane = copy % kPlanes, piece = copy / kPlanes;
        const int page_copy = __shfl_sync(0xffffffffu, page, min(piece * piece_rows >> 4, 7));
        const int page_row = __shfl_sync(0xffffffffu, page, thread >> 4);
        for (int side = 0; side < 2 && ok; ++side) {
          // Q after the first keys: its room is free only after the last tile's last scores.
          if (side == 1 && j == it.jb) loadQ();
          if (!ok) break;
          const int stage = (n & 1) * 2 + side;
          const uint32_t dst = kv_s + stage * G::kTileBytes;
          const fpk_heads_t& v = side == 0 ? a.k : a.v;
          const unsigned char* data = static_cast<const unsigned char*>(v.data);
          if constexpr (kKind == kPagedE4m3) {
            // A thread to a row. The next tile's records are on their way while
            // this one's are converted.
            uint4 codes[kPlanes / 2];
            const float scale = next_scale;
            const bool in = next_in;
#pragma unroll
            for (int p = 0; p < kPlanes / 2; ++p) codes[p] = next_codes[p];
            const int page_after = __shfl_sync(0xffffffffu, side == 0 ? page : page_next, thread >> 4);
            if (side == 0 || j + 1 < it.je) fetch(j + side, 1 - side, page_after);
            if (n >= 2) ok = wait(&sm.kv_empty[stage], ((n >> 1) - 1) & 1, sm, err, 54);
            if (!ok) break;
            const FastScale<T> fast(scale);
            const bool usual = !in || (scale >= FastScale<T>::low && scale <= FastScale<T>::high);
#pragma unroll
            for (int p = 0; p < kPlanes / 2; ++p) {
              const uint2 x = fast(codes[p].x), y = fast(codes[p].y), z = fast(codes[p].z), w4 = fast(codes[p].w);
              storeShared16(dst + 2 * p * kPlane + thread * 16, make_uint4(x.x, x.y, y.x, y.y));
              storeShared16(dst + (2 * p + 1) * kPlane + thread * 16, make_uint4(z.x, z.y, w4.x, w4.y));
            }
#pragma unroll
            for (int p = 0; p < kPlanes / 2; ++p) {
              if (!usual || hasNan(codes[p])) storeRecord<T>(dst + 2 * p * kPlane + thread * 16, codes[p], scale);
            }
            mbarArrive(&sm.kv_full[stage]);
          } else {
            if (n >= 2) ok = wait(&sm.kv_empty[stage], ((n >> 1) - 1) & 1, sm, err, 54);
            if (!ok) break;
            if (side == 0 ? k_planar : v_planar) {
              if (kKind == kPaged16 && piece_rows < kBulkRows) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                  const int rr = c * 32 + lane;
                  const int pg = __shfl_sync(0xffffffffu, page, rr >> 4);
                  const bool yes = rr < lim && pg >= 0;
                  const unsigned char* src =
                      yes ? record(v, it.head, (j * kKeys + rr) & ((1 << a.page_shift) - 1), w * kWarpPlanes) + pg * a.page_stride : data;
#pragma unroll
                  for (int p = 0; p < kWarpPlanes; ++p) {
                    copyAsync16(dst + (w * kWarpPlanes + p) * kPlane + rr * 16, src, yes);
                    if (yes) src += v.plane_stride;
                  }
                }
                copyArrive(&sm.kv_full[stage]);
                continue;
              }
              // Keys that nobody sees, or on no page, have no values.
              if (side == 1 && (thread >= lim || (kKind != kPacked16 && page_row < 0))) {
#pragma unroll 1
                for (int p = 0; p < kPlanes; ++p) storeShared16(dst + p * kPlane + thread * 16, make_uint4(0, 0, 0, 0));
              }
              const int rows_in = min(lim - piece * piece_rows, piece_rows);
              if (piece * piece_rows < kKeys && rows_in > 0 && (kKind == kPacked16 || page_copy >= 0)) {
                const unsigned char* src;
                if constexpr (kKind == kPacked16) {
                  src = record(v, it.head, static_cast<long long>(it.k0) + j * kKeys, plane);
                } else {
                  src = record(v, it.head, (j * kKeys + piece * piece_rows) & ((1 << a.page_shift) - 1), plane) + page_copy * a.page_stride;
                }
                copyBulk(dst + plane * kPlane + piece * piece_rows * 16, src, rows_in * 16, &sm.kv_full[stage]);
                in_flight = (in_flight & ~(17u << stage)) | (1u << stage) | (((n >> 1) & 1u) << (stage + 4));
              } else {
                mbarArrive(&sm.kv_full[stage]);
              }
            } else {
              const long long step = kRowStep * v.row_stride;
              const unsigned char* src = record(v, it.head, static_cast<long long>(it.k0) + j * kKeys + r_lane, p_lane);
#pragma unroll 4
              for (int x = 0; x < kKeys / kRowStep; ++x) {
                const bool yes = r_lane + x * kRowStep < lim;
                copyAsync16(dst + put_rows + x * kRowStep * 128, yes ? src : data, yes);
                src += step;
              }
              copyArrive(&sm.kv_full[stage]);
            }
          }
        }
      }
    }
    copyDrain();
    // After an error bulk copies may still be under way (otherwise all were waited for).
    if (!ok) {
      for (int stage = 0; stage < kStages; ++stage) {
        if ((in_flight >> stage) & 1u) drainBar(&sm.kv_full[stage], (in_flight >> (stage + 4)) & 1u);
      }
    }
  } else {
    // ---------------- softmax and output ----------------
    const int t = warp >> 2;
    const int rr = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_base = lane_base + t * kKeys;
    const uint32_t o_base = lane_base + kOCol + t * D;
    bool ok = true;
    int count = 0;  // blocks of this half
    for (int i = 0; ok; ++i) {
      const int slot = i % kItems;
      ok = wait(&sm.item_full[slot], (i / kItems) & 1, sm, err, 55);
      if (!ok) break;
      const Item it = sm.items[slot];
      __syncwarp();
      if (it.halves == 0) break;
      if (t >= it.halves) {
        if (lane == 0) mbarArrive(&sm.item_empty[slot]);
        continue;
      }
      const Sequence q{it.q0, it.nq, it.k0, it.nk};
      const int row_first = it.tile * kTileRows + t * kHalf;
      const int r = row_first + rr;
      const bool valid = r < it.nq * a.group;
      const int token = valid ? r / a.group : 0;
      const int vis = valid ? visible(a, q, token) : it.nk;
      const int min_vis = visible(a, q, row_first / a.group);
      float m = -INFINITY, l = 0.0f;
      int page_next = 0;
      auto pagesOf = [&](int j) -> int {
        if constexpr (kKind == kPacked16) return 0;
        const int key = j * kKeys + lane * 16;
        return lane < kKeys / 16 && key < it.lim ? pageOf(a, it.seq, key) : 0;
      };
      page_next = pagesOf(it.jb);
      for (int j = it.jb; j < it.je && ok; ++j, ++count) {
        const uint32_t bad = kKind == kPacked16 ? 0u : __ballot_sync(0xffffffffu, page_next < 0);
        if (j + 1 < it.je) page_next = pagesOf(j + 1);
        ok = wait(&sm.s_full[t], count & 1, sm, err, 58);
        if (!ok) break;
        tcFenceAfter();
        // 64 scores at a time, which registers hold, each read once. (A pass for
        // the maximum of all 128 before it, with the halves taking turns at the
        // exponentials, took 162 us for crops and 549 for planar prompts in place
        // of 150 and 530.)
        const bool edge = (j + 1) * kKeys > min_vis || bad != 0;  // the causal edge, the last keys, bad pages
        const int lim = vis - j * kKeys;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t sv[64];
          FPB_TMEM_LD32(s_base + 64 * c, sv);
          FPB_TMEM_LD32(s_base + 64 * c + 32, (sv + 32));
          tmemWaitLd();
          if (edge) hide(sv, lim - 64 * c, bad >> (4 * c));
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 64; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
          const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * a.scale_log2;
          if (j == it.jb && c == 0) {
            m = top - kHeadLog2;
          } else if (__any_sync(0xffffffffu, top > m + kGrowLog2)) {
            const float m_new = top > m + kGrowLog2 ? top - kHeadLog2 : m;
            const float f = m_new == m ? 1.0f : exp2Approx(m - m_new);
            // O takes in the products of the 64 keys before these.
            ok = wait(c == 0 ? &sm.pv_done[t] : &sm.pv_half[t], (c == 0 ? count - 1 : count) & 1, sm, err, 59);
            if (!ok) break;
            tcFenceAfter();
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              uint32_t ov[16];
              FPB_TMEM_LD16(o_base + d, ov);
              tmemWaitLd();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * f);
              FPB_TMEM_ST16(o_base + d, ov);
            }
            tmemStoreWait();
            l *= f;
            m = m_new;
          }
          const float neg = m == -INFINITY ? 0.0f : -m;  // a row that has seen no key yet
          const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), neg2 = pair(neg, neg);
          uint64_t sum[2] = {0, 0};
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float2 x = unpair(fma2(pair(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), scale2, neg2));
            const float p0 = exp2Approx(x.x), p1 = exp2Approx(x.y);
            sum[e & 1] = add2(sum[e & 1], pair(p0, p1));
            pk[e] = pack2<T>(p0, p1);
          }
          FPB_TMEM_ST32(s_base + 32 * c, pk);
          const float2 part = unpair(add2(sum[0], sum[1]));
          l += part.x + part.y;
          // The first 64 keys go ahead to the tensor core.
          tmemStoreWait();
          tcFenceBefore();
          __syncwarp();
          if (lane == 0) mbarArrive(c == 0 ? &sm.p_half[t] : &sm.p_full[t]);
        }
        if (!ok) break;
      }
      const Item end = sm.items[i % kItems];  // read again: registers are short in the loop above
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int h = end.head * a.group + (valid ? r - token * a.group : 0);
      float* part_at = end.part >= 0 ? partials + static_cast<size_t>(end.part) * partialFloats(D) : nullptr;
      const int tile_row = t * kHalf + rr;
      if (ok) ok = wait(&sm.pv_done[t], (count - 1) & 1, sm, err, 59);
      if (!ok) break;
      tcFenceAfter();
      if (a.causal && *const_cast<volatile int*>(&sm.hidden[i % kItems]) != 0) addHidden<D>(o_base, table, vis);
      float top = 0.0f;  // NaN if one of O is
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t ov[32];
        __syncwarp();  // the load is one of a whole warp, and lanes without a row skip the stores
        FPB_TMEM_LD32(o_base + c, ov);
        tmemWaitLd();
        if (a.causal) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) top = max3Nan(top, __uint_as_float(ov[e]), __uint_as_float(ov[e + 1]));
        }
        if (valid && part_at == nullptr) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(ov[g * 8 + e]) * inv;
            // A row that saw no key: whatever V held, the sum is empty.
            if (l == 0.0f) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            }
            *reinterpret_cast<uint4*>(record(a.out, h, end.q0 + token, (c >> 3) + g)) = pack8<T>(x);
          }
        } else if (valid) {
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            reinterpret_cast<uint4*>(part_at)[((c >> 2) + g) * kTileRows + tile_row] =
                make_uint4(ov[4 * g], ov[4 * g + 1], ov[4 * g + 2], ov[4 * g + 3]);
          }
        }
      }
      if (part_at != nullptr && valid) {
        part_at[kTileRows * D + tile_row] = m;
        part_at[kTileRows * D + kTileRows + tile_row] = l;
      }
      // NaN may come from values that this row does not see (0 * v): the item is
      // done again without them.
      if (valid && top != top && vis < end.lim && sm.again[i % kItems] == 0) sm.redo[i % kItems] = 1;
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) {
        mbarArrive(&sm.o_free[t]);
        mbarArrive(&sm.item_empty[i % kItems]);  // only now: the table is read, and whether to do it again known
      }
    }
  }
  tcFenceBefore();
  __syncthreads();
  if (tid == 0 && (sm.stop != 0 || static_cast<int>(blockIdx.x) == a.test_fail)) cuts[blockIdx.x].failed = 1;
  if (warp == 12) {
    tcFenceAfter();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

constexpr int kJoinGroups = 1;  // groups of 8 channels of a joining thread
constexpr int kJoinAhead = 4;   // pieces that it reads at a time

// Joins the pieces of a tile: CTA c looks after the tile that share c begins
// inside, if it is the first share to. A thread joins kJoinGroups x 8 channels
// of a row; the pieces lie [channel][row], so a warp reads whole lines. The
// pieces are counted first, so that several are read at a time: 237 rows over
// 5,077 keys, 4 heads, 20 pieces to a tile, take 20 us with both launches, and 33
// with the pieces one after the other. Two groups to a thread: 21.
template <typename T, int D, KvKind kKind>
__global__ void __launch_bounds__(kTileRows) joinTilesKernel(const Args a, int n_cta) {
  __shared__ int jb_s[kTileCtas + 1];  // where the tile's pieces begin, and its end
  tc::pdlTrigger();
  tc::pdlWait();
  const Cut* cuts = reinterpret_cast<const Cut*>(a.workspace);
  const float* partials = reinterpret_cast<const float*>(a.workspace + sizeof(Cut) * kTileCtas);
  const int c = blockIdx.x;
  const Cut cut = cuts[c];
  if (c == 0 || cut.tile_at < 0 || cuts[c - 1].tile_at == cut.tile_at) return;
  const int row = threadIdx.x, grp = blockIdx.y * kJoinGroups;
  // Shares c + 1, ... that begin in the same tile: they follow one another.
  static_assert(kTileCtas <= kTileRows, "a thread to each share");
  const int d = c + 1 + row;
  const bool same = d < n_cta && cuts[d].tile_at == cut.tile_at;
  if (same) jb_s[row + 1] = cuts[d].jb;
  const bool failed = (same && cuts[d].failed != 0) || (row == 0 && (cut.failed != 0 || cuts[c - 1].failed != 0));
  const int more = __syncthreads_count(same);
  if (row == 0) {
    jb_s[0] = cut.jb;
    jb_s[more + 1] = cut.blocks;
  }
  if (__syncthreads_or(failed)) return;  // a piece is missing: the tile is not stored
  const Sequence q = sequence<kKind>(a, cut.seq);
  const int r = cut.tile * kTileRows + row;
  if (r >= q.nq * a.group) return;
  float m = -INFINITY, l = 0.0f, x[kJoinGroups][8] = {};
  for (int p0 = 0; p0 <= more + 1; p0 += kJoinAhead) {
    float4 y[kJoinAhead][kJoinGroups][2];
    float pm[kJoinAhead], pl[kJoinAhead], top = m;
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      // Piece 0 is the last of CTA c - 1, piece p the first of CTA c + p - 1, unless that is empty.
      const int n = p0 + i;
      const bool in = n == 0 || (n <= more + 1 && jb_s[n] > jb_s[n - 1]);
      const float* p = partials + static_cast<size_t>(n == 0 || !in ? 2 * (c - 1) + 1 : 2 * (c + n - 1)) * partialFloats(D);
#pragma unroll
      for (int g = 0; g < kJoinGroups; ++g) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          y[i][g][z] = in ? reinterpret_cast<const float4*>(p)[(2 * (grp + g) + z) * kTileRows + row] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
      pm[i] = in ? p[kTileRows * D + row] : -INFINITY;
      pl[i] = in ? p[kTileRows * D + kTileRows + row] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) top = fmaxf(top, pm[i]);
    const float keep = m == top ? 1.0f : exp2Approx(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int g = 0; g < kJoinGroups; ++g) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[g][e] *= keep;
    }
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const float w = pm[i] == m ? 1.0f : exp2Approx(pm[i] - m);
      l = fmaf(pl[i], w, l);
#pragma unroll
      for (int g = 0; g < kJoinGroups; ++g) {
        const float z[8] = {y[i][g][0].x, y[i][g][0].y, y[i][g][0].z, y[i][g][0].w, y[i][g][1].x, y[i][g][1].y, y[i][g][1].z, y[i][g][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[g][e] = fmaf(z[e], w, x[g][e]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int token = r / a.group;
  const int h = cut.head * a.group + r - token * a.group;
#pragma unroll
  for (int g = 0; g < kJoinGroups; ++g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[g][e] = l == 0.0f ? 0.0f : x[g][e] * inv;
    *reinterpret_cast<uint4*>(record(a.out, h, q.q0 + token, grp + g)) = pack8<T>(x[g]);
  }
}

long long tilesWorkspaceBytes(int head_dim) {
  return static_cast<long long>(sizeof(Cut) * kTileCtas + 2 * kTileCtas * partialFloats(head_dim) * sizeof(float) + kTileCtas * 2 * head_dim * sizeof(int));
}

namespace {

template <typename T, int D, KvKind kKind>
cudaError_t launchOne(const Args& a, cudaStream_t s) {
  static DeviceOnce smem_attr;
  static DeviceValue sms;
  cudaError_t e = smem_attr.run([] {
    return cudaFuncSetAttribute(attentionTilesKernel<T, D, kKind>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Geo<D>::kSmem));
  });
  if (e != cudaSuccess) return e;
  const int ctas = sms.get([](int dev) {
    int n = kTileCtas;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return std::min(n, kTileCtas);
  });
  prof::countLaunch(prof::kAttention, 2);
  e = launchPdl(attentionTilesKernel<T, D, kKind>, dim3(ctas), dim3(kThreads), Geo<D>::kSmem, s, a);
  if (e != cudaSuccess) return e;
  return launchPdl(joinTilesKernel<T, D, kKind>, dim3(ctas, D / 8 / kJoinGroups), dim3(kTileRows), 0, s, a, ctas);
}

template <typename T, int D>
cudaError_t launchKind(const Args& a, KvKind kind, cudaStream_t s) {
  switch (kind) {
    case kPacked16: return launchOne<T, D, kPacked16>(a, s);
    case kPaged16: return launchOne<T, D, kPaged16>(a, s);
    default: return launchOne<T, D, kPagedE4m3>(a, s);
  }
}

}  // namespace

cudaError_t launchTiles(const Args& a, KvKind kind, int head_dim, int dtype, cudaStream_t s) {
  if (dtype == FPK_DTYPE_BF16) {
    return head_dim == 64 ? launchKind<__nv_bfloat16, 64>(a, kind, s) : launchKind<__nv_bfloat16, 128>(a, kind, s);
  }
  return head_dim == 64 ? launchKind<__half, 64>(a, kind, s) : launchKind<__half, 128>(a, kind, s);
}

}  // namespace seqattn
}  // namespace fpb
