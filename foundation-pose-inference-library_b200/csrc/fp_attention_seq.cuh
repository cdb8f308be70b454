// What the two kernels behind fpk_attention_packed and fpk_attention_paged
// share: the descriptor as the device sees it, a sequence's rows, and where its
// keys lie. fp_attention_stream.cu serves few query rows (decoding), bound by
// the keys' bytes; fp_attention_tiles.cu many (prompts, chunks), bound by the
// tensor cores; fp_attention_seq.cu checks the descriptors and chooses.
//
// Both order the query rows of one sequence and key head as r = token * group +
// g (g: the query heads that share the key head), and tile r. All of a tile's
// rows then read the same keys, whatever the group.
#pragma once

#include "fp_heads.cuh"

namespace fpb {
namespace seqattn {

using namespace heads;

enum KvKind { kPacked16, kPaged16, kPagedE4m3 };

struct Args {
  fpk_heads_t q, out;
  fpk_heads_t k, v;           // packed: rows [kv_rows]; paged: one page's strides
  const float* k_scale;       // e4m3
  const float* v_scale;
  const int32_t* q_starts;
  const int32_t* kv_starts;   // packed
  const int32_t* kv_lengths;  // paged
  const int32_t* page_table;
  long long page_stride;      // bytes of one page, all heads
  int table_pages, n_pages, page_shift;
  int n_seq, q_rows, kv_rows, kv_heads, group;
  int group_inv;              // ceil(2^16 / group): x * group_inv >> 16 = x / group for x * group < 2^16
  int causal;
  float scale_log2;           // scale * log2(e)
  int* error_flag;
  unsigned char* workspace;
  int test_fail;              // tile kernel: this CTA counts as one whose wait ran out (tests), else -1
};

struct Sequence {
  int q0, nq;  // first query row, query rows
  int k0, nk;  // first key row (packed), keys
};

// Rows of sequence s, clamped to the buffers.
template <KvKind kKind>
__device__ __forceinline__ Sequence sequence(const Args& a, int s) {
  Sequence q;
  const int b0 = a.q_starts[s], b1 = a.q_starts[s + 1];
  q.q0 = min(max(b0, 0), a.q_rows);
  const int q1 = min(max(b1, q.q0), a.q_rows);
  q.nq = q1 - q.q0;
  if (q.q0 != b0 || q1 != b1) reportIndex(a.error_flag, FPK_ERROR_STARTS);
  if constexpr (kKind == kPacked16) {
    const int c0 = a.kv_starts[s], c1 = a.kv_starts[s + 1];
    q.k0 = min(max(c0, 0), a.kv_rows);
    const int k1 = min(max(c1, q.k0), a.kv_rows);
    q.nk = k1 - q.k0;
    if (q.k0 != c0 || k1 != c1) reportIndex(a.error_flag, FPK_ERROR_STARTS);
  } else {
    const int n = a.kv_lengths[s];
    q.k0 = 0;
    q.nk = static_cast<int>(min(static_cast<long long>(max(n, 0)), static_cast<long long>(a.table_pages) << a.page_shift));
    if (q.nk != n) reportIndex(a.error_flag, FPK_ERROR_LENGTH);
  }
  return q;
}

// Keys that token i of a sequence sees: 0 .. visible - 1.
__device__ __forceinline__ int visible(const Args& a, const Sequence& q, int i) {
  if (!a.causal) return q.nk;
  return min(max(q.nk - q.nq + i + 1, 0), q.nk);
}

// Page of key `key` of sequence s, or -1 if the table holds no page there.
__device__ __forceinline__ int pageOf(const Args& a, int s, int key) {
  const int p = a.page_table[static_cast<long long>(s) * a.table_pages + (key >> a.page_shift)];
  return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages) ? p : -1;
}

// ---- launches ----

// Work that the launch helpers cannot see on the host (lengths live on the
// device) is bounded by these.
constexpr int kStreamCtas = 592;  // most CTAs of the streaming kernel: 4 on each of 148 SMs
constexpr int kStreamRows = 16;   // most query rows of its tile

constexpr int kTileCtas = 148;    // most CTAs of the tile kernel: one on each SM
constexpr int kTileRows = 256;    // query rows of its tile

long long streamWorkspaceBytes(int head_dim);
long long tilesWorkspaceBytes(int head_dim);
cudaError_t launchTiles(const Args& a, KvKind kind, int head_dim, int dtype, cudaStream_t s);
cudaError_t launchStream(const Args& a, KvKind kind, int head_dim, int dtype, cudaStream_t s);

}  // namespace seqattn
}  // namespace fpb
