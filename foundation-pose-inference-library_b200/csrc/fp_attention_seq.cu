// Host side of fpk_attention_packed and fpk_attention_paged (include/fpk.h):
// checks and the choice of the kernel.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "fp_attention_seq.cuh"

namespace fpb {
namespace seqattn {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// A CTA walks over sequences without rows one by one, some half a microsecond each,
// which the bounded waits (2 s) of those that it feeds have to outlast.
constexpr int kMostSequences = 1 << 20;
constexpr const char* kMisaligned = "starts, lengths, page_table and error_flag must be 4-byte aligned";

std::atomic<int> g_test_fail{-1};  // fpk_attention_test_fail_share

struct Shape {
  int q_heads, kv_heads, head_dim, n_seq, q_rows;
  long long keys;  // of a sequence: paged at most, packed four times the average
};

std::string shapeProblem(const Shape& n) {
  if (n.head_dim != 64 && n.head_dim != 128) return "head_dim must be 64 or 128";
  if (n.q_heads <= 0 || n.kv_heads <= 0 || n.q_heads % n.kv_heads || n.q_heads / n.kv_heads > 128 || n.q_heads > 65535) {
    return "q_heads must be a multiple of kv_heads, at most 128 to each";
  }
  if (n.n_seq < 0 || n.q_rows < 0) return "sizes must not be negative";
  if (n.n_seq > kMostSequences) return "at most 2^20 sequences";
  if (static_cast<long long>(n.q_rows) * (n.q_heads / n.kv_heads) + static_cast<long long>(n.n_seq) * 128 > kMost) {
    return "too many query rows (q_rows * q_heads / kv_heads + 128 * n_seq must be at most 2^31 - 1024)";
  }
  return std::string();
}

std::string scaleProblem(float scale) {
  // In the units of exp2 too.
  return scale >= 0.0f && std::isfinite(scale * kLog2e) ? std::string() : std::string("scale must be finite and not negative (at most 2^127)");
}

float scaleLog2(float scale, int head_dim) {
  return kLog2e * (scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(head_dim)));
}

// Which kernel, by what the host knows (lengths are on the device; either kernel
// is right for any). Rows are tokens x query heads to a key head, on average.
// Up to 16 rows are one tile of the streaming kernel, which reads the keys at
// the memory's rate; with more it reads them again for each 16 rows, while the
// tile kernel takes 256 at once but begins at some 18 us. Streaming against tiles
// (us, 8 key heads of 128, sequences x keys): 16 rows, 8 x 4000: 33 / 39, 8 x
// 16000: 86 / 113; 48 rows, 8 x 4000: 52 / 39; 64 rows, 1 x 600: 12.7 / 18.3, 8 x
// 600: 20 / 20, 1 x 4000: 22 / 21, 8 x 4000: 59 / 38; 128 rows, 1 x 600: 13.5 /
// 19.5, 8 x 600: 30 / 22, 1 x 4000: 28 / 22; 1,600 rows, 4 key heads, 1 x 400:
// 27 / 20.
constexpr int kStreamMostRows = kStreamRows;
constexpr int kStreamMostWork = 1 << 17;  // tiles of 16 rows x keys

bool useTiles(const Shape& n) {
  const long long rows = static_cast<long long>(n.q_rows) * (n.q_heads / n.kv_heads);  // below 2^31
  if (n.n_seq == 0 || rows <= static_cast<long long>(kStreamMostRows) * n.n_seq) return false;
  const double tiles = std::ceil(static_cast<double>(rows) / (static_cast<double>(kStreamRows) * n.n_seq)) * n.n_seq * n.kv_heads;
  return tiles * static_cast<double>(n.keys) > kStreamMostWork;
}

// Enough for either kernel: a workspace for one batch does for any other.
long long workspaceBytes(const Shape& n) { return std::max(tilesWorkspaceBytes(n.head_dim), streamWorkspaceBytes(n.head_dim)); }

int launch(const std::string& name, const Args& a, KvKind kind, const Shape& n, int dtype, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = useTiles(n) ? launchTiles(a, kind, n.head_dim, dtype, s) : launchStream(a, kind, n.head_dim, dtype, s);
  if (e != cudaSuccess) return fail(name + ": " + cudaGetErrorString(e));
  return 0;
}

std::string workspaceProblem(const void* p, long long have, long long need) {
  if (need > 0 && (p == nullptr || have < need)) return "workspace of " + std::to_string(need) + " bytes required";
  if (!aligned16(p)) return "workspace must be 16-byte aligned";
  return std::string();
}

Shape shapeOf(const fpk_attention_packed_desc_t& d) {
  const long long keys = d.n_seq > 0 ? std::min<long long>(d.kv_rows, 4LL * d.kv_rows / d.n_seq) : 0;
  return {d.q_heads, d.kv_heads, d.head_dim, d.n_seq, d.q_rows, keys};
}
Shape shapeOf(const fpk_attention_paged_desc_t& d) {
  const long long keys = static_cast<long long>(d.table_pages) * d.cache.page_rows;
  return {d.q_heads, d.cache.kv_heads, d.cache.head_dim, d.n_seq, d.q_rows, keys};
}

}  // namespace

}  // namespace seqattn
}  // namespace fpb

extern "C" long long fpk_attention_packed_workspace_bytes(const fpk_attention_packed_desc_t* d) {
  using namespace fpb::seqattn;
  return d == nullptr || !shapeProblem(shapeOf(*d)).empty() ? 0 : workspaceBytes(shapeOf(*d));
}

extern "C" long long fpk_attention_paged_workspace_bytes(const fpk_attention_paged_desc_t* d) {
  using namespace fpb::seqattn;
  return d == nullptr || !shapeProblem(shapeOf(*d)).empty() ? 0 : workspaceBytes(shapeOf(*d));
}

extern "C" int fpk_attention_packed(const fpk_attention_packed_desc_t* d, void* stream) {
  using namespace fpb;
  using namespace fpb::seqattn;
  const std::string name = "fpk_attention_packed";
  if (d == nullptr) return fail(name + ": null descriptor");
  if (!is16Bit(d->dtype)) return fail(name + ": dtype must be f16 or bf16");
  const Shape n = shapeOf(*d);
  std::string p = shapeProblem(n);
  if (p.empty()) p = scaleProblem(d->scale);
  if (p.empty() && d->kv_rows < 0) p = "sizes must not be negative";
  if (p.empty() && d->kv_rows > kMost) p = "kv_rows must be at most 2^31 - 1024";
  if (!p.empty()) return fail(name + ": " + p);
  if (d->n_seq == 0 || d->q_rows == 0) return 0;
  for (const fpk_heads_t* v : {&d->q, &d->out, &d->k, &d->v}) {
    if (d->kv_rows == 0 && (v == &d->k || v == &d->v)) continue;
    if (const char* q = headsProblem(*v)) return fail(name + ": " + q);
  }
  if (d->q_starts == nullptr || d->kv_starts == nullptr) return fail(name + ": q_starts and kv_starts are required");
  if (!aligned4(d->q_starts) || !aligned4(d->kv_starts) || !aligned4(d->error_flag)) return fail(name + ": " + kMisaligned);
  p = workspaceProblem(d->workspace, d->workspace_bytes, workspaceBytes(n));
  if (p.empty()) {
    const bool keys = d->kv_rows > 0;
    p = deviceProblem({d->q.data, d->out.data, keys ? d->k.data : nullptr, keys ? d->v.data : nullptr, d->q_starts, d->kv_starts,
                       d->error_flag, d->workspace});
  }
  if (!p.empty()) return fail(name + ": " + p);
  Args a{};
  a.q = d->q;
  a.out = d->out;
  a.k = d->k;
  a.v = d->v;
  a.q_starts = d->q_starts;
  a.kv_starts = d->kv_starts;
  a.n_seq = d->n_seq;
  a.q_rows = d->q_rows;
  a.kv_rows = d->kv_rows;
  a.kv_heads = d->kv_heads;
  a.group = d->q_heads / d->kv_heads;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.causal = d->causal != 0;
  a.scale_log2 = scaleLog2(d->scale, d->head_dim);
  a.error_flag = d->error_flag;
  a.workspace = static_cast<unsigned char*>(d->workspace);
  a.test_fail = g_test_fail.load();
  return launch(name, a, kPacked16, n, d->dtype, stream);
}

extern "C" int fpk_attention_paged(const fpk_attention_paged_desc_t* d, void* stream) {
  using namespace fpb;
  using namespace fpb::seqattn;
  const std::string name = "fpk_attention_paged";
  if (d == nullptr) return fail(name + ": null descriptor");
  if (!is16Bit(d->dtype)) return fail(name + ": dtype must be f16 or bf16");
  std::string p = cacheProblem(d->cache, d->dtype);
  const Shape n = shapeOf(*d);
  if (p.empty()) p = shapeProblem(n);
  if (p.empty()) p = scaleProblem(d->scale);
  if (p.empty() && d->table_pages < 0) p = "sizes must not be negative";
  if (p.empty() && n.keys > kMost) p = "table_pages * page_rows must be at most 2^31 - 1024";
  if (!p.empty()) return fail(name + ": " + p);
  if (d->n_seq == 0 || d->q_rows == 0) return 0;
  for (const fpk_heads_t* v : {&d->q, &d->out}) {
    if (const char* q = headsProblem(*v)) return fail(name + ": " + q);
  }
  if (d->q_starts == nullptr || d->kv_lengths == nullptr || (d->page_table == nullptr && d->table_pages > 0)) {
    return fail(name + ": q_starts, kv_lengths and page_table are required");
  }
  if (!aligned4(d->q_starts) || !aligned4(d->kv_lengths) || !aligned4(d->page_table) || !aligned4(d->error_flag)) {
    return fail(name + ": " + kMisaligned);
  }
  p = workspaceProblem(d->workspace, d->workspace_bytes, workspaceBytes(n));
  const fpk_kv_cache_t& c = d->cache;
  const bool e4m3 = c.dtype == FPK_DTYPE_E4M3;
  if (p.empty()) {
    p = deviceProblem({d->q.data, d->out.data, c.k, c.v, e4m3 ? c.k_scale : nullptr, e4m3 ? c.v_scale : nullptr, d->q_starts, d->kv_lengths,
                       d->table_pages > 0 ? d->page_table : nullptr, d->error_flag, d->workspace});
  }
  if (!p.empty()) return fail(name + ": " + p);
  Args a{};
  a.q = d->q;
  a.out = d->out;
  const long long plane = static_cast<long long>(c.page_rows) * 16;
  const long long head = plane * (c.head_dim / (e4m3 ? 16 : 8));
  a.k = {c.k, head, 16, plane};
  a.v = {c.v, head, 16, plane};
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  a.page_stride = head * c.kv_heads;
  a.n_pages = c.n_pages;
  while ((1 << a.page_shift) < c.page_rows) ++a.page_shift;
  a.q_starts = d->q_starts;
  a.kv_lengths = d->kv_lengths;
  a.page_table = d->page_table;
  a.table_pages = d->table_pages;
  a.n_seq = d->n_seq;
  a.q_rows = d->q_rows;
  a.kv_heads = c.kv_heads;
  a.group = d->q_heads / c.kv_heads;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.causal = d->causal != 0;
  a.scale_log2 = scaleLog2(d->scale, c.head_dim);
  a.error_flag = d->error_flag;
  a.workspace = static_cast<unsigned char*>(d->workspace);
  a.test_fail = g_test_fail.load();
  return launch(name, a, e4m3 ? kPagedE4m3 : kPaged16, n, d->dtype, stream);
}

extern "C" int fpk_attention_test_fail_share(int share) { return fpb::seqattn::g_test_fail.exchange(share < 0 ? -1 : share); }
