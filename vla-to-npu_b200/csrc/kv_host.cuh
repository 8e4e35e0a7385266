// Host side of the quantised key/value cache: argument checks, the choice of
// row tile and key splits, launches.
#pragma once
#include <cmath>

#include "host_common.cuh"
#include "kv_attention.cuh"
#include "kv_attention_tc.cuh"
#include "kvcache.cuh"

namespace vla {
namespace kv {

constexpr float kLog2e = 1.4426950408889634f;

static size_t block_bytes(int bits) {
  return bits == 4 ? (size_t)Block<4>::kBytes : bits == 8 ? (size_t)Block<8>::kBytes : 0;
}

static int check_cache(const vla_kv_cache* c, const char* what) {
  VLA_CHECK_ARG(c != nullptr, "%s: null cache", what);
  VLA_CHECK_ARG(c->bits == 4 || c->bits == 8, "%s: a cache holds 4 or 8 bits, not %d", what, c->bits);
  VLA_CHECK_ARG(c->head_dim == HD, "%s: head_dim must be 64", what);
  VLA_CHECK_ARG(c->batch >= 0 && c->kv_heads > 0 && c->pages >= 0 && c->max_pages >= 0, "%s: bad cache shape", what);
  // a block's first row may lie 255 positions before the first key, and its window starts below that
  VLA_CHECK_ARG((long long)c->max_pages * kPage <= (1ll << 31) - 512, "%s: %d pages per sequence are over 2^31 - 512 tokens",
                what, c->max_pages);
  VLA_CHECK_ARG(c->table_ld >= c->max_pages, "%s: table stride %lld below its %d columns", what,
                (long long)c->table_ld, c->max_pages);
  VLA_CHECK_ARG(c->batch == 0 || (c->pool != nullptr && c->table != nullptr), "%s: null pool or table", what);
  VLA_CHECK_ALIGN(aligned16(c->pool), "%s: the pool must be 16-byte aligned", what);
  return VLA_OK;
}

static Cache device_cache(const vla_kv_cache* c) {
  return Cache{(uint8_t*)c->pool, c->table, (long long)c->table_ld, c->pages, c->max_pages, c->batch, c->kv_heads};
}

// Row tensors [batch][n] of kv_heads * 64 (or heads * 64) elements.
static int check_rows(const void* x, int64_t row, int64_t batch, int64_t width, const char* what, const char* name) {
  VLA_CHECK_ARG(x != nullptr, "%s: null %s", what, name);
  VLA_CHECK_ARG(row >= width && batch >= 0, "%s: %s rows of stride %lld hold %lld elements", what, name,
                (long long)row, (long long)width);
  VLA_CHECK_ALIGN(aligned16(x) && row % 8 == 0 && batch % 8 == 0, "%s: 16-byte alignment of %s and its strides", what,
                  name);
  return VLA_OK;
}

// Output rows: no element may have two writers.  Sequences lie one after the
// other, or (rows of all sequences, then the next row of all) within a row's stride.
static int check_apart(const vla_kv_cache* c, int64_t n, int64_t row, int64_t batch, int64_t width, const char* what,
                       const char* name) {
  const int64_t b = c->batch - 1;
  VLA_CHECK_ARG(b == 0 || (batch >= width && (batch - width) / row >= n - 1) ||
                    (batch >= width && (row - width) / batch >= b),
                "%s: sequences of %s overlap: %lld rows of %lld elements, strides %lld and %lld", what, name,
                (long long)n, (long long)width, (long long)row, (long long)batch);
  return VLA_OK;
}

// Whether four groups of positions per warp leave a warp for each of the SMs' 64 places.
static bool wide_rows(const vla_kv_cache* c, int quads) {
  return (long long)c->batch * c->kv_heads * ((quads + 3ll) / 4) >= 64ll * device_info().num_sms;
}

#define VLA_TRY(expr)                \
  do {                               \
    const int _rc = (expr);          \
    if (_rc != VLA_OK) return _rc;   \
  } while (0)

static int append(const vla_kv_cache* c, const void* k, int64_t k_row, int64_t k_batch, const void* v, int64_t v_row,
                  int64_t v_batch, int32_t n, const int32_t* start, const int32_t* count, cudaStream_t st) {
  VLA_TRY(check_cache(c, "kv_append"));
  VLA_CHECK_ARG(n >= 0, "kv_append: n must not be negative");
  if (c->batch == 0 || n == 0) return VLA_OK;
  VLA_CHECK_ARG(start != nullptr, "kv_append: null start");
  const int64_t width = (int64_t)c->kv_heads * HD;
  VLA_TRY(check_rows(k, k_row, k_batch, width, "kv_append", "k"));
  VLA_TRY(check_rows(v, v_row, v_batch, width, "kv_append", "v"));
  AppendParams p{device_cache(c), (const bf16*)k, (const bf16*)v, (long long)k_row, (long long)v_row,
                 (long long)k_batch, (long long)v_batch, start, count, n, (int)(((long long)n + 6) / 4)};
  const bool many = wide_rows(c, p.quads);
  const long long items = ((long long)p.quads + (many ? 3 : 0)) / (many ? 4 : 1) * c->kv_heads;
  VLA_CHECK_ARG(items < (1ll << 31) - 8, "kv_append: too many rows");
  const dim3 grid((unsigned)((items + 7) / 8), c->batch < 65535 ? c->batch : 65535);
  prof_begin(st);
  launch_k(c->bits == 4 ? (many ? append_kernel<4, 4> : append_kernel<4, 1>)
                        : (many ? append_kernel<8, 4> : append_kernel<8, 1>),
           grid, dim3(256), 0, st, p);
  prof_end(st, VLA_KIND_LAYOUT, 0.0,
           (double)c->batch * n * c->kv_heads * (4.0 * HD + (double)block_bytes(c->bits) / kPage));
  return launch_status("kv_append");
}

static int read(const vla_kv_cache* c, void* k, int64_t k_row, int64_t k_batch, void* v, int64_t v_row,
                int64_t v_batch, int32_t n, const int32_t* start, const int32_t* count, cudaStream_t st) {
  VLA_TRY(check_cache(c, "kv_read"));
  VLA_CHECK_ARG(n >= 0, "kv_read: n must not be negative");
  if (c->batch == 0 || n == 0) return VLA_OK;
  const int64_t width = (int64_t)c->kv_heads * HD;
  VLA_TRY(check_rows(k, k_row, k_batch, width, "kv_read", "k"));
  VLA_TRY(check_rows(v, v_row, v_batch, width, "kv_read", "v"));
  VLA_TRY(check_apart(c, n, k_row, k_batch, width, "kv_read", "k"));
  VLA_TRY(check_apart(c, n, v_row, v_batch, width, "kv_read", "v"));
  VLA_CHECK_ARG(k != v, "kv_read: k and v are one output");
  ReadParams p{device_cache(c), (bf16*)k, (bf16*)v, (long long)k_row, (long long)v_row, (long long)k_batch,
               (long long)v_batch, start, count, n, (int)(((long long)n + 6) / 4),
               c->bits == 4 ? code_mask<4>() : code_mask<8>()};
  const bool many = wide_rows(c, p.quads);
  const long long items = ((long long)p.quads + (many ? 3 : 0)) / (many ? 4 : 1) * c->kv_heads;
  VLA_CHECK_ARG(items < (1ll << 31) - 8, "kv_read: too many rows");
  const dim3 grid((unsigned)((items + 7) / 8), c->batch < 65535 ? c->batch : 65535);
  prof_begin(st);
  launch_k(c->bits == 4 ? (many ? read_kernel<4, 4> : read_kernel<4, 1>)
                        : (many ? read_kernel<8, 4> : read_kernel<8, 1>),
           grid, dim3(256), 0, st, p);
  prof_end(st, VLA_KIND_LAYOUT, 0.0,
           (double)c->batch * n * c->kv_heads * (4.0 * HD + (double)block_bytes(c->bits) / kPage));
  return launch_status("kv_read");
}

// Row tile, split and workspace of a call; they depend on its sizes alone.
struct Plan {
  int nt;          // 8-row tiles of the mma.sync kernel, 0: the tcgen05 kernel
  int block, row_blocks, split;  // rows of a block, blocks per (sequence, kv head)
  int slots;       // rows of a part in the workspace
  size_t workspace;
};

template <int BITS, int NT>
static int resident_ctas() {
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& n = cached[dev & 63];
  if (n.load(std::memory_order_relaxed) == 0) {
    constexpr int smem = attend_smem<BITS, NT>();
    int per = 0;
    if (cudaFuncSetAttribute(attend_kernel<BITS, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaFuncSetAttribute(attend_kernel<BITS, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, attend_kernel<BITS, NT, false>, kWarps * 32, smem) != cudaSuccess ||
        per < 1) {
      cudaGetLastError();  // no device: sizes are still answered
      return 4 * device_info().num_sms;
    }
    n.store(per * device_info().num_sms, std::memory_order_relaxed);
  }
  return n.load(std::memory_order_relaxed);
}
static int resident_ctas(int bits, int nt) {
  if (bits == 4) return nt == 1 ? resident_ctas<4, 1>() : nt == 2 ? resident_ctas<4, 2>() : resident_ctas<4, 4>();
  return nt == 1 ? resident_ctas<8, 1>() : nt == 2 ? resident_ctas<8, 2>() : resident_ctas<8, 4>();
}

static int plan_attention(const vla_kv_cache* c, const vla_kv_attention_args* a, Plan* out) {
  const long long rows = (long long)a->Lq * (a->Hq / c->kv_heads);
  VLA_CHECK_ARG(rows < (1ll << 30), "kv_attention: too many query rows");
  const int G = a->Hq / c->kv_heads;
  // Few rows to mma.sync, by the least tile that holds them; above 32 to tcgen05, whose
  // blocks of 256 rows take nearly the same time however few are filled.  Both sides of the
  // border (us, 5 kv heads, 4 bits): 32 rows over 64 x 8000 keys 124 here and 250 there, 17
  // rows over 256 x 113 keys 45 and 42 (8 bits 42 and 43); in blocks of 32, 33 rows over 256
  // x 113 keys would take 78 and take 43 there, over 64 x 8000 keys 211 and 265, 96 rows 310
  // and 271.
  out->nt = rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 32 ? 4 : 0;
  const int block = out->nt > 0 ? 8 * out->nt : tc::kRows;
  const long long blocks = (rows + block - 1) / block;
  const long long room = (long long)c->max_pages * kPage;
  long long keys = a->max_len > 0 && a->max_len < room ? a->max_len : room;
  if (a->window > 0) {
    // the window of a block's rows and the first tokens, in whole pages
    const long long seen = (long long)a->window + a->sinks + (block - 1) / G + 3 * kUnit;
    if (seen < keys) keys = seen;
  }
  VLA_CHECK_ARG(c->batch * blocks * c->kv_heads <= ((1ll << 31) - 1) / (c->max_pages > 0 ? c->max_pages : 1) && c->batch * rows * c->kv_heads < (1ll << 31),
                "kv_attention: too many work items");
  out->block = block;
  out->slots = out->nt > 0 ? block : tc::kRows;
  out->row_blocks = (int)blocks;
  out->split = keys > 8 * kUnit;
  const size_t ctas = !out->split ? 0 : out->nt == 0 ? device_info().num_sms : resident_ctas(c->bits, out->nt);
  out->workspace = ctas * (2 * out->slots * (HD + 2) * sizeof(float) + sizeof(int4));
  return VLA_OK;
}

static int check_attention(const vla_kv_cache* c, const vla_kv_attention_args* a) {
  VLA_TRY(check_cache(c, "kv_attention"));
  VLA_CHECK_ARG(a != nullptr, "kv_attention: null args");
  VLA_CHECK_ARG(a->Lq >= 0 && a->Hq > 0 && a->Hq % c->kv_heads == 0, "kv_attention: %d query heads over %d kv heads",
                a->Hq, c->kv_heads);
  VLA_CHECK_ARG(a->window >= 0 && a->sinks >= 0 && a->max_len >= 0, "kv_attention: negative window, sinks or max_len");
  VLA_CHECK_ARG(std::isfinite(a->scale * kLog2e) && a->scale > 0.f,
                "kv_attention: scale (times log2 e) must be positive and finite");
  return VLA_OK;
}

template <int BITS, int NT>
static void launch_attend(const AttnParams& p, cudaStream_t st) {
  constexpr int smem = attend_smem<BITS, NT>();
  const int ctas = resident_ctas<BITS, NT>();
  const int items = p.c.batch * p.row_blocks * p.c.kv_heads;
  launch_k(p.split ? attend_kernel<BITS, NT, false> : attend_kernel<BITS, NT, true>, dim3(p.split ? ctas : items),
           dim3(kWarps * 32), smem, st, p);
  if (p.split) {  // a CTA per row that is there
    const int slices = p.row_blocks > 1 ? 8 * NT : p.Lq * p.G;
    launch_k(join_kernel<8 * NT, kJoinWarps>, dim3(slices, ctas), dim3(kJoinWarps * 32), 0, st, p, p.scale_log2);
  }
}

template <int BITS>
static int launch_tc(const AttnParams& p, cudaStream_t st) {
  constexpr int smem = tc::smem_bytes<BITS>();
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    VLA_CUDA_TRY(cudaFuncSetAttribute(tc::attend_kernel<BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaFuncAttributes fa{};
    VLA_CUDA_TRY(cudaFuncGetAttributes(&fa, tc::attend_kernel<BITS>));
    // setmaxnreg hands out exactly the launch's registers: only sound at the count it was sized for
    if (fa.numRegs != tc::kLaunchRegs)
      return set_error(VLA_E_CUDA, "kv_attention: built with %d registers per thread, sized for %d", fa.numRegs,
                       tc::kLaunchRegs);
    ready.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const int ctas = device_info().num_sms;
  launch_k(tc::attend_kernel<BITS>, dim3(ctas), dim3(tc::kThreads), smem, st, p);
  if (p.split) {
    const int slices = ((p.row_blocks > 1 ? p.block : p.Lq * p.G) + kJoinWarps - 1) / kJoinWarps;
    launch_k(join_kernel<tc::kRows, 1>, dim3(slices, ctas), dim3(kJoinWarps * 32), 0, st, p, 1.f);
  }
  return VLA_OK;
}

static size_t attention_workspace(const vla_kv_cache* c, const vla_kv_attention_args* a) {
  Plan pl;
  if (check_attention(c, a) != VLA_OK || c->batch == 0 || a->Lq == 0) return 0;
  return plan_attention(c, a, &pl) == VLA_OK ? pl.workspace : 0;
}

static int attention(const vla_kv_cache* c, const vla_kv_attention_args* a, cudaStream_t st) {
  VLA_TRY(check_attention(c, a));
  if (c->batch == 0 || a->Lq == 0) return VLA_OK;
  VLA_CHECK_ARG(a->lens != nullptr, "kv_attention: null lens");
  VLA_TRY(check_rows(a->q, a->q_row, a->q_batch, (int64_t)a->Hq * HD, "kv_attention", "q"));
  VLA_TRY(check_rows(a->o, a->o_row, a->o_batch, (int64_t)a->Hq * HD, "kv_attention", "o"));
  VLA_TRY(check_apart(c, a->Lq, a->o_row, a->o_batch, (int64_t)a->Hq * HD, "kv_attention", "o"));
  Plan pl;
  VLA_TRY(plan_attention(c, a, &pl));
  if (pl.workspace > 0) {
    if (a->workspace == nullptr || a->workspace_bytes < pl.workspace)
      return set_error(VLA_E_WORKSPACE, "kv_attention: needs %zu bytes of workspace, got %zu", pl.workspace,
                       a->workspace == nullptr ? (size_t)0 : a->workspace_bytes);
    VLA_CHECK_ALIGN(aligned16(a->workspace), "kv_attention: workspace alignment");
  }
  AttnParams p{};
  p.c = device_cache(c);
  p.q = (const bf16*)a->q;
  p.o = (bf16*)a->o;
  p.q_row = a->q_row;
  p.q_batch = a->q_batch;
  p.o_row = a->o_row;
  p.o_batch = a->o_batch;
  p.lens = a->lens;
  p.q_len = a->q_len;
  p.Lq = a->Lq;
  p.G = a->Hq / c->kv_heads;
  p.causal = a->causal != 0;
  // a window as long as the cache hides nothing, and first tokens mean nothing without one
  const long long room = (long long)c->max_pages * kPage;
  p.window = a->window > 0 && a->window < room ? a->window : 0;
  p.sinks = a->sinks < room ? a->sinks : (int)room;
  p.scale_log2 = a->scale * kLog2e;
  p.mask = c->bits == 4 ? code_mask<4>() : code_mask<8>();
  p.block = pl.block;
  p.row_blocks = pl.row_blocks;
  p.split = pl.split;
  p.part_o = (float*)a->workspace;
  if (pl.split) {
    const size_t rows = pl.workspace / (2 * pl.slots * (HD + 2) * sizeof(float) + sizeof(int4)) * 2 * pl.slots;
    p.part_ml = p.part_o + rows * HD;
    p.cut = reinterpret_cast<int4*>(p.part_ml + rows * 2);
  }
  prof_begin(st);
  if (pl.nt == 0) {
    VLA_TRY(c->bits == 4 ? launch_tc<4>(p, st) : launch_tc<8>(p, st));
  } else if (c->bits == 4) {
    if (pl.nt == 1) launch_attend<4, 1>(p, st);
    else if (pl.nt == 2) launch_attend<4, 2>(p, st);
    else launch_attend<4, 4>(p, st);
  } else {
    if (pl.nt == 1) launch_attend<8, 1>(p, st);
    else if (pl.nt == 2) launch_attend<8, 2>(p, st);
    else launch_attend<8, 4>(p, st);
  }
  // the lengths are on the device: the profile counts whole caches (or windows)
  const double keys = a->window > 0 && a->window < room ? (double)a->window + a->sinks : (double)room;
  prof_end(st, VLA_KIND_ATTENTION, 4.0 * c->batch * a->Hq * (double)a->Lq * keys * HD,
           c->batch * (keys * c->kv_heads * block_bytes(c->bits) / kPage + 4.0 * a->Lq * a->Hq * HD));
  return launch_status("kv_attention");
}

}  // namespace kv
}  // namespace vla
