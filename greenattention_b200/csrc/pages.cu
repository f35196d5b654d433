// C ABI of the pages' upkeep (kv_pages.cuh): argument checks and launches.
#include "../../include/green_attention.h"
#include "api_internal.h"
#include "kv_pages.cuh"

namespace {

using ga::api::fail;
using namespace ga::pages;

struct Call {
  PoolDev d;
  cudaStream_t st;
  int sm;
};

constexpr int kMaxRows = 32768;  // entries of one fork / grow call: their prefix sums lie in shared memory
constexpr int kMaxPages = 0x7fffffff - 2 * SPAN;  // a kernel's running page, a span further, is still an int

size_t up(size_t n) { return (n + 255) / 256 * 256; }

int fill(const GaPagePool* a, void* stream, Call* c) {
  int dev;
  if (ga::api::device(&dev, &c->sm)) return 1;
  if (!a) return fail("null pool");
  if (a->tensors <= 0 || a->chunks <= 0 || a->num_pages <= 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1)))
    return fail("pool of %d tensors, %d chunks, %d pages of %d tokens", a->tensors, a->chunks, a->num_pages, a->page_size);
  if (a->num_pages > kMaxPages) return fail("%d pages, at most %d", a->num_pages, kMaxPages);
  if (a->rows < 0 || a->cols < 0) return fail("page table of %d x %d", a->rows, a->cols);
  if (!a->base || !a->page_stride || !a->tok_bytes || !a->chunk_tensor || !a->chunk_first || !a->page_table || !a->seqlens ||
      !a->refs || !a->status)
    return fail("null tensor pointer");
  PoolDev& d = c->d;
  std::memset(&d, 0, sizeof(d));
  d.base = reinterpret_cast<const unsigned long long*>(a->base);
  d.stride = reinterpret_cast<const long long*>(a->page_stride);
  d.tok_bytes = a->tok_bytes;
  d.chunk_tensor = a->chunk_tensor;
  d.chunk_first = a->chunk_first;
  d.tensors = a->tensors, d.chunks = a->chunks;
  d.num_pages = a->num_pages, d.page_size = a->page_size, d.page_shift = __builtin_ctz(a->page_size);
  d.table = a->page_table;
  d.t_s0 = a->pt_stride_row, d.t_s1 = a->pt_stride_col;
  d.rows = a->rows, d.cols = a->cols;
  d.lens = a->seqlens;
  d.refs = a->refs;
  d.status = a->status;
  c->st = static_cast<cudaStream_t>(stream);
  return 0;
}

int scratch_of(const GaPagePool* a, size_t need, uint8_t** out) {
  if (!a->scratch || a->scratch_bytes < need) return fail("scratch too small: %zu < %zu bytes", a->scratch_bytes, need);
  if (reinterpret_cast<uintptr_t>(a->scratch) % 256) return fail("scratch must be 256-byte aligned");
  *out = static_cast<uint8_t*>(a->scratch);
  return 0;
}

// CTAs of a copy kernel for at most so many pieces.
unsigned copy_grid(long long items, int sm) {
  const long long most = static_cast<long long>(COPY_CTAS) * sm;
  return static_cast<unsigned>(items < most ? (items > 0 ? items : 1) : most);
}

size_t copy_bytes(int pages, int n) { return up(static_cast<size_t>(pages) * 4) + up(static_cast<size_t>(n) * 8); }
size_t fork_bytes(int rows, int n) { return up(static_cast<size_t>(rows) * 4) + up(static_cast<size_t>(n) * 16) + up(static_cast<size_t>(n) * 4); }
int spans_of(int pages) { return (pages + SPAN - 1) / SPAN; }
size_t compact_bytes(int pages) { return up(static_cast<size_t>(spans_of(pages)) * 4) + 2 * up(static_cast<size_t>(pages) * 4) + 256; }

int release(const GaPagePool* a, const void* rows, int is64, int n, int evict, int window, int sinks, void* stream) {
  Call c;
  if (fill(a, stream, &c)) return 1;
  if (n < 0 || n > kMaxRows || (n > 0 && !rows)) return fail("rows: at most %d entries", kMaxRows);
  ga::api::launches(n > 0);
  if (n == 0) return 0;
  GA_TRY(ga::api::launch_serial(release_kernel, dim3(n), dim3(256), 0, c.st, c.d, rows, is64, n, evict, window, sinks));
  return 0;
}

}  // namespace

int ga::api::init_pages() {
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(grow_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRows * 4));
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(fork_plan_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRows * 4));
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(copy_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, COPY_SMEM));
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(fork_apply_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, COPY_SMEM));
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(compact_apply_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, COPY_SMEM));
  return 0;
}

extern "C" {

size_t ga_pages_scratch_bytes(const GaPagePool* a, int n) {
  if (!a || n < 0) return 0;
  size_t most = copy_bytes(a->num_pages, n);
  if (fork_bytes(a->rows, n) > most) most = fork_bytes(a->rows, n);
  if (compact_bytes(a->num_pages) > most) most = compact_bytes(a->num_pages);
  return most;
}

int ga_pages_copy(const GaPagePool* a, const void* src, const void* dst, int is64, int n, void* stream) {
  Call c;
  if (fill(a, stream, &c)) return 1;
  if (n < 0 || (n > 0 && (!src || !dst))) return fail("src / dst");
  ga::api::launches(n > 0 ? 2 : 0);
  if (n == 0) return 0;
  uint8_t* s;
  if (scratch_of(a, copy_bytes(c.d.num_pages, n), &s)) return 1;
  int* mark = reinterpret_cast<int*>(s);
  int2* list = reinterpret_cast<int2*>(s + up(static_cast<size_t>(c.d.num_pages) * 4));
  GA_TRY(ga::api::launch_serial(copy_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, c.st, c.d, src, dst, is64, n, mark, list));
  GA_TRY(ga::api::launch_serial(copy_kernel, dim3(copy_grid(static_cast<long long>(n) * c.d.chunks, c.sm)), dim3(COPY_THREADS), COPY_SMEM, c.st,
                                c.d, const_cast<const int2*>(list), n));
  return 0;
}

int ga_pages_free(const GaPagePool* a, const void* rows, int is64, int n, void* stream) {
  return release(a, rows, is64, n, 0, 0, 0, stream);
}

int ga_pages_evict(const GaPagePool* a, const void* rows, int is64, int n, int window_left, int sink_tokens, void* stream) {
  if (window_left < 0 || sink_tokens < 0) return fail("window_left %d, sink_tokens %d", window_left, sink_tokens);
  return release(a, rows, is64, n, 1, window_left, sink_tokens, stream);
}

int ga_pages_grow(const GaPagePool* a, const void* rows, const void* lens, int is64, int lens64, int n, void* stream) {
  Call c;
  if (fill(a, stream, &c)) return 1;
  if (n < 0 || n > kMaxRows || (n > 0 && (!rows || !lens))) return fail("rows / lens: at most %d entries", kMaxRows);
  ga::api::launches(n > 0);
  if (n == 0) return 0;
  uint8_t* s;
  if (scratch_of(a, fork_bytes(c.d.rows, 0), &s)) return 1;
  GA_TRY(ga::api::launch_serial(grow_kernel, dim3(1), dim3(PLAN_THREADS), static_cast<size_t>(n) * 4, c.st, c.d, rows, lens, is64, lens64,
                                n, reinterpret_cast<int*>(s)));
  return 0;
}

int ga_pages_fork(const GaPagePool* a, const void* parents, const void* children, int is64, int n, void* stream) {
  Call c;
  if (fill(a, stream, &c)) return 1;
  if (n < 0 || n > kMaxRows || (n > 0 && (!parents || !children))) return fail("parents / children: at most %d entries", kMaxRows);
  ga::api::launches(n > 0 ? 2 : 0);
  if (n == 0) return 0;
  uint8_t* s;
  if (scratch_of(a, fork_bytes(c.d.rows, n), &s)) return 1;
  int4* list = reinterpret_cast<int4*>(s + up(static_cast<size_t>(c.d.rows) * 4));
  int* ends = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(list) + up(static_cast<size_t>(n) * 16));
  if (static_cast<long long>(n) * c.d.chunks > 0x7fffffffLL) return fail("%d forks of %d pieces a page", n, c.d.chunks);
  GA_TRY(ga::api::launch_serial(fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), static_cast<size_t>(n) * 4, c.st, c.d, parents, children,
                                is64, n, reinterpret_cast<int*>(s), list, ends));
  GA_TRY(ga::api::launch_serial(fork_apply_kernel, dim3(copy_grid(n + static_cast<long long>(n) * c.d.chunks, c.sm)), dim3(COPY_THREADS),
                                COPY_SMEM, c.st, c.d, parents, children, is64, n, const_cast<const int4*>(list), const_cast<const int*>(ends)));
  return 0;
}

int ga_pages_compact(const GaPagePool* a, int32_t* map, int32_t* live, void* stream) {
  Call c;
  if (fill(a, stream, &c)) return 1;
  if (!map || !live) return fail("map / live");
  const int pages = c.d.num_pages, spans = spans_of(pages);
  uint8_t* s;
  if (scratch_of(a, compact_bytes(pages), &s)) return 1;
  int* moved = reinterpret_cast<int*>(s);
  int* counts = reinterpret_cast<int*>(s + 256);
  int* movers = reinterpret_cast<int*>(s + 256 + up(static_cast<size_t>(spans) * 4));
  int* gaps = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(movers) + up(static_cast<size_t>(pages) * 4));
  if (spans > 1)
    GA_TRY(ga::api::launch_serial(compact_count_kernel, dim3(spans), dim3(PLAN_THREADS), 0, c.st, c.d, counts));
  GA_TRY(ga::api::launch_serial(compact_rank_kernel, dim3(spans), dim3(PLAN_THREADS), 0, c.st, c.d, const_cast<const int*>(counts), map,
                                movers, gaps, live, moved));
  const long long bound = c.d.rows + static_cast<long long>(pages / 2) * c.d.chunks;
  GA_TRY(ga::api::launch_serial(compact_apply_kernel, dim3(copy_grid(bound, c.sm)), dim3(COPY_THREADS), COPY_SMEM, c.st, c.d, map,
                                const_cast<const int*>(movers), const_cast<const int*>(gaps), const_cast<const int*>(moved)));
  ga::api::launches(spans > 1 ? 3 : 2);
  return 0;
}

}  // extern "C"
