// C ABI of the attention over 16-bit and e4m3 paged caches with first tokens kept visible (attn_paged.cuh): argument
// checks, choice of the instance, launches.
#include <algorithm>
#include <mutex>
#include <vector>

#include "../../include/green_attention.h"
#include "api_internal.h"
#include "attn_paged.cuh"
#include "attn_paged_tc.cuh"

namespace {

using ga::api::fail;
using ga::paged::PagedDev;

struct Launch {
  PagedDev d;
  cudaStream_t st;
  int sm;
  long long max_tokens;  // keys a page-table row can address
  bool prompt;
};

size_t prefix_bytes(int batch) { return (static_cast<size_t>(batch) + 1 + 63) / 64 * 256; }
size_t slots_bytes(int sm) {
  return (static_cast<size_t>(2 * sm) * (ga::paged::SLOT_FLOATS + ga::paged::SLOT_ROWS) + static_cast<size_t>(sm) * (ga::paged::SEG_FLOATS + 1)) * 4;
}

template <class I>
int limits() {
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(ga::paged::attn_paged_kernel<I, 0>),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, I::SMEM));
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(ga::paged::attn_paged_kernel<I, 1>),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, I::SMEM));
  return 0;
}

// Tensor maps of paged pools [pages, page, kv_heads, head_dim] of 16-bit values, dimensions as (dim, token, head, page), for
// boxes of 64 dims x `box` tokens. A map is a function of its key; the few last ones are kept.
struct MapKey {
  const void* base;
  long long s_page, s_tok, s_head;
  int pages, page, kvh, hd, box, pad;
};
struct MapEntry {
  MapKey key;
  CUtensorMap map;
};
std::mutex g_maps_mu;
std::vector<MapEntry> g_maps;

bool pool_map(const MapKey& key, CUtensorMap* out) {
  std::lock_guard<std::mutex> lock(g_maps_mu);
  for (const MapEntry& e : g_maps)
    if (std::memcmp(&e.key, &key, sizeof(MapKey)) == 0) {
      *out = e.map;
      return true;
    }
  MapEntry e;
  std::memset(&e, 0, sizeof(e));
  e.key = key;
  if (!ga::api::encode_map(&e.map, key.base, key.hd, key.page, key.kvh, key.pages, key.s_tok, key.s_head, key.s_page, key.box)) return false;
  if (g_maps.size() >= 64) g_maps.erase(g_maps.begin());
  g_maps.push_back(e);
  *out = e.map;
  return true;
}

// Whether an instance of the tensor-core kernel was built with the registers that its split between the roles draws on. Where
// a compiler gave it fewer its calls go to the warp-level kernel, and the rest of the library is not concerned.
template <class I>
bool g_tc_built = false;

template <class I>
int limits_tc() {
  cudaFuncAttributes at;
  GA_TRY(cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(ga::paged::tc::attn_paged_tc_kernel<I>)));
  g_tc_built<I> = at.numRegs >= I::REGS;
  if (!g_tc_built<I>) return 0;
  GA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(ga::paged::tc::attn_paged_tc_kernel<I>),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, I::SMEM));
  return 0;
}

// Maps of the call's K and V pools; false: the tensor-core kernel gathers without them.
template <class I>
bool pool_maps(const PagedDev& d, CUtensorMap (&maps)[2]) {
  std::memset(maps, 0, sizeof(maps));
  const int page = d.page_mask + 1;
  if (page < 8 || d.num_pages <= 0 || I::KV == ga::paged::KV_E4M3) return false;
  MapKey kk, vk;
  std::memset(&kk, 0, sizeof(kk));
  kk.base = d.k, kk.s_page = d.k_s0, kk.s_tok = d.k_s1, kk.s_head = d.k_s2;
  kk.pages = d.num_pages, kk.page = page, kk.kvh = d.kvh, kk.hd = I::HD;
  kk.box = page < ga::paged::tc::GK ? page : ga::paged::tc::GK;
  vk = kk;
  vk.base = d.v, vk.s_page = d.v_s0, vk.s_tok = d.v_s1, vk.s_head = d.v_s2;
  return pool_map(kk, &maps[0]) && pool_map(vk, &maps[1]);  // not for strides that a map cannot hold
}

// What the tensor-core kernel takes: its query rows go through 16-byte copies, and it takes the maximum before the scale
// (a k_descale comes with e4m3 caches, where the queries can take its sign).
template <class I>
bool tc_takes(const PagedDev& d) {
  const bool e4m3 = I::KV == ga::paged::KV_E4M3;
  const int el = e4m3 && d.q_kind == ga::paged::Q_SAME ? 1 : 2;
  return g_tc_built<I> && (!d.kd || e4m3) && d.scale_log2 > 0.f && d.q_s0 * el % 16 == 0 && d.q_s1 * el % 16 == 0 && reinterpret_cast<uintptr_t>(d.q) % 16 == 0;
}

// Enough CTAs to spread the rows of a small call over the SMs.
unsigned combine_shares(long long pairs, int rows, int sm) {
  const long long z = (2LL * sm + pairs - 1) / pairs;
  return static_cast<unsigned>(z < 1 ? 1 : (z > rows ? rows : z));
}

// Whether a call of at most 128 rows per kv head goes to the tensor-core kernel in slices. Both sides measured (bf16,
// device time, warp-level kernel / tensor-core kernel): 32 x 8192 tokens, 8 kv heads, head_dim 128: 16 rows 176 / 190 us,
// 20 rows 294 / 194, 128 rows (8 requests) 297 / 80; head_dim 64: 20 rows 145 / 215, 64 rows 44 / 35 (8 x 2000);
// head_dim 256 (32 x 4096): 2 rows 265 / 174, 20 rows 527 / 183; pages of one token (32 x 4096), 20 rows: 161 / 201; 4 x 300
// tokens, head_dim 256: 27 / 28, both bound by the host. So: where the warp-level kernel would read the keys more than once (over 32 rows, 16 at
// head_dim 256); at head_dim 128 from 17 rows and at 256 always, if pages are whole boxes and the call is not a small one.
// An e4m3 cache is converted on the way into the stages, which costs more than reading it again a few times (16 x 8192
// tokens: head_dim 128 64 rows 260 / 384 us, 128 rows 475 / 403; head_dim 256 64 rows 564 / 886, 128 rows 1088 / 911; head_dim
// 64 64 rows 143 / 223, 128 rows 266 / 233): from 65 rows on.
template <int KV>
bool split_on_tensor_cores(const Launch& a, int hd) {
  const long long rows = static_cast<long long>(a.d.max_q) * a.d.gqa;
  if (rows > ga::paged::tc::TM) return false;
  if (rows > (KV == ga::paged::KV_E4M3 ? 64 : (hd == 256 ? 16 : 32))) return true;
  const double most_bytes = 4.0 * a.d.batch * a.max_tokens * a.d.kvh * hd;
  return KV != ga::paged::KV_E4M3 && a.d.page_mask >= 7 && most_bytes >= 8e6 && (hd == 256 || (hd == 128 && rows > 16));
}

// Verify on the tensor cores (at most 128 rows of a kv head): gangs of kv_heads CTAs, slices of the requests' tiles, and the
// combine kernel; -1: the call is not one for it.
template <class I>
int run_tc_split(Launch& a) {
  PagedDev& d = a.d;
  if (!tc_takes<I>(d) || d.kvh > a.sm) return -1;
  CUtensorMap maps[2];
  const bool boxes = pool_maps<I>(d, maps);
  const int gangs = a.sm / d.kvh;
  d.nrb = 1;
  int4* list = reinterpret_cast<int4*>(d.ws_lse + static_cast<size_t>(2 * a.sm) * ga::paged::tc::TM);
  static_assert(ga::paged::SLOT_ROWS >= ga::paged::tc::TM + 16 && I::HD * ga::paged::tc::TM <= ga::paged::SLOT_FLOATS &&
                    I::SOFT_WARPS * 32 <= ga::paged::SEG_FLOATS, "workspace");
  GA_TRY(ga::api::launch_serial(ga::paged::tc::plan_split_kernel<I>, dim3(1), dim3(1024), 0, a.st, d, gangs, list));
  GA_TRY(ga::api::launch_serial(ga::paged::tc::attn_paged_tc_kernel<I>, dim3(gangs * d.kvh), dim3(I::NT), I::SMEM, a.st, d,
                                static_cast<const int*>(nullptr), const_cast<const int4*>(list), maps[0], maps[1], static_cast<int>(boxes)));
  const int rows = d.max_q * d.gqa;
  GA_TRY(ga::api::launch_serial(ga::paged::attn_paged_combine<I>, dim3(d.batch, d.kvh, combine_shares(static_cast<long long>(d.batch) * d.kvh, rows, a.sm)),
                                dim3(128), 0, a.st, d, gangs));
  ga::api::launches(3);
  return 0;
}

// Prompts on the tensor cores; -1: the call is not one for them.
template <class I>
int run_tc(Launch& a) {
  PagedDev& d = a.d;
  if (!tc_takes<I>(d)) return -1;
  const long long blocks = static_cast<long long>(d.total_q) * d.gqa / I::ROWS + d.batch;
  // the list in front, O of the segments before (one slot a CTA) in the back half of the slots
  float* room = d.ws_o + static_cast<size_t>(a.sm) * ga::paged::SLOT_FLOATS;
  static_assert(I::ROWS * I::HD <= ga::paged::SLOT_FLOATS && I::SOFT_WARPS * 32 <= ga::paged::SEG_FLOATS, "workspace");
  const size_t need = 256 + static_cast<size_t>(blocks) * 16;
  if (need > static_cast<size_t>(reinterpret_cast<uint8_t*>(room) - reinterpret_cast<uint8_t*>(d.prefix)) || blocks * d.kvh > 0x7fffffffLL) return -1;
  d.ws_o = room;
  int* count = d.prefix;
  int4* list = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(d.prefix) + 256);
  const long long items = blocks * d.kvh;
  CUtensorMap maps[2];
  const bool boxes = pool_maps<I>(d, maps);
  GA_TRY(ga::api::launch_serial(ga::paged::tc::plan_prompts_kernel<I::ROWS>, dim3(1), dim3(1024), 0, a.st, d, count, list,
                                static_cast<int>(blocks)));
  GA_TRY(ga::api::launch_serial(ga::paged::tc::attn_paged_tc_kernel<I>, dim3(static_cast<unsigned>(items < a.sm ? items : a.sm)), dim3(I::NT),
                                I::SMEM, a.st, d, const_cast<const int*>(count), const_cast<const int4*>(list), maps[0], maps[1],
                                static_cast<int>(boxes)));
  ga::api::launches(2);
  return 0;
}

template <class I>
int run(Launch& a) {
  PagedDev& d = a.d;
  static_assert(I::NW * I::RC * I::HD <= ga::paged::SLOT_FLOATS && I::NW * I::RC <= ga::paged::SLOT_ROWS, "slot");
  if (d.kvh > a.sm * I::NW) return fail("%d kv heads: more than a gang can hold", d.kvh);
  const long long rows = static_cast<long long>(d.max_q) * d.gqa;
  if (a.prompt) {
    // a request of n tokens has ceil(n * gqa / RC) row blocks
    const long long blocks = static_cast<long long>(d.total_q) * d.gqa / I::RC + d.batch;
    const long long grid = (blocks * d.kvh + I::NW - 1) / I::NW;
    if (grid > 0x7fffffffLL || blocks > 0x7fffffffLL) return fail("too many row blocks");
    d.nrb = 1;
    GA_TRY(cudaMemsetAsync(d.ws_spoilt, 0, 4, a.st));
    GA_TRY(ga::api::launch_serial(ga::paged::attn_paged_kernel<I, 1>, dim3(static_cast<unsigned>(grid)), dim3(I::NT), I::SMEM, a.st, d));
    GA_TRY(ga::api::launch_serial(ga::paged::attn_paged_mend<I::KV, I::HD, I::RC>, dim3(a.sm), dim3(128), 0, a.st, d));
    ga::api::launches(2);
    return 0;
  }
  d.nrb = static_cast<int>((rows + I::RC - 1) / I::RC);
  const long long units = static_cast<long long>(d.batch) * d.nrb;
  if (units > 0x7fffffffLL) return fail("too many (request, row block) units");
  const long long tiles = units * ((a.max_tokens + I::T - 1) / I::T);  // at most, of each kv head
  const long long want = (tiles * d.kvh + I::NW - 1) / I::NW;
  const int least = (d.kvh + I::NW - 1) / I::NW;
  const int grid = static_cast<int>(want < least ? least : (want < a.sm ? want : a.sm));
  GA_TRY(ga::api::launch_serial(ga::paged::attn_paged_kernel<I, 0>, dim3(grid), dim3(I::NT), I::SMEM, a.st, d));
  const int block_rows = rows < I::RC ? static_cast<int>(rows) : I::RC;
  const unsigned z = combine_shares(units * d.kvh, block_rows, a.sm);
  GA_TRY(ga::api::launch_serial(ga::paged::attn_paged_combine<I>, dim3(static_cast<unsigned>(units), d.kvh, z), dim3(128), 0, a.st, d,
                                grid * I::NW / d.kvh));
  ga::api::launches(2);
  return 0;
}

template <int KV>
int run_tc_kv(Launch& a, int hd) {
  using namespace ga::paged::tc;
  if (hd == 64) return run_tc<TcInst<64, KV, false>>(a);
  if (hd == 128) return run_tc<TcInst<128, KV, false>>(a);
  return run_tc<TcInst<256, KV, false>>(a);
}

template <int KV>
int run_tc_split_kv(Launch& a, int hd) {
  using namespace ga::paged::tc;
  if (hd == 64) return run_tc_split<TcInst<64, KV, true>>(a);
  if (hd == 128) return run_tc_split<TcInst<128, KV, true>>(a);
  return run_tc_split<TcInst<256, KV, true>>(a);
}

template <int KV>
int run_kv(Launch& a, int hd) {
  using namespace ga::paged;
  const long long rows = static_cast<long long>(a.d.max_q) * a.d.gqa;
  if (hd == 64) return a.prompt || rows > 16 ? run<Inst<64, KV, 2>>(a) : run<Inst<64, KV, 1>>(a);
  if (hd == 128) return a.prompt || rows > 16 ? run<Inst<128, KV, 2>>(a) : run<Inst<128, KV, 1>>(a);
  return run<Inst<256, KV, 1>>(a);
}

template <int KV>
int route(Launch& a, int hd) {
  int rc = -1;
  if (split_on_tensor_cores<KV>(a, hd)) rc = run_tc_split_kv<KV>(a, hd);
  else if (a.prompt) rc = run_tc_kv<KV>(a, hd);
  return rc >= 0 ? rc : run_kv<KV>(a, hd);
}

template <int KV>
int limits_tc_kv() {
  using namespace ga::paged::tc;
  return limits_tc<TcInst<64, KV, true>>() || limits_tc<TcInst<128, KV, true>>() || limits_tc<TcInst<256, KV, true>>() ||
         limits_tc<TcInst<64, KV, false>>() || limits_tc<TcInst<128, KV, false>>() || limits_tc<TcInst<256, KV, false>>();
}

template <int KV>
int limits_kv() {
  using namespace ga::paged;
  return limits<Inst<64, KV, 1>>() || limits<Inst<64, KV, 2>>() || limits<Inst<128, KV, 1>>() ||
         limits<Inst<128, KV, 2>>() || limits<Inst<256, KV, 1>>();
}

}  // namespace

int ga::api::init_paged() {
  return limits_kv<ga::paged::KV_BF16>() || limits_kv<ga::paged::KV_FP16>() || limits_kv<ga::paged::KV_E4M3>() ||
         limits_tc_kv<ga::paged::KV_BF16>() || limits_tc_kv<ga::paged::KV_FP16>() || limits_tc_kv<ga::paged::KV_E4M3>();
}

extern "C" {

size_t ga_paged_workspace_bytes(int device, int max_batch) {
  const int sm = ga_sm_count(device);
  return prefix_bytes(max_batch) + slots_bytes(sm > 0 ? sm : 160);
}

int ga_paged_attend(const GaPagedParams* a, void* stream) {
  Launch l;
  int dev;
  if (ga::api::device(&dev, &l.sm)) return 1;
  if (!a) return fail("null params");
  if (a->kv_type < 0 || a->kv_type > 2) return fail("kv_type %d", a->kv_type);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return fail("head_dim %d: only 64, 128 and 256 are built", a->head_dim);
  if (a->kv_heads <= 0 || a->q_heads <= 0 || a->q_heads % a->kv_heads) return fail("q_heads %d / kv_heads %d", a->q_heads, a->kv_heads);
  if (a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return fail("page_size %d is not a power of two", a->page_size);
  if (a->batch <= 0 || a->num_pages < 0 || a->pt_cols < 0) return fail("batch %d, num_pages %d, pt_cols %d", a->batch, a->num_pages, a->pt_cols);
  if (a->total_q < 0 || a->total_q > 0x7fffffffLL) return fail("total_q %lld", (long long)a->total_q);
  if (a->max_seqlen_q < 1) return fail("max_seqlen_q %d", a->max_seqlen_q);
  if (a->sink_tokens < 0) return fail("sink_tokens %d", a->sink_tokens);
  if (a->total_q * (a->q_heads / a->kv_heads) > 0x7fffffffLL) return fail("%lld query rows of a kv head", (long long)a->total_q * (a->q_heads / a->kv_heads));
  if (a->total_q == 0) {
    ga::api::launches(0);
    return 0;
  }
  if (!a->q || !a->k_cache || !a->v_cache || !a->page_table || !a->cache_seqlens || !a->cu_seqlens_q || !a->out || !a->status)
    return fail("null tensor pointer");
  const int el = a->kv_type == ga::paged::KV_E4M3 ? 1 : 2;
  const int64_t kv[6] = {a->k_stride_page, a->k_stride_tok, a->k_stride_head, a->v_stride_page, a->v_stride_tok, a->v_stride_head};
  for (int64_t s : kv)
    if (s < 0 || s * el % 16) return fail("k/v cache strides must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return fail("k/v cache base must be 16-byte aligned");
  const bool q8 = el == 1 && !a->q_is_bf16;
  if (a->q_stride_tok % 4 || a->q_stride_head % 4 || reinterpret_cast<uintptr_t>(a->q) % (q8 ? 4 : 8)) return fail("q strides/base must allow 4-element vector loads");
  if (a->o_stride_tok % 4 || a->o_stride_head % 4 || reinterpret_cast<uintptr_t>(a->out) % 8) return fail("out strides/base must allow 4-element vector stores");
  // Only the route without split units needs no workspace, but which route a call takes is not the caller's business.
  if (!a->workspace || a->workspace_bytes < prefix_bytes(a->batch) + slots_bytes(l.sm))
    return fail("workspace too small: %zu < %zu bytes", a->workspace_bytes, prefix_bytes(a->batch) + slots_bytes(l.sm));
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256) return fail("workspace must be 256-byte aligned");

  PagedDev& d = l.d;
  std::memset(&d, 0, sizeof(d));
  d.q = static_cast<const uint8_t*>(a->q);
  d.q_kind = el == 1 && a->q_is_bf16 ? ga::paged::Q_BF16_TO_E4M3 : ga::paged::Q_SAME;
  d.q_s0 = a->q_stride_tok, d.q_s1 = a->q_stride_head;
  d.k = static_cast<const uint8_t*>(a->k_cache);
  d.v = static_cast<const uint8_t*>(a->v_cache);
  d.k_s0 = a->k_stride_page * el, d.k_s1 = a->k_stride_tok * el, d.k_s2 = a->k_stride_head * el;
  d.v_s0 = a->v_stride_page * el, d.v_s1 = a->v_stride_tok * el, d.v_s2 = a->v_stride_head * el;
  d.page_shift = __builtin_ctz(a->page_size);
  d.page_mask = a->page_size - 1;
  d.num_pages = a->num_pages;
  d.kvh = a->kv_heads, d.gqa = a->q_heads / a->kv_heads, d.q_heads = a->q_heads;
  d.pt = a->page_table;
  d.pt_s0 = a->pt_stride_row, d.pt_s1 = a->pt_stride_col, d.pt_cols = a->pt_cols;
  d.seqlens = a->cache_seqlens;
  d.cu = a->cu_seqlens_q;
  d.kd = a->k_descale, d.kd_s0 = a->kd_stride_b, d.kd_s1 = a->kd_stride_h;
  d.vd = a->v_descale, d.vd_s0 = a->vd_stride_b, d.vd_s1 = a->vd_stride_h;
  d.out = a->out;
  d.o_s0 = a->o_stride_tok, d.o_s1 = a->o_stride_head;
  d.lse = a->lse;
  d.total_q = static_cast<int>(a->total_q);
  d.batch = a->batch;
  d.max_q = a->max_seqlen_q < d.total_q ? a->max_seqlen_q : d.total_q;
  constexpr int kFar = ga::paged::MAX_KEYS;  // no position is further away
  d.window = a->window_left < 0 ? -1 : (a->window_left < kFar ? a->window_left : kFar);
  d.sinks = d.window < 0 ? 0 : (a->sink_tokens < kFar ? a->sink_tokens : kFar);
  d.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  d.status = a->status;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  d.prefix = reinterpret_cast<int*>(ws);
  d.ws_lse = reinterpret_cast<float*>(ws + prefix_bytes(a->batch));
  d.ws_o = d.ws_lse + static_cast<size_t>(2 * l.sm) * ga::paged::SLOT_ROWS;
  d.ws_seg = d.ws_o + static_cast<size_t>(2 * l.sm) * ga::paged::SLOT_FLOATS;
  d.ws_spoilt = reinterpret_cast<int*>(d.ws_seg + static_cast<size_t>(l.sm) * ga::paged::SEG_FLOATS);
  l.st = static_cast<cudaStream_t>(stream);
  l.max_tokens = std::min<long long>(static_cast<long long>(a->pt_cols) * a->page_size, kFar);
  l.prompt = d.max_q > 16;
  if (a->kv_type == ga::paged::KV_BF16) return route<ga::paged::KV_BF16>(l, a->head_dim);
  if (a->kv_type == ga::paged::KV_FP16) return route<ga::paged::KV_FP16>(l, a->head_dim);
  return route<ga::paged::KV_E4M3>(l, a->head_dim);
}

}  // extern "C"
