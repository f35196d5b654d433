// Upkeep of the pages of a paged cache: copying pages inside every layer's pool, sharing a request's pages with its
// forks, releasing, allocating and closing gaps, all on the device (no host round trip, capturable).
//
// Books: refs[page] = number of page-table entries that hold the page; a page is free while its count is 0. A row of
// the page table holds ceil(len / page_size) entries; -1 stands for a released page. New pages are the lowest free
// ones, handed out in the order of the call's rows, so the outcome does not depend on scheduling (counts are changed
// with integer atomics, whose order does not matter).
//
// What bounds it: the bytes of the copied tokens, read once and written once. The decisions (a few integers per row,
// one count per page) are made by small kernels in front; a copy kernel then moves pieces of pages of up to 16 KB, all
// layers of all pairs in one launch. A CTA takes a contiguous range of the pieces and one of its threads streams them
// through shared memory with bulk copies (global to shared, shared to global), up to three loads ahead of the stores, so
// that the reads of a piece's descriptors hide behind the pieces in flight. Measured: 250 pages of 128 KB in 16 tensors (1.05
// GB read and written) 178 us = 5.9 TB/s, 0.91 of a plain copy (186 us with vector loads and stores by 256 threads a piece); a
// call that has nothing to do 4 - 5 us, compaction 11.
#pragma once

#include "ga_common.cuh"

namespace ga {
namespace pages {

enum : int { ST_BAD_PAGE = GA_ST_BAD_PAGE, ST_LEN_RANGE = GA_ST_LEN_RANGE, ST_BAD_INDEX = 7, ST_NO_PAGES = 8, ST_REFS = 9, ST_CLASH = 10 };

constexpr int CHUNK = 16384;      // bytes of a copy item
constexpr int COPY_THREADS = 128;
constexpr int COPY_SLOTS = 4;    // pieces of a CTA in shared memory
constexpr int COPY_CTAS = 3;     // CTAs per SM
constexpr int COPY_SMEM = COPY_SLOTS * CHUNK;
constexpr int PLAN_THREADS = 1024;
constexpr int SPAN = 16384;       // pages that a CTA looks through at a time (16 per thread)

struct PoolDev {
  const unsigned long long* base;  // [tensors] address of page 0
  const long long* stride;         // [tensors] bytes between pages
  const int* tok_bytes;            // [tensors] bytes of a token
  const int* chunk_tensor;         // [chunks] tensor of a page's chunk
  const int* chunk_first;          // [tensors] first chunk of a tensor
  int tensors, chunks;
  int num_pages, page_shift, page_size;
  int* table;
  long long t_s0, t_s1;
  int rows, cols;
  int* lens;
  int* refs;
  int* status;
};

__device__ __forceinline__ int pages_of(const PoolDev& p, int len) { return len <= 0 ? 0 : (len - 1) / p.page_size + 1; }
__device__ __forceinline__ void flag(const PoolDev& p, int what) { atomicExch(p.status, what); }

// Exclusive prefix of `v` over the CTA's threads, and the sum. `tmp`: 33 numbers of shared memory.
template <int NT, typename N>
__device__ __forceinline__ N block_scan(N v, N* tmp, N& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const N o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) tmp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    N w = lane < NT / 32 ? tmp[lane] : 0, wi = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const N o = __shfl_up_sync(0xffffffffu, wi, d);
      if (lane >= d) wi += o;
    }
    if (lane < NT / 32) tmp[lane] = wi - w;
    if (lane == NT / 32 - 1) tmp[32] = wi;
  }
  __syncthreads();
  const N before = tmp[warp] + incl - v;
  total = tmp[32];
  __syncthreads();
  return before;
}

// ------------------------------------------------------------------------------------------------------ copying

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, int bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, int bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ int pieces(const PoolDev& p, int t, int tokens) { return (tokens * p.tok_bytes[t] + CHUNK - 1) / CHUNK; }

// Pieces [from, to) of the call by one thread. Pair i is `pair(i, src, dst, tokens)`: false for one that is not carried
// out; its pieces are those of `tokens` tokens of every tensor, tensor by tensor; (i0, skip): the pair that holds piece
// `from` and how many of its pieces come before. `ring`: COPY_SMEM bytes, `bars`: COPY_SLOTS initialised barriers.
template <typename Pair>
__device__ __forceinline__ void copy_pieces(const PoolDev& p, long long from, long long to, int i0, long long skip, Pair pair, uint32_t ring,
                                            uint32_t bars) {
  if (from >= to) return;
  int i = i0, t = 0, src, dst, tokens;
  bool real = pair(i, src, dst, tokens);
  int per = pieces(p, 0, tokens);
  while (skip >= per) {
    skip -= per;
    per = pieces(p, ++t, tokens);
  }
  int c = static_cast<int>(skip);
  uint8_t* to_at[COPY_SLOTS];
  int size[COPY_SLOTS];
  int loads = 0, stores = 0;  // pieces so far
  bool failed = false;
  auto store = [&]() {  // the oldest piece that has not been stored; after a wait that ran out pieces are only waited for
#pragma unroll
    for (int k = 0; k < COPY_SLOTS; ++k)
      if (k == stores % COPY_SLOTS) {
        if (!mbar_wait(bars + 8 * k, (stores / COPY_SLOTS) & 1)) {
          failed = true;
          flag(p, GA_ST_WAIT_FULL);
        }
        if (!failed) bulk_store(to_at[k], ring + k * CHUNK, size[k]);
      }
    ++stores;
  };
  for (long long at = from; at < to && !failed; ++at) {
    if (real) {
      const int off = c * CHUNK;
      const int n = min(tokens * p.tok_bytes[t] - off, CHUNK);
      const long long stride = p.stride[t];
      uint8_t* base = reinterpret_cast<uint8_t*>(p.base[t]) + off;
      // the slot's last piece was stored two turns ago: at most the store behind it may still be reading
      if (loads >= COPY_SLOTS) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
#pragma unroll
      for (int k = 0; k < COPY_SLOTS; ++k)
        if (k == loads % COPY_SLOTS) {
          to_at[k] = base + dst * stride;
          size[k] = n;
          mbar_expect_tx(bars + 8 * k, n);
          bulk_load(ring + k * CHUNK, base + src * stride, n, bars + 8 * k);
        }
      ++loads;
      if (loads - stores == COPY_SLOTS - 1) store();
    }
    if (++c == per) {
      c = 0;
      do {
        if (++t == p.tensors) {
          t = 0;
          if (at + 1 >= to) break;
          do real = pair(++i, src, dst, tokens);
          while (tokens <= 0);  // pairs without pieces
        }
        per = pieces(p, t, tokens);
      } while (per == 0);
    }
  }
  while (stores < loads) store();
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// A CTA's barriers; the thread that copies is thread 0.
__device__ __forceinline__ void copy_setup(uint32_t bars) {
  if (threadIdx.x == 0) {
    for (int k = 0; k < COPY_SLOTS; ++k) mbar_init(bars + 8 * k, 1);
    mbar_fence_init();
  }
}

__device__ __forceinline__ long long index_at(const void* p, int is64, int i) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// Which pairs of a copy call are carried out: list[i] = (src, dst), src -1: not. Of several pairs with one destination
// the last counts; a pair whose source another pair writes is not carried out (its content would depend on the order)
// and flagged, and so is one that names no page. `mark`: num_pages ints.
__global__ void __launch_bounds__(PLAN_THREADS) copy_plan_kernel(const __grid_constant__ PoolDev p, const void* src,
                                                                 const void* dst, int is64, int n, int* mark, int2* list) {
  grid_dep_wait();
  grid_dep_launch();
  auto get = [&](int i, int& s, int& d) {
    const long long a = index_at(src, is64, i), b = index_at(dst, is64, i);
    const bool ok = a >= 0 && a < p.num_pages && b >= 0 && b < p.num_pages;
    s = ok ? static_cast<int>(a) : -1;
    d = ok ? static_cast<int>(b) : -1;
    return ok;
  };
  int s, d;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
    if (get(i, s, d)) mark[s] = mark[d] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
    if (get(i, s, d) && s != d) atomicMax(mark + d, i);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const bool ok = get(i, s, d);
    int use = ok && s != d && __ldcg(mark + d) == i ? s : -1;
    if (!ok) flag(p, ST_BAD_INDEX);
    if (use >= 0 && __ldcg(mark + s) >= 0) {
      flag(p, ST_CLASH);
      use = -1;
    }
    list[i] = make_int2(use, d);
  }
}

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const __grid_constant__ PoolDev p, const int2* list, int n) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[COPY_SLOTS];
  copy_setup(smem_u32(bars));
  grid_dep_wait();
  grid_dep_launch();
  if (threadIdx.x != 0) return;
  const long long all = static_cast<long long>(n) * p.chunks;
  const long long from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
  copy_pieces(p, from, to, static_cast<int>(from / p.chunks), from % p.chunks, [&](int i, int& src, int& dst, int& tokens) {
    const int2 e = list[i];
    src = e.x, dst = e.y, tokens = p.page_size;
    return e.x >= 0;
  }, smem_u32(ring), smem_u32(bars));
}

// ---------------------------------------------------------------------------------------------------- releasing

// One CTA per entry of `rows`. Releases the row's entries [first, last) that hold a page: all of them and the row's
// length (evict = 0), or those whose keys lie behind the first `sinks` and before the window of the next query at
// position len (evict = 1).
__global__ void __launch_bounds__(256) release_kernel(const __grid_constant__ PoolDev p, const void* rows, int is64, int n,
                                                      int evict, int window, int sinks) {
  grid_dep_wait();
  grid_dep_launch();
  const int i = blockIdx.x;
  const long long row64 = index_at(rows, is64, i);
  if (row64 < 0 || row64 >= p.rows) {
    if (threadIdx.x == 0) flag(p, ST_BAD_INDEX);
    return;
  }
  bool again = false;  // a row named twice is released once
  for (int k = threadIdx.x; k < i; k += blockDim.x) again |= index_at(rows, is64, k) == row64;
  if (__syncthreads_or(again)) return;
  const int row = static_cast<int>(row64);
  const int len = p.lens[row];
  int held = pages_of(p, len);
  if (held > p.cols) {
    held = p.cols;
    if (threadIdx.x == 0) flag(p, ST_LEN_RANGE);
  }
  int first = 0, last = held;
  if (evict) {
    first = (sinks >> p.page_shift) + ((sinks & (p.page_size - 1)) != 0);
    const int gone = len > window ? (len - window) >> p.page_shift : 0;
    last = gone < held ? gone : held;
    first = min(first, last);  // so that no thread's index passes 32 bits
  }
  int* t = p.table + row * p.t_s0;
  for (int j = first + threadIdx.x; j < last; j += blockDim.x) {
    const int page = t[j * p.t_s1];
    if (page < 0) continue;
    t[j * p.t_s1] = -1;
    if (page >= p.num_pages) {
      flag(p, ST_BAD_PAGE);
    } else if (atomicSub(p.refs + page, 1) <= 0) {
      atomicAdd(p.refs + page, 1);
      flag(p, ST_REFS);
    }
  }
  __syncthreads();
  if (!evict && threadIdx.x == 0) p.lens[row] = 0;
}

// --------------------------------------------------------------------------------------------------- allocating

// Hands the lowest free pages to ranks 0, 1, ... < want: give(rank, page) by the thread that found it. Returns how
// many there were. One CTA of PLAN_THREADS; stops as soon as enough are found.
template <typename Give>
__device__ __forceinline__ int hand_out(const PoolDev& p, int want, int* tmp, Give give) {
  int found = 0;
  for (int p0 = 0; p0 < p.num_pages && found < want; p0 += SPAN) {
    const int at = p0 + threadIdx.x * 16;
    unsigned free_bits = 0;
    if (at + 16 <= p.num_pages && (reinterpret_cast<uintptr_t>(p.refs + at) & 15) == 0) {
      int4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __ldcg(reinterpret_cast<const int4*>(p.refs + at) + u);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        free_bits |= ((v[u].x == 0) | (v[u].y == 0) << 1 | (v[u].z == 0) << 2 | (v[u].w == 0) << 3) << (4 * u);
    } else {
      for (int u = 0; u < 16; ++u)
        if (at + u < p.num_pages && __ldcg(p.refs + at + u) == 0) free_bits |= 1u << u;
    }
    int total;
    int rank = found + block_scan<PLAN_THREADS>(__popc(free_bits), tmp, total);
    while (free_bits && rank < want) {
      const int u = __ffs(free_bits) - 1;
      free_bits &= free_bits - 1;
      give(rank++, at + u);
    }
    found += total;
  }
  __syncthreads();
  return found < want ? found : want;
}
// First i in [0, n) with incl[i] > rank (incl: non-decreasing inclusive prefix of the needs).
__device__ __forceinline__ int holder(const int* incl, int n, int rank) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (incl[mid] > rank) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// Only the first entry of a call that names a row counts: mark[row] = lowest i. `mark`: rows ints.
template <typename RowOf>
__device__ __forceinline__ void mark_first(int n, int* mark, RowOf row_of) {
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int r = row_of(i);
    if (r >= 0) mark[r] = 0x7fffffff;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int r = row_of(i);
    if (r >= 0) atomicMin(mark + r, i);
  }
  __syncthreads();
}

// Rows grow to the given lengths with the lowest free pages, in the call's order. From the first row on whose pages
// are not there, rows that need some are left as they were (flagged). One CTA; dynamic shared memory: n ints, the inclusive
// prefix of the needs, cut where it is past every page (rows times columns may pass 32 bits).
__global__ void __launch_bounds__(PLAN_THREADS) grow_kernel(const __grid_constant__ PoolDev p, const void* rows,
                                                            const void* to, int is64, int to64, int n, int* mark) {
  extern __shared__ int incl[];
  __shared__ long long tmp[33];
  __shared__ int found[33];
  grid_dep_wait();
  grid_dep_launch();
  auto row_of = [&](int i) {
    const long long r = index_at(rows, is64, i);
    return r >= 0 && r < p.rows ? static_cast<int>(r) : -1;
  };
  const long long most = min(static_cast<long long>(p.cols) << p.page_shift, 0x7fffffffLL);  // tokens of a row
  const long long all = p.num_pages + 1LL;
  mark_first(n, mark, row_of);
  long long sum = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int r = row_of(i);
      if (r < 0) {
        flag(p, ST_BAD_INDEX);
      } else if (__ldcg(mark + r) != i) {
        flag(p, ST_CLASH);
      } else {
        const long long want = index_at(to, to64, i);
        if (want > most) flag(p, ST_LEN_RANGE);
        else need = max(0, pages_of(p, static_cast<int>(want < 0 ? 0 : want)) - pages_of(p, p.lens[r]));
      }
    }
    long long total;
    const long long before = block_scan<PLAN_THREADS>(static_cast<long long>(need), tmp, total);
    if (i < n) incl[i] = static_cast<int>(min(sum + before + need, all));
    sum += total;
  }
  __syncthreads();
  const int got = hand_out(p, static_cast<int>(min(sum, all)), found, [&](int rank, int page) {
    const int i = holder(incl, n, rank);
    const int r = row_of(i), j = pages_of(p, p.lens[r]) + rank - (i ? incl[i - 1] : 0);
    p.table[r * p.t_s0 + j * p.t_s1] = page;
    p.refs[page] = 1;
  });
  __syncthreads();
  if (got < sum) {  // the row that ran out gives back what it got
    const int i = holder(incl, n, got);
    const int r = row_of(i), j0 = pages_of(p, p.lens[r]);
    for (int k = threadIdx.x; k < got - (i ? incl[i - 1] : 0); k += PLAN_THREADS) {
      int* e = p.table + r * p.t_s0 + (j0 + k) * p.t_s1;
      p.refs[*e] = 0;
      *e = -1;
    }
    if (threadIdx.x == 0) flag(p, ST_NO_PAGES);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int r = row_of(i);
    if (r < 0 || __ldcg(mark + r) != i) continue;
    const long long want = index_at(to, to64, i);
    if (want <= p.lens[r] || want > most) continue;
    if (incl[i] <= got || pages_of(p, static_cast<int>(want)) <= pages_of(p, p.lens[r])) p.lens[r] = static_cast<int>(want);
  }
}

// ------------------------------------------------------------------------------------------------------ forking

// list[i] = (source of the partial last page or -1, its copy, tokens of the parent, 1 if the pair is carried out), ends[i]
// = pieces to copy of the pairs up to i. A child is an empty row that the call names once; a parent is taken as it was
// before the call. One CTA; dynamic shared memory: n ints.
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(const __grid_constant__ PoolDev p, const void* parents,
                                                                 const void* children, int is64, int n, int* mark, int4* list,
                                                                 int* ends) {
  extern __shared__ int incl[];
  __shared__ int tmp[33];
  grid_dep_wait();
  grid_dep_launch();
  auto child_of = [&](int i) {
    const long long r = index_at(children, is64, i);
    return r >= 0 && r < p.rows ? static_cast<int>(r) : -1;
  };
  mark_first(n, mark, child_of);
  int sum = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      int4 e = make_int4(-1, -1, 0, 0);
      const int c = child_of(i);
      const long long a = index_at(parents, is64, i);
      if (c < 0 || a < 0 || a >= p.rows) {
        flag(p, ST_BAD_INDEX);
      } else if (__ldcg(mark + c) != i || p.lens[c] != 0) {
        flag(p, ST_CLASH);
      } else {
        const int len = p.lens[a], tail = len & (p.page_size - 1);
        if (pages_of(p, len) > p.cols) {
          flag(p, ST_LEN_RANGE);
        } else if (len > 0) {
          e = make_int4(-1, -1, len, 1);
          if (tail) {
            const int src = p.table[a * p.t_s0 + (len >> p.page_shift) * p.t_s1];
            if (src < 0 || src >= p.num_pages) {
              flag(p, ST_BAD_PAGE);
              e.w = 0;
            } else {
              e.x = src;
              need = 1;
            }
          }
        }
      }
      list[i] = e;
    }
    int total;
    const int before = block_scan<PLAN_THREADS>(need, tmp, total);
    if (i < n) incl[i] = sum + before + need;
    sum += total;
  }
  __syncthreads();
  const int got = hand_out(p, sum, tmp, [&](int rank, int page) {
    const int i = holder(incl, n, rank);
    p.table[child_of(i) * p.t_s0 + (list[i].z >> p.page_shift) * p.t_s1] = page;
    p.refs[page] = 1;
    list[i].y = page;
  });
  __syncthreads();
  int before_all = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    int count = 0;
    if (i < n) {
      int4 e = list[i];
      if (e.x >= 0 && e.y < 0) {  // no page left for its copy
        flag(p, ST_NO_PAGES);
        e = make_int4(-1, -1, 0, 0);
        list[i] = e;
      }
      if (e.w) p.lens[child_of(i)] = e.z;
      if (e.x >= 0)
        for (int t = 0; t < p.tensors; ++t) count += pieces(p, t, e.z & (p.page_size - 1));
    }
    int total;
    const int before = block_scan<PLAN_THREADS>(count, tmp, total);
    if (i < n) ends[i] = before_all + before + count;
    before_all += total;
  }
}

// The pairs' full pages are shared (all threads), then the tokens of the partial pages copied.
__global__ void __launch_bounds__(COPY_THREADS) fork_apply_kernel(const __grid_constant__ PoolDev p, const void* parents,
                                                                  const void* children, int is64, int n, const int4* list,
                                                                  const int* ends) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[COPY_SLOTS];
  copy_setup(smem_u32(bars));
  grid_dep_wait();
  grid_dep_launch();
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int4 e = list[i];
    if (!e.w) continue;
    const int* from = p.table + index_at(parents, is64, i) * p.t_s0;
    int* to = p.table + index_at(children, is64, i) * p.t_s0;
    for (int j = threadIdx.x; j < e.z >> p.page_shift; j += COPY_THREADS) {
      const int page = from[j * p.t_s1];
      to[j * p.t_s1] = page;
      if (page >= p.num_pages) flag(p, ST_BAD_PAGE);
      else if (page >= 0) atomicAdd(p.refs + page, 1);
    }
  }
  if (threadIdx.x != 0) return;
  const long long all = ends[n - 1];
  const long long from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
  if (from >= to) return;
  const int i0 = holder(ends, n, static_cast<int>(from));
  copy_pieces(p, from, to, i0, from - (i0 ? ends[i0 - 1] : 0), [&](int i, int& src, int& dst, int& tokens) {
    const int4 e = list[i];
    src = e.x, dst = e.y, tokens = e.x >= 0 ? e.z & (p.page_size - 1) : 0;
    return e.x >= 0;
  }, smem_u32(ring), smem_u32(bars));
}

// --------------------------------------------------------------------------------------------------- compacting

// Live pages of each span of SPAN pages.
__device__ __forceinline__ unsigned live_bits(const PoolDev& p, int at) {
  unsigned bits = 0;
  if (at + 16 <= p.num_pages && (reinterpret_cast<uintptr_t>(p.refs + at) & 15) == 0) {
    int4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __ldcg(reinterpret_cast<const int4*>(p.refs + at) + u);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      bits |= ((v[u].x > 0) | (v[u].y > 0) << 1 | (v[u].z > 0) << 2 | (v[u].w > 0) << 3) << (4 * u);
  } else {
    for (int u = 0; u < 16; ++u)
      if (at + u < p.num_pages && __ldcg(p.refs + at + u) > 0) bits |= 1u << u;
  }
  return bits;
}
__global__ void __launch_bounds__(PLAN_THREADS) compact_count_kernel(const __grid_constant__ PoolDev p, int* counts) {
  __shared__ int tmp[33];
  grid_dep_wait();
  grid_dep_launch();
  int total;
  block_scan<PLAN_THREADS>(__popc(live_bits(p, blockIdx.x * SPAN + threadIdx.x * 16)), tmp, total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}
// With L live pages, the live pages at L and above move, in order, to the free ones below L. map[page] = its new id,
// -1 for a free page, -2 - k for the k-th page that moves (to gaps[k]; the apply kernel puts the id there).
__global__ void __launch_bounds__(PLAN_THREADS) compact_rank_kernel(const __grid_constant__ PoolDev p, const int* counts,
                                                                    int* map, int* movers, int* gaps, int* live, int* moved) {
  __shared__ int tmp[33];
  __shared__ int below;  // live pages before this CTA's span
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x;
  int mine = 0, before = 0;
  for (int s = tid; s < static_cast<int>(gridDim.x) && gridDim.x > 1; s += PLAN_THREADS) {
    mine += counts[s];
    if (s < static_cast<int>(blockIdx.x)) before += counts[s];
  }
  int L, B;
  if (gridDim.x == 1) mine = __popc(live_bits(p, tid * 16));  // a pool of one span is counted here
  block_scan<PLAN_THREADS>(mine, tmp, L);
  block_scan<PLAN_THREADS>(before, tmp, B);
  if (tid == 0) below = B;
  // live pages below L: the spans before L's, whose counts are there if there are several, and the part of the one L lies in
  const int ls = gridDim.x == 1 ? 0 : L / SPAN;
  int low = 0;
  for (int s = tid; s < ls; s += PLAN_THREADS) low += counts[s];
  if (L > ls * SPAN) {
    const int at = ls * SPAN + tid * 16;
    unsigned bits = live_bits(p, at);
    if (at + 16 > L) bits &= at >= L ? 0u : (1u << (L - at)) - 1;
    low += __popc(bits);
  }
  int low_total;
  block_scan<PLAN_THREADS>(low, tmp, low_total);
  if (blockIdx.x == 0 && tid == 0) {
    *live = L;
    *moved = L - low_total;
  }
  const int at = blockIdx.x * SPAN + tid * 16;
  const unsigned bits = live_bits(p, at);
  int total;
  int rank = below + block_scan<PLAN_THREADS>(__popc(bits), tmp, total);  // live pages before page `at`
  for (int u = 0; u < 16; ++u) {
    const int id = at + u;
    if (id >= p.num_pages) break;
    if (bits >> u & 1) {
      if (id >= L) {
        movers[rank - low_total] = id;
        map[id] = -2 - (rank - low_total);
      } else {
        map[id] = id;
      }
      ++rank;
    } else {
      if (id < L) gaps[id - rank] = id;
      map[id] = -1;
    }
  }
}
// Rewrites the page table, moves the counts (all threads), then copies the pages.
__global__ void __launch_bounds__(COPY_THREADS) compact_apply_kernel(const __grid_constant__ PoolDev p, int* map, const int* movers,
                                                                     const int* gaps, const int* moved) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[COPY_SLOTS];
  copy_setup(smem_u32(bars));
  grid_dep_wait();
  grid_dep_launch();
  // at most half of the pages move; pairs that do not name two pages of the pool are left alone whatever the books say
  const int n = min(*moved, p.num_pages / 2);
  auto pair = [&](int i, int& src, int& dst) {
    src = movers[i], dst = gaps[i];
    return static_cast<unsigned>(src) < static_cast<unsigned>(p.num_pages) && static_cast<unsigned>(dst) < static_cast<unsigned>(p.num_pages);
  };
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int held = min(pages_of(p, p.lens[row]), p.cols);
    int* t = p.table + row * p.t_s0;
    for (int j = threadIdx.x; j < held; j += COPY_THREADS) {
      const int page = t[j * p.t_s1];
      if (page < 0) continue;
      if (page >= p.num_pages) {
        flag(p, ST_BAD_PAGE);
        continue;
      }
      const int to = __ldcg(map + page);
      if (to == -1) flag(p, ST_REFS);  // the books say that the page is free: left alone
      else if (to <= -2 && -2 - to < n) t[j * p.t_s1] = gaps[-2 - to];
      else if (to <= -2) flag(p, ST_REFS);
      else if (to != page) t[j * p.t_s1] = to;
    }
  }
  for (int i = blockIdx.x * COPY_THREADS + threadIdx.x; i < n; i += gridDim.x * COPY_THREADS) {
    int src, dst;
    if (!pair(i, src, dst)) continue;
    p.refs[dst] = p.refs[src];
    p.refs[src] = 0;
    map[src] = dst;
  }
  if (threadIdx.x != 0) return;
  const long long all = static_cast<long long>(n) * p.chunks;
  const long long from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
  copy_pieces(p, from, to, static_cast<int>(from / p.chunks), from % p.chunks, [&](int i, int& src, int& dst, int& tokens) {
    tokens = p.page_size;
    return pair(i, src, dst);
  }, smem_u32(ring), smem_u32(bars));
}

}  // namespace pages
}  // namespace ga
