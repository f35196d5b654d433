// Attention over paged caches of 16-bit (bf16, fp16) or e4m3 keys and values, with an optional left window and first
// tokens that stay visible beside it. Decode, verify and (row block by row block) prompts.
//
// Mathematics, per query row i at position p_i = len - new + t of its request and for one kv head:
//     s_ij = scale * k_descale * q_i . k_j,   key j visible iff j <= p_i and (W < 0 or j >= p_i - W or j < S)
//     o_i  = v_descale * sum_j softmax_j(s_ij) v_j,   lse_i = ln sum_j exp s_ij;  a row without keys: o = 0, lse = -inf
// evaluated in one pass with the running maximum m and sum l of the row (log2 domain):
//     m' = max(m, max_j s_ij),  l' = l 2^(m - m') + sum_j 2^(s_ij - m'),  O' = O 2^(m - m') + sum_j 2^(s_ij - m') v_j.
// Products run on the warp-level 16-bit tensor path with 32-bit accumulators; m, l, O and the partial results are
// 32 bits. P is rounded to the cache's 16-bit type before P V, by at most 2^-8 (bf16) or 2^-11 (fp16) of each probability:
// as much again as the rounding of a 16-bit output. fp16 P are taken up to 2^15 (P_TOP), which the sum and the LSE take
// back: they are subnormal only from 2^-29 of the row's largest down, and a key loses at most 2^-40 of it (2^-25 with P up
// to 1, so that a long flat tail under one dominant key was lost). An e4m3 value is an exact fp16 value, so an e4m3 cache
// runs on the fp16 path with P in fp16. Queries beside an e4m3 cache are e4m3, or bf16 rounded to e4m3 (the contract of the
// FP8 kernels next to this one).
//
// What bounds it: the cache's bytes. A warp owns one kv head and a private ring of tiles in shared memory that it fills
// with 16-byte cp.async and drains itself, so there is no barrier between warps: the kv_heads warps of a gang (neighbours
// in the grid, whatever CTAs they are in) walk the same tokens, one kv head each, which makes the bytes of a token run
// contiguous in DRAM within a short window whatever the page size (from one token up), strides and alignment. The call is
// one stream of tiles ordered by (request, row block), cut evenly over the gangs on the device from the live lengths; a
// unit that is cut leaves normalised 32-bit partials and their log2 LSE in the workspace, folded in slice order by
// attn_paged_combine (no atomics: results do not depend on scheduling).
//
// Tiles of 16 or 32 tokens (8 KB of K and V; 4 or 16 KB where a row is narrow or wide) in three stages: two in flight per
// warp are 128 KB per SM, three times what latency times bandwidth asks for. Measured: 64 requests of 1k..8k tokens, 64 / 8
// heads, head_dim 128, bf16 (1.29 GB): 202 us = 6.4 TB/s in a burst, 232 us in a long run at the power cap; 128 streams
// with a 4096-key window and 4 first tokens (2.15 GB) 331 us; 48 requests over pages of one token, 5 kv heads of 64 dims
// (145 MB) 40 us, of which planner, fill and combine are 12. Cutting by gangs of warps and not of CTAs took the last from
// 57 to 45 us (5 of 8 warps worked before), checking page ids an iteration after their load from 45 to 40.
#pragma once

#include <cuda_fp16.h>

#include "ga_common.cuh"

namespace ga {
namespace paged {

enum : int { KV_BF16 = 0, KV_FP16 = 1, KV_E4M3 = 2 };
enum : int { Q_SAME = 0, Q_BF16_TO_E4M3 = 1 };

constexpr int MAX_WARPS = 8;
constexpr int MAX_KEYS = 1 << 30;   // keys of a request: sums of two positions, and a tile behind the last, stay ints
// Keys after which O and the sum are put aside, normalised, and begun anew: the tensor cores cut every product to the last place
// of the accumulator that it goes into, so that over 2^20 keys of equal weight a single accumulator lost 0.4 % of O (2.3 % over
// 2^22). Rounding every 16 keys' products into O instead (as MODE 1 does, which has no workspace) made decode 3 % slower and
// 32-row blocks 16 %.
constexpr int FOLD_KEYS = 32768;
constexpr int SLOT_FLOATS = 32768;  // O floats of a CTA's workspace slot: warps x rows x head_dim of every instance
constexpr int SLOT_ROWS = 256;      // rows of a CTA's workspace slot, at most
constexpr int SEG_FLOATS = 512;     // softmax threads of a CTA of the tensor-core kernel, at most

struct PagedDev {
  const uint8_t* q;
  int q_kind;
  long long q_s0, q_s1;  // elements
  const uint8_t* k;
  const uint8_t* v;
  long long k_s0, k_s1, k_s2, v_s0, v_s1, v_s2;  // page, token, head (bytes)
  int page_shift, page_mask, num_pages;
  int kvh, gqa, q_heads;
  const int* pt;
  long long pt_s0, pt_s1;
  int pt_cols;
  const int* seqlens;
  const int* cu;
  const float* kd;
  const float* vd;
  long long kd_s0, kd_s1, vd_s0, vd_s1;
  void* out;
  long long o_s0, o_s1;  // elements
  float* lse;
  int total_q, batch, max_q;
  int window, sinks;  // window < 0: none (sinks is 0 then)
  float scale_log2;
  int nrb;           // row blocks = units of a request (split mode)
  int* status;
  int* prefix;
  float* ws_o;
  float* ws_lse;
  int* ws_spoilt;  // whether a result is no number: a word a CTA of the tensor-core kernel's slices, one in MODE 1
  float* ws_seg;  // tensor-core kernel: LSE of an item's segments before, a float for each softmax thread
};

// What the query tokens [t0, t0 + nt) of request b see: tiles of T tokens, the sinks' first, then one run that ends
// with the last visible key. Tile i starts at token T * (i < ns ? i : tlo + i - ns).
struct Req {
  int q0, nq;    // first query row and tokens of the request
  int pos0;      // position of token 0
  int kend;      // keys from here on are invisible to every row
  int lower;     // first key of the run (window) some row sees
  int ns, tlo, cnt;
};
__device__ __forceinline__ int new_tokens(const PagedDev& p, int b, int& q0) {
  q0 = p.cu[b];
  int q1 = p.cu[b + 1];
  if (q0 < 0 || q0 > p.total_q) return 0;
  if (q1 > p.total_q) q1 = p.total_q;
  return q1 - q0;
}
template <int T>
__device__ __forceinline__ Req req_info(const PagedDev& p, int b, int t0, int nt) {
  Req r;
  int L = p.seqlens[b];
  const long long cap = min(static_cast<long long>(p.pt_cols) << p.page_shift, static_cast<long long>(MAX_KEYS));
  if (L > cap) {
    L = static_cast<int>(cap);
    atomicExch(p.status, GA_ST_LEN_RANGE);
  }
  const int ql = new_tokens(p, b, r.q0);
  r.nq = ql < p.max_q ? ql : p.max_q;
  r.pos0 = L - ql;
  if (nt > r.nq - t0) nt = r.nq - t0;
  r.kend = r.pos0 + t0 + nt;
  r.lower = 0;
  r.ns = r.tlo = r.cnt = 0;
  if (L <= 0 || nt <= 0 || r.kend <= 0) return r;
  if (p.window >= 0) {
    const int lo = r.pos0 + t0 - p.window;
    r.lower = lo > 0 ? lo : 0;
  }
  r.tlo = r.lower / T;
  const int send = p.sinks < r.lower ? p.sinks : r.lower;
  const int ns = (send + T - 1) / T;
  r.ns = ns < r.tlo ? ns : r.tlo;
  r.cnt = r.ns + (r.kend + T - 1) / T - r.tlo;
  return r;
}

// T tiles are cut over at most G gangs, each of which gets MIN_TILES tiles at least; first tile of gang c's slice.
constexpr int MIN_TILES = 2;
__device__ __forceinline__ int gangs_for(long long T, int G) {
  const long long most = T / MIN_TILES;
  return most < G ? (most > 0 ? static_cast<int>(most) : 1) : G;
}
__device__ __forceinline__ long long slice(long long T, int G, int c) {
  if (c >= G) return T;
  const unsigned long long x = static_cast<unsigned long long>(T) * c;
  return x <= 0xffffffffull ? static_cast<unsigned>(x) / static_cast<unsigned>(G) : x / G;  // 32 bits: a third of the latency
}

// Exclusive prefix over the requests' counts, by the whole CTA (NT threads), and the request that holds item g0[s] for
// each of the gangs vc0 + s of the CTA's warps. find_b < 0: past the end. `publish`: this CTA writes p.prefix.
template <int NT, typename CountFn>
__device__ __forceinline__ long long plan(const PagedDev& p, CountFn count_of, int mul, long long (*g_of)(long long, int, int),
                                          int G, int vc0, int gangs, int* find_b, long long* find_pre, bool publish) {
  __shared__ long long wsum[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + NT - 1) / NT;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  const int first = b0 < b1 ? count_of(b0) : 0;  // a thread's first request, the only one in most calls, is read once
  auto count = [&](int b) { return b == b0 ? first : count_of(b); };
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += count(b);
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) wsum[warp] = incl;
  if (tid < MAX_WARPS) find_b[tid] = -1;
  __syncthreads();
  long long base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) base += wsum[w];
    total += wsum[w];
  }
  const long long T = total * mul;
  const long long pre = base + incl - mine;
  for (int s = 0; s < gangs; ++s) {
    const long long g0 = g_of(T, G, vc0 + s);
    if (g0 < T && mine > 0 && pre * mul <= g0 && g0 < (pre + mine) * mul) {
      long long at = pre;
      for (int b = b0; b < b1; ++b) {
        const int c = count(b);
        if (g0 < (at + c) * mul) {
          find_b[s] = b;
          find_pre[s] = at;
          break;
        }
        at += c;
      }
    }
  }
  if (publish) {
    long long at = pre;
    for (int b = b0; b < b1; ++b) {
      p.prefix[b] = static_cast<int>(at);
      at += count(b);
    }
    if (tid == 0) p.prefix[p.batch] = static_cast<int>(total);
  }
  __syncthreads();
  return T;
}
__device__ __forceinline__ long long at_cut(long long T, int G, int c) { return slice(T, gangs_for(T, G), c); }
__device__ __forceinline__ long long at_index(long long, int, int c) { return c; }

// ---------------------------------------------------------------------------------------------------- fragments

template <int KV>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (KV == KV_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same for O. APART: the sum of the 16 products is rounded to nearest on its way into d.
template <int KV, bool APART>
__device__ __forceinline__ void pv16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (!APART) {
    mma16<KV>(d, a, b0, b1);
  } else {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    mma16<KV>(c, a, b0, b1);
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] += c[e];
  }
}
template <int KV>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (KV == KV_BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// log2 of the largest P.
template <int KV>
constexpr float P_TOP = KV == KV_BF16 ? 0.f : 15.f;
// Two e4m3 values (the low 16 bits) as two fp16 values: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(v)));
  return r;
}
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------------------------------- values that are no numbers

// P of a key that a row does not see is 0, and 0 times an infinity or NaN is NaN: a V row with such values spoils, in a matrix
// product, rows that do not see it. So the results of calls with several new tokens are looked at, by the kernel behind or (prompts)
// as they are written; where one is no number the V rows with such values that only some rows of the block see are looked for, and
// the rows that do not see all of them are computed anew. (Looking at every such V row ahead of the product instead cost
// prompts 3 to 20 %.)

// The places of a word that hold infinities or NaN, as bits 15 and 31 (16-bit types) or 7, 15, 23 and 31 (e4m3, NaN).
template <int KV>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t EXP = KV == KV_BF16 ? 0x7f807f80u : (KV == KV_FP16 ? 0x7c007c00u : 0x7f7f7f7fu);
  constexpr uint32_t ONE = KV == KV_BF16 ? 0x00800080u : (KV == KV_FP16 ? 0x04000400u : 0x01010101u);
  return ((w & EXP) + ONE) & (KV == KV_E4M3 ? 0x80808080u : 0x80008000u);
}
// Products of two words' 16-bit values with 0, added up: no number once one of them was none.
template <int KV>
__device__ __forceinline__ void look_at(uint32_t& acc, uint32_t x, uint32_t y) {
  if (KV == KV_FP16)
    asm("fma.rn.f16x2 %0, %1, %3, %0;\n\tfma.rn.f16x2 %0, %2, %3, %0;" : "+r"(acc) : "r"(x), "r"(y), "r"(0u));
  else
    asm("fma.rn.bf16x2 %0, %1, %3, %0;\n\tfma.rn.bf16x2 %0, %2, %3, %0;" : "+r"(acc) : "r"(x), "r"(y), "r"(0u));
}
// Value `d` of a row of the cache.
template <int KV>
__device__ __forceinline__ float value_at(const uint8_t* row, int d) {
  if (KV == KV_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[d]);
  if (KV == KV_FP16) return __half2float(reinterpret_cast<const __half*>(row)[d]);
  const uint32_t two = e4m3x2_to_f16x2(row[d]);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(two)));
}

// Whether every query between positions pmin and pmax sees the keys [n0, n0 + n).
__device__ __forceinline__ bool all_see(const PagedDev& p, int n0, int n, int pmin, int pmax) {
  return n0 + n - 1 <= pmin && (p.window < 0 || n0 >= pmax - p.window || n0 + n <= p.sinks);
}
// Rows of K and V of request b's key in head h; null: a page that does not exist.
__device__ __forceinline__ void rows_of(const PagedDev& p, int b, int h, int key, const uint8_t*& k, const uint8_t*& v) {
  const int page = p.pt[b * p.pt_s0 + (key >> p.page_shift) * p.pt_s1];
  const bool real = page >= 0 && page < p.num_pages;
  k = real ? p.k + page * p.k_s0 + (key & p.page_mask) * p.k_s1 + h * p.k_s2 : nullptr;
  v = real ? p.v + page * p.v_s0 + (key & p.page_mask) * p.v_s1 + h * p.v_s2 : nullptr;
}
__device__ __forceinline__ const uint8_t* shfl_ptr(const uint8_t* x, int lane) {
  return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(x), lane));
}

// By one warp, up to 16 rows of request b and kv head h anew, row i being base + i * step < n of the block that begins at row0: steps
// of 16 keys whose fragments come straight from global memory. V rows that only some of the rows see go into the product
// without values that are no numbers; those are added to the rows that see them afterwards.
template <int KV, int HD>
__device__ __forceinline__ void redo16(const PagedDev& p, const Req& r, int b, int h, int row0, int base, int step, int n) {
  constexpr int EB = KV == KV_E4M3 ? 1 : 2, OKV = KV == KV_E4M3 ? KV_BF16 : KV;
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const int rows = min((n - base + step - 1) / step, 16);
  const float sl2 = p.scale_log2 * (p.kd ? p.kd[b * p.kd_s0 + h * p.kd_s1] : 1.f);
  const float vds = p.vd ? p.vd[b * p.vd_s0 + h * p.vd_s1] : 1.f;
  auto tok_of = [&](int i) { return (row0 + base + i * step) / p.gqa; };
  auto head_of = [&](int i) { return h * p.gqa + (row0 + base + i * step) % p.gqa; };
  auto out_of = [&](int i) { return static_cast<uint8_t*>(p.out) + ((r.q0 + tok_of(i)) * p.o_s0 + head_of(i) * p.o_s1) * 2; };
  const int pmin = r.pos0 + tok_of(0), pmax = r.pos0 + tok_of(rows - 1);
  int pos[2];
  uint32_t qf[HD / 16][4];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int i = hf * 8 + g;
    const bool real = i < rows;
    pos[hf] = real ? r.pos0 + tok_of(i) : -1;
    const bool q8 = KV == KV_E4M3 && p.q_kind == Q_SAME;
    const uint8_t* q = p.q + (real ? ((r.q0 + tok_of(i)) * p.q_s0 + head_of(i) * p.q_s1) * (q8 ? 1 : 2) : 0);
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) {  // dims 8 x + 2 tq, + 1
      uint32_t w = 0;
      if (real) {
        if (q8) {
          w = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(q + x * 8 + tq * 2));
        } else {
          w = *reinterpret_cast<const uint32_t*>(q + (x * 8 + tq * 2) * 2);
          if (KV == KV_E4M3) w = e4m3x2_to_f16x2(pack_e4m3x2(bf16_bits_to_f32(w & 0xffffu), bf16_bits_to_f32(w >> 16)));
        }
      }
      qf[x / 2][(x & 1) * 2 + hf] = w;
    }
  }
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  const int low = p.window >= 0 ? max(0, pmin - p.window) : 0, sinks = min(p.sinks, low);
  const int seen = pmax < 0 ? 0 : sinks + pmax + 1 - low;
  auto key_at = [&](int i) { return i < sinks ? i : low + i - sinks; };
#pragma unroll 1
  for (int i0 = 0; i0 < seen; i0 += 16) {
    const uint8_t *kp = nullptr, *vp = nullptr;
    bool part = false;
    if (lane < 16 && i0 + lane < seen) {
      const int key = key_at(i0 + lane);
      rows_of(p, b, h, key, kp, vp);
      part = !all_see(p, key, 1, pmin, pmax);
    }
    const uint32_t parts = __ballot_sync(0xffffffffu, part);
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      const uint8_t* k = shfl_ptr(kp, j * 8 + g);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t w[2] = {0u, 0u};
        if (k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint8_t* at = k + (ks * 16 + x * 8 + tq * 2) * EB;
            w[x] = KV == KV_E4M3 ? e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(at)) : *reinterpret_cast<const uint32_t*>(at);
          }
        mma16<KV>(s[j], qf[ks], w[0], w[1]);
      }
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + j * 8 + tq * 2 + (e & 1), key = key_at(i), at = pos[e >> 1];
        const bool sees = i < seen && key <= at && (p.window < 0 || key >= at - p.window || key < p.sinks);
        s[j][e] = sees ? s[j][e] * sl2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[j][e]);
      }
    float mu[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
      top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
      const float f = top[hf] == -INFINITY ? 1.f : ex2(m[hf] - top[hf]);
      m[hf] = top[hf];
      mu[hf] = top[hf] == -INFINITY ? 0.f : top[hf] - P_TOP<KV>;
      l[hf] *= f;
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) o[j][hf * 2] *= f, o[j][hf * 2 + 1] *= f;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2(s[j][e] - mu[e >> 1]);
        l[e >> 1] += s[j][e];
      }
    const uint32_t a[4] = {pack16<KV>(s[0][0], s[0][1]), pack16<KV>(s[0][2], s[0][3]), pack16<KV>(s[1][0], s[1][1]), pack16<KV>(s[1][2], s[1][3])};
    const uint8_t* v[4];  // of keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9
    uint32_t keep = 0;    // bits of a word that stay whatever they are: those of keys that all rows see
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int at = tq * 2 + (x & 1) + (x >> 1) * 8;
      v[x] = shfl_ptr(vp, at);
      keep |= (parts >> at & 1) ? 0u : 1u << x;
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      uint32_t w[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t u[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint8_t* row = v[x * 2 + y];
          u[y] = 0u;
          if (row) u[y] = KV == KV_E4M3 ? row[j * 8 + g] : reinterpret_cast<const uint16_t*>(row)[j * 8 + g];
          if (!(keep >> (x * 2 + y) & 1) && (not_finite<KV>(u[y]) & (KV == KV_E4M3 ? 0x80u : 0x8000u))) u[y] = 0u;
        }
        w[x] = KV == KV_E4M3 ? e4m3x2_to_f16x2(u[0] | u[1] << 8) : (u[0] | u[1] << 16);
      }
      pv16<KV, true>(o[j], a, w[0], w[1]);
    }
  }
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    float sum = l[hf];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int i = hf * 8 + g;
    if (i < rows) {
      uint8_t* out = out_of(i);
      const float f = vds / sum;
#pragma unroll
      for (int j = 0; j < HD / 8; ++j)
        *reinterpret_cast<uint32_t*>(out + (j * 8 + tq * 2) * 2) = sum == 0.f ? 0u : pack16<OKV>(o[j][hf * 2] * f, o[j][hf * 2 + 1] * f);
    }
  }
  __syncwarp();
  auto add = [&](int from, int to, int least) {
#pragma unroll 1
    for (int key = max(max(from, 0), least); key < to; ++key) {
      const uint8_t *k, *v;
      rows_of(p, b, h, key, k, v);
      if (!v) continue;
#pragma unroll 1
      for (int d = lane; d < HD; d += 32) {
        const float x = value_at<KV>(v, d);
        if (fabsf(x) <= 3.4028234663852886e38f) continue;
#pragma unroll 1
        for (int y = 0; y < rows; ++y) {
          const int at = r.pos0 + tok_of(y);
          if (key > at || (p.window >= 0 && key < at - p.window && key >= p.sinks)) continue;
          if (OKV == KV_FP16) {
            __half* w = reinterpret_cast<__half*>(out_of(y)) + d;
            *w = __float2half_rn(__half2float(*w) + x * vds);
          } else {
            __nv_bfloat16* w = reinterpret_cast<__nv_bfloat16*>(out_of(y)) + d;
            *w = __float2bfloat16_rn(__bfloat162float(*w) + x * vds);
          }
        }
      }
    }
  };
  add(pmin + 1, pmax + 1, 0);
  if (p.window >= 0) add(low, min(pmax - p.window, pmin + 1), p.sinks);
  __syncwarp();
}

// By one warp, a row of request b and kv head h anew, with few registers: for the kernels that fold pieces, where blocks are of few
// rows. `sq`: HD floats of shared memory.
template <int KV, int HD>
__device__ __forceinline__ void redo1(const PagedDev& p, const Req& r, int b, int h, int rr, float* sq) {
  constexpr int OKV = KV == KV_E4M3 ? KV_BF16 : KV;
  const int lane = threadIdx.x & 31;
  const int tok = rr / p.gqa, head = h * p.gqa + rr - tok * p.gqa, pos = r.pos0 + tok;
  uint8_t* out = static_cast<uint8_t*>(p.out) + ((r.q0 + tok) * p.o_s0 + head * p.o_s1) * 2;
  const float sl2 = p.scale_log2 * (p.kd ? p.kd[b * p.kd_s0 + h * p.kd_s1] : 1.f);
  const float vds = p.vd ? p.vd[b * p.vd_s0 + h * p.vd_s1] : 1.f;
      // the row anew: a lane a key for the scores, lanes over the dims for O
      const uint8_t* q = p.q + ((r.q0 + tok) * p.q_s0 + head * p.q_s1) * (KV == KV_E4M3 && p.q_kind == Q_SAME ? 1 : 2);
      __syncwarp();
      for (int d = lane; d < HD; d += 32) {
        float x;
        if (KV == KV_E4M3 && p.q_kind == Q_BF16_TO_E4M3) {
          const uint32_t two = e4m3x2_to_f16x2(pack_e4m3x2(value_at<KV_BF16>(q, d), 0.f));
          x = __half2float(__ushort_as_half(static_cast<unsigned short>(two)));
        } else {
          x = value_at<KV>(q, d);
        }
        sq[d] = x;
      }
      __syncwarp();
      float o[HD / 32], m = -INFINITY, l = 0.f;
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) o[x] = 0.f;
      const int low = p.window >= 0 ? max(0, pos - p.window) : 0, sinks = min(p.sinks, low);
      const int seen = pos < 0 ? 0 : sinks + pos + 1 - low;
#pragma unroll 1
      for (int i0 = 0; i0 < seen; i0 += 32) {
        const int i = i0 + lane;
        const uint8_t *k = nullptr, *v = nullptr;
        float s = -INFINITY;
        if (i < seen) {
          rows_of(p, b, h, i < sinks ? i : low + i - sinks, k, v);
          s = 0.f;
          if (k)
#pragma unroll 4
            for (int d = 0; d < HD; ++d) s += value_at<KV>(k, d) * sq[d];
          s *= sl2;
        }
        float top = s;
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, m);
        const float f = top == -INFINITY ? 1.f : ex2(m - top), e = i < seen ? ex2(s - (top == -INFINITY ? 0.f : top)) : 0.f;
        m = top;
        l = l * f + e;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) o[x] *= f;
#pragma unroll 1
        for (int x = 0; x < 32 && i0 + x < seen; ++x) {
          const float w = __shfl_sync(0xffffffffu, e, x);
          const uint8_t* row_v = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), x));
          if (row_v)
#pragma unroll
            for (int y = 0; y < HD / 32; ++y) {
              const float u = value_at<KV>(row_v, y * 32 + lane);
              o[y] += fabsf(u) <= 3.4028234663852886e38f ? w * u : u + w;  // (w: its score may be no number)
            }
        }
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      const float one = l == 0.f ? 0.f : vds / l;
#pragma unroll
      for (int y = 0; y < HD / 32; ++y) {
        const float u = l == 0.f ? 0.f : o[y] * one;
        if (OKV == KV_FP16) reinterpret_cast<__half*>(out)[y * 32 + lane] = __float2half_rn(u);
        else reinterpret_cast<__nv_bfloat16*>(out)[y * 32 + lane] = __float2bfloat16_rn(u);
      }
}

constexpr int MEND_KEYS = 64;
struct MendSmem {
  int keys[MEND_KEYS];   // V rows that are no numbers
  int n;
  float q[4][256];       // ROWS 1: a warp's query row
};
// By the NW first warps of a CTA, which meet in `sync`: request b's rows row0 .. row0 + n of kv head h (row = token * GQA + head), of
// which a warp has first, first + step, ..., and takes 16 or one at a time (ROWS); `r`: what the block's tiles were made of.
template <int KV, int HD, int NW, int ROWS, typename Sync>
__device__ __forceinline__ void mend(const PagedDev& p, const Req& r, int b, int h, int row0, int n, int first, int step, MendSmem& sm, Sync sync) {
  constexpr int OKV = KV == KV_E4M3 ? KV_BF16 : KV;
  const int lane = threadIdx.x & 31;
  const int pmin = r.pos0 + row0 / p.gqa, pmax = r.pos0 + (row0 + n - 1) / p.gqa;
  sync();
  if (threadIdx.x == 0) sm.n = 0;
  sync();
  // keys that are seen, but not by all rows: new tokens, and those that the window leaves behind
  auto look = [&](int from, int to, int least) {
#pragma unroll 1
    for (int key = max(from, 0) + threadIdx.x; key < to; key += NW * 32) {
      const uint8_t *k, *v;
      if (key < least) continue;
      rows_of(p, b, h, key, k, v);
      uint32_t any = 0;
      if (v) {
#pragma unroll 1
        for (int c = 0; c < HD * (KV == KV_E4M3 ? 1 : 2) / 16; ++c) {
          const uint4 w = reinterpret_cast<const uint4*>(v)[c];
          any |= not_finite<KV>(w.x) | not_finite<KV>(w.y) | not_finite<KV>(w.z) | not_finite<KV>(w.w);
        }
      }
      if (any) {
        const int at = atomicAdd(&sm.n, 1);
        if (at < MEND_KEYS) sm.keys[at] = key;
      }
    }
  };
  look(pmin + 1, r.kend, 0);
  if (p.window >= 0) look(r.lower, min(pmax - p.window, pmin + 1), p.sinks);
  sync();
  const int found = sm.n;
  if (found == 0) return;
#pragma unroll 1
  for (int base = first; base < n; base += ROWS * step) {
    // whether one of these rows is no number somewhere, and does not see all that was found
    bool redo = false;
#pragma unroll 1
    for (int row = base; row < n && row < base + ROWS * step; row += step) {
      const int rr = row0 + row, tok = rr / p.gqa, pos = r.pos0 + tok;
      const uint8_t* out = static_cast<const uint8_t*>(p.out) + ((r.q0 + tok) * p.o_s0 + (h * p.gqa + rr - tok * p.gqa) * p.o_s1) * 2;
      bool odd = found > MEND_KEYS, none = false;
      for (int i = lane; i < found && i < MEND_KEYS; i += 32) {
        const int key = sm.keys[i];
        odd |= key > pos || (p.window >= 0 && key < pos - p.window && key >= p.sinks);
      }
      for (int d = lane * 2; d < HD; d += 64) none |= not_finite<OKV>(*reinterpret_cast<const uint32_t*>(out + d * 2)) != 0;
      redo |= __any_sync(0xffffffffu, odd) && __any_sync(0xffffffffu, none);
    }
    if (!redo) continue;
    if (ROWS == 16) redo16<KV, HD>(p, r, b, h, row0, base, step, n);
    else redo1<KV, HD>(p, r, b, h, row0 + base, sm.q[threadIdx.x >> 5]);
  }
}

// The same by a CTA of four warps, as a call: it is rare, and the kernel around it short.
template <int KV, int HD, int ROWS>
__device__ __noinline__ void mend_call(const PagedDev& p, const Req& r, int b, int h, int row0, int n, int first, int step) {
  __shared__ MendSmem sm;
  mend<KV, HD, 4, ROWS>(p, r, b, h, row0, n, first, step, sm, [] { __syncthreads(); });
}

// Byte offset of 16-byte chunk `c` of row `r` in a tile whose rows hold RB bytes: rows lie one after the other in
// 128-byte lines, and the chunks of a line are permuted so that eight rows' chunks c fall into different banks.
template <int RB>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  if (RB >= 128) return r * RB + (c >> 3) * 128 + (((c & 7) ^ (r & 7)) << 4);
  const int line = r >> 1, cc = (r & 1) * 4 + c;  // RB == 64
  return line * 128 + (((cc ^ line) & 7) << 4);
}

template <int HD_, int KV_, int MT_>
struct Inst {
  static constexpr int HD = HD_, KV = KV_, MT = MT_;
  static constexpr int EB = KV == KV_E4M3 ? 1 : 2;
  static constexpr int RB = HD * EB;                       // bytes of a row of one head
  static constexpr int T = RB >= 256 ? 16 : 32;            // tokens per tile
  static constexpr int CPR = RB / 16;                      // 16-byte chunks per row
  static constexpr int KTILE = T * RB;
  static constexpr int STAGE = 2 * KTILE;                  // K then V: 4, 8 or 16 KB
  static constexpr int NW = STAGE > 8192 ? 4 : 8;          // warps
  static constexpr int NST = STAGE <= 4096 ? 6 : 3;        // stages of a warp's ring: 192 KB of shared memory in all
  static constexpr int SMEM = NW * NST * STAGE;
  static constexpr int RC = 16 * MT;                       // rows of a unit
  static constexpr bool LOOKS = false;                     // whether the kernel looks at the results that it writes itself
  static constexpr int NT = NW * 32;
  static __device__ __forceinline__ Req req(const PagedDev& p, int b) { return req_info<T>(p, b, 0, p.max_q); }
};

// ------------------------------------------------------------------------------------------------------- kernel

// A walker's place in the tile stream.
struct Cursor {
  int b, block;    // request, row block
  Req r;
  int t, t_end;    // tiles of the current segment
  long long rem;   // tiles of the slice after this segment
  bool live, first;
  bool whole;      // the slice holds all of the unit
  bool more;       // the unit's segments before were put aside
};

// A segment of tiles of the current unit from t_off on; at most FOLD_KEYS of them where there is a workspace for what is put aside.
template <class I, int MODE>
__device__ __forceinline__ void open_segment(const PagedDev& p, Cursor& c, int t_off, bool more) {
  const long long left = c.r.cnt - t_off;
  long long n = left < c.rem ? left : c.rem;
  if (!more) c.whole = t_off == 0 && n == left;
  c.more = more;
  if (MODE == 0 && n > FOLD_KEYS / I::T) n = FOLD_KEYS / I::T;
  c.t = t_off;
  c.t_end = t_off + static_cast<int>(n);
  c.rem -= n;
}
// To the next tile; to the next segment behind the last one.
template <class I, int MODE>
__device__ __forceinline__ void advance(const PagedDev& p, Cursor& c) {
  if (++c.t < c.t_end) return;
  if (MODE == 1 || c.rem <= 0) {
    c.live = false;
    return;
  }
  if (c.t < c.r.cnt) {
    open_segment<I, MODE>(p, c, c.t, true);
    return;
  }
  c.first = false;
  if (++c.block == p.nrb) {
    c.block = 0;
    do {
      if (++c.b >= p.batch) {
        c.live = false;
        return;
      }
      c.r = req_info<I::T>(p, c.b, 0, p.max_q);
    } while (c.r.cnt == 0);
  }
  open_segment<I, MODE>(p, c, 0, false);
}

// MODE 0: the tile stream cut evenly over all gangs (decode, verify). MODE 1: a gang takes one row block with the tiles that
// block sees (prompts; blocks from the last to the first, the longest first).
template <class I, int MODE>
__global__ void __launch_bounds__(I::NT, 1) attn_paged_kernel(const __grid_constant__ PagedDev p) {
  constexpr int T = I::T, RB = I::RB, HD = I::HD, KV = I::KV, MT = I::MT;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ int find_b[MAX_WARPS];
  __shared__ long long find_pre[MAX_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // This warp's gang and kv head, and the gangs that the CTA's warps belong to (the grid's last, incomplete one is left out).
  const long long w0 = static_cast<long long>(blockIdx.x) * I::NW;
  const int G = static_cast<int>(static_cast<long long>(gridDim.x) * I::NW / p.kvh);
  const int vc0 = static_cast<int>(w0 / p.kvh), vc = static_cast<int>((w0 + warp) / p.kvh);
  const int h = static_cast<int>(w0 + warp - static_cast<long long>(vc) * p.kvh);
  const int gangs = min(static_cast<int>((w0 + I::NW - 1) / p.kvh), G - 1) - vc0 + 1;
  const int me = vc - vc0;
  const int g = lane >> 2, tq = lane & 3;
  grid_dep_wait();
  grid_dep_launch();

  Cursor ci;
  ci.live = false;
  if (MODE == 0) {
    const long long total = plan<I::NT>(p, [&](int b) { return req_info<T>(p, b, 0, p.max_q).cnt; }, p.nrb, at_cut, G, vc0,
                                        gangs, find_b, find_pre, blockIdx.x == 0);
    if (vc >= G || find_b[me] < 0) return;
    const int used = gangs_for(total, G);
    const long long g0 = slice(total, used, vc), g1 = slice(total, used, vc + 1);
    if (g1 <= g0) return;
    ci.b = find_b[me];
    ci.r = req_info<T>(p, ci.b, 0, p.max_q);
    const long long in = g0 - find_pre[me] * p.nrb;
    const int unit = static_cast<int>(in / ci.r.cnt);
    ci.block = unit;
    ci.rem = g1 - g0;
    ci.live = ci.first = true;
    open_segment<I, MODE>(p, ci, static_cast<int>(in - static_cast<long long>(unit) * ci.r.cnt), false);
  } else {
    auto blocks = [&](int b) {
      int q0;
      const int ql = new_tokens(p, b, q0);
      return ql > 0 ? static_cast<int>((static_cast<long long>(min(ql, p.max_q)) * p.gqa + I::RC - 1) / I::RC) : 0;
    };
    const long long total = plan<I::NT>(p, blocks, 1, at_index, G, vc0, gangs, find_b, find_pre, false);
    if (vc >= G || vc >= total || find_b[me] < 0) return;
    ci.b = find_b[me];
    ci.block = blocks(ci.b) - 1 - static_cast<int>(vc - find_pre[me]);
    const int t0 = ci.block * I::RC / p.gqa, t1 = (ci.block * I::RC + I::RC - 1) / p.gqa;
    ci.r = req_info<T>(p, ci.b, t0, t1 - t0 + 1);
    ci.rem = ci.r.cnt;
    ci.live = ci.r.cnt > 0;
    open_segment<I, MODE>(p, ci, 0, false);
  }

  const uint32_t ring = smem_u32(smem_raw) + warp * (I::NST * I::STAGE);

  // Page of this lane's token of the tile the cursor stands on; UNSEEN where no row sees the token (its page-table entry may
  // be a released page's, or padding). It is looked at when the tile is issued, an iteration later, so that the load has
  // that long: a check here cost every tile the latency of a load. Unseen rows, and those of pages that do not exist, are
  // filled with zeros.
  constexpr int UNSEEN = static_cast<int>(0x80000000);
  auto fetch_pages = [&](const Cursor& c) -> int {
    if (!c.live || lane >= T) return UNSEEN;
    const int n = (c.t < c.r.ns ? c.t : c.r.tlo + c.t - c.r.ns) * T + lane;
    if (n >= c.r.kend || (n < c.r.lower && n >= p.sinks)) return UNSEEN;
    return p.pt[c.b * p.pt_s0 + (n >> p.page_shift) * p.pt_s1];
  };
  auto issue = [&](const Cursor& c, int pages, int stage) {
    if (c.live) {
      if (static_cast<unsigned>(pages) >= static_cast<unsigned>(p.num_pages)) {
        if (pages != UNSEEN) atomicExch(p.status, GA_ST_BAD_PAGE);
        pages = -1;
      }
      const int n0 = (c.t < c.r.ns ? c.t : c.r.tlo + c.t - c.r.ns) * T;
      const uint32_t dst = ring + stage * I::STAGE;
      constexpr int RPI = 32 / I::CPR;  // rows per instruction
      const int chunk = lane % I::CPR;
      const uint8_t* kb = p.k + h * p.k_s2 + chunk * 16;
      const uint8_t* vb = p.v + h * p.v_s2 + chunk * 16;
#pragma unroll
      for (int it = 0; it < T / RPI; ++it) {
        const int row = it * RPI + lane / I::CPR;
        const int page = __shfl_sync(0xffffffffu, pages, row);
        const bool real = page >= 0;
        const long long pg = real ? page : 0, tk = real ? ((n0 + row) & p.page_mask) : 0;
        const uint32_t d = dst + swz<RB>(row, chunk);
        cp_async_16_or_zero(d, kb + pg * p.k_s0 + tk * p.k_s1, real);
        cp_async_16_or_zero(d + I::KTILE, vb + pg * p.v_s0 + tk * p.v_s1, real);
      }
    }
    cp_async_commit();
  };

  Cursor cc = ci;  // the tile to consume; ci: the tile to load
  int pages = fetch_pages(ci);
#pragma unroll
  for (int i = 0; i < I::NST - 1; ++i) {
    issue(ci, pages, i);
    if (ci.live) advance<I, MODE>(p, ci);
    pages = fetch_pages(ci);
  }

  uint32_t qf[MT][HD / 16][4];
  float o[MT][HD / 8][4];
  float m[MT][2], l[MT][2];
  int pos[MT][2];
  float sl2 = 0.f;
  int stage = 0, pos_first = 0, pos_last = 0;
  bool fresh = true;
  // A prompt's row block without a single visible key still has rows to write (zeros).
  const bool blank = MODE == 1 && !cc.live;
  while (cc.live || (blank && fresh)) {
    const int block = cc.block;
    const int rows = cc.r.nq * p.gqa - block * I::RC;  // rows of this block, may exceed RC
    if (fresh) {
      fresh = false;
      sl2 = p.scale_log2 * (p.kd ? p.kd[cc.b * p.kd_s0 + h * p.kd_s1] : 1.f);
      pos_first = cc.r.pos0 + block * I::RC / p.gqa;
      pos_last = cc.r.pos0 + (block * I::RC + min(rows, I::RC) - 1) / p.gqa;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = mt * 16 + hf * 8 + g;
          const bool real = row < rows;
          const int rr = block * I::RC + row;
          const int tok = rr / p.gqa;
          pos[mt][hf] = real ? cc.r.pos0 + tok : -1;
          m[mt][hf] = -INFINITY;
          l[mt][hf] = 0.f;
          const long long qo = real ? (cc.r.q0 + tok) * p.q_s0 + (h * p.gqa + rr - tok * p.gqa) * p.q_s1 : 0;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t a0 = 0, a1 = 0;
            if (real) {
              if (KV != KV_E4M3) {
                const uint8_t* s = p.q + (qo + ks * 16 + tq * 2) * 2;
                a0 = *reinterpret_cast<const uint32_t*>(s);
                a1 = *reinterpret_cast<const uint32_t*>(s + 16);
              } else {
                // the contraction's dims are taken in the order in which a thread finds them in an e4m3 K row: its
                // four values 16 ks + 4 tq .. + 3
                uint32_t raw;
                if (p.q_kind == Q_BF16_TO_E4M3) {
                  const uint2 w = *reinterpret_cast<const uint2*>(p.q + (qo + ks * 16 + tq * 4) * 2);
                  raw = pack_e4m3x4(bf16_bits_to_f32(w.x & 0xffffu), bf16_bits_to_f32(w.x >> 16),
                                    bf16_bits_to_f32(w.y & 0xffffu), bf16_bits_to_f32(w.y >> 16));
                } else {
                  raw = *reinterpret_cast<const uint32_t*>(p.q + qo + ks * 16 + tq * 4);
                }
                a0 = e4m3x2_to_f16x2(raw & 0xffffu);
                a1 = e4m3x2_to_f16x2(raw >> 16);
              }
            }
            qf[mt][ks][hf] = a0;
            qf[mt][ks][2 + hf] = a1;
          }
        }
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
      }
    }
    bool last = blank;
    if (cc.live) {
      cp_async_wait<I::NST - 2>();
      __syncwarp();  // the tile of every lane is there, and every lane is done with the stage that is refilled next
      {
        int st = stage + I::NST - 1;
        if (st >= I::NST) st -= I::NST;
        issue(ci, pages, st);
        if (ci.live) advance<I, MODE>(p, ci);
        pages = fetch_pages(ci);
      }
      const uint32_t ka = ring + stage * I::STAGE, va = ka + I::KTILE;
      const int n0 = (cc.t < cc.r.ns ? cc.t : cc.r.tlo + cc.t - cc.r.ns) * T;
      float s[MT][T / 8][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < T / 8; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
      if (KV != KV_E4M3) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks += 2) {
#pragma unroll
          for (int j = 0; j < T / 8; ++j) {
            uint32_t r0, r1, r2, r3;
            ldsm_x4(ka + swz<RB>(j * 8 + (lane & 7), ks * 2 + (lane >> 3)), r0, r1, r2, r3);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma16<KV>(s[mt][j], qf[mt][ks], r0, r1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma16<KV>(s[mt][j], qf[mt][ks + 1], r2, r3);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks += 4) {
#pragma unroll
          for (int j = 0; j < T / 8; ++j) {
            uint32_t r[4];
            ldsm_x4(ka + swz<RB>(j * 8 + (lane & 7), ks + (lane >> 3)), r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t b0 = e4m3x2_to_f16x2(r[i] & 0xffffu), b1 = e4m3x2_to_f16x2(r[i] >> 16);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) mma16<KV>(s[mt][j], qf[mt][ks + i], b0, b1);
            }
          }
        }
      }
      const bool open = all_see(p, n0, T, pos_first, pos_last);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < T / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = s[mt][j][e] * sl2;
            if (!open) {
              const int key = n0 + j * 8 + tq * 2 + (e & 1), at = pos[mt][e >> 1];
              if (key > at || (p.window >= 0 && key < at - p.window && key >= p.sinks)) x = -INFINITY;
            }
            s[mt][j][e] = x;
            mx[e >> 1] = fmaxf(mx[e >> 1], x);
          }
        float mu[2];
        bool moved = false;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
          moved |= mx[hf] > m[mt][hf];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float nm = fmaxf(m[mt][hf], mx[hf]);
            const float f = nm == -INFINITY ? 1.f : ex2(m[mt][hf] - nm);
            m[mt][hf] = nm;
            l[mt][hf] *= f;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
              o[mt][j][hf * 2] *= f;
              o[mt][j][hf * 2 + 1] *= f;
            }
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) mu[hf] = m[mt][hf] == -INFINITY ? 0.f : m[mt][hf] - P_TOP<KV>;
#pragma unroll
        for (int j = 0; j < T / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = ex2(s[mt][j][e] - mu[e >> 1]);
            s[mt][j][e] = x;
            l[mt][e >> 1] += x;
          }
      }
#pragma unroll
      for (int ts = 0; ts < T / 16; ++ts) {
        uint32_t a[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          a[mt][0] = pack16<KV>(s[mt][2 * ts][0], s[mt][2 * ts][1]);
          a[mt][1] = pack16<KV>(s[mt][2 * ts][2], s[mt][2 * ts][3]);
          a[mt][2] = pack16<KV>(s[mt][2 * ts + 1][0], s[mt][2 * ts + 1][1]);
          a[mt][3] = pack16<KV>(s[mt][2 * ts + 1][2], s[mt][2 * ts + 1][3]);
        }
        const int row = ts * 16 + (lane & 15), cx = lane >> 4;
        if (KV != KV_E4M3) {
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t r0, r1, r2, r3;
            ldsm_x4_trans(va + swz<RB>(row, d * 2 + cx), r0, r1, r2, r3);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              pv16<KV, MODE == 1>(o[mt][2 * d], a[mt], r0, r1);
              pv16<KV, MODE == 1>(o[mt][2 * d + 1], a[mt], r2, r3);
            }
          }
        } else {
#pragma unroll
          for (int d = 0; d < HD / 32; ++d) {
            uint32_t r[4];
            ldsm_x4_trans(va + swz<RB>(row, d * 2 + cx), r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // chunk 2 d + i: its even dims, its odd dims
              const uint32_t e0 = e4m3x2_to_f16x2(prmt(r[2 * i], 0, 0x4420)), e1 = e4m3x2_to_f16x2(prmt(r[2 * i + 1], 0, 0x4420));
              const uint32_t o0 = e4m3x2_to_f16x2(prmt(r[2 * i], 0, 0x4431)), o1 = e4m3x2_to_f16x2(prmt(r[2 * i + 1], 0, 0x4431));
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                pv16<KV, MODE == 1>(o[mt][4 * d + 2 * i], a[mt], e0, e1);
                pv16<KV, MODE == 1>(o[mt][4 * d + 2 * i + 1], a[mt], o0, o1);
              }
            }
          }
        }
      }
      if (++stage == I::NST) stage = 0;
      last = cc.t + 1 >= cc.t_end;
    }
    if (last) {
      const float vds = p.vd ? p.vd[cc.b * p.vd_s0 + h * p.vd_s1] : 1.f;
      const int slot = 2 * vc + (cc.first ? 0 : 1);
      const bool on = MODE == 0 && cc.t_end < cc.r.cnt && cc.rem > 0;  // the unit goes on in this slice
      if (MODE == 0 && (cc.more || on)) {
        // One of several segments of a unit: what there is so far goes where the unit's piece goes or would have gone.
        const bool piece = on || !cc.whole;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float sum = l[mt][hf];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = mt * 16 + hf * 8 + g;
            if (row >= rows) continue;
            const long long wr = (static_cast<long long>(slot) * p.kvh + h) * I::RC + row;
            float* w = p.ws_o + wr * HD;
            const float one = piece ? 1.f : vds;
            float lse2 = sum == 0.f ? -INFINITY : m[mt][hf] + (lg2(sum) - P_TOP<KV>);
            float f = one / sum, theirs = one;
            if (cc.more) {
              const float before = __ldcg(p.ws_lse + wr);
              if (sum == 0.f) {
                lse2 = before;
              } else {
                const float top = fmaxf(before, lse2), wb = before == -INFINITY ? 0.f : ex2(before - top), wm = ex2(lse2 - top);
                f *= wm / (wb + wm);
                theirs *= wb / (wb + wm);
                lse2 = top + lg2(wb + wm);
              }
            }
            // columns of n8 tiles j and, beside an e4m3 cache, j + 1: this thread's two or four dims
#pragma unroll
            for (int j = 0; j < HD / 8; j += (KV == KV_E4M3 ? 2 : 1)) {
              float v[4];
              if (KV != KV_E4M3) {
                v[0] = o[mt][j][hf * 2], v[1] = o[mt][j][hf * 2 + 1];
              } else {
                v[0] = o[mt][j][hf * 2], v[1] = o[mt][j + 1][hf * 2], v[2] = o[mt][j][hf * 2 + 1], v[3] = o[mt][j + 1][hf * 2 + 1];
              }
              constexpr int N = KV == KV_E4M3 ? 4 : 2;
              const int at = j * 8 + tq * N;
#pragma unroll
              for (int e = 0; e < N; ++e) v[e] = sum == 0.f ? 0.f : v[e] * f;
              if (cc.more) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] += w[at + e] * theirs;
              }
              if (piece) {
                if (KV != KV_E4M3) *reinterpret_cast<float2*>(w + at) = make_float2(v[0], v[1]);
                else *reinterpret_cast<float4*>(w + at) = make_float4(v[0], v[1], v[2], v[3]);
              } else {
                const int rr = block * I::RC + row, tok = rr / p.gqa;
                uint8_t* dst = static_cast<uint8_t*>(p.out) + ((cc.r.q0 + tok) * p.o_s0 + (h * p.gqa + rr - tok * p.gqa) * p.o_s1 + at) * 2;
                if (KV != KV_E4M3) *reinterpret_cast<uint32_t*>(dst) = pack16<KV>(v[0], v[1]);
                else *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<KV_BF16>(v[0], v[1]), pack16<KV_BF16>(v[2], v[3]));
              }
            }
            if (tq == 0) {
              const int rr = block * I::RC + row, tok = rr / p.gqa, qh = h * p.gqa + rr - tok * p.gqa;
              if (piece) p.ws_lse[wr] = lse2;
              else if (p.lse) p.lse[static_cast<long long>(qh) * p.total_q + cc.r.q0 + tok] = lse2 * 0.6931471805599453f;
            }
          }
        }
        __syncwarp();  // a row's LSE is written by one lane and read by four
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float sum = l[mt][hf];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = mt * 16 + hf * 8 + g;
            if (row >= rows) continue;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const float lse2 = sum == 0.f ? -INFINITY : m[mt][hf] + (lg2(sum) - P_TOP<KV>);
            if (MODE == 0 && !cc.whole) {
              const long long wr = (static_cast<long long>(slot) * p.kvh + h) * I::RC + row;
              float* w = p.ws_o + wr * HD;
#pragma unroll
              for (int j = 0; j < HD / 8; j += (KV == KV_E4M3 ? 2 : 1)) {
                if (KV != KV_E4M3) {
                  *reinterpret_cast<float2*>(w + j * 8 + tq * 2) = make_float2(o[mt][j][hf * 2] * inv, o[mt][j][hf * 2 + 1] * inv);
                } else {
                  *reinterpret_cast<float4*>(w + j * 8 + tq * 4) =
                      make_float4(o[mt][j][hf * 2] * inv, o[mt][j + 1][hf * 2] * inv, o[mt][j][hf * 2 + 1] * inv, o[mt][j + 1][hf * 2 + 1] * inv);
                }
              }
              if (tq == 0) p.ws_lse[wr] = lse2;
            } else {
              const int rr = block * I::RC + row, tok = rr / p.gqa;
              const int qrow = cc.r.q0 + tok, qh = h * p.gqa + rr - tok * p.gqa;
              uint8_t* dst = static_cast<uint8_t*>(p.out) + (qrow * p.o_s0 + qh * p.o_s1) * 2;
              const float f = sum == 0.f ? 0.f : inv * vds;
              uint32_t acc = 0;
#pragma unroll
              for (int j = 0; j < HD / 8; j += (KV == KV_E4M3 ? 2 : 1)) {
                if (KV != KV_E4M3) {
                  const uint32_t w = pack16<KV>(o[mt][j][hf * 2] * f, o[mt][j][hf * 2 + 1] * f);
                  *reinterpret_cast<uint32_t*>(dst + (j * 8 + tq * 2) * 2) = w;
                  if (MODE == 1) look_at<KV>(acc, w, 0u);
                } else {
                  uint2 w;
                  w.x = pack16<KV_BF16>(o[mt][j][hf * 2] * f, o[mt][j + 1][hf * 2] * f);
                  w.y = pack16<KV_BF16>(o[mt][j][hf * 2 + 1] * f, o[mt][j + 1][hf * 2 + 1] * f);
                  *reinterpret_cast<uint2*>(dst + (j * 8 + tq * 4) * 2) = w;
                  if (MODE == 1) look_at<KV_BF16>(acc, w.x, w.y);
                }
              }
              if (MODE == 1 && not_finite<KV == KV_E4M3 ? KV_BF16 : KV>(acc)) *p.ws_spoilt = 1;
              if (tq == 0 && p.lse) p.lse[static_cast<long long>(qh) * p.total_q + qrow] = lse2 * 0.6931471805599453f;
            }
          }
        }
      }
      fresh = true;
      if (blank) break;
    }
    advance<I, MODE>(p, cc);
  }
  cp_async_wait<0>();
}

// Behind the kernels that write every row themselves (prompts): nothing, unless a result is no number. RC: rows of their blocks.
template <int KV, int HD, int RC>
__global__ void __launch_bounds__(128) attn_paged_mend(const __grid_constant__ PagedDev p) {
  grid_dep_wait();
  grid_dep_launch();
  if (__ldcg(p.ws_spoilt) == 0) return;
  long long before = 0;  // (block, kv head) items of the requests before
  for (int b = 0; b < p.batch; ++b) {
    int q0;
    const int ql = new_tokens(p, b, q0);
    const long long rows = ql > 0 ? static_cast<long long>(min(ql, p.max_q)) * p.gqa : 0;
    const long long n = (rows + RC - 1) / RC * p.kvh;
    for (long long x = (blockIdx.x + gridDim.x - before % gridDim.x) % gridDim.x; x < n; x += gridDim.x) {
      const int block = static_cast<int>(x / p.kvh), h = static_cast<int>(x - static_cast<long long>(block) * p.kvh);
      const int t0 = block * RC / p.gqa, t1 = (block * RC + RC - 1) / p.gqa;
      const Req r = req_info<32>(p, b, t0, t1 - t0 + 1);
      mend_call<KV, HD, 16>(p, r, b, h, block * RC, static_cast<int>(min(rows - static_cast<long long>(block) * RC, static_cast<long long>(RC))),
                        threadIdx.x >> 5, 4);
    }
    before += n;
  }
}

// Folds the pieces of every unit that the main kernel cut, in slice order, and writes the rows of requests without
// visible keys. grid = (batch * nrb, kv heads, row shares); 4 warps. A row's pieces are spread over the warps
// when there are many of them (one long sequence), the rows are when there are few.
template <class I>
__global__ void __launch_bounds__(128) attn_paged_combine(const __grid_constant__ PagedDev p, int G) {
  constexpr int HD = I::HD, VEC = HD / 32, UNR = 8;
  const int b = blockIdx.x / p.nrb, block = blockIdx.x - b * p.nrb;
  const int h = blockIdx.y;
  const Req r = I::req(p, b);
  const int rows = min(r.nq * p.gqa - block * I::RC, I::RC);
  const float vds = p.vd ? p.vd[b * p.vd_s0 + h * p.vd_s1] : 1.f;
  grid_dep_wait();
  grid_dep_launch();
  if (rows <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int OKV = I::KV == KV_E4M3 ? KV_BF16 : I::KV;
  bool none = false;  // a result is no number
  auto store = [&](int row, const float (&v)[VEC], float f, float lse2) {
    const int rr = block * I::RC + row, tok = rr / p.gqa;
    const int qrow = r.q0 + tok, qh = h * p.gqa + rr - tok * p.gqa;
    uint8_t* dst = static_cast<uint8_t*>(p.out) + (qrow * p.o_s0 + qh * p.o_s1 + lane * VEC) * 2;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const uint32_t w = pack16<OKV>(v[i] * f, v[i + 1] * f);
      *reinterpret_cast<uint32_t*>(dst + i * 2) = w;
      none |= not_finite<OKV>(w) != 0;
    }
    if (lane == 0 && p.lse) p.lse[static_cast<long long>(qh) * p.total_q + qrow] = lse2 * 0.6931471805599453f;
  };
  const int share = gridDim.z;
  if (r.cnt == 0) {
    const float zero[VEC] = {};
    for (int row = blockIdx.z * 4 + warp; row < rows; row += 4 * share) store(row, zero, 0.f, -INFINITY);
    return;
  }
  const long long total = static_cast<long long>(p.prefix[p.batch]) * p.nrb;
  G = gangs_for(total, G);
  const long long u0 = static_cast<long long>(p.prefix[b]) * p.nrb + static_cast<long long>(block) * r.cnt, u1 = u0 + r.cnt;
  auto owner = [&](long long x) {  // the gang whose slice holds tile x
    const unsigned long long at = static_cast<unsigned long long>(x + 1) * G - 1;
    long long c = at <= 0xffffffffull && total <= 0xffffffffll ? static_cast<unsigned>(at) / static_cast<unsigned>(total) : at / total;
    while (c > 0 && slice(total, G, static_cast<int>(c)) > x) --c;
    while (c < G - 1 && slice(total, G, static_cast<int>(c) + 1) <= x) ++c;
    return static_cast<int>(c);
  };
  const int c0 = owner(u0), c1 = owner(u1 - 1);
  if (c0 == c1) {  // its gang has written the rows
    if (p.max_q == 1) return;
    if (I::LOOKS) {
      if (__ldcg(p.ws_spoilt + c0 * p.kvh + h))
        mend_call<I::KV, HD, 1>(p, r, b, h, block * I::RC, rows, blockIdx.z * 4 + warp, 4 * share);
      return;
    }
    constexpr int LPR = HD / 8;  // lanes a row, 16 bytes each
    const int row0 = (blockIdx.z * 4 + warp) * (32 / LPR) + lane / LPR;
    for (int row = row0; row < rows; row += 4 * share * (32 / LPR)) {
      const int rr = block * I::RC + row, tok = rr / p.gqa;
      const uint8_t* at = static_cast<const uint8_t*>(p.out) + ((r.q0 + tok) * p.o_s0 + (h * p.gqa + rr - tok * p.gqa) * p.o_s1 + lane % LPR * 8) * 2;
      const uint2 x = __ldcg(reinterpret_cast<const uint2*>(at)), y = __ldcg(reinterpret_cast<const uint2*>(at + 8));
      none |= (not_finite<OKV>(x.x) | not_finite<OKV>(x.y) | not_finite<OKV>(y.x) | not_finite<OKV>(y.y)) != 0;
    }
    if (__syncthreads_or(none))
      for (int s = 0; s < 32 / LPR; ++s)
        mend_call<I::KV, HD, 1>(p, r, b, h, block * I::RC, rows, (blockIdx.z * 4 + warp) * (32 / LPR) + s, 4 * share * (32 / LPR));
    return;
  }
  const int n = c1 - c0 + 1;  // every gang between them holds a piece too
  const int e0 = u0 <= slice(total, G, c0) ? 0 : 1;
  auto piece = [&](int i) {  // workspace row 0 of the unit's piece i
    return (static_cast<long long>(2 * (c0 + i) + (i == 0 ? e0 : 0)) * p.kvh + h) * I::RC;
  };
  __shared__ float red_o[4][HD], red_m[4], red_l[4];
  const bool many = n > UNR;
  for (int row = many ? blockIdx.z : blockIdx.z * 4 + warp; row < rows; row += many ? share : 4 * share) {
    float mx = -INFINITY, den = 0.f, acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    const int step = many ? 4 : 1;
#pragma unroll 1
    for (int i0 = many ? warp : 0; i0 < n; i0 += step * UNR) {
      float w[UNR], v[UNR][VEC];
      float mc = mx;
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const int i = i0 + u * step;
        w[u] = -INFINITY;
        if (i < n) {
          const long long at = piece(i);
          w[u] = __ldcg(p.ws_lse + at + row);
#pragma unroll
          for (int x = 0; x < VEC; x += 2) {
            const float2 t = __ldcg(reinterpret_cast<const float2*>(p.ws_o + (at + row) * HD + lane * VEC + x));
            v[u][x] = t.x;
            v[u][x + 1] = t.y;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UNR; ++u) mc = fmaxf(mc, w[u]);
      if (mc != mx) {
        const float f = ex2(mx - mc);
        den *= f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] *= f;
        mx = mc;
      }
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        if (w[u] == -INFINITY) continue;
        const float f = ex2(w[u] - mx);
        den += f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] += f * v[u][x];
      }
    }
    if (many) {
#pragma unroll
      for (int x = 0; x < VEC; ++x) red_o[warp][lane * VEC + x] = acc[x];
      if (lane == 0) red_m[warp] = mx, red_l[warp] = den;
      __syncthreads();
      if (warp == 0) {
        const float top = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
        den = 0.f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = red_m[w] == -INFINITY && red_l[w] == 0.f ? 0.f : ex2(red_m[w] - top);
          den += f * red_l[w];
#pragma unroll
          for (int x = 0; x < VEC; ++x) acc[x] += f * red_o[w][lane * VEC + x];
        }
        store(row, acc, den == 0.f ? 0.f : vds / den, den == 0.f ? -INFINITY : top + lg2(den));
      }
      __syncthreads();
    } else {
      store(row, acc, den == 0.f ? 0.f : vds / den, den == 0.f ? -INFINITY : mx + lg2(den));
    }
  }
  if (p.max_q > 1 && __syncthreads_or(none))
    mend_call<I::KV, HD, 1>(p, r, b, h, block * I::RC, rows, many ? (warp ? rows : blockIdx.z) : blockIdx.z * 4 + warp, many ? share : 4 * share);
}

}  // namespace paged
}  // namespace ga
