// Prompts and verify over paged caches on the tensor cores (tcgen05, kind::f16, accumulators in tensor memory): the same
// mathematics as attn_paged.cuh. Prompts are cut into row blocks; verify (SPLIT_KV: at most 128 rows of a kv head) along
// the keys, with the pieces folded by attn_paged_combine.
//
// A persistent CTA takes work items of NQ tiles of 128 query rows (row = token * GQA + head, one kv head) against tiles of
// 128 keys. Roles: softmax warps (two threads a row, each with half of the keys; four in verify at head_dim 128), one or two
// lanes that issue the MMAs, four or five warps that gather K and V, one to four that gather Q.
//   * S = Q K^T into one of two 128-column score buffers, softmax in place, P as 16-bit pairs over the front half of the
//     buffer it came from, O += P V with P as the A operand from tensor memory and V as an MN-major B operand, i.e. the
//     page's [token, dim] layout as it is. Score buffers alternate job by job; a job is (key tile, query tile): at
//     head_dim <= 128 two query tiles share every K and V tile (NQ = 2), at 256 one query tile (O alone takes half of
//     tensor memory) has two key tiles in flight.
//   * The MMAs are issued in an order that needs few barriers: PV(n), then QK(n + 2) into the same buffer. With NQ 2 one
//     lane issues them all and the pipe runs them in order; with NQ 1 a second lane issues the QK MMAs and waits for the PV
//     two jobs before. Either way scores that are ready say that the PV two jobs before is done.
//   * The row's reference maximum moves only when a tile exceeds it by more than 2^8 (the lazy rescaling of online softmax),
//     so O is rescaled in tensor memory in few tiles. At the reference fp16 P are 2^7, so that they stay within 2^15 and a
//     key loses at most 2^-32 of the row's largest to subnormals; the 16-bit rounding of P is relative otherwise.
//   * An item's tiles come in segments of at most 256 (32768 keys): O and the sum are read out, normalised and folded with the
//     segments before in 32 bits. The tensor cores cut every product to the accumulator's last place, so that over 2^20 keys of
//     equal weight a single accumulator lost 0.4 % of O (2.3 % over 2^22); and no wait lasts longer than a segment.
//   * K and V come through one ring of 16 KB stages in the order in which the MMAs use them: a K stage is 128 keys x 64
//     dims, a V stage 8192 / head_dim keys x all dims, in the 128-byte swizzle that the MMA descriptors name. Where every
//     key of a stage is seen by some query, TMA boxes of up to a page each fill it (pages of 8 tokens and more); edges of
//     what is seen and smaller pages are filled with 16-byte cp.async, rows no query of the item sees (released pages
//     among them) with zeros. Values of an e4m3 cache go through registers, converted to fp16.
// Keys are taken in groups of 32: the sinks' groups, then those of the run that ends with the item's last visible key (Req);
// a tile is the next four, so a few first tokens cost 32 keys of a tile and not one of their own. Items come from a list that a
// small kernel lays out, later row blocks of a request first (they see more keys), all kv heads of a block side by side
// (they share pages).
//
// What bounds it: a key tile is 2 x 1024 tensor cycles at head_dim 256 and takes about 4600, because scores, softmax, P and
// PV follow one another over two score buffers, and the QK MMAs (both operands from shared memory) use all of its 128
// bytes a clock. Measured (bf16): 4 causal prompts of 4096 tokens, head_dim 256, 16 heads 652 us = 842 TFLOP/s, head_dim 128,
// 32 heads 802 us = 685; 8 x 2048 tokens on 16k, head_dim 256, window 1024 and 4 first tokens 431 us; verify in slices, 32 x
// 8192 tokens, 20 rows of 8 kv heads (1.07 GB) 191 us = 5.6 TB/s (299 on the warp-level kernel). Over an e4m3 cache the
// gathering warps convert (exactly, to fp16), which bounds it: the windowed extend takes 1150 us.
#pragma once

#include "attn_paged.cuh"

namespace ga {
namespace paged {
namespace tc {

constexpr int TM = 128;          // query rows of a tile = tensor memory lanes
constexpr int TK = 128;          // keys of a tile
constexpr int GK = 32;           // keys of a group
constexpr int STAGE = 16384;
constexpr int SEG_TILES = FOLD_KEYS / TK;  // tiles of a segment, at most
constexpr float RISE = 8.f;      // log2: how far a row's maximum may exceed the reference before O is rescaled
template <int KV>
constexpr float P_REF = KV == KV_BF16 ? 0.f : P_TOP<KV> - RISE;  // log2 of P at the reference

// SPLIT_KV: at most 128 rows of each (request, kv head), its keys cut over CTAs (verify). Else row blocks of prompts.
template <int HD_, int KV_, bool SPLIT_KV_>
struct TcInst {
  static constexpr int HD = HD_, KV = KV_;
  static constexpr bool SPLIT_KV = SPLIT_KV_;
  static constexpr int NQ = HD == 256 || SPLIT_KV ? 1 : 2;
  static constexpr int SLABS = HD / 64;            // K stages of a tile, and V stages
  static constexpr int KC = 8192 / HD;             // keys of a V stage
  static constexpr int ROWS = NQ * TM;
  static constexpr int Q_BYTES = NQ * SLABS * STAGE;
  static constexpr int NST = HD == 64 ? (NQ == 1 ? 12 : 8) : 10;
  static constexpr int EG = SLABS < 2 ? SLABS : 2;  // stages that are filled and released together
  // Threads that share a row. With few rows only the warps of the first lanes have any (tensor memory lanes belong to the
  // warps of one place in their group of four), so there more threads take part in a row.
  static constexpr int SPLIT = SPLIT_KV && HD == 128 ? 4 : 2;  // (head_dim 256: no shared memory for it)
  static constexpr int SOFT_WARPS = 4 * NQ * SPLIT;
  // Gathering warps. A stage is always filled by the same warp: one that waits for use u of a stage to be released has
  // filled that use itself, so the barrier cannot be a whole phase behind the wait (stages are not released in ring order
  // when K and V are released by different lanes, and a parity cannot tell phase u - 2 from phase u).
  static constexpr int KV_WARPS = NST % 5 == 0 ? 5 : 4;
  static constexpr int Q_WARPS = SOFT_WARPS == 16 ? 6 - KV_WARPS : 4;
  static_assert(NST % KV_WARPS == 0, "gathering warps");
  static constexpr int WARPS = (SOFT_WARPS + 2 + KV_WARPS + Q_WARPS + 3) / 4 * 4;  // whole warpgroups
  static constexpr int NT = WARPS * 32;
  // Registers a thread: what the block is launched with (limit of the launch bounds), and its split between the softmax
  // warps and the others. The shares add up to no more than the launch's.
  static constexpr int REGS = SOFT_WARPS == 16 ? 80 : 96;
  static constexpr int REGS_SOFT = SOFT_WARPS == 16 ? 88 : 120, REGS_REST = SOFT_WARPS == 16 ? 64 : 80;
  static_assert(SOFT_WARPS * REGS_SOFT + (WARPS - SOFT_WARPS) * REGS_REST <= WARPS * REGS, "register split");
  // Row maxima that the halves of a row exchange: at NQ 1 two jobs' in turn; at NQ 2 a query tile's next scores are ready
  // only after both halves are done with the job before.
  static constexpr int TURNS = 3 - NQ;
  static constexpr int X_BYTES = (NQ == 1 ? 2 * SPLIT : 2 * 2) * TM * 4;
  // Operands first: they need the 1024-byte alignment that dynamic shared memory starts with (the kernel checks it).
  static constexpr int SMEM = Q_BYTES + NST * STAGE + X_BYTES + 512;
  static_assert(NST % EG == 0, "ring");
  static constexpr int O_COL = 256;
  static constexpr int RC = ROWS;  // rows of a unit, for the combine kernel
  static constexpr bool LOOKS = true;
  static __device__ __forceinline__ Req req(const PagedDev& p, int b) {
    Req r = req_info<GK>(p, b, 0, p.max_q);
    r.cnt = (r.cnt + TK / GK - 1) / (TK / GK);
    return r;
  }
  static_assert(SMEM <= 232448, "shared memory");
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// kind::f16: f32 accumulators, A and B of one 16-bit type, A K-major, B K-major or MN-major.
__device__ __forceinline__ uint32_t instr_desc(int kv, int m, int n, int b_mn_major) {
  const uint32_t f = kv == KV_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0)
      : "memory");
}
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void mbar_expect_tx_only(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// A wait that runs out is recorded, and every later wait of the thread is skipped: all warps still reach the exit.
__device__ __forceinline__ void wait_or_flag(uint32_t bar, uint32_t parity, bool& failed, int* status, int code) {
  if (failed) return;
  if (!mbar_wait(bar, parity)) {
    failed = true;
    atomicExch(status, code);
  }
}

// 16 e4m3 values as fp16 into chunks `ch` and ch + 1 of a 128-byte row whose chunks are permuted by `sw`.
__device__ __forceinline__ void store_e4m3x16(uint32_t row, int ch, int sw, uint4 v, uint32_t flip) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(row + (((ch + k) ^ sw) << 4)), "r"(e4m3x2_to_f16x2(w[2 * k] & 0xffffu) ^ flip),
                 "r"(e4m3x2_to_f16x2(w[2 * k] >> 16) ^ flip), "r"(e4m3x2_to_f16x2(w[2 * k + 1] & 0xffffu) ^ flip),
                 "r"(e4m3x2_to_f16x2(w[2 * k + 1] >> 16) ^ flip)
                 : "memory");
}

// One warp fills a stage with KEYS keys of CPK 16-byte chunks each, in slabs of eight chunks (128 bytes a key), swizzled by
// key. n0[u] is the first token of the stage's group u, page[u]
// the page of its token `lane`, or -1 for a row of zeros. Its own instruction stream is what a stage costs
// here (32 copies a lane), so a copy is its address step and little else: within 32 keys of one page the source advances
// by a constant, and the swizzle of the destination is a constant flipped in. Smaller pages and edges pass each row's
// offset from the lane that looked it up.
template <int CPK, int KEYS>
__device__ __forceinline__ void gather(uint32_t dst, const uint8_t* base, long long s0, long long s1, const int (&n0)[4], int page_shift,
                                       int page_mask, const int (&page)[4], int lane) {
  constexpr int KPI = 32 / CPK;  // keys an instruction
  const int c = lane % CPK, k0 = lane / CPK;
  const uint32_t d0 = (c >> 3) * (KEYS * 128) + k0 * 128 + (((c ^ k0) & 7) << 4);
  base += c * 16;
  const long long step = s1 * KPI;
#pragma unroll
  for (int u = 0; u < (KEYS + 31) / 32; ++u) {
    const int tok = n0[u] & page_mask;
    if (page_shift >= 5 && __all_sync(0xffffffffu, page[u] >= 0)) {
      const uint8_t* src = base + page[u] * s0 + (tok + k0) * s1;
#pragma unroll
      for (int i = 0; i < CPK; ++i, src += step)
        cp_async_16(dst + (u * 32 + i * KPI) * 128 + (d0 ^ (((i * KPI) & 7) << 4)), src);
    } else {
      const long long off = page[u] >= 0 ? page[u] * s0 + ((n0[u] + lane) & page_mask) * s1 : -1;
#pragma unroll 4
      for (int i = 0; i < CPK; ++i) {
        const long long o = __shfl_sync(0xffffffffu, off, i * KPI + k0);
        cp_async_16_or_zero(dst + (u * 32 + i * KPI) * 128 + (d0 ^ (((i * KPI) & 7) << 4)), base + (o >= 0 ? o : 0), o >= 0);
      }
    }
  }
}

// Where each gang's slice of the call's tiles begins: (request, tile, tiles of the slice), tiles 0: none. A unit is a whole
// request; gang g is the CTAs g * kv_heads + h, one kv head each, which walk the same pages at the same time.
template <class I>
__global__ void __launch_bounds__(1024) plan_split_kernel(const __grid_constant__ PagedDev p, int G, int4* list) {
  __shared__ long long wsum[32];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + 1023) / 1024;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += I::req(p, b).cnt;
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  long long at = incl - mine, total = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) at += wsum[w];
    total += wsum[w];
  }
  for (int b = b0; b < b1; ++b) {
    p.prefix[b] = static_cast<int>(at);
    at += I::req(p, b).cnt;
  }
  if (tid == 0) p.prefix[p.batch] = static_cast<int>(total);
  __syncthreads();
  const int used = gangs_for(total, G);
  for (int g = tid; g < G; g += 1024) {
    const long long g0 = slice(total, used, g), g1 = slice(total, used, g + 1);
    int4 e = make_int4(0, 0, 0, 0);
    if (g1 > g0) {
      int lo = 0, hi = p.batch - 1;  // the last request whose tiles begin at g0 or before
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.prefix[mid] <= g0) lo = mid;
        else hi = mid - 1;
      }
      e = make_int4(lo, static_cast<int>(g0 - p.prefix[lo]), static_cast<int>(g1 - g0), 0);
    }
    list[g] = e;
  }
  for (int g = tid; g < G * p.kvh; g += 1024) p.ws_spoilt[g] = 0;
}

// The same for an e4m3 cache: 16 values of a key a load, converted to fp16 (exact) on the way into the stage. CPK: loads a key.
template <int CPK, int KEYS>
__device__ __forceinline__ void gather_e4m3(uint32_t dst, const uint8_t* base, long long s0, long long s1, const int (&n0)[4], int page_mask,
                                            const int (&page)[4], int lane) {
  constexpr int KPI = 32 / CPK;  // keys an instruction
  const int c = lane % CPK, k0 = lane / CPK;
  base += c * 16;
  constexpr int U = 4;
#pragma unroll
  for (int i0 = 0; i0 < KEYS / KPI; i0 += U) {
    uint4 v[U];
    const int u = i0 * KPI / 32;  // a batch of loads lies within a group
    const long long off = page[u] >= 0 ? page[u] * s0 + ((n0[u] + lane) & page_mask) * s1 : -1;
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const long long o = __shfl_sync(0xffffffffu, off, ((i0 + x) * KPI + k0) & 31);
      v[x] = make_uint4(0u, 0u, 0u, 0u);
      if (o >= 0) v[x] = *reinterpret_cast<const uint4*>(base + o);
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int key = (i0 + x) * KPI + k0;
      const uint32_t row = dst + (c >> 2) * (KEYS * 128) + key * 128;
      store_e4m3x16(row, (c & 3) * 2, key & 7, v[x], 0u);
    }
  }
}

// The call's row blocks: *count = how many, then (request, row block), a request's last block first.
template <int ROWS>
__global__ void __launch_bounds__(1024) plan_prompts_kernel(const __grid_constant__ PagedDev p, int* count, int4* blocks, int cap) {
  __shared__ int wsum[32];
  __shared__ int base;
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) base = 0;
  __syncthreads();
  for (int b0 = 0; b0 < p.batch; b0 += 1024) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.batch) {
      int q0;
      const int ql = new_tokens(p, b, q0);
      n = ql > 0 ? static_cast<int>((static_cast<long long>(min(ql, p.max_q)) * p.gqa + ROWS - 1) / ROWS) : 0;
    }
    int incl = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int at = base, total = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += wsum[w];
      total += wsum[w];
    }
    at += incl - n;
    // a warp lays out its requests' blocks together
    for (int src = 0; src < 32; ++src) {
      const int m = __shfl_sync(0xffffffffu, n, src), to = __shfl_sync(0xffffffffu, at, src);
      // query offsets that do not ascend could ask for more blocks than the list holds: they are left out
      for (int k = lane; k < m && to + k < cap; k += 32) blocks[to + k] = make_int4(b0 + warp * 32 + src, m - 1 - k, 0, 0);
    }
    __syncthreads();
    if (tid == 0) base = min(base + total, cap);
    __syncthreads();
  }
  if (tid == 0) *count = min(base, cap);
}

// Two products and sums, two sums an instruction: the exponential pass issues 5 instructions for two scores instead of 7
// (full causal head_dim 256 680 -> 652 us, head_dim 128 816 -> 802).
__device__ __forceinline__ float2 fma2(float x, float y, float s, float t) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x), "f"(y), "f"(s), "f"(t));
  return r;
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

// What a row sees: keys in [lo, pos], and those below `sinks` that are not behind pos. pmin, pmax: positions of the first
// and the last row of the thread's warp, which decide for 32 keys at a time whether any row has to look at them.
struct View {
  int pos, lo, sinks, pmin, pmax, window;
};
enum : int { ALL, SOME, NONE };
__device__ __forceinline__ int chunk_class(const View& w, int base) {
  if (base > w.pmax) return NONE;
  if (base + 31 <= w.pmin && (w.window < 0 || base >= w.pmax - w.window || base + 31 < w.sinks)) return ALL;
  if (w.window >= 0 && base + 31 < w.pmin - w.window && base >= w.sinks) return NONE;
  return SOME;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t seen_bits(const View& w, int base) {
  return low_bits(w.pos + 1 - base) & (~low_bits(w.lo - base) | low_bits(w.sinks - base));
}

// Largest visible score of a thread's KEYS keys of a row; base[c]: first token of its group c.
template <int KEYS>
__device__ __forceinline__ float part_max(uint32_t tS, const int (&base)[KEYS / GK], const View& w) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < KEYS / 32; ++c) {
    const int cls = chunk_class(w, base[c]);
    if (cls == NONE) continue;
    uint32_t v[32];
    tmem_ld32(tS + c * 32, v);
    wait_ld();
    if (cls == SOME) {
      const uint32_t seen = seen_bits(w, base[c]);
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (!(seen >> k & 1)) v[k] = 0xff800000u;
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) mx[k & 3] = fmaxf(mx[k & 3], __uint_as_float(v[k]));
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// P = 2^(s * sl2 - mu) as 16-bit pairs over the front of the thread's scores; returns the sum of the unrounded P.
template <int KV, int KEYS>
__device__ __forceinline__ float part_exp(uint32_t tS, float sl2, float mu, const int (&base)[KEYS / GK], const View& w) {
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < KEYS / 32; ++c) {
    const int cls = chunk_class(w, base[c]);
    uint32_t out[16];
    if (cls == NONE) {
#pragma unroll
      for (int k = 0; k < 16; ++k) out[k] = 0u;
    } else {
      uint32_t v[32];
      tmem_ld32(tS + c * 32, v);
      wait_ld();
      if (cls == SOME) {
        const uint32_t seen = seen_bits(w, base[c]);
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (!(seen >> k & 1)) v[k] = 0xff800000u;
      }
#pragma unroll
      for (int k = 0; k < 32; k += 2) {
        const float2 a = fma2(__uint_as_float(v[k]), __uint_as_float(v[k + 1]), sl2, -mu);
        const float e0 = ex2(a.x), e1 = ex2(a.y);
        add2(part[k & 2], part[(k & 2) + 1], e0, e1);
        out[k / 2] = pack16<KV>(e0, e1);
      }
    }
    tmem_st16(tS + c * 16, out);
  }
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// What the softmax warps do when a result is no number: a call, so that it takes no registers from the tiles (in line prompts hd128
// took 429 us instead of 300; a kernel behind, which finds nothing to do, costs every call 15 us).
template <class I>
__device__ __noinline__ void mend_tail(const PagedDev& p, const Req& r, int b, int h, int row0, int n, MendSmem& sm) {
  mend<I::KV, I::HD, I::SOFT_WARPS, 16>(p, r, b, h, row0, n, threadIdx.x >> 5, I::SOFT_WARPS, sm, [] { named_bar_sync(3, I::SOFT_WARPS * 32); });
}

template <class I>
__global__ void __launch_bounds__(I::NT, 1) attn_paged_tc_kernel(const __grid_constant__ PagedDev p, const int* count, const int4* list,
                                                                 const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int boxes) {
  constexpr int HD = I::HD, KV = I::KV, NQ = I::NQ, SLABS = I::SLABS, NST = I::NST, KC = I::KC;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sQ = smem_u32(smem_raw);
  const uint32_t ring = sQ + I::Q_BYTES;
  const uint32_t sX = ring + NST * STAGE;
  const uint32_t head = sX + I::X_BYTES;                     // barriers
  if (sQ & 1023u) {
    if (threadIdx.x == 0) atomicExch(p.status, GA_ST_WAIT_TMEM);
    return;
  }
  const uint32_t b_full = head, b_empty = b_full + 8 * NST;  // ring stages
  const uint32_t b_qfull = b_empty + 8 * NST, b_qempty = b_qfull + 8;
  const uint32_t b_s = b_qempty + 8, b_p = b_s + 16;         // [2] scores ready, [2] P ready
  const uint32_t b_pv = b_p + 16;                            // NQ 1: PV out of a buffer done
  const uint32_t b_ofull = b_pv + 16, b_ofree = b_ofull + 16; // [2] O complete / read
  const uint32_t slot_at = b_ofree + 16;
  const uint32_t spoilt = slot_at + 8;                       // prompts [2]: a result is no number, a wait of the softmax warps ran out
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int MMA_WARP = I::SOFT_WARPS, KV_WARP = MMA_WARP + 2, Q_WARP = KV_WARP + I::KV_WARPS;

  if (tid == 0) {
    for (int i = 0; i < NST / I::EG; ++i) {
      mbar_init(b_full + 8 * i, 32 * I::EG);
      mbar_init(b_empty + 8 * i, 1);
    }
    mbar_init(b_qfull, I::Q_WARPS * 32);
    mbar_init(b_qempty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_pv + 8 * i, 1);
      mbar_init(b_s + 8 * i, 1);
      mbar_init(b_p + 8 * i, I::SPLIT * 4);
      mbar_init(b_ofull + 8 * i, 1);
      mbar_init(b_ofree + 8 * i, I::SPLIT * 4);
    }
    mbar_fence_init();
    asm volatile("st.shared.v2.b32 [%0], {%1,%1};" ::"r"(spoilt), "r"(0) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_at), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot_at));
  grid_dep_wait();
  grid_dep_launch();

  bool failed = false;
  // The CTA's segments: parts of a row block of a prompt, or of what its gang's slice holds of a request. What the softmax warps
  // need behind a segment's tiles follows from few numbers (opens, last): they have no registers to spare.
  struct Seg {
    int b, block, h;
    int i0, i1;  // tiles of the segment
    int slot;    // split: workspace slot of the piece, or -1 - the one that a whole request's piece would have gone to
    bool first;  // split: the piece's first segment
    Req r;       // r.cnt = i1 - i0
  };
  struct Work {
    int x, end;                 // prompts: item and their number
    int b, rem, gang, h, slot;  // split: request and place in the slice, slot of the piece
    int off, left;              // first tile of the item's next segment, 0 behind its last; split: tiles left of the piece
    bool first;
  };
  auto begin = [&]() {
    Work w;
    w.off = w.left = 0;
    if (I::SPLIT_KV) {
      w.gang = blockIdx.x / p.kvh;
      w.h = blockIdx.x - w.gang * p.kvh;
      const int4 e = list[w.gang];
      w.b = e.x, w.off = e.y, w.rem = e.z;
      w.first = true;
    } else {
      w.x = blockIdx.x;
      w.end = *count * p.kvh;
    }
    return w;
  };
  auto next = [&](Work& w, Seg& s) {
    if (I::SPLIT_KV) {
      s.first = w.left == 0;
      if (s.first) {  // the next request of the slice
        if (w.rem <= 0) return false;
        s.r = I::req(p, w.b);
        while (s.r.cnt == 0) {  // requests without visible keys
          if (++w.b >= p.batch) return false;
          s.r = I::req(p, w.b);
        }
        w.left = min(s.r.cnt - w.off, w.rem);
        w.rem -= w.left;
        w.slot = (2 * w.gang + (w.first ? 0 : 1)) * p.kvh + w.h;
        if (w.left == s.r.cnt) w.slot = -1 - w.slot;
        w.first = false;
      } else {
        s.r = I::req(p, w.b);
      }
      s.b = w.b, s.block = 0, s.h = w.h;
      s.slot = w.slot;
      s.i0 = w.off, s.i1 = w.off + min(w.left, SEG_TILES);
      w.left -= s.i1 - s.i0;
      w.off = s.i1;
      if (w.left == 0) {
        w.off = 0;
        if (++w.b >= p.batch) w.rem = 0;
      }
    } else {
      if (w.x >= w.end) return false;
      const int k = w.x / p.kvh;
      s.h = w.x - k * p.kvh;
      const int4 e = list[k];
      s.b = e.x, s.block = e.y;
      const int t0 = s.block * I::ROWS / p.gqa, t1 = (s.block * I::ROWS + I::ROWS - 1) / p.gqa;
      s.r = req_info<GK>(p, s.b, t0, t1 - t0 + 1);
      const int all = (s.r.cnt + TK / GK - 1) / (TK / GK);
      s.i0 = w.off, s.i1 = min(all, w.off + SEG_TILES);
      w.off = s.i1;
      if (s.i1 == all) w.off = 0, w.x += gridDim.x;
    }
    s.r.cnt = s.i1 - s.i0;
    return true;
  };
  auto opens = [&](const Seg& s) { return I::SPLIT_KV ? s.first : s.i1 <= SEG_TILES; };
  auto last = [&](const Work& w) { return (I::SPLIT_KV ? w.left : w.off) == 0; };
  // first token of a group; groups behind the last one lie past every visible key
  auto group_at = [](const Req& r, int i) { return (i < r.ns ? i : r.tlo + i - r.ns) * GK; };

  if (warp < I::SOFT_WARPS) {
    // ------------------------------------------------------------------------------------------ softmax, epilogue
    regs_up<I::REGS_SOFT>();
    constexpr int OKV = KV == KV_E4M3 ? KV_BF16 : KV;
    constexpr int SPLIT = I::SPLIT, KEYS = TK / SPLIT, DIMS = HD / SPLIT;
    const int g = warp / (4 * SPLIT), half = (warp >> 2) % SPLIT;  // query tile, part of its keys
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lanes + I::O_COL + g * HD + half * DIMS;  // this thread's part of the output dims
    const uint32_t xm = sX + (g * 2 * TM + row) * 4;                         // [turn or query tile][half][row]
    int n = NQ == 2 ? g : 0;  // running job
    int done = 0;             // segments with jobs so far
    uint32_t turn = 0;
    auto exchange = [&](float mine, bool add) {  // maximum or sum over the threads that have the row's parts
      const uint32_t at = xm + turn * (SPLIT * TM * 4);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + half * (TM * 4)), "f"(mine) : "memory");
      named_bar_sync(1 + g, SPLIT * TM);
      float all = add ? 0.f : mine;
#pragma unroll
      for (int k = 0; k < SPLIT; ++k) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at + k * (TM * 4)) : "memory");
        all = add ? all + v : fmaxf(all, v);
      }
      if (I::TURNS == 2) turn ^= 1;  // the slot is written again behind a barrier that its reader has passed
      return all;
    };
    Work work = begin();
    Seg seg;
    while (next(work, seg)) {
      const int b = seg.b, block = seg.block, h = seg.h;
      const Req& r = seg.r;
      const int rr0 = block * I::ROWS + g * TM + (warp & 3) * 32, rr = rr0 + lane;
      const bool real = rr < r.nq * p.gqa;
      const int tok = rr / p.gqa;
      View w;
      w.pos = real ? r.pos0 + tok : -1;
      w.lo = p.window >= 0 ? w.pos - p.window : -(1 << 30);
      w.sinks = p.sinks;
      w.window = p.window;
      const bool any = rr0 < r.nq * p.gqa;  // a warp of padding rows sees nothing and looks at nothing
      w.pmin = any ? r.pos0 + rr0 / p.gqa : -1;
      w.pmax = any ? r.pos0 + (rr0 + 31) / p.gqa : -1;
      // with a negative descale the queries' signs are flipped as they are gathered; a zero one leaves every score at 0 (the
      // masked ones stay below it), one that is no number makes every score none
      float sl2 = p.scale_log2;
      if (KV == KV_E4M3 && p.kd) {
        sl2 *= fabsf(p.kd[b * p.kd_s0 + h * p.kd_s1]);
        if (sl2 == 0.f) sl2 = 1e-30f;
      }
      float ref = -INFINITY, sum = 0.f;
      for (int i = seg.i0; i < seg.i1; ++i, n += NQ) {
        const int buf = n & 1;
        const uint32_t tS = tmem + lanes + buf * TK + half * KEYS;
        wait_or_flag(b_s + 8 * buf, (n >> 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
        __syncwarp();
        fence_after();
        int base[KEYS / GK];
#pragma unroll
        for (int c = 0; c < KEYS / GK; ++c) base[c] = group_at(r, i * (TK / GK) + half * (KEYS / GK) + c);
        float mx = part_max<KEYS>(tS, base, w);
        mx = exchange(mx, false) * sl2;
        bool scale = false;
        float f = 1.f;
        if (mx > ref + RISE || (ref == -INFINITY && mx > ref)) {
          scale = ref != -INFINITY;  // until then O holds nothing of this row
          f = scale ? ex2(ref - mx) : 1.f;
          sum *= f;
          ref = mx;
        }
        if (__any_sync(0xffffffffu, scale)) {
          // NQ == 1: the PV before this job's may still be adding to O (it is waited for only here, where the barrier
          // is at most one phase ahead of what is waited for)
          if (NQ == 1) {
            wait_or_flag(b_pv + 8 * ((n - 1) & 1), ((n - 1) >> 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
            __syncwarp();
            fence_after();
          }
#pragma unroll 1
          for (int c = 0; c < DIMS / 32; ++c) {
            uint32_t v[32];
            tmem_ld32(tO + c * 32, v);
            wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
            tmem_st32(tO + c * 32, v);
          }
        }
        sum += part_exp<KV, KEYS>(tS, sl2, ref == -INFINITY ? 0.f : ref - P_REF<KV>, base, w);
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_p + 8 * buf);
      }
      if (I::TURNS == 1) named_bar_sync(1 + g, SPLIT * TM);
      sum = exchange(sum, true);
      if (I::TURNS == 1) named_bar_sync(1 + g, SPLIT * TM);
      const int qrow = r.q0 + tok, qh = h * p.gqa + rr - tok * p.gqa;
      uint8_t* dst = static_cast<uint8_t*>(p.out) +
                     (static_cast<long long>(qrow) * p.o_s0 + static_cast<long long>(qh) * p.o_s1 + half * DIMS) * 2;
      // O of the segments before, and their log2 LSE (each thread's own): in the piece's slot, or the CTA's room
      const int room = !I::SPLIT_KV ? static_cast<int>(blockIdx.x) : (seg.slot < 0 ? -1 - seg.slot : seg.slot);
      float* ws = p.ws_o + (static_cast<long long>(room) * I::ROWS + g * TM + row) * HD + half * DIMS;
      float* ws_before = p.ws_seg + static_cast<long long>(blockIdx.x) * (SPLIT * NQ * TM) + tid;
      const bool has = seg.i1 > 0;
      const bool piece = !last(work) || (I::SPLIT_KV && seg.slot >= 0);
      const float before = opens(seg) ? -INFINITY : *ws_before;
      // what is added of this segment's O and of the one before: their shares, and 1 / sum
      const bool some = sum != 0.f, more = before != -INFINITY;
      const float vds = !piece && p.vd ? p.vd[b * p.vd_s0 + h * p.vd_s1] : 1.f;
      float lse2 = some ? ref + (lg2(sum) - P_REF<KV>) : -INFINITY, mine = vds / sum, theirs = vds;
      if (more && some) {
        const float top = fmaxf(before, lse2), wb = ex2(before - top), wm = ex2(lse2 - top), one = 1.f / (wb + wm);
        mine *= wm * one;
        theirs *= wb * one;
        lse2 = top + lg2(wb + wm);
      } else if (more) {
        lse2 = before;
      }
      if (!last(work)) *ws_before = lse2;
      if (has) {
        wait_or_flag(b_ofull + 8 * g, done & 1, failed, p.status, GA_ST_WAIT_FULL);
        __syncwarp();
        fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < DIMS / 32; ++c) {
        uint32_t acc = 0;
        uint32_t v[32];
        if (has) {
          tmem_ld32(tO + c * 32, v);
          wait_ld();
        }
        if (real && !piece && !more) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            uint2 o = make_uint2(0u, 0u);
            if (some) {
              o.x = pack16<OKV>(__uint_as_float(v[k]) * mine, __uint_as_float(v[k + 1]) * mine);
              o.y = pack16<OKV>(__uint_as_float(v[k + 2]) * mine, __uint_as_float(v[k + 3]) * mine);
            }
            *reinterpret_cast<uint2*>(dst + (c * 32 + k) * 2) = o;
            look_at<OKV>(acc, o.x, o.y);
          }
        } else if (real && !more) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(ws + c * 32 + k) =
                some ? make_float4(__uint_as_float(v[k]) * mine, __uint_as_float(v[k + 1]) * mine, __uint_as_float(v[k + 2]) * mine,
                                   __uint_as_float(v[k + 3]) * mine)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (real) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (some)
              o = make_float4(__uint_as_float(v[k]) * mine, __uint_as_float(v[k + 1]) * mine, __uint_as_float(v[k + 2]) * mine,
                              __uint_as_float(v[k + 3]) * mine);
            float4* at = reinterpret_cast<float4*>(ws + c * 32 + k);
            const float4 w = *at;
            o.x += w.x * theirs, o.y += w.y * theirs, o.z += w.z * theirs, o.w += w.w * theirs;
            if (piece) {
              *at = o;
            } else {
              const uint2 u = make_uint2(pack16<OKV>(o.x, o.y), pack16<OKV>(o.z, o.w));
              *reinterpret_cast<uint2*>(dst + (c * 32 + k) * 2) = u;
              look_at<OKV>(acc, u.x, u.y);
            }
          }
        }
        if (not_finite<OKV>(acc)) {
          if (I::SPLIT_KV) p.ws_spoilt[blockIdx.x] = 1;  // for the combine kernel
          else asm volatile("st.shared.b32 [%0], %1;" ::"r"(spoilt), "r"(1) : "memory");
        }
      }
      if (real && half == 0 && last(work)) {
        if (I::SPLIT_KV && seg.slot >= 0) p.ws_lse[static_cast<long long>(seg.slot) * TM + row] = lse2;
        else if (p.lse) p.lse[static_cast<long long>(qh) * p.total_q + qrow] = lse2 * 0.6931471805599453f;
      }
      if (has) {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_ofree + 8 * g);
        ++done;
      }
    }
    if (!I::SPLIT_KV) {  // the CTA's blocks once more if need be; the operands' shared memory is free
      if (failed) asm volatile("st.shared.b32 [%0], %1;" ::"r"(spoilt + 4), "r"(1) : "memory");
      named_bar_sync(3, I::SOFT_WARPS * 32);
      uint32_t any, lost;  // (where a wait ran out copies may still be on their way)
      asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(any), "=r"(lost) : "r"(spoilt) : "memory");
      if (any && !lost) {
        auto& sm = *reinterpret_cast<MendSmem*>(smem_raw);
        Work again = begin();
        Seg s;
        while (next(again, s)) {
          const int row0 = s.block * I::ROWS;
          if (last(again)) mend_tail<I>(p, s.r, s.b, s.h, row0, min(s.r.nq * p.gqa - row0, I::ROWS), sm);
        }
      }
    }
  } else {
  regs_down<I::REGS_REST>();
  if (warp < KV_WARP) {
    // ------------------------------------------------------------------------------------------------- MMA issue
    // NQ 2: one lane issues for both query tiles in turn (a lane for each: 4 x 4096 causal tokens 1064 us instead of 897). NQ 1: one lane for the QK
    // MMAs, one for the PV MMAs; a QK waits for the PV two tiles before, whose P it overwrites.
    const int role = warp - MMA_WARP;
    if (lane == 0 && (NQ == 1 || role == 0)) {
      const uint32_t id_qk = instr_desc(KV, TM, TK, 0), id_pv = instr_desc(KV, TM, HD, 1);
      const uint64_t dq = smem_desc(sQ, 16, 1024);
      const uint64_t dk = smem_desc(ring, 16, 1024), dv = smem_desc(ring, KC * 128, 1024);
      // column of P's key `key` in its buffer: every part of the keys lies over the front of its own scores
      auto p_col = [](int key) { return key / (TK / I::SPLIT) * (TK / I::SPLIT) + key % (TK / I::SPLIT) / 2; };
      int unit = 0;         // K and V tiles of the items before, in ring order
      int n = 0, done = 0;  // NQ 1: first job of the item; items with jobs so far
      auto qk = [&](int u, int g, int buf, bool release) {
        int at = u * SLABS % NST;
        uint32_t par = (u * SLABS / NST) & 1;
#pragma unroll
        for (int s = 0; s < SLABS; s += I::EG) {
          wait_or_flag(b_full + 8 * (at / I::EG), par, failed, p.status, GA_ST_WAIT_FULL);
          if (failed) return;
          fence_after();
#pragma unroll
          for (int e = 0; e < I::EG; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(tmem + buf * TK, dq + (((g * SLABS + s + e) * STAGE + k * 32) >> 4), dk + (((at + e) * STAGE + k * 32) >> 4), id_qk, s + e > 0 || k > 0);
          if (s + I::EG == SLABS) commit(b_s + 8 * buf);
          if (release) commit(b_empty + 8 * (at / I::EG));
          at += I::EG;
          if (at == NST) at = 0, par ^= 1;
        }
      };
      auto pv = [&](int u, int g, int buf, bool opens, bool release) {
        int at = u * SLABS % NST;
        uint32_t par = (u * SLABS / NST) & 1;
#pragma unroll
        for (int s = 0; s < SLABS; s += I::EG) {
          wait_or_flag(b_full + 8 * (at / I::EG), par, failed, p.status, GA_ST_WAIT_FULL);
          if (failed) return;
          fence_after();
#pragma unroll
          for (int e = 0; e < I::EG; ++e)
#pragma unroll
            for (int k = 0; k < KC / 16; ++k)
              mma_ts(tmem + I::O_COL + g * HD, tmem + buf * TK + p_col((s + e) * KC + k * 16), dv + (((at + e) * STAGE + k * 2048) >> 4), id_pv,
                     !opens || s + e > 0 || k > 0);
          if (release) commit(b_empty + 8 * (at / I::EG));
          at += I::EG;
          if (at == NST) at = 0, par ^= 1;
        }
      };
      Work work = begin();
      Seg seg;
      while (!failed && next(work, seg)) {
        const Req& r = seg.r;
        if (r.cnt == 0) continue;
        if (NQ == 2) {
          wait_or_flag(b_qfull, done & 1, failed, p.status, GA_ST_WAIT_FULL);
          fence_after();
          qk(unit, 0, 0, false);
          qk(unit, 1, 1, true);
          if (r.cnt == 1 && !failed) commit(b_qempty);
          for (int j = 0; j < 2 * r.cnt && !failed; ++j) {
            const int g = j & 1, i = j >> 1;
            if (i == 0 && done > 0) wait_or_flag(b_ofree + 8 * g, (done - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
            wait_or_flag(b_p + 8 * g, (n + i) & 1, failed, p.status, GA_ST_WAIT_FULL);
            if (failed) break;
            fence_after();
            pv(unit + 2 * i + 1, g, g, i == 0, g == 1);
            if (i == r.cnt - 1) commit(b_ofull + 8 * g);
            if (i + 1 < r.cnt) qk(unit + 2 * i + 2, g, g, g == 1);
            if (j == 2 * r.cnt - 3) commit(b_qempty);
          }
        } else if (role == 0) {
          wait_or_flag(b_qfull, done & 1, failed, p.status, GA_ST_WAIT_FULL);
          fence_after();
          for (int i = 0; i < r.cnt && !failed; ++i) {
            const int buf = (n + i) & 1;
            if (n + i >= 2) wait_or_flag(b_pv + 8 * buf, ((n + i - 2) >> 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
            qk(unit + (i == 0 ? 0 : 2 * i - 1), 0, buf, true);
          }
          if (!failed) commit(b_qempty);
        } else {
          for (int i = 0; i < r.cnt && !failed; ++i) {
            const int buf = (n + i) & 1;
            if (i == 0 && done > 0) wait_or_flag(b_ofree, (done - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
            wait_or_flag(b_p + 8 * buf, ((n + i) >> 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
            fence_after();
            pv(unit + (i == r.cnt - 1 ? 2 * i + 1 : 2 * i + 2), 0, buf, i == 0, true);
            commit(b_pv + 8 * buf);
          }
          if (!failed) commit(b_ofull);
        }
        n += r.cnt;
        unit += 2 * r.cnt;
        ++done;
      }
    }
    __syncwarp();
  } else if (warp < Q_WARP) {
    // ------------------------------------------------------------------------------------------------ K / V gather
    const int w = warp - KV_WARP;
    int q = 0;           // running stage
    int pending = -1;    // stage filled by cp.async that are still in flight
    auto signal = [&]() {
      fence_proxy_async();
      mbar_arrive(b_full + 8 * (pending % NST / I::EG));
      pending = -1;
    };
    auto wait_stage = [&](int at, int turn) {
      const uint32_t empty = b_empty + 8 * (at / I::EG);
      if (turn > 0 && !failed && !mbar_test_wait(empty, (turn - 1) & 1)) {
        if (pending >= 0) {  // nothing may wait for what this warp holds back
          cp_async_wait<0>();
          signal();
        }
        wait_or_flag(empty, (turn - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
      }
      failed = __any_sync(0xffffffffu, failed);
    };
    auto stage_for = [&](const Req& r, int b, int h, int tile, int part, bool is_v) {
      if (q % I::KV_WARPS == w) {
        constexpr int MOST = TK / GK;
        const int keys = is_v ? KC : TK;
        int n0[MOST];
        bool inside = boxes != 0;  // every key of the stage is a real one
#pragma unroll
        for (int u = 0; u < MOST; ++u) {
          n0[u] = group_at(r, tile * MOST + (is_v ? part * (KC / GK) : 0) + u);
          if (KV != KV_E4M3 && u * GK < keys) inside &= n0[u] + GK <= r.kend && (n0[u] >= r.lower || n0[u] + GK <= p.sinks);
        }
        if (KV != KV_E4M3 && inside) {  // whole boxes of pages by TMA
          const int box = min(p.page_mask + 1, GK), nb = keys / box;
          const int k = lane % nb, slab = lane / nb;
          const int gu = k * box / GK;
          const int at_key = (gu == 0 ? n0[0] : gu == 1 ? n0[1] : gu == 2 ? n0[2] : n0[3]) + k * box % GK;
          const int pg = p.pt[b * p.pt_s0 + (at_key >> p.page_shift) * p.pt_s1];
          const int at = q % NST, turn = q / NST;
          wait_stage(at, turn);
          if (__all_sync(0xffffffffu, pg >= 0 && pg < p.num_pages)) {
            const uint32_t full = b_full + 8 * (at / I::EG);
            if (lane == 0) mbar_expect_tx_only(full, STAGE);
            __syncwarp();
            if (slab < (is_v ? SLABS : 1))
              tma_load_4d(ring + at * STAGE + slab * (KC * 128) + k * box * 128, is_v ? &vmap : &kmap, full, (is_v ? slab : part) * 64,
                          at_key & p.page_mask, h, pg);
            if (pending >= 0) {
              cp_async_wait<0>();
              signal();
            }
            mbar_arrive(full);
            ++q;
            return;
          }
        }
        int page[MOST];
#pragma unroll
        for (int u = 0; u < MOST; ++u) {
          const int n = n0[u] + lane;
          page[u] = -1;
          if (u * GK < keys && n < r.kend && (n >= r.lower || n < p.sinks)) {
            page[u] = p.pt[b * p.pt_s0 + (n >> p.page_shift) * p.pt_s1];
            if (page[u] < 0 || page[u] >= p.num_pages) {
              atomicExch(p.status, GA_ST_BAD_PAGE);
              page[u] = -1;
            }
          }
        }
        const int at = q % NST, turn = q / NST;
        wait_stage(at, turn);
        const uint32_t dst = ring + at * STAGE;
        if (KV == KV_E4M3) {
          if (!is_v) gather_e4m3<4, TK>(dst, p.k + h * p.k_s2 + part * 64, p.k_s0, p.k_s1, n0, p.page_mask, page, lane);
          else gather_e4m3<HD / 16, KC>(dst, p.v + h * p.v_s2, p.v_s0, p.v_s1, n0, p.page_mask, page, lane);
          pending = q;
          signal();
          ++q;
          return;
        }
        if (!is_v) gather<8, TK>(dst, p.k + h * p.k_s2 + part * 128, p.k_s0, p.k_s1, n0, p.page_shift, p.page_mask, page, lane);
        else gather<HD / 8, KC>(dst, p.v + h * p.v_s2, p.v_s0, p.v_s1, n0, p.page_shift, p.page_mask, page, lane);
        cp_async_commit();
        if (pending >= 0) {
          cp_async_wait<1>();
          signal();
        }
        pending = q;
      }
      ++q;
    };
    Work work = begin();
    Seg seg;
    while (!failed && next(work, seg)) {
      const int b = seg.b, h = seg.h;
      const Req& r = seg.r;
      constexpr int AHEAD = NQ == 1 ? 2 : 1;  // K tiles in front of the V tile they go with
      for (int i = 0; i < r.cnt + AHEAD; ++i) {
        if (i >= AHEAD)
          for (int s = 0; s < SLABS; ++s) stage_for(r, b, h, seg.i0 + i - AHEAD, s, true);
        if (i < r.cnt)
          for (int s = 0; s < SLABS; ++s) stage_for(r, b, h, seg.i0 + i, s, false);
      }
    }
    if (pending >= 0) {
      cp_async_wait<0>();
      signal();
    }
  } else if (warp < Q_WARP + I::Q_WARPS) {
    // ---------------------------------------------------------------------------------------------------- Q gather
    const int w = warp - Q_WARP;
    int done = 0;
    Work work = begin();
    Seg seg;
    while (!failed && next(work, seg)) {
      const int block = seg.block, h = seg.h;
      const Req& r = seg.r;
      if (r.cnt == 0) continue;
      if (done > 0) wait_or_flag(b_qempty, (done - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
      failed = __any_sync(0xffffffffu, failed);
      const int rows = r.nq * p.gqa - block * I::ROWS;
      const int c = lane & 7;
      for (int part = w; part < NQ * 4; part += I::Q_WARPS) {  // 32 rows
        const int mine = part * 32 + lane;
        const int rr = block * I::ROWS + mine, tok = rr / p.gqa;
        const long long off = mine < rows ? static_cast<long long>(r.q0 + tok) * p.q_s0 + static_cast<long long>(h * p.gqa + rr - tok * p.gqa) * p.q_s1 : -1;
        const uint32_t tile = sQ + (part >> 2) * (SLABS * STAGE);
        if (KV == KV_E4M3) {
          constexpr int CPR = HD / 16;  // 16 values at a time
          const uint32_t flip = p.kd && p.kd[seg.b * p.kd_s0 + h * p.kd_s1] < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
          for (int it = 0; it < CPR; ++it) {
            const int e = it * 32 + lane, k = e / CPR, ch = e % CPR;
            const long long o = __shfl_sync(0xffffffffu, off, k);
            const int row = (part & 3) * 32 + k;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (o >= 0 && p.q_kind == Q_BF16_TO_E4M3) {
              const uint4* s = reinterpret_cast<const uint4*>(p.q + (o + ch * 16) * 2);
              const uint4 a = s[0], b = s[1];
              auto four = [](uint32_t x, uint32_t y) {
                return pack_e4m3x4(bf16_bits_to_f32(x & 0xffffu), bf16_bits_to_f32(x >> 16), bf16_bits_to_f32(y & 0xffffu), bf16_bits_to_f32(y >> 16));
              };
              v = make_uint4(four(a.x, a.y), four(a.z, a.w), four(b.x, b.y), four(b.z, b.w));
            } else if (o >= 0) {
              v = *reinterpret_cast<const uint4*>(p.q + o + ch * 16);
            }
            store_e4m3x16(tile + (ch >> 2) * STAGE + row * 128, (ch & 3) * 2, row & 7, v, flip);
          }
          continue;
        }
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int k = it * 4 + (lane >> 3);
          const long long o = __shfl_sync(0xffffffffu, off, k);
          const int row = (part & 3) * 32 + k;
#pragma unroll
          for (int s = 0; s < SLABS; ++s)
            cp_async_16_or_zero(tile + s * STAGE + row * 128 + ((c ^ (row & 7)) << 4), p.q + (o >= 0 ? o * 2 : 0) + s * 128 + c * 16, o >= 0);
        }
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_proxy_async();
      mbar_arrive(b_qfull);
      ++done;
    }
  }
  }
  // Every MMA has completed where its result was waited for: the softmax groups waited for O of the last item.
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace tc
}  // namespace paged
}  // namespace ga
