// Prompts over paged 16-bit caches on the tensor cores (tcgen05, kind::f16, accumulators in tensor memory): the same
// mathematics as attn_paged.cuh, for calls with enough query rows to fill 128-row tiles.
//
// A persistent CTA takes work items of NQ tiles of 128 query rows (row = token * GQA + head, one kv head) against tiles of
// 128 keys. Roles: a softmax group of four warps per query tile (a thread owns one row), one warp whose elected lane
// issues every MMA, four warps that gather K and V, two that gather Q.
//   * S = Q K^T into one of two 128-column score buffers, softmax in place, P as 16-bit pairs over the front half of the
//     buffer it came from, O += P V with P as the A operand from tensor memory and V as an MN-major B operand, i.e. the
//     page's [token, dim] layout as it is. Score buffers alternate job by job; a job is (key tile, query tile): at
//     head_dim <= 128 two query tiles share every K and V tile (NQ = 2), at 256 one query tile (O alone takes half of
//     tensor memory) has two key tiles in flight.
//   * The MMAs of a job are issued in an order that needs few barriers: PV(n), then QK(n + 2) into the same buffer. One
//     thread issues them all and the pipe runs them in order, so scores that are ready say that the PV two jobs before is.
//   * The row's reference maximum moves only when a tile exceeds it by more than 2^8 (P stays below 256, exact in the
//     sums; the 16-bit rounding of P is relative), so O is rescaled in tensor memory in few tiles.
//   * K and V come through one ring of 16 KB stages in the order in which the MMAs use them: a K stage is 128 keys x 64
//     dims, a V stage 8192 / head_dim keys x all dims. Stages are filled with 16-byte cp.async (any page size, stride and
//     alignment of 16 bytes; rows no query of the item sees, released pages among them, are filled with zeros), in the
//     128-byte swizzle that the MMA descriptors name.
// Tiles are the sinks' first, then the run that ends with the item's last visible key (Req). Items come from a list that a
// small kernel lays out, later row blocks of a request first (they see more keys), all kv heads of a block side by side
// (they share pages).
#pragma once

#include "attn_paged.cuh"

namespace ga {
namespace paged {
namespace tc {

constexpr int TM = 128;          // query rows of a tile = tensor memory lanes
constexpr int TK = 128;          // keys of a tile
constexpr int STAGE = 16384;
constexpr int KV_WARPS = 4, Q_WARPS = 2;
constexpr float RISE = 8.f;      // log2: how far a row's maximum may exceed the reference before O is rescaled

template <int HD_, int KV_>
struct TcInst {
  static constexpr int HD = HD_, KV = KV_;
  static constexpr int NQ = HD == 256 ? 1 : 2;
  static constexpr int SLABS = HD / 64;            // K stages of a tile, and V stages
  static constexpr int KC = 8192 / HD;             // keys of a V stage
  static constexpr int ROWS = NQ * TM;
  static constexpr int Q_BYTES = NQ * SLABS * STAGE;
  static constexpr int NST = HD == 64 ? 8 : 10;
  static constexpr int SOFT_WARPS = 4 * NQ;
  static constexpr int WARPS = SOFT_WARPS + 1 + KV_WARPS + Q_WARPS;
  static constexpr int NT = WARPS * 32;
  static constexpr int SMEM = 2048 + Q_BYTES + NST * STAGE;  // barriers, 1024-byte alignment
  static constexpr int O_COL = 256;
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

// The call's row blocks: blocks[0] = how many, then (request, row block) pairs, a request's last block first.
template <int ROWS>
__global__ void __launch_bounds__(1024) plan_prompts_kernel(const __grid_constant__ PagedDev p, int* count, int2* blocks) {
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
      for (int k = lane; k < m; k += 32) blocks[to + k] = make_int2(b0 + warp * 32 + src, m - 1 - k);
    }
    __syncthreads();
    if (tid == 0) base += total;
    __syncthreads();
  }
  if (tid == 0) *count = base;
}

template <class I>
__global__ void __launch_bounds__(I::NT, 1) attn_paged_tc_kernel(const __grid_constant__ PagedDev p, const int* count, const int2* blocks) {
  constexpr int HD = I::HD, KV = I::KV, NQ = I::NQ, SLABS = I::SLABS, NST = I::NST, KC = I::KC;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t head = (raw + 15u) & ~15u;                  // barriers
  const uint32_t sQ = (head + 512 + 1023u) & ~1023u;
  const uint32_t ring = sQ + I::Q_BYTES;
  const uint32_t b_full = head, b_empty = b_full + 8 * NST;  // ring stages
  const uint32_t b_qfull = b_empty + 8 * NST, b_qempty = b_qfull + 8;
  const uint32_t b_s = b_qempty + 8, b_p = b_s + 16;         // [2] scores ready, [2] P ready
  const uint32_t b_pv = b_p + 16;                            // PV of a job done
  const uint32_t b_ofull = b_pv + 8, b_ofree = b_ofull + 16; // [2] O complete / read
  const uint32_t slot_at = b_ofree + 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int MMA_WARP = I::SOFT_WARPS, KV_WARP = MMA_WARP + 1, Q_WARP = KV_WARP + KV_WARPS;

  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(b_full + 8 * i, 32);
      mbar_init(b_empty + 8 * i, 1);
    }
    mbar_init(b_qfull, Q_WARPS * 32);
    mbar_init(b_qempty, 1);
    mbar_init(b_pv, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_s + 8 * i, 1);
      mbar_init(b_p + 8 * i, TM);
      mbar_init(b_ofull + 8 * i, 1);
      mbar_init(b_ofree + 8 * i, TM);
    }
    mbar_fence_init();
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

  const int items = *count * p.kvh;
  bool failed = false;
  auto item_of = [&](int x, int& b, int& block, int& h, Req& r) {
    const int k = x / p.kvh;
    h = x - k * p.kvh;
    const int2 e = blocks[k];
    b = e.x;
    block = e.y;
    const int t0 = block * I::ROWS / p.gqa, t1 = (block * I::ROWS + I::ROWS - 1) / p.gqa;
    r = req_info<TK>(p, b, t0, t1 - t0 + 1);
  };
  auto tile_at = [](const Req& r, int i) { return (i < r.ns ? i : r.tlo + i - r.ns) * TK; };

  if (warp < I::SOFT_WARPS) {
    // ------------------------------------------------------------------------------------------ softmax, epilogue
    const int g = warp >> 2;  // query tile
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lanes + I::O_COL + g * HD;
    int n = NQ == 2 ? g : 0;  // running job
    int done = 0;             // items with jobs so far
    for (int x = blockIdx.x; x < items; x += gridDim.x) {
      int b, block, h;
      Req r;
      item_of(x, b, block, h, r);
      const int rr = block * I::ROWS + g * TM + row;
      const bool real = rr < r.nq * p.gqa;
      const int tok = rr / p.gqa;
      const int pos = real ? r.pos0 + tok : -1;
      const int first = r.pos0 + (block * I::ROWS + g * TM) / p.gqa;  // positions of the tile's first and last row
      const int last = r.pos0 + (block * I::ROWS + g * TM + TM - 1) / p.gqa;
      const int lo = p.window >= 0 ? pos - p.window : -(1 << 30);
      const float sl2 = p.scale_log2;
      float ref = -INFINITY, sum = 0.f;
      for (int i = 0; i < r.cnt; ++i, n += NQ) {
        const int buf = n & 1;
        const uint32_t tS = tmem + lanes + buf * TK;
        wait_or_flag(b_s + 8 * buf, (n >> 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
        __syncwarp();
        fence_after();
        const int n0 = tile_at(r, i);
        const bool open = n0 + TK - 1 <= first && (p.window < 0 || n0 >= last - p.window || n0 + TK <= p.sinks);
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(tS + c * 32, v);
          wait_ld();
          if (open) {
#pragma unroll
            for (int k = 0; k < 32; ++k) mx = fmaxf(mx, __uint_as_float(v[k]));
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const int key = n0 + c * 32 + k;
              if (key <= pos && (key >= lo || key < p.sinks)) mx = fmaxf(mx, __uint_as_float(v[k]));
            }
          }
        }
        mx *= sl2;
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
            wait_or_flag(b_pv, (n - 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
            __syncwarp();
            fence_after();
          }
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t v[32];
            tmem_ld32(tO + c * 32, v);
            wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
            tmem_st32(tO + c * 32, v);
          }
        }
        const float mu = ref == -INFINITY ? 0.f : ref;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32], w[16];
          tmem_ld32(tS + c * 32, v);
          wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float e[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float a = fmaf(__uint_as_float(v[k + u]), sl2, -mu);
              if (!open) {
                const int key = n0 + c * 32 + k + u;
                if (!(key <= pos && (key >= lo || key < p.sinks))) a = -INFINITY;
              }
              e[u] = ex2(a);
              part[(k + u) & 3] += e[u];
            }
            w[k / 2] = pack16<KV>(e[0], e[1]);
          }
          tmem_st16(tS + c * 16, w);
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        wait_st();
        fence_before();
        mbar_arrive(b_p + 8 * buf);
      }
      const int qrow = r.q0 + tok, qh = h * p.gqa + rr - tok * p.gqa;
      uint8_t* dst = static_cast<uint8_t*>(p.out) + (static_cast<long long>(qrow) * p.o_s0 + static_cast<long long>(qh) * p.o_s1) * 2;
      const float vds = p.vd ? p.vd[b * p.vd_s0 + h * p.vd_s1] : 1.f;
      const float inv = sum == 0.f ? 0.f : vds / sum;
      if (r.cnt > 0) {
        wait_or_flag(b_ofull + 8 * g, done & 1, failed, p.status, GA_ST_WAIT_FULL);
        __syncwarp();
        fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        if (r.cnt > 0) {
          tmem_ld32(tO + c * 32, v);
          wait_ld();
        }
        if (real) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            uint2 w = make_uint2(0u, 0u);
            if (r.cnt > 0 && sum != 0.f) {
              w.x = pack16<KV>(__uint_as_float(v[k]) * inv, __uint_as_float(v[k + 1]) * inv);
              w.y = pack16<KV>(__uint_as_float(v[k + 2]) * inv, __uint_as_float(v[k + 3]) * inv);
            }
            *reinterpret_cast<uint2*>(dst + (c * 32 + k) * 2) = w;
          }
        }
      }
      if (real && p.lse)
        p.lse[static_cast<long long>(qh) * p.total_q + qrow] = sum == 0.f ? -INFINITY : (ref + lg2(sum)) * 0.6931471805599453f;
      if (r.cnt > 0) {
        fence_before();
        mbar_arrive(b_ofree + 8 * g);
        ++done;
      }
    }
  } else if (warp == MMA_WARP) {
    // -------------------------------------------------------------------------------------------------- MMA issue
    if (lane == 0) {
      const uint32_t id_qk = instr_desc(KV, TM, TK, 0), id_pv = instr_desc(KV, TM, HD, 1);
      const uint64_t dq = smem_desc(sQ, 16, 1024);
      const uint64_t dk = smem_desc(ring, 16, 1024), dv = smem_desc(ring, KC * 128, 1024);
      int rp = 0, use = 0;  // ring position of the next stage and how often the ring went round
      int n = 0, done = 0;  // first job of the item, items with jobs so far
      auto take = [&]() {   // the next stage in ring order, filled
        const int at = rp;
        wait_or_flag(b_full + 8 * at, use & 1, failed, p.status, GA_ST_WAIT_FULL);
        if (++rp == NST) rp = 0, ++use;
        return at;
      };
      for (int x = blockIdx.x; x < items && !failed; x += gridDim.x) {
        int b, block, h;
        Req r;
        item_of(x, b, block, h, r);
        if (r.cnt == 0) continue;
        const int jobs = r.cnt * NQ;
        int ks[SLABS], vs[SLABS];
        auto qk = [&](int j) {
          const int g = NQ == 2 ? j & 1 : 0, buf = (n + j) & 1;
          if (NQ == 1 || g == 0) {
#pragma unroll
            for (int s = 0; s < SLABS; ++s) ks[s] = take();
            fence_after();
          }
          if (failed) return;
#pragma unroll
          for (int s = 0; s < SLABS; ++s)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(tmem + buf * TK, dq + (((g * SLABS + s) * STAGE + k * 32) >> 4), dk + ((ks[s] * STAGE + k * 32) >> 4), id_qk, s > 0 || k > 0);
          commit(b_s + 8 * buf);
          if (NQ == 1 || g == 1)
#pragma unroll
            for (int s = 0; s < SLABS; ++s) commit(b_empty + 8 * ks[s]);
          if (j == jobs - 1) commit(b_qempty);
        };
        wait_or_flag(b_qfull, done & 1, failed, p.status, GA_ST_WAIT_FULL);
        fence_after();
        qk(0);
        if (jobs > 1) qk(1);
        for (int j = 0; j < jobs && !failed; ++j) {
          const int g = NQ == 2 ? j & 1 : 0, buf = (n + j) & 1;
          const bool opens = j < NQ;
          if (NQ == 1 || g == 0) {
#pragma unroll
            for (int s = 0; s < SLABS; ++s) vs[s] = take();
          }
          if (opens && done > 0) wait_or_flag(b_ofree + 8 * g, (done - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
          wait_or_flag(b_p + 8 * buf, ((n + j) >> 1) & 1, failed, p.status, GA_ST_WAIT_FULL);
          if (failed) break;
          fence_after();
#pragma unroll
          for (int s = 0; s < SLABS; ++s)
#pragma unroll
            for (int k = 0; k < KC / 16; ++k)
              mma_ts(tmem + I::O_COL + g * HD, tmem + buf * TK + s * (KC / 2) + k * 8, dv + ((vs[s] * STAGE + k * 2048) >> 4), id_pv,
                     !opens || s > 0 || k > 0);
          if (NQ == 1) commit(b_pv);
          if (NQ == 1 || g == 1)
#pragma unroll
            for (int s = 0; s < SLABS; ++s) commit(b_empty + 8 * vs[s]);
          if (j >= jobs - NQ) commit(b_ofull + 8 * g);
          if (j + 2 < jobs) qk(j + 2);
        }
        n += jobs;
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
      mbar_arrive(b_full + 8 * (pending % NST));
      pending = -1;
    };
    auto stage_for = [&](const Req& r, int b, int h, int tile, int part, bool is_v) {
      if (q % KV_WARPS == w) {
        const int at = q % NST, turn = q / NST;
        if (turn > 0 && !failed && !mbar_test_wait(b_empty + 8 * at, (turn - 1) & 1)) {
          if (pending >= 0) {  // nothing may wait for what this warp holds back
            cp_async_wait<0>();
            signal();
          }
          wait_or_flag(b_empty + 8 * at, (turn - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
        }
        failed = __any_sync(0xffffffffu, failed);
        const uint32_t dst = ring + at * STAGE;
        const int n0 = tile_at(r, tile) + (is_v ? part * KC : 0);
        constexpr int MOST = 128 / 32;
        int page[MOST];
        const int keys = is_v ? KC : TK;
#pragma unroll
        for (int u = 0; u < MOST; ++u) {
          const int n = n0 + u * 32 + lane;
          page[u] = -1;
          if (u * 32 < keys && n < r.kend && (n >= r.lower || n < p.sinks)) {
            page[u] = p.pt[b * p.pt_s0 + (n >> p.page_shift) * p.pt_s1];
            if (page[u] < 0 || page[u] >= p.num_pages) {
              atomicExch(p.status, GA_ST_BAD_PAGE);
              page[u] = -1;
            }
          }
        }
        const uint8_t* base = (is_v ? p.v + h * p.v_s2 : p.k + h * p.k_s2 + part * 128);
        const long long s0 = is_v ? p.v_s0 : p.k_s0, s1 = is_v ? p.v_s1 : p.k_s1;
        if (!is_v) {
          // 128 keys x 64 dims: eight chunks a key, four keys an instruction
          const int c = lane & 7;
#pragma unroll
          for (int it = 0; it < 32; ++it) {
            const int key = it * 4 + (lane >> 3);
            const int pg = __shfl_sync(0xffffffffu, page[it / 8], key & 31);
            const bool real = pg >= 0;
            const uint8_t* src = base + (real ? pg * s0 + ((n0 + key) & p.page_mask) * s1 : 0) + c * 16;
            cp_async_16_or_zero(dst + key * 128 + ((c ^ (key & 7)) << 4), src, real);
          }
        } else {
          // KC keys x HD dims: HD / 8 chunks a key
          constexpr int CPK = HD / 8, KPI = 32 / CPK;  // chunks a key, keys an instruction
          const int c = lane % CPK;
#pragma unroll
          for (int it = 0; it < KC / KPI; ++it) {
            const int key = it * KPI + lane / CPK;
            const int pg = __shfl_sync(0xffffffffu, page[it * KPI / 32], key & 31);
            const bool real = pg >= 0;
            const uint8_t* src = base + (real ? pg * s0 + ((n0 + key) & p.page_mask) * s1 : 0) + c * 16;
            cp_async_16_or_zero(dst + (c >> 3) * (KC * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4), src, real);
          }
        }
        cp_async_commit();
        if (pending >= 0) {
          cp_async_wait<1>();
          signal();
        }
        pending = q;
      }
      ++q;
    };
    for (int x = blockIdx.x; x < items && !failed; x += gridDim.x) {
      int b, block, h;
      Req r;
      item_of(x, b, block, h, r);
      constexpr int AHEAD = NQ == 1 ? 2 : 1;  // K tiles in front of the V tile they go with
      for (int i = 0; i < r.cnt + AHEAD; ++i) {
        if (i >= AHEAD)
          for (int s = 0; s < SLABS; ++s) stage_for(r, b, h, i - AHEAD, s, true);
        if (i < r.cnt)
          for (int s = 0; s < SLABS; ++s) stage_for(r, b, h, i, s, false);
      }
    }
    if (pending >= 0) {
      cp_async_wait<0>();
      signal();
    }
  } else {
    // ---------------------------------------------------------------------------------------------------- Q gather
    const int w = warp - Q_WARP;
    int done = 0;
    for (int x = blockIdx.x; x < items && !failed; x += gridDim.x) {
      int b, block, h;
      Req r;
      item_of(x, b, block, h, r);
      if (r.cnt == 0) continue;
      if (done > 0) wait_or_flag(b_qempty, (done - 1) & 1, failed, p.status, GA_ST_WAIT_EMPTY);
      failed = __any_sync(0xffffffffu, failed);
      const int rows = r.nq * p.gqa - block * I::ROWS;
      const int c = lane & 7;
      for (int part = w; part < NQ * 4; part += Q_WARPS) {  // 32 rows
        const int mine = part * 32 + lane;
        const int rr = block * I::ROWS + mine, tok = rr / p.gqa;
        const long long off = mine < rows ? static_cast<long long>(r.q0 + tok) * p.q_s0 + static_cast<long long>(h * p.gqa + rr - tok * p.gqa) * p.q_s1 : -1;
        const uint32_t tile = sQ + (part >> 2) * (SLABS * STAGE);
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
  // Every MMA has completed where its result was waited for: the softmax groups waited for O of the last item.
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace tc
}  // namespace paged
}  // namespace ga
