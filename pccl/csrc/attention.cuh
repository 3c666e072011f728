// What the attention kernels share: tensor-core instructions on 128-row tiles, the walk over packed sequences, bounded
// waits, tensor maps.
//
// Tiles.  A tile is 128 rows (queries or keys) of one head, staged by TMA as DP / 64 blocks of 128 rows x 64 columns (rows of
// 128 bytes, 128-byte swizzle); DP is the head size rounded up to 64 or 128, and the copy fills the missing columns with
// zeros, which add nothing to any product.  The same bytes serve as an operand whose contraction runs along the columns
// (K-major: q k^T, do v^T) and as one whose contraction runs along the rows (MN-major: p v, ds k, p^T do, ds^T q).
// Probabilities and score gradients never leave the SM: they are written as 16-bit words over the accumulator columns
// that they were computed from, and the second product reads them from tensor memory as its first operand.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "act.cuh"
#include "attention.h"
#include "bulk.cuh"
#include "pdl.cuh"
#include "primitives.cuh"

namespace pccl {
namespace attn {

constexpr uint32_t kBlockBytes = 128 * 128;          // 128 rows x 64 columns of 16 bits
constexpr uint64_t kWaitNs = 4ull * 1000 * 1000 * 1000;
constexpr int kErrLoad = 1, kErrMma = 2, kErrCompute = 3;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Bounded wait that also gives up when another role has failed.  The clock is first read after some polls: reading the
// global timer takes longer than most waits here.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 255u) == 255u) {
      if (*abort_flag != 0) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > kWaitNs) return false;
    }
  }
}
// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag)) != 0;
}

__device__ __forceinline__ void load_block(void* dst, const CUtensorMap* map, int col, int head, int row, int batch, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(col), "r"(head), "r"(row), "r"(batch)
      : "memory");
}
// One tile of DP columns; the barrier's transaction count has been raised by the caller.
template <int DP>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, int head, int row, int batch, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) load_block(dst + c * kBlockBytes, map, c * 64, head, row, batch, bar);
}
// Rows [first, 128) of a tile to zero, by the whole warp.  Rows behind a packed sequence belong to its neighbour, and as the
// contraction index of a product they meet weights of zero there: what is infinite or NaN in them would make the product NaN.
template <int DP>
__device__ __forceinline__ void clear_rows(unsigned char* tile, int first) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < DP / 64; ++c)
    for (int i = first * 8 + lane; i < 128 * 8; i += 32) reinterpret_cast<uint4*>(tile + c * kBlockBytes)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// Shared-memory descriptors as two words; only the low one (address, leading byte offset) changes.  Stride byte offset 1024
// (eight rows of 128 bytes); leading byte offset of a row-contracted tile: from one block of 64 columns to the next.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) + (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) + ((kBlockBytes >> 4) << 16); }

// Instruction descriptor: fp32 accumulator, 16-bit operands of one type, 128 rows, N columns.
__host__ __device__ constexpr uint32_t idesc(bool bf16, int n, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(id), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(id), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// True in one lane of a converged warp, the same one every time.  The issuing warp runs as a whole and only its products and commits
// stand behind this: in a branch on the lane number every operand of every product is moved into the
// uniform registers anew (128 x 16 x 16 products back to back: 57 against 42-46 cycles each).
__device__ __forceinline__ bool elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Columns of a head in steps of 16, as the products take them: the rest of a tile's DP columns is zeros.
__device__ __forceinline__ int steps_of(int D) { return (D + 15) / 16; }
// d[128, 128] = a b^T, both tiles contracted along their first `steps` x 16 columns.
template <int DP>
__device__ __forceinline__ void mma_columns(uint32_t d, uint32_t a_addr, uint32_t b_addr, uint32_t id, int steps) {
  const uint32_t a = desc_k(a_addr), b = desc_k(b_addr);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint32_t off = (k >> 2) * (kBlockBytes >> 4) + (k & 3) * (32 >> 4);
    if (k == 0 || k < steps) mma_ss(d, a + off, b + off, id, k > 0 ? 1u : 0u);
  }
}
// d[128, columns of id] (+)= a b, a: 128 x 128 of 16 bits in tensor memory, b: a tile contracted along its 128 rows, in steps of 16 of
// which this takes [FROM, TO).  GROUP steps of a lie side by side (8 columns each), the next GROUP from STRIDE columns further on.
template <int FROM, int TO, int GROUP, int STRIDE>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b_addr, uint32_t id, bool accumulate) {
  const uint32_t b = desc_mn(b_addr);
#pragma unroll
  for (int k = FROM; k < TO; ++k)
    mma_ts(d, a + (k / GROUP) * STRIDE + (k % GROUP) * 8, b + k * (2048 >> 4), id, (accumulate || k > FROM) ? 1u : 0u);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Waits for the loads issued so far.  The registers pass through it, so that nothing that reads them can be moved before it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}

// Two fp32 values as one word of 16-bit elements, the first in the low half.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---- work that is taken over at run time.  A grid has one CTA per tile; a CTA that is done with its tile takes the place of one
// that has not started yet (cluster launch control), so that loads of its next tile overlap the end of the last and
// the hardware's order of CTAs, which is the order in which tiles are listed, is kept.
struct alignas(16) Handle {
  uint32_t w[4];
};
__device__ __forceinline__ void ask_for_work(Handle* slot, uint64_t* bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(slot)),
               "r"(smem_u32(bar))
               : "memory");
}
// The number of the CTA whose place was taken, or -1: there is none left.
__device__ __forceinline__ int work_taken(const Handle* slot) {
  int taken, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.s32 %0, 1, 0, p;\n\t"
      "mov.s32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(taken), "=r"(x)
      : "r"(smem_u32(slot))
      : "memory");
  fence_proxy_async_smem();              // the slot is written again through the other proxy
  return taken ? x : -1;
}

// ---- which rows a CTA works on.  Packed sequences are cut into tiles of `rows` each on its own.  Tiles are numbered by what is
// left of their sequence behind them (keys: that many query tiles see them) or lies before them (queries: they see that many
// key tiles), most first, so that with a causal mask the longest come first, whatever the order of the sequences.  A kernel of
// one block per table writes down which is which.  The starts are clamped into [0, limit], so that starts that are out of
// order or out of range make tiles fewer, shorter or equal, never out of range.
struct Span {
  int batch, first_q, len_q, first_k, len_k;   // the sequence
  int tile;                                    // tile number within it, or -1: no tile left
};
__device__ __forceinline__ int clamp_start(int x, int limit) { return x < 0 ? 0 : (x > limit ? limit : x); }
__host__ __device__ __forceinline__ int64_t max_tiles(int64_t limit, int64_t nseq, int rows) { return limit / rows + nseq + 1; }

// order[t] = (sequence, tile), or (-1, how many tiles of the tail lie before it) behind the last one.  A sequence of n tiles has one on each
// of the levels 1 to n; levels are listed from the highest on, sequences in order on each.  A warp takes a level.
__device__ __forceinline__ void write_order(const int* cu, int nseq, int limit, int rows, bool of_keys, int2* order) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int entries = (int)max_tiles(limit, nseq, rows);
  auto tiles_of = [&](int s) {
    if (s >= nseq) return 0;
    const int len = clamp_start(cu[s + 1], limit) - clamp_start(cu[s], limit);
    return len > 0 ? (len + rows - 1) / rows : 0;
  };
  // how many tiles are on level r or above (starts that overlap may make more than there are entries)
  auto above = [&](int r) {
    int64_t n = 0;
    for (int s = lane; s < nseq; s += 32) {
      const int m = tiles_of(s) - r + 1;
      n += m > 0 ? m : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  };
  int most = 0;                                                // the longest sequence's tiles
  for (int s = lane; s < nseq; s += 32) most = max(most, tiles_of(s));
  most = __reduce_max_sync(0xffffffffu, most);
  for (int level = warp + 1; level <= most; level += warps) {
    int64_t at = above(level + 1);
    for (int s0 = 0; s0 < nseq && at < entries; s0 += 32) {
      const int n = tiles_of(s0 + lane);
      const unsigned hit = __ballot_sync(0xffffffffu, n >= level);
      const int64_t t = at + __popc(hit & ((1u << lane) - 1u));
      if (n >= level && t < entries) order[t] = make_int2(s0 + lane, of_keys ? n - level : level - 1);
      at += __popc(hit);
    }
  }
  const int64_t total = above(1);
  for (int64_t t = total + threadIdx.x; t < entries; t += blockDim.x) order[t] = make_int2(-1, (int)(t - total));
}
// What an earlier kernel has written, read where all SMs meet.  For a kernel that reads before its pdl_wait() (the dq kernel): an
// ordinary load may return what this SM's first-level cache still holds from before that kernel.
__device__ __forceinline__ int load_past_l1(const int* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float load_past_l1(const float* p) {
  float v;
  asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
template <bool PAST_L1>
__device__ __forceinline__ Span find_span(const AttnArgs& a, int t, int rows, bool of_keys) {
  auto read = [](const int* p) { return PAST_L1 ? load_past_l1(p) : *p; };
  const int2* entry = (of_keys ? a.order_k : a.order_q) + t;
  const int2 e = PAST_L1 ? make_int2(load_past_l1(&entry->x), load_past_l1(&entry->y)) : *entry;
  Span sp;
  sp.batch = 0;
  if (e.x < 0) {
    const int limit = of_keys ? a.Sk : a.Sq;
    const int64_t first = (int64_t)clamp_start(read((of_keys ? a.cu_k : a.cu_q) + a.nseq), limit) + (int64_t)e.y * rows;
    sp.len_q = sp.len_k = 0;
    sp.tile = -1;
    sp.first_q = sp.first_k = first > limit ? limit : (int)first;
    return sp;
  }
  sp.first_q = clamp_start(read(a.cu_q + e.x), a.Sq);
  sp.len_q = clamp_start(read(a.cu_q + e.x + 1), a.Sq) - sp.first_q;
  sp.first_k = clamp_start(read(a.cu_k + e.x), a.Sk);
  sp.len_k = clamp_start(read(a.cu_k + e.x + 1), a.Sk) - sp.first_k;
  if (sp.len_q < 0) sp.len_q = 0;
  if (sp.len_k < 0) sp.len_k = 0;
  sp.tile = e.y;
  return sp;
}

// Rows [first, min(first + rows, limit)) of one head to zero, by `threads` threads.
__device__ __forceinline__ void zero_rows(const AttnTensor& t, int head, int first, int rows, int limit, int D, int tid, int threads) {
  const int n = limit - first < rows ? limit - first : rows;
  const int vecs = D >> 3;
  for (int i = tid; i < n * vecs; i += threads) {
    const int r = i / vecs, c = i - r * vecs;
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(const_cast<void*>(t.p)) +
                              2 * ((int64_t)(first + r) * t.ss + (int64_t)head * t.sh + c * 8)) = make_uint4(0, 0, 0, 0);
  }
}

// Eight words to a 32-byte boundary.
__device__ __forceinline__ void store_words(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// 32 accumulator columns of one row, times f, as 16-bit elements; only columns below D exist.  wide: the row starts on a
// 32-byte boundary, and a store of 32 bytes writes one whole sector.
template <bool BF16>
__device__ __forceinline__ void store32(uint16_t* row, int col0, int D, const uint32_t* r, float f, bool wide) {
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = pack2<BF16>(__uint_as_float(r[v * 16 + 2 * e]) * f, __uint_as_float(r[v * 16 + 2 * e + 1]) * f);
    const int col = col0 + v * 16;
    if (wide && col + 16 <= D) {
      store_words(row + col, w);
    } else {
      if (col < D) *reinterpret_cast<uint4*>(row + col) = make_uint4(w[0], w[1], w[2], w[3]);
      if (col + 8 < D) *reinterpret_cast<uint4*>(row + col + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
}
__device__ __forceinline__ bool rows_are_wide(const AttnTensor& t) {
  return ((reinterpret_cast<uintptr_t>(t.p) | (uintptr_t)(t.sb * 2) | (uintptr_t)(t.ss * 2) | (uintptr_t)(t.sh * 2)) & 31u) == 0;
}
__device__ __forceinline__ uint16_t* row_ptr(const AttnTensor& t, int batch, int head, int row) {
  return reinterpret_cast<uint16_t*>(const_cast<void*>(t.p)) + (int64_t)batch * t.sb + (int64_t)row * t.ss + (int64_t)head * t.sh;
}
// Where the row of one part's sums starts (H heads of S rows).
__device__ __forceinline__ float* part_row(float* partial, int part, int B, int H, int S, int D, int batch, int head, int row) {
  return partial + ((((int64_t)part * B + batch) * H + head) * S + row) * D;
}
// 32 accumulator columns of one row, times f, in fp32.
__device__ __forceinline__ void store32_f32(float* row, int col0, int D, const uint32_t* r, float f) {
#pragma unroll
  for (int v = 0; v < 8; ++v)
    if (col0 + v * 4 < D)
      *reinterpret_cast<float4*>(row + col0 + v * 4) = make_float4(__uint_as_float(r[v * 4]) * f, __uint_as_float(r[v * 4 + 1]) * f,
                                                                   __uint_as_float(r[v * 4 + 2]) * f, __uint_as_float(r[v * 4 + 3]) * f);
}
// Where the row statistics of one head start.
__device__ __forceinline__ int64_t stat_row(const AttnArgs& a, int batch, int head) { return ((int64_t)batch * a.H + head) * a.Sq; }

// ---- host
// An early launch that is counted.
template <typename K, typename... A>
cudaError_t launch_counted(int64_t& kernels, K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const A&... args) {
  const cudaError_t e = launch_pdl(kernel, grid, block, smem, stream, args...);
  if (e == cudaSuccess) ++kernels;
  return e;
}
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
inline EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return static_cast<EncodeFn>(nullptr);
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}
// Boxes of 128 rows x 64 columns of one head; columns from D on and rows from S on read as zero.
inline bool make_map(CUtensorMap* map, const AttnTensor& t, bool bf16, int D, int H, int S, int B) {
  EncodeFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)S, (cuuint64_t)B};
  // the stride of an extent of one is never used, but has to be a valid one
  const cuuint64_t strides[3] = {H > 1 ? (cuuint64_t)t.sh * 2 : (cuuint64_t)256, S > 1 ? (cuuint64_t)t.ss * 2 : (cuuint64_t)256,
                                 B > 1 ? (cuuint64_t)t.sb * 2 : (cuuint64_t)256};
  const cuuint32_t box[4] = {64, 1, 128, 1}, one[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(t.p), dims, strides, box,
            one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace attn
}  // namespace pccl
