// Attention, backward pass: a kernel for the row sums <do_i, o_i>, one for dk and dv, one for dq (attention.h has the formulas,
// attention.cuh the tiles).
//
// Two kernels share the work so that every gradient has one owner: a CTA keeps 128 keys (dk, dv) or 128 queries (dq) and walks
// over the others, and its sums stay in tensor memory until they are complete.  Scores and do v^T are computed twice, seven
// products instead of five; what is saved are fp32 atomic additions of a whole dq per key tile, and results are the same bits
// from run to run.  (Leaving the score gradients in memory for dq instead was tried: 2 to 4 % faster for 4 x 2048 x 16 heads, up to 50 %
// slower for small calls, and up to 1 GiB of memory.)  The heads of a group are walked over one after the other by the CTA that
// owns their shared key head.
//
//   warps 0-7   probabilities and score gradients: two warpgroups, each with half of a tile's 128 columns
//   warp 8      TMA; asks for the next tile of the grid (attention.cuh)
//   warp 9      tensor memory; one thread issues the products
//   warp 10     dk, dv: the row statistics of each query tile, into shared memory
//
// dk, dv: scores are computed transposed, S = K Q^T, so that a thread owns a key and the 16-bit P^T and dS^T lie in tensor memory
// as the first operand of dv += P^T dO and dk += dS^T Q.  The products of one tile run while the other operand is being made:
//   S(i) | P(i): dv += P^T dO, S(i+1) | dS(i): dk += dS^T Q, dP(i+1) | ...
// dq: S = Q K^T and dP = dO V^T as in the forward pass, dq += dS K; S is kept twice, so that its next tile is ready when the
// exponentials of the last one are done.
//
// What bounds it.  4 x 2048 x 16 heads of 128 causal take 250 us in runs of some 30 calls (302 on a card that has been busy for seconds,
// whose clock is lower), 687 TFLOP/s by the five products that the formulas need and 960 by the seven computed: row sums 10 us (6.4 TB/s),
// dk and dv 132, dq 103.  With the exponentials and conversions left out the products alone take 110 and 87, 1330 and 1260 TFLOP/s, at
// heads of 64 81 instead of 110 for dk and dv; without the loads of query tiles the whole takes 249.  A product of 128 x 128 x 16 takes 64.6 cycles, with 64 columns 32.5 (48.5 with both operands in shared memory),
// so the four of a step need 2070 cycles, at heads of 64 1040; with the conversions left out a step still takes 3200 and 2400.  So most
// of the rest is the hand-over between warps at every tile, and the start and end of each walk, here of 8.5 steps on average.
// Sixteen compute warps for eight: 253, at heads of 64 197 instead of 201; a second tile of scores at heads of 64: 199.  The
// clock is at 1.69 GHz by the power limit.  16 heads of 4096 223 us (768 TFLOP/s), heads of 64 200.
#include "attention.cuh"

namespace pccl {

namespace {

using namespace attn;

constexpr int kCompute = 8;                     // warps that make probabilities and score gradients, 512 / kCompute columns each
constexpr int kCols = 512 / kCompute;
constexpr int kThreads = kCompute * 32 + 128;

// ---------------------------------------------------------------- row sums
// delta_i = <do_i, o_i>: sixteen lanes per row.  One read of both tensors.
template <bool BF16>
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y) {
  const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
  float acc = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x0, x1, y0, y1;
    if constexpr (BF16) {
      split(unpack2(xw[e]), x0, x1);
      split(unpack2(yw[e]), y0, y1);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(xw + e)), q = __half22float2(*reinterpret_cast<const __half2*>(yw + e));
      x0 = p.x, x1 = p.y, y0 = q.x, y1 = q.y;
    }
    acc = fmaf(x0, y0, fmaf(x1, y1, acc));
  }
  return acc;
}
// A block takes 64 rows of one head, a warp eight of them, two at once; all loads first.
template <bool BF16>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x & 15, half = (threadIdx.x >> 4) & 1, warp = threadIdx.x >> 5;
  const int s0 = (int)blockIdx.x * 64 + warp * 8 + half, h = (int)blockIdx.y, b = (int)blockIdx.z;
  const bool on = sub * 8 < a.D;
  uint4 x[4], y[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int s = s0 + u * 2;
    const bool here = on && s < a.Sq;
    x[u] = here ? *reinterpret_cast<const uint4*>(row_ptr(a.dout, b, h, s) + sub * 8) : make_uint4(0, 0, 0, 0);
    y[u] = here ? *reinterpret_cast<const uint4*>(row_ptr(a.o, b, h, s) + sub * 8) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int s = s0 + u * 2;
    float acc = dot8<BF16>(x[u], y[u]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (s < a.Sq && sub == 0) a.delta[stat_row(a, b, h) + s] = acc;
  }
}

__global__ void __launch_bounds__(1024) attention_orders_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0) write_order(a.cu_k, a.nseq, a.Sk, 128, true, a.order_k);
  else write_order(a.cu_q, a.nseq, a.Sq, 128, false, a.order_q);
}

// ---------------------------------------------------------------- dk, dv
template <int DP>
struct Dkv {
  // Stages of the two rings.  A query tile is last read by the fourth product of its step and wanted again by the first, two
  // products later with two stages: less than a load takes.
  static constexpr int kNq = DP == 128 ? 3 : 4, kNdo = DP == 128 ? 2 : 4;
  static constexpr uint32_t kTile = (DP / 64) * kBlockBytes;
  static constexpr uint32_t kQ = 2 * kTile, kDo = kQ + kNq * kTile;
  static constexpr uint32_t kStat = kDo + kNdo * kTile;      // [2][lse, delta][128] floats
  static constexpr uint32_t kBars = kStat + 2 * 2 * 128 * 4;
  static constexpr uint32_t kSmem = kBars + 512;              // 231,936 of 232,448: no room to move the base to a boundary
  static constexpr uint32_t kS = 0, kDp = 128, kDv = 256, kDk = 256 + DP;      // tensor memory columns
  static constexpr int kOutWarps = kCompute;                 // that read the finished sums
  static constexpr int kReaders = kCompute + 3;              // of the next tile's number: all warps but the last
};
struct DkvBars {
  Handle next[2];
  uint64_t next_full[2], next_empty[2];
  uint64_t k_full, k_empty, v_full, v_empty, q_full[4], q_empty[4], do_full[4], do_empty[4], stat_full[2], stat_empty[2];
  uint64_t s, dp, p_ready, ds_ready, out_full, out_empty, fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(DkvBars) <= 512, "the barriers' part of shared memory");

// The keys of one tile number, and the query tiles that see one of them: per_head of them from tile `first` on, for each head
// of the group.  Of that sequence of steps, `total` from i0 on are this part's.
struct DkvWork {
  Span sp;
  int kv_head, key0, offset, first, per_head, part, i0, total;
};
template <bool SPLIT>
__device__ __forceinline__ DkvWork dkv_work_at(const AttnArgs& a, unsigned id) {
  DkvWork w;
  w.part = 0;
  if constexpr (SPLIT) {
    w.part = (int)(id % (unsigned)a.parts_dkv);
    id /= (unsigned)a.parts_dkv;
  }
  if (a.cu_q != nullptr) {
    w.kv_head = (int)(id % (unsigned)a.Hk);
    w.sp = find_span<false>(a, (int)(id / (unsigned)a.Hk), 128, true);
  } else {
    // with a causal mask the first tiles are seen by the most queries: they come first
    const unsigned heads = (unsigned)(a.B * a.Hk), bh = id % heads;
    w.kv_head = (int)(bh % (unsigned)a.Hk);
    w.sp.batch = (int)(bh / (unsigned)a.Hk);
    w.sp.first_q = w.sp.first_k = 0;
    w.sp.len_q = a.Sq;
    w.sp.len_k = a.Sk;
    w.sp.tile = (int)(id / heads);
  }
  w.key0 = w.sp.tile * 128;
  w.offset = w.sp.len_k - w.sp.len_q;
  w.first = a.causal && w.key0 - w.offset > 0 ? (w.key0 - w.offset) / 128 : 0;
  const int tiles = (w.sp.len_q + 127) / 128;
  w.per_head = w.sp.tile >= 0 && tiles > w.first ? tiles - w.first : 0;
  w.i0 = 0;
  w.total = a.H / a.Hk * w.per_head;
  if constexpr (SPLIT) {
    w.i0 = (int)((int64_t)w.total * w.part / a.parts_dkv);
    w.total = (int)((int64_t)w.total * (w.part + 1) / a.parts_dkv) - w.i0;
  }
  return w;
}

template <int DP, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                         const __grid_constant__ AttnArgs a) {
  using C = Dkv<DP>;
  extern __shared__ __align__(1024) unsigned char smem[];   // the swizzled tiles want 1024 bytes; without static variables it starts there
  if ((smem_u32(smem) & 1023u) != 0u) {
    pdl_wait();                                              // this block too lets the dq kernel in only when the row sums are complete
    if (threadIdx.x == 0) atomicCAS(a.error, 0, kErrLoad);
    return;
  }
  DkvBars& b = *reinterpret_cast<DkvBars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.H / a.Hk;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kNq; ++i) {
      mbar_init(b.q_full + i, 1);
      mbar_init(b.q_empty + i, 1);
    }
    for (int i = 0; i < C::kNdo; ++i) {
      mbar_init(b.do_full + i, 1);
      mbar_init(b.do_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(b.next_full + i, 1);
      mbar_init(b.next_empty + i, C::kReaders);
      mbar_init(b.stat_full + i, 1);
      mbar_init(b.stat_empty + i, kCompute);
    }
    mbar_init(&b.k_full, 1);
    mbar_init(&b.k_empty, 1);
    mbar_init(&b.v_full, 1);
    mbar_init(&b.v_empty, 1);
    mbar_init(&b.s, 1);
    mbar_init(&b.dp, 1);
    mbar_init(&b.p_ready, kCompute);
    mbar_init(&b.ds_ready, kCompute);
    mbar_init(&b.out_full, 1);
    mbar_init(&b.out_empty, C::kOutWarps);
    mbar_init(&b.fix, 1);
    mbar_init(&b.drain, 1);
    b.abort = 0;
    fence_mbar_init();
  }
  if (warp == kCompute + 1) tmem_alloc(&b.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = b.tmem;
  pdl_wait();
  pdl_trigger();                                             // behind the wait of every block: the dq kernel relies on it

  // The tile after the k-th, for every role alike: -1 none, -2 a wait gave up.  Whole warps.
  auto next_tile = [&](int k) {
    if (!wait_warp(b.next_full + (k & 1), (k >> 1) & 1u, abort_flag)) return -2;
    const int id = work_taken(b.next + (k & 1));
    __syncwarp();
    if (lane == 0) mbar_arrive(b.next_empty + (k & 1));
    return id;
  };
  auto fail = [&](int code) {
    if (lane == 0) {
      atomicCAS(a.error, 0, code);
      *abort_flag = 1;
    }
  };

  // 384 threads start with 168 registers each, 64,512 together: 256 x 208 + 128 x 88.
  if (warp >= kCompute) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kCompute) {
      // ---------------------------------------------------------- loads, and the tiles to come
      bool ok = true;
      uint32_t n = 0, items = 0, fixes = 0;                  // query tiles, key tiles so far
      int id = (int)blockIdx.x;
      for (int k = 0; ok; ++k) {
        if (k >= 2 && !(ok = wait_warp(b.next_empty + (k & 1), ((k >> 1) - 1) & 1u, abort_flag))) break;
        if (lane == 0) ask_for_work(b.next + (k & 1), b.next_full + (k & 1));
        const DkvWork w = dkv_work_at<SPLIT>(a, (unsigned)id);
        for (int i = 0; i < w.total && ok; ++i, ++n) {
          const int hg = (w.i0 + i) / w.per_head, head = w.kv_head * group + hg, row = (w.first + w.i0 + i - hg * w.per_head) * 128;
          // the rows behind a packed sequence are its neighbour's, and both tiles are contracted along their rows
          const bool ragged = a.cu_q != nullptr && row + 128 > w.sp.len_q;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            if (i == 0) {                                    // the keys (values) of the last tile may still be in use
              uint64_t *full = which == 0 ? &b.k_full : &b.v_full, *empty = which == 0 ? &b.k_empty : &b.v_empty;
              if (!(ok = wait_warp(empty, (items & 1u) ^ 1u, abort_flag))) break;
              if (lane == 0) {
                mbar_expect_tx(full, C::kTile);
                load_tile<DP>(smem + which * C::kTile, which == 0 ? &map_k : &map_v, w.kv_head, w.sp.first_k + w.key0, w.sp.batch, full);
              }
            }
            const uint32_t stages = which == 0 ? C::kNq : C::kNdo, st = n % stages, ph = (n / stages) & 1u;
            uint64_t* full = (which == 0 ? b.q_full : b.do_full) + st;
            if (!(ok = wait_warp((which == 0 ? b.q_empty : b.do_empty) + st, ph ^ 1u, abort_flag))) break;
            unsigned char* dst = smem + (which == 0 ? C::kQ : C::kDo) + st * C::kTile;
            uint64_t* bar = ragged ? &b.fix : full;
            if (lane == 0) {
              mbar_expect_tx(bar, C::kTile);
              load_tile<DP>(dst, which == 0 ? &map_q : &map_do, head, w.sp.first_q + row, w.sp.batch, bar);
            }
            if (ragged) {
              if (!(ok = wait_warp(&b.fix, fixes++ & 1u, abort_flag))) break;
              clear_rows<DP>(dst, w.sp.len_q - row);
              if (lane == 0) mbar_arrive(full);
            }
          }
        }
        if (!ok) break;
        items += w.total > 0;
        id = next_tile(k);
        ok = id != -2;
        if (id < 0) break;
      }
      if (!ok) {
        fail(kErrLoad);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);    // which copies are on their way is not known: the time that they can take
      }
    } else if (warp == kCompute + 1) {
      // ---------------------------------------------------------- products
      constexpr uint32_t id_s = idesc(BF16, 128, false);
      const int steps = steps_of(a.D);
      const uint32_t id_o = idesc(BF16, steps * 16, true);
      const uint32_t k_addr = smem_u32(smem), v_addr = k_addr + C::kTile;
      const uint32_t q_ring = smem_u32(smem + C::kQ), do_ring = smem_u32(smem + C::kDo);
      bool ok = true;
      uint32_t n = 0, items = 0;
      int id = (int)blockIdx.x;
      for (int k = 0;; ++k) {
        const DkvWork w = dkv_work_at<SPLIT>(a, (unsigned)id);
        if (w.total > 0) {
          auto q_at = [&](uint32_t m) { return q_ring + (m % C::kNq) * C::kTile; };
          auto do_at = [&](uint32_t m) { return do_ring + (m % C::kNdo) * C::kTile; };
          auto scores = [&](int i) {
            const uint32_t m = n + (uint32_t)i;
            if (!wait_warp(b.q_full + m % C::kNq, (m / C::kNq) & 1u, abort_flag)) return false;
            if (elect()) {
              mma_columns<DP>(tmem + C::kS, k_addr, q_at(m), id_s, steps);
              commit(&b.s);
              if (i + 1 == w.total) commit(&b.k_empty);
            }
            __syncwarp();
            return true;
          };
          auto dprobs = [&](int i) {
            const uint32_t m = n + (uint32_t)i;
            if (!wait_warp(b.do_full + m % C::kNdo, (m / C::kNdo) & 1u, abort_flag)) return false;
            if (elect()) {
              mma_columns<DP>(tmem + C::kDp, v_addr, do_at(m), id_s, steps);
              commit(&b.dp);
              if (i + 1 == w.total) commit(&b.v_empty);
            }
            __syncwarp();
            return true;
          };
          ok = wait_warp(&b.k_full, items & 1u, abort_flag) && scores(0) && wait_warp(&b.v_full, items & 1u, abort_flag) && dprobs(0);
          for (int i = 0; i < w.total && ok; ++i) {
            const uint32_t m = n + (uint32_t)i;
            // the last tile's sums have been read before this one's are begun
            if (i == 0 && !(ok = wait_warp(&b.out_empty, (items & 1u) ^ 1u, abort_flag))) break;
            if (!(ok = wait_warp(&b.p_ready, m & 1u, abort_flag))) break;
            fence_after();
            if (elect()) {
              mma_rows<0, 8, kCols / 16, kCols>(tmem + C::kDv, tmem + C::kS, do_at(m), id_o, i > 0);
              commit(b.do_empty + m % C::kNdo);
            }
            __syncwarp();
            if (i + 1 < w.total && !(ok = scores(i + 1))) break;
            if (!(ok = wait_warp(&b.ds_ready, m & 1u, abort_flag))) break;
            fence_after();
            if (elect()) {
              mma_rows<0, 8, kCols / 16, kCols>(tmem + C::kDk, tmem + C::kDp, q_at(m), id_o, i > 0);
              commit(b.q_empty + m % C::kNq);
              if (i + 1 == w.total) commit(&b.out_full);
            }
            __syncwarp();
            if (i + 1 < w.total) ok = dprobs(i + 1);
          }
          n += (uint32_t)w.total;
          ++items;
        }
        if (!ok) break;
        id = next_tile(k);
        ok = id != -2;
        if (id < 0) break;
      }
      if (!ok) fail(kErrMma);
      __syncwarp();
      if (elect()) commit(&b.drain);
      __syncwarp();
      mbar_wait(&b.drain, 0, kWaitNs);
    } else if (warp == kCompute + 2) {
      // ---------------------------------------------------------- statistics: -lse in powers of two, -delta.  Queries that do not
      // exist or see no key get probabilities of zero.
      bool ok = true;
      uint32_t n = 0;
      int id = (int)blockIdx.x;
      for (int k = 0; ok; ++k) {
        const DkvWork w = dkv_work_at<SPLIT>(a, (unsigned)id);
        for (int i = 0; i < w.total; ++i, ++n) {
          const int hg = (w.i0 + i) / w.per_head, head = w.kv_head * group + hg, row = (w.first + w.i0 + i - hg * w.per_head) * 128;
          const int64_t at = stat_row(a, w.sp.batch, head) + w.sp.first_q;
          float x[4], y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = row + e * 32 + lane;
            const bool exists = r < w.sp.len_q;
            const float l = exists ? a.lse[at + r] : -INFINITY;
            x[e] = l == -INFINITY ? -INFINITY : l * -kLog2e;
            y[e] = exists ? -a.delta[at + r] : 0.f;
          }
          if (!(ok = wait_warp(b.stat_empty + (n & 1), ((n >> 1) & 1u) ^ 1u, abort_flag))) break;
          float* st = reinterpret_cast<float*>(smem + C::kStat) + (n & 1) * 256;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st[e * 32 + lane] = x[e];
            st[128 + e * 32 + lane] = y[e];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(b.stat_full + (n & 1));
        }
        if (!ok) break;
        id = next_tile(k);
        ok = id != -2;
        if (id < 0) break;
      }
      if (!ok) fail(kErrLoad);
    }
  } else {
    // ------------------------------------------------------------ probabilities and score gradients: thread = key
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + C::kS + g * kCols + lanes, t_dp = tmem + C::kDp + g * kCols + lanes;
    const F2 scale2 = f2(a.scale * kLog2e);
    bool ok = true;
    uint32_t n = 0, items = 0;
    int id = (int)blockIdx.x;
    for (int k = 0; ok; ++k) {
      const DkvWork w = dkv_work_at<SPLIT>(a, (unsigned)id);
      const int key = w.key0 + (warp & 3) * 32 + lane;
      int tile = w.first + (w.per_head > 0 ? w.i0 % w.per_head : 0);            // query tile within its head
      for (int i = 0; i < w.total; ++i, ++n) {
        const float* st = reinterpret_cast<const float*>(smem + C::kStat) + (n & 1) * 256 + g * kCols;
        const int q0 = tile * 128 + g * kCols;
        if (++tile == w.first + w.per_head) tile = w.first;
        const int hidden = a.causal ? key - w.offset - q0 : 0;               // this key is not seen by the first so many queries
        const bool masked = a.causal && w.key0 + (warp & 3) * 32 + 31 - w.offset - q0 > 0;
        if (!(ok = wait_warp(b.stat_full + (n & 1), (n >> 1) & 1u, abort_flag))) break;
        if (!(ok = wait_warp(&b.s, n & 1u, abort_flag))) break;
        fence_after();
        float p[kCols];
        uint32_t s[kCols / 32][32];
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld32(t_s + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_wait_ld(s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t wd[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float4 base = *reinterpret_cast<const float4*>(st + c * 32 + 2 * e);
            float x[4];
            split(fma2(f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, f2(base.x, base.y)), x[0], x[1]);
            split(fma2(f2(__uint_as_float(s[c][2 * e + 2]), __uint_as_float(s[c][2 * e + 3])), scale2, f2(base.z, base.w)), x[2], x[3]);
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = ex2_hw(x[v]);
            if (masked) {
#pragma unroll
              for (int v = 0; v < 4; ++v) x[v] = c * 32 + 2 * e + v < hidden ? 0.f : x[v];
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) p[c * 32 + 2 * e + v] = x[v];
            wd[e] = pack2<BF16>(x[0], x[1]);
            wd[e + 1] = pack2<BF16>(x[2], x[3]);
          }
          tmem_st16(t_s + c * 16, wd);
        }
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.p_ready);

        if (!(ok = wait_warp(&b.dp, n & 1u, abort_flag))) break;
        fence_after();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld32(t_dp + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_wait_ld(s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t wd[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float4 d = *reinterpret_cast<const float4*>(st + 128 + c * 32 + 2 * e);
            const int i0 = c * 32 + 2 * e;
            float x[4];
            split(f2(p[i0], p[i0 + 1]) * (f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])) + f2(d.x, d.y)), x[0], x[1]);
            split(f2(p[i0 + 2], p[i0 + 3]) * (f2(__uint_as_float(s[c][2 * e + 2]), __uint_as_float(s[c][2 * e + 3])) + f2(d.z, d.w)), x[2],
                  x[3]);
            if (masked) {
#pragma unroll
              for (int v = 0; v < 4; ++v) x[v] = i0 + v < hidden ? 0.f : x[v];
            }
            wd[e] = pack2<BF16>(x[0], x[1]);
            wd[e + 1] = pack2<BF16>(x[2], x[3]);
          }
          tmem_st16(t_dp + c * 16, wd);
        }
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&b.ds_ready);
          mbar_arrive(b.stat_empty + (n & 1));
        }
      }
      if (ok && w.total > 0) {
        ok = wait_warp(&b.out_full, items & 1u, abort_flag);
        ++items;
        fence_after();
      }
      if (!ok) break;
      if (w.sp.tile < 0) {
        if (a.zero_tail) {
          zero_rows(a.dk, w.kv_head, w.sp.first_k, 128, a.Sk, a.D, threadIdx.x, kCompute * 32);
          zero_rows(a.dv, w.kv_head, w.sp.first_k, 128, a.Sk, a.D, threadIdx.x, kCompute * 32);
        }
      } else {
        // the first half of the warps writes dv, the second dk, each warpgroup its share of the columns
        constexpr int per = DP * 2 / (kCompute / 4);
        const bool keys_grad = g >= kCompute / 8;
        const AttnTensor& dst = keys_grad ? a.dk : a.dv;
        const int col0 = (g % (kCompute / 8)) * per;
        const bool exists = key < w.sp.len_k, wide = rows_are_wide(dst);
        uint16_t* out = row_ptr(dst, w.sp.batch, w.kv_head, w.sp.first_k + key);
        const uint32_t t_out = tmem + (keys_grad ? C::kDk : C::kDv) + lanes + col0;
#pragma unroll
        for (int c = 0; c < per / 32; ++c) {
          uint32_t o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
          if (w.total > 0) {
            tmem_ld32(t_out + c * 32, o);
            tmem_wait_ld(o);
            if (c == per / 32 - 1) {                         // the sums may be written again
              fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&b.out_empty);
            }
          }
          if (!exists) continue;
          if constexpr (SPLIT) {
            // dv's parts first, then dk's
            float* sums = part_row(a.partial, keys_grad ? a.parts_dkv + w.part : w.part, a.B, a.Hk, a.Sk, a.D, w.sp.batch, w.kv_head, key);
            store32_f32(sums, col0 + c * 32, a.D, o, keys_grad ? a.scale : 1.f);
          } else {
            store32<BF16>(out, col0 + c * 32, a.D, o, keys_grad ? a.scale : 1.f, wide);
          }
        }
      }
      id = next_tile(k);
      ok = id != -2;
      if (id < 0) break;
    }
    if (!ok) fail(kErrCompute);
  }
  fence_before();
  __syncthreads();
  if (warp == kCompute + 1) {
    fence_after();
    tmem_free(tmem, 512);
  }
}

// ---------------------------------------------------------------- dq
template <int DP>
struct Dq {
  static constexpr int kK = DP == 128 ? 3 : 4, kV = DP == 128 ? 2 : 3;        // ring stages
  static constexpr uint32_t kTile = (DP / 64) * kBlockBytes;
  static constexpr uint32_t kKRing = 2 * kTile, kVRing = kKRing + kK * kTile;
  static constexpr uint32_t kBars = kVRing + kV * kTile;
  static constexpr uint32_t kSmem = kBars + 512 + 1024;
  static constexpr uint32_t kS = 0, kDp = 256, kDq = 384;
  static constexpr int kOutWarps = DP / 32 * 4 < kCompute ? DP / 32 * 4 : kCompute;   // that read the finished sums, 32 columns or more each
  static constexpr int kReaders = kCompute + 2;              // of the next tile's number: all warps but the last two
};
struct DqBars {
  Handle next[2];
  uint64_t next_full[2], next_empty[2];
  uint64_t q_full, q_empty, do_full, do_empty, k_full[4], k_empty[4], v_full[3], v_empty[3], s[2], dp, dp_read, ds_ready[2];
  uint64_t out_full, out_empty, fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(DqBars) <= 512, "the barriers' part of shared memory");

// The queries of one tile number, and the key tiles that this part of them has to do with: n of them from tile j0 on.
struct DqWork {
  Span sp;
  int head, row0, offset, part, j0, n;
};
template <bool SPLIT>
__device__ __forceinline__ DqWork dq_work_at(const AttnArgs& a, unsigned id, int tiles) {
  DqWork w;
  w.part = 0;
  if constexpr (SPLIT) {
    w.part = (int)(id % (unsigned)a.parts_dq);
    id /= (unsigned)a.parts_dq;
  }
  if (a.cu_q != nullptr) {
    w.head = (int)(id % (unsigned)a.H);
    w.sp = find_span<true>(a, (int)(id / (unsigned)a.H), 128, false);
  } else {
    const unsigned heads = (unsigned)(a.B * a.H), bh = id % heads, t = id / heads;
    w.head = (int)(bh % (unsigned)a.H);
    w.sp.batch = (int)(bh / (unsigned)a.H);
    w.sp.first_q = w.sp.first_k = 0;
    w.sp.len_q = a.Sq;
    w.sp.len_k = a.Sk;
    w.sp.tile = a.causal ? tiles - 1 - (int)t : (int)t;                       // most keys first
  }
  w.row0 = w.sp.tile * 128;
  w.offset = w.sp.len_k - w.sp.len_q;
  const int last = w.row0 + 127 < w.sp.len_q - 1 ? w.row0 + 127 : w.sp.len_q - 1;
  const int keys = !a.causal ? w.sp.len_k : (last + w.offset + 1 < w.sp.len_k ? last + w.offset + 1 : w.sp.len_k);
  w.n = w.sp.tile >= 0 && keys > 0 ? (keys + 127) / 128 : 0;
  w.j0 = 0;
  if constexpr (SPLIT) {
    w.j0 = w.n * w.part / a.parts_dq;
    w.n = w.n * (w.part + 1) / a.parts_dq - w.j0;
  }
  return w;
}

template <int DP, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ AttnArgs a, int tiles, bool beside) {
  using C = Dq<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  DqBars& b = *reinterpret_cast<DqBars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kK; ++i) {
      mbar_init(b.k_full + i, 1);
      mbar_init(b.k_empty + i, 1);
    }
    for (int i = 0; i < C::kV; ++i) {
      mbar_init(b.v_full + i, 1);
      mbar_init(b.v_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(b.next_full + i, 1);
      mbar_init(b.next_empty + i, C::kReaders);
      mbar_init(b.s + i, 1);
      mbar_init(b.ds_ready + i, kCompute);
    }
    mbar_init(&b.q_full, 1);
    mbar_init(&b.q_empty, 1);
    mbar_init(&b.do_full, 1);
    mbar_init(&b.do_empty, 1);
    mbar_init(&b.dp, 1);
    mbar_init(&b.dp_read, kCompute);
    mbar_init(&b.out_full, 1);
    mbar_init(&b.out_empty, C::kOutWarps);
    mbar_init(&b.fix, 1);
    mbar_init(&b.drain, 1);
    b.abort = 0;
    fence_mbar_init();
  }
  if (warp == kCompute + 1) tmem_alloc(&b.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = b.tmem;
  // beside: the kernel in front is the one for dk and dv, which shares nothing with this one but what both read.  All of that,
  // the row sums among it, was complete when its blocks let this one's in, since each of them has passed its own wait before (or
  // left behind it), so these begin on the SMs that it leaves, and wait for it at their end.  Completeness is not yet visibility
  // to this grid, which has not waited: what earlier kernels of the call have written (row sums, tile list) and the other words that it
  // reads by ordinary loads (lse, starts) are read past the first-level cache, and tiles come by TMA, which does not use it.
  if (!beside) pdl_wait();

  // The tile after the k-th, for every role alike: -1 none, -2 a wait gave up.  Whole warps.
  auto next_tile = [&](int k) {
    if (!wait_warp(b.next_full + (k & 1), (k >> 1) & 1u, abort_flag)) return -2;
    const int id = work_taken(b.next + (k & 1));
    __syncwarp();
    if (lane == 0) mbar_arrive(b.next_empty + (k & 1));
    return id;
  };
  auto fail = [&](int code) {
    if (lane == 0) {
      atomicCAS(a.error, 0, code);
      *abort_flag = 1;
    }
  };

  // 384 threads start with 168 registers each, 64,512 together: 256 x 208 + 128 x 88.
  if (warp >= kCompute) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kCompute) {
      // ---------------------------------------------------------- loads, and the tiles to come
      bool ok = true;
      uint32_t n = 0, items = 0, fixes = 0;                  // key tiles, query tiles so far
      int id = (int)blockIdx.x;
      for (int k = 0; ok; ++k) {
        if (k >= 2 && !(ok = wait_warp(b.next_empty + (k & 1), ((k >> 1) - 1) & 1u, abort_flag))) break;
        if (lane == 0) ask_for_work(b.next + (k & 1), b.next_full + (k & 1));
        const DqWork w = dq_work_at<SPLIT>(a, (unsigned)id, tiles);
        const int kv_head = w.head / (a.H / a.Hk);
        for (int j = 0; j < w.n; ++j, ++n) {
          const uint32_t ks = n % C::kK, vs = n % C::kV;
          if (!(ok = wait_warp(b.k_empty + ks, ((n / C::kK) & 1u) ^ 1u, abort_flag))) break;
          unsigned char* dst = smem + C::kKRing + ks * C::kTile;
          // the rows behind a packed sequence are its neighbour's
          const int row = (w.j0 + j) * 128;
          const bool ragged = a.cu_q != nullptr && row + 128 > w.sp.len_k;
          uint64_t* bar = ragged ? &b.fix : b.k_full + ks;
          if (lane == 0) {
            mbar_expect_tx(bar, C::kTile);
            load_tile<DP>(dst, &map_k, kv_head, w.sp.first_k + row, w.sp.batch, bar);
          }
          if (ragged) {
            if (!(ok = wait_warp(&b.fix, fixes++ & 1u, abort_flag))) break;
            clear_rows<DP>(dst, w.sp.len_k - row);
            if (lane == 0) mbar_arrive(b.k_full + ks);
          }
          if (j == 0) {                                      // behind the first keys: the queries of the last tile may still be in use
            if (!(ok = wait_warp(&b.q_empty, (items & 1u) ^ 1u, abort_flag))) break;
            if (lane == 0) {
              mbar_expect_tx(&b.q_full, C::kTile);
              load_tile<DP>(smem, &map_q, w.head, w.sp.first_q + w.row0, w.sp.batch, &b.q_full);
            }
          }
          if (!(ok = wait_warp(b.v_empty + vs, ((n / C::kV) & 1u) ^ 1u, abort_flag))) break;
          if (lane == 0) {
            mbar_expect_tx(b.v_full + vs, C::kTile);
            load_tile<DP>(smem + C::kVRing + vs * C::kTile, &map_v, kv_head, w.sp.first_k + row, w.sp.batch, b.v_full + vs);
          }
          if (j == 0) {
            if (!(ok = wait_warp(&b.do_empty, (items & 1u) ^ 1u, abort_flag))) break;
            if (lane == 0) {
              mbar_expect_tx(&b.do_full, C::kTile);
              load_tile<DP>(smem + C::kTile, &map_do, w.head, w.sp.first_q + w.row0, w.sp.batch, &b.do_full);
            }
          }
        }
        if (!ok) break;
        items += w.n > 0;
        id = next_tile(k);
        ok = id != -2;
        if (id < 0) break;
      }
      if (!ok) {
        fail(kErrLoad);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);    // which copies are on their way is not known: the time that they can take
      }
    } else if (warp == kCompute + 1) {
      // ---------------------------------------------------------- products
      constexpr uint32_t id_s = idesc(BF16, 128, false);
      const int steps = steps_of(a.D);
      const uint32_t id_o = idesc(BF16, steps * 16, true);
      const uint32_t q_addr = smem_u32(smem), do_addr = q_addr + C::kTile;
      const uint32_t k_ring = smem_u32(smem + C::kKRing), v_ring = smem_u32(smem + C::kVRing);
      bool ok = true;
      uint32_t n = 0, items = 0;
      int id = (int)blockIdx.x;
      for (int k = 0;; ++k) {
        const DqWork w = dq_work_at<SPLIT>(a, (unsigned)id, tiles);
        if (w.n > 0) {
          auto scores = [&](int j) {
            const uint32_t m = n + (uint32_t)j;
            if (!wait_warp(b.k_full + m % C::kK, (m / C::kK) & 1u, abort_flag)) return false;
            if (elect()) {
              mma_columns<DP>(tmem + C::kS + (m & 1) * 128, q_addr, k_ring + (m % C::kK) * C::kTile, id_s, steps);
              commit(b.s + (m & 1));
              if (j + 1 == w.n) commit(&b.q_empty);
            }
            __syncwarp();
            return true;
          };
          auto dprobs = [&](int j) {
            const uint32_t m = n + (uint32_t)j;
            if (!wait_warp(b.v_full + m % C::kV, (m / C::kV) & 1u, abort_flag)) return false;
            if (elect()) {
              mma_columns<DP>(tmem + C::kDp, do_addr, v_ring + (m % C::kV) * C::kTile, id_s, steps);
              commit(&b.dp);
              commit(b.v_empty + m % C::kV);
              if (j + 1 == w.n) commit(&b.do_empty);
            }
            __syncwarp();
            return true;
          };
          ok = wait_warp(&b.q_full, items & 1u, abort_flag) && scores(0);
          if (ok) ok = wait_warp(&b.do_full, items & 1u, abort_flag) && dprobs(0);
          if (ok && w.n > 1) ok = scores(1);
          for (int j = 0; j < w.n && ok; ++j) {
            const uint32_t m = n + (uint32_t)j;
            if (!(ok = wait_warp(&b.dp_read, m & 1u, abort_flag))) break;
            if (j + 1 < w.n) {
              fence_after();
              if (!(ok = dprobs(j + 1))) break;
            }
            // the last tile's sums have been read before this one's are begun
            if (j == 0 && !(ok = wait_warp(&b.out_empty, (items & 1u) ^ 1u, abort_flag))) break;
            if (!(ok = wait_warp(b.ds_ready + (m & 1), (m >> 1) & 1u, abort_flag))) break;
            fence_after();
            if (elect()) {
              const uint32_t ds = tmem + C::kS + (m & 1) * 128;
              mma_rows<0, 8, kCols / 16, kCols>(tmem + C::kDq, ds, k_ring + (m % C::kK) * C::kTile, id_o, j > 0);
              commit(b.k_empty + m % C::kK);
              if (j + 1 == w.n) commit(&b.out_full);
            }
            __syncwarp();
            if (j + 2 < w.n) ok = scores(j + 2);
          }
          n += (uint32_t)w.n;
          ++items;
        }
        if (!ok) break;
        id = next_tile(k);
        ok = id != -2;
        if (id < 0) break;
      }
      if (!ok) fail(kErrMma);
      __syncwarp();
      if (elect()) commit(&b.drain);
      __syncwarp();
      mbar_wait(&b.drain, 0, kWaitNs);
    }
  } else {
    // ------------------------------------------------------------ probabilities and score gradients: thread = query
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_dp = tmem + C::kDp + g * kCols + lanes;
    const F2 scale2 = f2(a.scale * kLog2e);
    bool ok = true;
    uint32_t n = 0, items = 0;
    int id = (int)blockIdx.x;
    for (int k = 0; ok; ++k) {
      const DqWork w = dq_work_at<SPLIT>(a, (unsigned)id, tiles);
      const int row = w.row0 + (warp & 3) * 32 + lane;
      const bool exists = w.sp.tile >= 0 && row < w.sp.len_q;
      float lse2 = INFINITY, delta = 0.f;
      if (exists) {
        const int64_t at = stat_row(a, w.sp.batch, w.head) + w.sp.first_q + row;
        const float x = load_past_l1(a.lse + at);
        lse2 = x == -INFINITY ? INFINITY : x * kLog2e;
        delta = load_past_l1(a.delta + at);
      }
      const int keys = !a.causal ? w.sp.len_k : (row + w.offset + 1 < w.sp.len_k ? row + w.offset + 1 : w.sp.len_k);
      const int keys_all = __shfl_sync(0xffffffffu, keys, 0);
      const F2 base2 = f2(-lse2), delta2 = f2(-delta);
      for (int j = 0; j < w.n; ++j, ++n) {
        const int key0 = (w.j0 + j) * 128 + g * kCols;
        const bool masked = keys_all < key0 + kCols;
        const int left = keys - key0;
        if (!(ok = wait_warp(b.s + (n & 1), (n >> 1) & 1u, abort_flag))) break;
        fence_after();
        const uint32_t t_s = tmem + C::kS + (n & 1) * 128 + g * kCols + lanes;
        F2 p[kCols / 2];
        uint32_t s[kCols / 32][32];
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld32(t_s + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_wait_ld(s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            split(fma2(f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, base2), x0, x1);
            p[c * 16 + e] = f2(ex2_hw(x0), ex2_hw(x1));
          }
        if (!(ok = wait_warp(&b.dp, n & 1u, abort_flag))) break;
        fence_after();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld32(t_dp + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_wait_ld(s[c]);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.dp_read);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t wd[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            split(p[c * 16 + e] * (f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])) + delta2), x0, x1);
            if (masked) {
              x0 = c * 32 + 2 * e < left ? x0 : 0.f;
              x1 = c * 32 + 2 * e + 1 < left ? x1 : 0.f;
            }
            wd[e] = pack2<BF16>(x0, x1);
          }
          tmem_st16(t_s + c * 16, wd);
        }
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b.ds_ready + (n & 1));
      }
      if (ok && w.n > 0) {
        ok = wait_warp(&b.out_full, items & 1u, abort_flag);
        ++items;
        fence_after();
      }
      if (!ok) break;
      if (w.sp.tile < 0) {
        if (a.zero_tail) zero_rows(a.dq, w.head, w.sp.first_q, 128, a.Sq, a.D, threadIdx.x, kCompute * 32);
      } else {
        // each warpgroup writes its share of the columns
        constexpr int per = DP * 4 / C::kOutWarps;
        const bool wide = rows_are_wide(a.dq);
        uint16_t* out = row_ptr(a.dq, w.sp.batch, w.head, w.sp.first_q + row);
        if (warp < C::kOutWarps) {
#pragma unroll
          for (int c = 0; c < per / 32; ++c) {
            const int col = g * per + c * 32;
            uint32_t o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
            if (w.n > 0) {
              tmem_ld32(tmem + C::kDq + lanes + col, o);
              tmem_wait_ld(o);
              if (c == per / 32 - 1) {                       // the sums may be written again
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.out_empty);
              }
            }
            if (!exists) continue;
            if constexpr (SPLIT) store32_f32(part_row(a.partial, w.part, a.B, a.H, a.Sq, a.D, w.sp.batch, w.head, row), col, a.D, o, a.scale);
            else store32<BF16>(out, col, a.D, o, a.scale, wide);
          }
        }
      }
      id = next_tile(k);
      ok = id != -2;
      if (id < 0) break;
    }
    if (!ok) fail(kErrCompute);
  }
  if (beside) pdl_wait();
  fence_before();
  __syncthreads();
  if (warp == kCompute + 1) {
    fence_after();
    tmem_free(tmem, 512);
  }
}

// A gradient from its parts, added up in order: dst = sum of `parts` arrays of [batch][head][row][D].  Sixteen lanes per row.
template <bool BF16>
__global__ void __launch_bounds__(256) attention_sum_kernel(const float* partial, int parts, AttnTensor dst, int B, int H, int S, int D) {
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x & 15;
  const int64_t rows = (int64_t)B * H * S, r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (r >= rows || sub * 8 >= D) return;
  const int64_t bh = r / S;
  const int row = (int)(r - bh * S), b = (int)(bh / H), h = (int)(bh - (int64_t)b * H);
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float4* v = reinterpret_cast<const float4*>(partial + (p * rows + r) * D + sub * 8);
    const float4 u = v[0], w = v[1];
    o[0] += u.x, o[1] += u.y, o[2] += u.z, o[3] += u.w;
    o[4] += w.x, o[5] += w.y, o[6] += w.z, o[7] += w.w;
  }
  *reinterpret_cast<uint4*>(row_ptr(dst, b, h, row) + sub * 8) =
      make_uint4(pack2<BF16>(o[0], o[1]), pack2<BF16>(o[2], o[3]), pack2<BF16>(o[4], o[5]), pack2<BF16>(o[6], o[7]));
}
template <bool BF16>
cudaError_t add_parts(const float* partial, int parts, const AttnTensor& dst, int B, int H, int S, int D, cudaStream_t stream,
                      int64_t& kernels) {
  const int64_t blocks = ((int64_t)B * H * S + 15) / 16;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return launch_counted(kernels, attention_sum_kernel<BF16>, dim3((unsigned)blocks), dim3(256), 0, stream, partial, parts, dst, B, H, S, D);
}

// The shared-memory limit is an attribute of the function on the current device.
template <auto KERNEL>
cudaError_t allow_smem(uint32_t bytes) {
  static thread_local bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && configured[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev] = true;
  return e;
}

template <int DP, bool BF16, bool SPLIT>
cudaError_t launch_dkv(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mdo, const AttnArgs& a,
                       cudaStream_t stream, int64_t& kernels) {
  const cudaError_t e = allow_smem<attention_dkv_kernel<DP, BF16, SPLIT>>(Dkv<DP>::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t tiles = a.cu_q != nullptr ? max_tiles(a.Sk, a.nseq, 128) : ((int64_t)a.Sk + 127) / 128;
  const int64_t ctas = tiles * a.Hk * a.B * a.parts_dkv;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  return launch_counted(kernels, attention_dkv_kernel<DP, BF16, SPLIT>, dim3((unsigned)ctas), dim3(kThreads), Dkv<DP>::kSmem, stream, mq,
                        mk, mv, mdo, a);
}
template <int DP, bool BF16, bool SPLIT>
cudaError_t launch_dq(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mdo, const AttnArgs& a,
                      cudaStream_t stream, int64_t& kernels) {
  const cudaError_t e = allow_smem<attention_dq_kernel<DP, BF16, SPLIT>>(Dq<DP>::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t tiles = a.cu_q != nullptr ? max_tiles(a.Sq, a.nseq, 128) : ((int64_t)a.Sq + 127) / 128;
  const int64_t ctas = tiles * a.H * a.B * a.parts_dq;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  const bool beside = a.Sk > 0 && a.parts_dkv == 1;          // the dk/dv kernel is right in front, and no part of its work is in this one's memory
  return launch_counted(kernels, attention_dq_kernel<DP, BF16, SPLIT>, dim3((unsigned)ctas), dim3(kThreads), Dq<DP>::kSmem, stream, mq, mk,
                        mv, mdo, a, (int)tiles, beside);
}

template <int DP, bool BF16>
cudaError_t launch(const AttnArgs& a, cudaStream_t stream, int64_t& kernels) {
  const bool packed = a.cu_q != nullptr;
  CUtensorMap mq, mk, mv, mdo;
  if (a.Sq > 0 && (!make_map(&mq, a.q, BF16, a.D, a.H, a.Sq, a.B) || !make_map(&mdo, a.dout, BF16, a.D, a.H, a.Sq, a.B)))
    return cudaErrorInvalidValue;
  if (a.Sk > 0 && (!make_map(&mk, a.k, BF16, a.D, a.Hk, a.Sk, a.B) || !make_map(&mv, a.v, BF16, a.D, a.Hk, a.Sk, a.B)))
    return cudaErrorInvalidValue;
  if (a.Sq == 0) mq = mdo = mk;                              // nothing of what is missing is ever loaded
  if (a.Sk == 0) mk = mv = mq;
  if (packed) {
    const cudaError_t e = launch_counted(kernels, attention_orders_kernel, dim3(2), dim3(1024), 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  if (a.Sq > 0) {
    if (a.B > 65535) return cudaErrorInvalidValue;
    const cudaError_t e = launch_counted(kernels, attention_delta_kernel<BF16>,
                                         dim3((unsigned)((a.Sq + 63) / 64), (unsigned)a.H, (unsigned)a.B), dim3(256), 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  if (a.Sk > 0) {
    cudaError_t e = a.parts_dkv > 1 ? launch_dkv<DP, BF16, true>(mq, mk, mv, mdo, a, stream, kernels)
                                    : launch_dkv<DP, BF16, false>(mq, mk, mv, mdo, a, stream, kernels);
    if (e != cudaSuccess) return e;
    if (a.parts_dkv > 1) {
      if ((e = add_parts<BF16>(a.partial, a.parts_dkv, a.dv, a.B, a.Hk, a.Sk, a.D, stream, kernels)) != cudaSuccess) return e;
      const float* dk = a.partial + (int64_t)a.parts_dkv * a.B * a.Hk * a.Sk * a.D;
      if ((e = add_parts<BF16>(dk, a.parts_dkv, a.dk, a.B, a.Hk, a.Sk, a.D, stream, kernels)) != cudaSuccess) return e;
    }
  }
  if (a.Sq > 0) {
    cudaError_t e = a.parts_dq > 1 ? launch_dq<DP, BF16, true>(mq, mk, mv, mdo, a, stream, kernels)
                                   : launch_dq<DP, BF16, false>(mq, mk, mv, mdo, a, stream, kernels);
    if (e != cudaSuccess) return e;
    if (a.parts_dq > 1 && (e = add_parts<BF16>(a.partial, a.parts_dq, a.dq, a.B, a.H, a.Sq, a.D, stream, kernels)) != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

}  // namespace

// Tiles are split where they alone leave SMs without work and the longest walk is of sixteen steps or more, into parts of four steps
// or more: the parts' sums take another launch each and part the kernels for dk, dv and dq, about eight steps' time.  A group of many
// heads on few key heads makes few and long tiles: those are cut until there are two for each SM.  Both kernels use the same
// memory for their parts, one after the other.  Measured, whole / split (us): 2048 x 16 heads on one key head (18 parts for dk, dv)
// 443 / 116; 256 queries on 4096 keys, 8 heads (8 for dq) 63 / 43; 1021 on 4093, 16 heads on 4 of 80 (2 for dk, dv) 132 / 122; 2 x 1000,
// 12 heads on 3 (6 for dk, dv) 54 / 51.  Below the line, in two parts: 128 queries on 1024 keys, 4 heads (dq) 16.7 / 14.9;
// 512 x 4 heads (dq) 14.0 / 16.1, (dk, dv) 24.6; 1024 x 8 heads (dq) 24.1 / 27.9.
AttnScratch plan_attention_backward(AttnArgs& a, int sm_count) {
  a.parts_dq = a.parts_dkv = 1;
  AttnScratch need = {0, 0, 0, 0};
  if (a.cu_q != nullptr) {
    need.order_q = max_tiles(a.Sq, a.nseq, 128);
    need.order_k = max_tiles(a.Sk, a.nseq, 128);
    return need;
  }
  if (a.Sq <= 0 || a.Sk <= 0 || a.B <= 0) return need;
  const int64_t q_tiles = ((int64_t)a.Sq + 127) / 128, k_tiles = ((int64_t)a.Sk + 127) / 128;
  const int64_t dq = q_tiles * a.H * a.B, dkv = k_tiles * a.Hk * a.B, steps = q_tiles * (a.H / a.Hk);
  auto parts = [](int64_t room, int64_t steps) {
    const int64_t p = room < steps / 4 ? room : steps / 4;
    return steps >= 16 && p > 1 ? (int)p : 1;
  };
  if (dq < sm_count) a.parts_dq = parts(sm_count / dq, k_tiles);
  if (dkv < sm_count) a.parts_dkv = parts((a.H > a.Hk ? 2 : 1) * sm_count / dkv, steps);
  const int64_t dq_floats = a.parts_dq > 1 ? (int64_t)a.parts_dq * a.B * a.H * a.Sq * a.D : 0;
  const int64_t dkv_floats = a.parts_dkv > 1 ? (int64_t)2 * a.parts_dkv * a.B * a.Hk * a.Sk * a.D : 0;
  need.partial = dq_floats > dkv_floats ? dq_floats : dkv_floats;
  return need;
}

cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream, int64_t& kernels) {
  if (a.B <= 0 || a.H <= 0 || (a.Sq <= 0 && a.Sk <= 0)) return cudaSuccess;
  if (a.Hk <= 0 || a.H % a.Hk != 0 || a.D <= 0 || a.D % 8 != 0 || a.D > kAttnMaxDim || a.Sk < 0 || a.Sq < 0 || a.parts_dq < 1 || a.parts_dkv < 1)
    return cudaErrorInvalidValue;
  if (a.D <= 64) return a.is_bf16 ? launch<64, true>(a, stream, kernels) : launch<64, false>(a, stream, kernels);
  return a.is_bf16 ? launch<128, true>(a, stream, kernels) : launch<128, false>(a, stream, kernels);
}

}  // namespace pccl
