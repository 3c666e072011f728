// Attention, forward pass: one CTA per 256 queries of one head, a running maximum and sum per query, keys and values in one
// pass (attention.h has the formulas, attention.cuh the tiles).
//
//   warps 0-3   softmax of queries 0-127: one query per thread, its 128 scores of a key tile in registers
//   warps 4-7   the same for queries 128-255
//   warp 8      TMA: the query tiles, then key and value tiles into a ring; asks for the next tile of the grid
//   warp 9      tensor memory; one thread issues the products
// The products of one half run while the other half is in its softmax:
//   S0(j)  S1(j) | P0(j) V -> O0, S0(j+1) | P1(j) V -> O1, S1(j+1) | ...
// Tensor memory: S0, S1 (128 columns each, P over the first 64 of them), O0, O1 (DP columns each).  Products of one CTA run in
// the order of issue, so S0(j+1) may be written over P0(j), and a finished S0(j+1) says that O0 holds the sum up to j.
// P is handed over in two halves, so that its product begins while the other half is still in its exponentials.
//
// What bounds it.  16 heads of 16384 causal take 870 us, 1265 TFLOP/s; with the softmax left out the products alone take 735
// (1495 TFLOP/s, 0.91 of the measured rate: both operands of Q K^T come from shared memory, 128 bytes per cycle for 128 x 128 tiles).
// The exponentials are not the limit: without them the same call takes as long, and moving a quarter of them to the
// multiply-add units as a polynomial made it slower (928 us).  The chain product - maximum - exponentials - product is, and
// the clock, which the power limit takes down to 1.69 GHz.
// Shorter sequences pay for the start and the end of each tile: 4 x 2048 x 16 heads of 128 causal 82 us (838 TFLOP/s), 63
// without softmax; heads of 64 69 us.  These are runs of some 30 calls; on a card that has been busy for seconds, whose clock is lower, the
// first takes 94 us (731 TFLOP/s).  The grid's tiles are taken over at run time (attention.cuh), so that the loads of the next
// tile overlap the end of the last: one CTA per tile took a seventh longer, two passes over the scores in tensor memory a quarter.
//
// The running maximum and sum of a softmax in one pass are Milakov and Gimelshein's (2018); to let the maximum lag is a published idea for
// this hardware, where reading O back costs more than headroom in the exponent.  It only follows the true one when it has fallen
// behind by a factor of 2^8: sums and products are then at most 2^8 times larger than with the true maximum, far inside fp32 and inside the range of 16-bit probabilities, and O, which
// would have to be read and written to be rescaled, is left alone for all but the first few tiles.  Probabilities are rounded
// to 16 bits for the product (half a step of the inputs' own type); their sum is taken before that, in 32 bits.
#include "attention.cuh"

namespace pccl {

namespace {

using namespace attn;

constexpr int kThreads = 384;                   // warps 10 and 11 only complete the third warpgroup
constexpr float kBehind = 8.f;                  // binary orders of magnitude that the running maximum may fall behind
constexpr int kReaders = 10;                    // of the next tile's number: eight softmax warps, loads, products

template <int DP>
struct Fwd {
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr uint32_t kTile = (DP / 64) * kBlockBytes;
  static constexpr uint32_t kRing = 2 * kTile;
  static constexpr uint32_t kBars = kRing + kStages * kTile;
  static constexpr uint32_t kSmem = kBars + 512 + 1024;     // barriers, slack for the alignment of the swizzled tiles
  static constexpr uint32_t kS = 0, kO = 256;               // tensor memory columns
  static constexpr uint32_t kCols = 512;
};

struct Bars {
  Handle next[2];
  uint64_t next_full[2], next_empty[2];
  uint64_t full[8], empty[8], q_full[2], q_empty[2], s[2], p0[2], p1[2], o_full[2], o_empty[2], fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= 512, "the barriers' part of shared memory");

// Scores from place `left` on become -inf.
__device__ __forceinline__ void mask32(uint32_t* r, int left) {
#pragma unroll
  for (int e = 0; e < 32; ++e) r[e] = e < left ? r[e] : 0xff800000u;
}

// The queries of one tile number, and the key tiles that each half of them has to do with: n[h] of them from tile j0 on.
struct Work {
  Span sp;
  int head, row0, offset, j0, part, n[2];
};
template <bool SPLIT>
__device__ __forceinline__ Work work_at(const AttnArgs& a, unsigned id, int tiles) {
  Work w;
  w.part = 0;
  if constexpr (SPLIT) {
    w.part = (int)(id % (unsigned)a.parts_o);
    id /= (unsigned)a.parts_o;
  }
  if (a.cu_q != nullptr) {
    w.head = (int)(id % (unsigned)a.H);
    w.sp = find_span<false>(a, (int)(id / (unsigned)a.H), 256, false);
  } else {
    // with a causal mask the last tiles have the most keys: they come first
    const unsigned heads = (unsigned)(a.B * a.H), bh = id % heads, t = id / heads;
    w.head = (int)(bh % (unsigned)a.H);
    w.sp.batch = (int)(bh / (unsigned)a.H);
    w.sp.first_q = w.sp.first_k = 0;
    w.sp.len_q = a.Sq;
    w.sp.len_k = a.Sk;
    w.sp.tile = a.causal ? tiles - 1 - (int)t : (int)t;
  }
  w.row0 = w.sp.tile * 256;
  w.offset = w.sp.len_k - w.sp.len_q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int first = w.row0 + h * 128;
    const int last = first + 127 < w.sp.len_q - 1 ? first + 127 : w.sp.len_q - 1;
    const int keys = !a.causal ? w.sp.len_k : (last + w.offset + 1 < w.sp.len_k ? last + w.offset + 1 : w.sp.len_k);
    w.n[h] = w.sp.tile >= 0 && first < w.sp.len_q && keys > 0 ? (keys + 127) / 128 : 0;
  }
  w.j0 = 0;
  if constexpr (SPLIT) {                                     // an even share of the longer half's key tiles
    const int most = w.n[0] > w.n[1] ? w.n[0] : w.n[1];
    w.j0 = most * w.part / a.parts_o;
    const int j1 = most * (w.part + 1) / a.parts_o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int end = w.n[h] < j1 ? w.n[h] : j1;
      w.n[h] = end > w.j0 ? end - w.j0 : 0;
    }
  }
  return w;
}

template <int DP, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attention_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a, int tiles) {
  using C = Fwd<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Bars& b = *reinterpret_cast<Bars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(b.full + i, 1);
      mbar_init(b.empty + i, 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(b.next_full + h, 1);
      mbar_init(b.next_empty + h, kReaders);
      mbar_init(b.q_full + h, 1);
      mbar_init(b.q_empty + h, 1);
      mbar_init(b.s + h, 1);
      mbar_init(b.p0 + h, 4);
      mbar_init(b.p1 + h, 4);
      mbar_init(b.o_full + h, 1);
      mbar_init(b.o_empty + h, 4);
    }
    mbar_init(&b.fix, 1);
    mbar_init(&b.drain, 1);
    b.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(&b.tmem, C::kCols);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = b.tmem;
  pdl_wait();
  pdl_trigger();

  // The tile after the k-th, for every role alike: -1 none, -2 a wait gave up.  Whole warps.
  auto next_tile = [&](int k) {
    if (!wait_warp(b.next_full + (k & 1), (k >> 1) & 1u, abort_flag)) return -2;
    const int id = work_taken(b.next + (k & 1));
    __syncwarp();
    if (lane == 0) mbar_arrive(b.next_empty + (k & 1));
    return id;
  };

  // Registers: 384 threads start with 168 each, 64,512 together.  A thread that holds 128 scores wants more, the issuing warps
  // less: 256 x 216 + 128 x 72 = 64,512.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ---------------------------------------------------------- loads, and the tiles to come
      bool ok = true;
      uint32_t it = 0, fixes = 0, q_count[2] = {0, 0};
      int k = 0;
      for (int id = (int)blockIdx.x;; ++k) {
        if (k >= 2 && !wait_warp(b.next_empty + (k & 1), ((k >> 1) - 1) & 1u, abort_flag)) {
          ok = false;
          break;
        }
        if (lane == 0) ask_for_work(b.next + (k & 1), b.next_full + (k & 1));
        const Work w = work_at<SPLIT>(a, (unsigned)id, tiles);
        const int kv_head = w.head / (a.H / a.Hk), nmax = w.n[0] > w.n[1] ? w.n[0] : w.n[1];
        for (int i = 0; i < 2 * nmax && ok; ++i, ++it) {     // K0, V0, K1, V1, ...
          const uint32_t st = it % C::kStages, ph = (it / C::kStages) & 1u;
          if (!(ok = wait_warp(b.empty + st, ph ^ 1u, abort_flag))) break;
          const int row = (w.j0 + (i >> 1)) * 128;
          const bool value = (i & 1) != 0;
          unsigned char* dst = smem + C::kRing + st * C::kTile;
          // the rows behind a packed sequence are its neighbour's
          const bool ragged = value && a.cu_q != nullptr && row + 128 > w.sp.len_k;
          uint64_t* bar = ragged ? &b.fix : b.full + st;
          if (lane == 0) {
            mbar_expect_tx(bar, C::kTile);
            load_tile<DP>(dst, value ? &map_v : &map_k, kv_head, w.sp.first_k + row, w.sp.batch, bar);
          }
          if (ragged) {
            ok = wait_warp(&b.fix, fixes++ & 1u, abort_flag);
            clear_rows<DP>(dst, w.sp.len_k - row);
            if (lane == 0) mbar_arrive(b.full + st);
          }
          if (i == 0) {                                      // behind the first key tile: the queries of the last tile may still be in use
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (w.n[h] == 0 || !ok) continue;
              if (!(ok = wait_warp(b.q_empty + h, (q_count[h] & 1u) ^ 1u, abort_flag))) continue;
              ++q_count[h];
              if (lane == 0) {
                mbar_expect_tx(b.q_full + h, C::kTile);
                load_tile<DP>(smem + h * C::kTile, &map_q, w.head, w.sp.first_q + w.row0 + h * 128, w.sp.batch, b.q_full + h);
              }
            }
          }
        }
        if (!ok) break;
        id = next_tile(k);
        if (id < 0) {
          ok = id == -1;
          break;
        }
      }
      if (!ok) {
        if (lane == 0) {
          atomicCAS(a.error, 0, kErrLoad);
          *abort_flag = 1;
        }
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);    // which copies are on their way is not known: the time that they can take
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- products
      constexpr uint32_t id_s = idesc(BF16, 128, false);
      const int steps = steps_of(a.D);
      const uint32_t id_o = idesc(BF16, steps * 16, true);
      const uint32_t q_addr = smem_u32(smem), ring = smem_u32(smem + C::kRing);
      bool ok = true;
      uint32_t it = 0, s_count[2] = {0, 0}, items[2] = {0, 0};     // ring position; tiles and work items of each half
      int id = (int)blockIdx.x;
      for (int k = 0;; ++k) {
        const Work w = work_at<SPLIT>(a, (unsigned)id, tiles);
        const int nmax = w.n[0] > w.n[1] ? w.n[0] : w.n[1];
        if (nmax > 0) {
          auto tile_at = [&](uint32_t i) { return ring + (i % C::kStages) * C::kTile; };
          auto loaded = [&](uint32_t i) { return wait_warp(b.full + i % C::kStages, (i / C::kStages) & 1u, abort_flag); };
          auto scores = [&](int h, int j) {
            if (elect()) {
              mma_columns<DP>(tmem + C::kS + h * 128, q_addr + h * C::kTile, tile_at(it + 2 * j), id_s, steps);
              commit(b.s + h);
              if (j + 1 == w.n[h]) commit(b.q_empty + h);    // the queries are not read again
            }
            __syncwarp();
          };
          auto release = [&](uint32_t i) {
            if (elect()) commit(b.empty + i % C::kStages);
            __syncwarp();
          };
          ok = loaded(it);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (ok && w.n[h] > 0) {
              ok = wait_warp(b.q_full + h, items[h] & 1u, abort_flag);
              if (ok) scores(h, 0);
            }
          if (ok) release(it);
          for (int j = 0; j < nmax && ok; ++j) {
            if (!(ok = loaded(it + 2 * j + 1))) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!ok) break;
              if (j < w.n[h]) {
                // the last tile's sums have been read out of O before this one's are begun
                if (j == 0 && !(ok = wait_warp(b.o_empty + h, (items[h] & 1u) ^ 1u, abort_flag))) break;
                const uint32_t ph = (s_count[h] + (uint32_t)j) & 1u, p = tmem + C::kS + h * 128, v = tile_at(it + 2 * j + 1);
                if (!(ok = wait_warp(b.p0 + h, ph, abort_flag))) break;
                fence_after();
                if (elect()) mma_rows<0, 4, 8, 0>(tmem + C::kO + h * 128, p, v, id_o, j > 0);
                __syncwarp();
                if (!(ok = wait_warp(b.p1 + h, ph, abort_flag))) break;
                fence_after();
                if (elect()) {
                  mma_rows<4, 8, 8, 0>(tmem + C::kO + h * 128, p, v, id_o, true);
                  if (j + 1 == w.n[h]) commit(b.o_full + h);
                }
                __syncwarp();
              }
              if (h == 0 && j + 1 < nmax) ok = loaded(it + 2 * j + 2);
              if (ok && j + 1 < w.n[h]) scores(h, j + 1);
            }
            if (!ok) break;
            release(it + 2 * j + 1);
            if (j + 1 < nmax) release(it + 2 * j + 2);
          }
          it += 2 * (uint32_t)nmax;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (w.n[h] > 0) {
              s_count[h] += (uint32_t)w.n[h];
              ++items[h];
            }
        }
        if (!ok) break;
        id = next_tile(k);
        if (id < 0) {
          ok = id == -1;
          break;
        }
      }
      if (!ok && lane == 0) {
        atomicCAS(a.error, 0, kErrMma);
        *abort_flag = 1;
      }
      __syncwarp();
      if (elect()) commit(&b.drain);
      __syncwarp();
      mbar_wait(&b.drain, 0, kWaitNs);
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = query
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int h = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + C::kS + h * 128 + lanes, t_o = tmem + C::kO + h * 128 + lanes;
    const float sl2 = a.scale * kLog2e;
    const float behind = kBehind / sl2;
    bool ok = true;
    uint32_t s_count = 0, items = 0;
    int id = (int)blockIdx.x;
    for (int k = 0;; ++k) {
      const Work w = work_at<SPLIT>(a, (unsigned)id, tiles);
      const int n = h == 0 ? w.n[0] : w.n[1];
      const int row = w.row0 + h * 128 + (warp & 3) * 32 + lane;         // within the sequence
      const int keys = !a.causal ? w.sp.len_k : (row + w.offset + 1 < w.sp.len_k ? row + w.offset + 1 : w.sp.len_k);   // that this query sees
      const int keys_all = __shfl_sync(0xffffffffu, keys, 0);           // that every query of the warp sees
      const int keys_left = keys - w.j0 * 128, all_left = keys_all - w.j0 * 128;      // from the first of its key tiles on
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++s_count) {
        if (!(ok = wait_warp(b.s + h, s_count & 1u, abort_flag))) break;
        fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld(s[c]);
        const bool masked = all_left < (j + 1) * 128;
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask32(s[c], keys_left - j * 128 - c * 32);
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = fmaxf(fmaxf(top[i], __uint_as_float(s[c][e + i])), __uint_as_float(s[c][e + 4 + i]));
        const float m_new = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m);
        if (__any_sync(0xffffffffu, m_new > m + behind)) {
          const float f = m_new == m ? 1.f : ex2_hw((m - m_new) * sl2);
          m = m_new;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + c * 32, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(t_o + c * 32, o);
            }
          }
        }
        const F2 scale2 = f2(sl2), base2 = f2(m == -INFINITY ? 0.f : -m * sl2);
        F2 sum2[2] = {f2(0.f), f2(0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t wd[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const F2 x = fma2(f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, base2);
            float x0, x1;
            split(x, x0, x1);
            x0 = ex2_hw(x0);
            x1 = ex2_hw(x1);
            sum2[e & 1] = sum2[e & 1] + f2(x0, x1);
            wd[e] = pack2<BF16>(x0, x1);
          }
          tmem_st16(t_s + c * 16, wd);
          if (c == 1) {                                                // the product may begin with the first half
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b.p0 + h);
          }
        }
        float a0, a1;
        split(sum2[0] + sum2[1], a0, a1);
        l += a0 + a1;
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b.p1 + h);
      }
      if (ok && n > 0) {
        ok = wait_warp(b.o_full + h, items & 1u, abort_flag);
        ++items;
        fence_after();
      }
      if (!ok) break;
      if (w.sp.tile < 0) {                                             // behind the last sequence
        if (a.zero_tail) zero_rows(a.o, w.head, w.sp.first_q, 256, a.Sq, a.D, threadIdx.x, 256);
        const int r = w.sp.first_q + (int)threadIdx.x;
        if (r < a.Sq) a.lse[stat_row(a, 0, w.head) + r] = -INFINITY;
      } else {
        const bool exists = row < w.sp.len_q, wide = rows_are_wide(a.o);
        const bool none = l == 0.f;                                    // no key is seen (scores that are NaN leave l NaN)
        const float inv = none ? 0.f : 1.f / l;
        uint16_t* out = row_ptr(a.o, w.sp.batch, w.head, w.sp.first_q + row);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
          if (n > 0) {
            tmem_ld32(t_o + c * 32, o);
            tmem_wait_ld(o);
            if (c == DP / 32 - 1) {                                    // O may be written again
              fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(b.o_empty + h);
            }
          }
          if (none) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          if (!exists) continue;
          if constexpr (SPLIT) store32_f32(part_row(a.partial, w.part, a.B, a.H, a.Sq, a.D, w.sp.batch, w.head, row), c * 32, a.D, o, inv);
          else store32<BF16>(out, c * 32, a.D, o, inv, wide);
        }
        if (exists) {
          float* lse = SPLIT ? a.partial_lse + (int64_t)w.part * a.B * a.H * a.Sq : a.lse;
          lse[stat_row(a, w.sp.batch, w.head) + w.sp.first_q + row] = none ? -INFINITY : m * a.scale + logf(l);
        }
      }
      id = next_tile(k);
      if (id < 0) {
        ok = id == -1;
        break;
      }
    }
    if (!ok && lane == 0) {
      atomicCAS(a.error, 0, kErrCompute);
      *abort_flag = 1;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    tmem_free(tmem, C::kCols);
  }
}

__global__ void __launch_bounds__(1024) attention_order_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  write_order(a.cu_q, a.nseq, a.Sq, 256, false, a.order_q);
}

// The parts of one row joined: lse = log(sum of exp(lse_part)), o = sum of exp(lse_part - lse) o_part.  Sixteen lanes per row.
template <bool BF16>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x & 15;
  const int64_t rows = (int64_t)a.B * a.H * a.Sq, r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (r >= rows) return;
  const int64_t bh = r / a.Sq;
  const int row = (int)(r - bh * a.Sq), b = (int)(bh / a.H), h = (int)(bh - (int64_t)b * a.H);
  float top = -INFINITY;
  for (int p = 0; p < a.parts_o; ++p) {
    const float x = a.partial_lse[p * rows + r];
    top = x > top || x != x ? x : top;                       // NaN stays
  }
  float sum = 0.f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  const bool on = sub * 8 < a.D;
  if (top != -INFINITY) {
    for (int p = 0; p < a.parts_o; ++p) {
      const float x = a.partial_lse[p * rows + r];
      if (x == -INFINITY) continue;                          // a part in which this query sees no key
      const float f = ex2_hw((x - top) * kLog2e);
      sum += f;
      if (on) {
        const float4* v = reinterpret_cast<const float4*>(a.partial + (p * rows + r) * a.D + sub * 8);
        const float4 u = v[0], w = v[1];
        o[0] = fmaf(f, u.x, o[0]), o[1] = fmaf(f, u.y, o[1]), o[2] = fmaf(f, u.z, o[2]), o[3] = fmaf(f, u.w, o[3]);
        o[4] = fmaf(f, w.x, o[4]), o[5] = fmaf(f, w.y, o[5]), o[6] = fmaf(f, w.z, o[6]), o[7] = fmaf(f, w.w, o[7]);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (on)
    *reinterpret_cast<uint4*>(row_ptr(a.o, b, h, row) + sub * 8) =
        make_uint4(pack2<BF16>(o[0] * inv, o[1] * inv), pack2<BF16>(o[2] * inv, o[3] * inv), pack2<BF16>(o[4] * inv, o[5] * inv),
                   pack2<BF16>(o[6] * inv, o[7] * inv));
  if (sub == 0) a.lse[r] = top == -INFINITY ? -INFINITY : top + logf(sum);
}

template <int DP, bool BF16, bool SPLIT>
cudaError_t launch(const AttnArgs& a, cudaStream_t stream, int64_t& kernels) {
  using C = Fwd<DP>;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, a.q, BF16, a.D, a.H, a.Sq, a.B)) return cudaErrorInvalidValue;
  if (a.Sk == 0) mk = mv = mq;                               // no key is ever loaded
  else if (!make_map(&mk, a.k, BF16, a.D, a.Hk, a.Sk, a.B) || !make_map(&mv, a.v, BF16, a.D, a.Hk, a.Sk, a.B)) return cudaErrorInvalidValue;
  auto kernel = attention_fwd_kernel<DP, BF16, SPLIT>;
  static thread_local bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t tiles = a.cu_q != nullptr ? max_tiles(a.Sq, a.nseq, 256) : ((int64_t)a.Sq + 255) / 256;
  const int64_t ctas = tiles * a.H * a.B * a.parts_o;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  if (a.cu_q != nullptr) {
    if ((e = launch_counted(kernels, attention_order_kernel, dim3(1), dim3(1024), 0, stream, a)) != cudaSuccess) return e;
  }
  e = launch_counted(kernels, kernel, dim3((unsigned)ctas), dim3(kThreads), C::kSmem, stream, mq, mk, mv, a, (int)tiles);
  if (e != cudaSuccess || !SPLIT) return e;
  const int64_t blocks = ((int64_t)a.B * a.H * a.Sq + 15) / 16;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return launch_counted(kernels, attention_join_kernel<BF16>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

template <int DP, bool BF16>
cudaError_t launch_type(const AttnArgs& a, cudaStream_t stream, int64_t& kernels) {
  return a.parts_o > 1 ? launch<DP, BF16, true>(a, stream, kernels) : launch<DP, BF16, false>(a, stream, kernels);
}

}  // namespace

// A tile's keys are split where the tiles alone leave SMs without work, into as many parts as the device has room for, of four
// key tiles or more; the join takes another launch.  Measured, whole / split (us): 1021 queries on 4093 keys, 16 heads of 80
// (2 parts) 60 / 45; 256 on 4096, 8 heads (8 parts) 61 / 24, in 16 parts 27; 128 on 1024, 4 heads (2 parts) 15.2 / 13.9, in 8 parts
// 11.6.  Causal calls, whose tiles are of different lengths, gain little or nothing near the line: 1024 x 8 heads (2 parts)
// 20.4 / 21.9; below it, in parts of two tiles, 512 x 4 heads 11.6 / 12.9.
AttnScratch plan_attention_forward(AttnArgs& a, int sm_count) {
  a.parts_o = 1;
  const int64_t tiles = ((int64_t)a.Sq + 255) / 256 * a.H * a.B, key_tiles = ((int64_t)a.Sk + 127) / 128;
  if (a.cu_q == nullptr && tiles > 0 && tiles < sm_count) {
    const int64_t room = sm_count / tiles, most = key_tiles / 4;
    a.parts_o = (int)(room < most ? room : most);
    if (a.parts_o < 1) a.parts_o = 1;
  }
  AttnScratch need = {0, 0, 0, 0};
  if (a.cu_q != nullptr) need.order_q = max_tiles(a.Sq, a.nseq, 256);
  if (a.parts_o > 1) {
    need.partial_lse = (int64_t)a.parts_o * a.B * a.H * a.Sq;
    need.partial = need.partial_lse * a.D;
  }
  return need;
}

cudaError_t launch_attention_forward(const AttnArgs& a, cudaStream_t stream, int64_t& kernels) {
  if (a.B <= 0 || a.H <= 0 || a.Sq <= 0) return cudaSuccess;
  if (a.Hk <= 0 || a.H % a.Hk != 0 || a.D <= 0 || a.D % 8 != 0 || a.D > kAttnMaxDim || a.Sk < 0 || a.parts_o < 1) return cudaErrorInvalidValue;
  if (a.D <= 64) return a.is_bf16 ? launch_type<64, true>(a, stream, kernels) : launch_type<64, false>(a, stream, kernels);
  return a.is_bf16 ? launch_type<128, true>(a, stream, kernels) : launch_type<128, false>(a, stream, kernels);
}

}  // namespace pccl
