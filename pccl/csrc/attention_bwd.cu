// Attention, backward pass: a kernel for the row sums <do_i, o_i>, one for dk and dv, one for dq (attention.h has the formulas,
// attention.cuh the tiles).
//
// Two kernels share the work so that every gradient has one owner: a CTA keeps 128 keys (dk, dv) or 128 queries (dq) and walks
// over the others, and its sums stay in tensor memory until they are complete.  Scores and do v^T are computed twice, seven
// products instead of five; what is saved are fp32 atomic additions of a whole dq per key tile, and results are the same bits
// from run to run.  The heads of a group are walked over one after the other by the CTA that owns their shared key head.
//
//   warps 0-7   probabilities and score gradients: two warpgroups, each with half of a tile's 128 columns
//   warp 8      TMA
//   warp 9      tensor memory; one thread issues the products
//
// dk, dv: scores are computed transposed, S = K Q^T, so that a thread owns a key and the 16-bit P^T and dS^T lie in tensor memory
// as the first operand of dv += P^T dO and dk += dS^T Q.  The products of one tile run while the other operand is being made:
//   S(i) | P(i): dv += P^T dO, S(i+1) | dS(i): dk += dS^T Q, dP(i+1) | ...
// dq: S = Q K^T and dP = dO V^T as in the forward pass, dq += dS K; S is kept twice, so that its next tile is ready when the
// exponentials of the last one are done.
#include "attention.cuh"

namespace pccl {

namespace {

using namespace attn;

constexpr int kThreads = 320;

// ---------------------------------------------------------------- row sums
// delta_i = <do_i, o_i>: sixteen lanes per row, two rows per warp and step.  One read of both tensors.
template <bool BF16>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ AttnArgs a) {
  const int sub = threadIdx.x & 15;
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  const bool on = sub * 8 < a.D;
  for (int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4; r < ((rows + 1) & ~(int64_t)1); r += (int64_t)gridDim.x * 16) {
    const int64_t bs = r / a.H;
    const int h = (int)(r - bs * a.H), b = (int)(bs / a.Sq), s = (int)(bs - (int64_t)b * a.Sq);
    float acc = 0.f;
    if (r < rows && on) {
      const uint4 x = *reinterpret_cast<const uint4*>(row_ptr(a.dout, b, h, s) + sub * 8);
      const uint4 y = *reinterpret_cast<const uint4*>(row_ptr(a.o, b, h, s) + sub * 8);
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
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
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (r < rows && sub == 0) a.delta[stat_row(a, b, h) + s] = acc;
  }
}

// ---------------------------------------------------------------- dk, dv
template <int DP>
struct Dkv {
  static constexpr int kStages = DP == 128 ? 2 : 4;          // of each of the two rings
  static constexpr uint32_t kTile = (DP / 64) * kBlockBytes;
  static constexpr uint32_t kQ = 2 * kTile, kDo = kQ + kStages * kTile;
  static constexpr uint32_t kStat = kDo + kStages * kTile;   // [2][warpgroup][lse, delta][64] floats
  static constexpr uint32_t kBars = kStat + 2 * 2 * 2 * 64 * 4;
  static constexpr uint32_t kSmem = kBars + 256 + 1024;
  static constexpr uint32_t kS = 0, kDp = 128, kDv = 256, kDk = 256 + DP;      // tensor memory columns
};
struct DkvBars {
  uint64_t kv, q_full[4], q_empty[4], do_full[4], do_empty[4], s, dp, p_ready, ds_ready, out, fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(DkvBars) <= 256, "the barriers' part of shared memory");

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                         const __grid_constant__ AttnArgs a) {
  using C = Dkv<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  DkvBars& b = *reinterpret_cast<DkvBars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  Span sp;
  int kv_head;
  if (a.cu_q != nullptr) {
    kv_head = (int)(blockIdx.x % (unsigned)a.Hk);
    sp = find_span(a, (int)(blockIdx.x / (unsigned)a.Hk), 128, true);
    if (sp.tile < 0) {
      if (a.zero_tail) {
        zero_rows(a.dk, kv_head, sp.first_k, 128, a.Sk, a.D, threadIdx.x, kThreads);
        zero_rows(a.dv, kv_head, sp.first_k, 128, a.Sk, a.D, threadIdx.x, kThreads);
      }
      return;
    }
  } else {
    // with a causal mask the first tiles are seen by the most queries: they come first
    const unsigned bh = blockIdx.x % (unsigned)(a.B * a.Hk);
    kv_head = (int)(bh % (unsigned)a.Hk);
    sp.batch = (int)(bh / (unsigned)a.Hk);
    sp.first_q = sp.first_k = 0;
    sp.len_q = a.Sq;
    sp.len_k = a.Sk;
    sp.tile = (int)(blockIdx.x / (unsigned)(a.B * a.Hk));
  }
  const int group = a.H / a.Hk, key0 = sp.tile * 128, offset = sp.len_k - sp.len_q;
  const int first = a.causal && key0 - offset > 0 ? (key0 - offset) / 128 : 0;      // first query tile that sees a key of this one
  const int tiles = (sp.len_q + 127) / 128;
  const int per_head = tiles > first ? tiles - first : 0;
  const int total = group * per_head;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(b.q_full + i, 1);
      mbar_init(b.q_empty + i, 1);
      mbar_init(b.do_full + i, 1);
      mbar_init(b.do_empty + i, 1);
    }
    mbar_init(&b.kv, 1);
    mbar_init(&b.s, 1);
    mbar_init(&b.dp, 1);
    mbar_init(&b.p_ready, 8);
    mbar_init(&b.ds_ready, 8);
    mbar_init(&b.out, 1);
    mbar_init(&b.fix, 1);
    mbar_init(&b.drain, 1);
    b.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(&b.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = b.tmem;

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    bool ok = true;
    if (lane == 0 && total > 0) {
      mbar_expect_tx(&b.kv, 2 * C::kTile);
      load_tile<DP>(smem, &map_k, kv_head, sp.first_k + key0, sp.batch, &b.kv);
      load_tile<DP>(smem + C::kTile, &map_v, kv_head, sp.first_k + key0, sp.batch, &b.kv);
    }
    int it = 0;
    uint32_t fixes = 0;
    for (; it < total && ok; ++it) {
      const uint32_t st = (uint32_t)it % C::kStages, ph = ((uint32_t)it / C::kStages) & 1u;
      const int head = kv_head * group + it / per_head, row = (first + it % per_head) * 128;
      // the rows behind a packed sequence are its neighbour's, and both tiles are contracted along their rows
      const bool ragged = a.cu_q != nullptr && row + 128 > sp.len_q;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint64_t* full = (w == 0 ? b.q_full : b.do_full) + st;
        uint64_t* empty = (w == 0 ? b.q_empty : b.do_empty) + st;
        if (!wait_warp(empty, ph ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        unsigned char* dst = smem + (w == 0 ? C::kQ : C::kDo) + st * C::kTile;
        uint64_t* bar = ragged ? &b.fix : full;
        if (lane == 0) {
          mbar_expect_tx(bar, C::kTile);
          load_tile<DP>(dst, w == 0 ? &map_q : &map_do, head, sp.first_q + row, sp.batch, bar);
        }
        if (ragged) {
          if (!wait_warp(&b.fix, fixes++ & 1u, abort_flag)) ok = false;
          clear_rows<DP>(dst, sp.len_q - row);
          if (lane == 0) mbar_arrive(full);
        }
      }
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.error, 0, kErrLoad);
        *abort_flag = 1;
      }
      // how far the two rings got is not known any more: give their copies the time that they can take
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else {
      for (int m = it > C::kStages ? it - C::kStages : 0; m < it; ++m) {
        mbar_wait(b.q_full + m % C::kStages, (m / C::kStages) & 1u, kWaitNs);
        mbar_wait(b.do_full + m % C::kStages, (m / C::kStages) & 1u, kWaitNs);
      }
    }
    if (total > 0) mbar_wait(&b.kv, 0, kWaitNs);
  } else if (warp == 9) {
    // ------------------------------------------------------------ products
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(BF16, 128, false), id_o = idesc(BF16, DP, true);
      const uint32_t k_addr = smem_u32(smem), v_addr = k_addr + C::kTile;
      const uint32_t q_ring = smem_u32(smem + C::kQ), do_ring = smem_u32(smem + C::kDo);
      bool ok = total == 0 || wait(&b.kv, 0, abort_flag);
      auto at = [&](uint32_t ring, int it) { return ring + ((uint32_t)it % C::kStages) * C::kTile; };
      auto scores = [&](int it) {
        if (!wait(b.q_full + it % C::kStages, ((uint32_t)it / C::kStages) & 1u, abort_flag)) return false;
        mma_columns<DP>(tmem + C::kS, k_addr, at(q_ring, it), id_s);
        commit(&b.s);
        return true;
      };
      auto dprobs = [&](int it) {
        if (!wait(b.do_full + it % C::kStages, ((uint32_t)it / C::kStages) & 1u, abort_flag)) return false;
        mma_columns<DP>(tmem + C::kDp, v_addr, at(do_ring, it), id_s);
        commit(&b.dp);
        return true;
      };
      if (ok && total > 0) ok = scores(0) && dprobs(0);
      for (int it = 0; it < total && ok; ++it) {
        if (!(ok = wait(&b.p_ready, it & 1u, abort_flag))) break;
        fence_after();
        mma_rows<0, 8>(tmem + C::kDv, tmem + C::kS, tmem + C::kS + 64, at(do_ring, it), id_o, it > 0);
        commit(b.do_empty + it % C::kStages);
        if (it + 1 < total && !(ok = scores(it + 1))) break;
        if (!(ok = wait(&b.ds_ready, it & 1u, abort_flag))) break;
        fence_after();
        mma_rows<0, 8>(tmem + C::kDk, tmem + C::kDp, tmem + C::kDp + 64, at(q_ring, it), id_o, it > 0);
        commit(b.q_empty + it % C::kStages);
        if (it + 1 < total) ok = dprobs(it + 1);
      }
      if (ok) commit(&b.out);
      else {
        atomicCAS(a.error, 0, kErrMma);
        *abort_flag = 1;
      }
      commit(&b.drain);
      mbar_wait(&b.drain, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ probabilities and score gradients: thread = key
    const int g = warp >> 2, t = threadIdx.x & 127;
    const int key = key0 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + C::kS + g * 64 + lanes, t_dp = tmem + C::kDp + g * 64 + lanes;
    const float sl2 = a.scale * kLog2e;
    float* stat = reinterpret_cast<float*>(smem + C::kStat) + g * 128;       // + (it & 1) * 256
    const F2 scale2 = f2(sl2);
    // one statistic per thread and step: lse (in powers of two) of this half's 64 queries, then their deltas.  Queries that
    // do not exist or see no key get probabilities of zero.
    auto fetch = [&](int it) {
      const int head = kv_head * group + it / per_head, q = (first + it % per_head) * 128 + g * 64 + (t & 63);
      if (q >= sp.len_q) return t < 64 ? INFINITY : 0.f;
      const float x = (t < 64 ? a.lse : a.delta)[stat_row(a, sp.batch, head) + sp.first_q + q];
      return t < 64 ? (x == -INFINITY ? INFINITY : x * kLog2e) : x;
    };
    float next = total > 0 ? fetch(0) : 0.f;
    bool ok = true;
    int it = 0;
    for (; it < total; ++it) {
      float* st = stat + (it & 1) * 256;
      st[t] = next;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
      if (it + 1 < total) next = fetch(it + 1);
      const int q0 = (first + it % per_head) * 128 + g * 64;
      const int hidden = a.causal ? key - offset - q0 : 0;                    // this key is not seen by the first so many queries
      const bool masked = a.causal && key0 + (warp & 3) * 32 + 31 - offset - q0 > 0;
      if (!(ok = wait_warp(&b.s, it & 1u, abort_flag))) break;
      fence_after();
      float p[64];
      uint32_t s[2][32];
      tmem_ld32(t_s, s[0]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_wait_ld(s[c]);
        if (c == 0) tmem_ld32(t_s + 32, s[1]);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 base = *reinterpret_cast<const float4*>(st + c * 32 + 2 * e);
          float x[4];
          split(fma2(f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, f2(-base.x, -base.y)), x[0], x[1]);
          split(fma2(f2(__uint_as_float(s[c][2 * e + 2]), __uint_as_float(s[c][2 * e + 3])), scale2, f2(-base.z, -base.w)), x[2], x[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = ex2_hw(x[i]);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = c * 32 + 2 * e + i < hidden ? 0.f : x[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) p[c * 32 + 2 * e + i] = x[i];
          w[e] = pack2<BF16>(x[0], x[1]);
          w[e + 1] = pack2<BF16>(x[2], x[3]);
        }
        tmem_st16(t_s + c * 16, w);
      }
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.p_ready);

      if (!(ok = wait_warp(&b.dp, it & 1u, abort_flag))) break;
      fence_after();
      tmem_ld32(t_dp, s[0]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_wait_ld(s[c]);
        if (c == 0) tmem_ld32(t_dp + 32, s[1]);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 d = *reinterpret_cast<const float4*>(st + 64 + c * 32 + 2 * e);
          const int i0 = c * 32 + 2 * e;
          float x[4];
          split(f2(p[i0], p[i0 + 1]) * (f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])) + f2(-d.x, -d.y)), x[0], x[1]);
          split(f2(p[i0 + 2], p[i0 + 3]) * (f2(__uint_as_float(s[c][2 * e + 2]), __uint_as_float(s[c][2 * e + 3])) + f2(-d.z, -d.w)), x[2],
                x[3]);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = i0 + i < hidden ? 0.f : x[i];
          }
          w[e] = pack2<BF16>(x[0], x[1]);
          w[e + 1] = pack2<BF16>(x[2], x[3]);
        }
        tmem_st16(t_dp + c * 16, w);
      }
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.ds_ready);
    }
    // a warp that gave up still meets the others of its warpgroup at the barriers that are left
    for (++it; it < total; ++it) asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
    if (ok && total > 0) {
      ok = wait_warp(&b.out, 0, abort_flag);
      fence_after();
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.error, 0, kErrCompute);
        *abort_flag = 1;
      }
    } else {
      // the first warpgroup writes dv, the second dk
      const bool exists = key < sp.len_k;
      uint16_t* out = row_ptr(g == 0 ? a.dv : a.dk, sp.batch, kv_head, sp.first_k + key);
      const uint32_t t_out = tmem + (g == 0 ? C::kDv : C::kDk) + lanes;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (total > 0) {
          tmem_ld32(t_out + c * 32, o);
          tmem_wait_ld(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (exists) store32<BF16>(out, c * 32, a.D, o, g == 0 ? 1.f : a.scale, rows_are_wide(g == 0 ? a.dv : a.dk));
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
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
  static constexpr uint32_t kSmem = kBars + 256 + 1024;
  static constexpr uint32_t kS = 0, kDp = 256, kDq = 384;
};
struct DqBars {
  uint64_t q, k_full[4], k_empty[4], v_full[3], v_empty[3], s[2], dp, dp_read, ds_ready[2], out, fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(DqBars) <= 256, "the barriers' part of shared memory");

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ AttnArgs a, int tiles) {
  using C = Dq<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  DqBars& b = *reinterpret_cast<DqBars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  Span sp;
  int head;
  if (a.cu_q != nullptr) {
    head = (int)(blockIdx.x % (unsigned)a.H);
    sp = find_span(a, (int)(blockIdx.x / (unsigned)a.H), 128, false);
    if (sp.tile < 0) {
      if (a.zero_tail) zero_rows(a.dq, head, sp.first_q, 128, a.Sq, a.D, threadIdx.x, kThreads);
      return;
    }
  } else {
    const unsigned bh = blockIdx.x % (unsigned)(a.B * a.H), t = blockIdx.x / (unsigned)(a.B * a.H);
    head = (int)(bh % (unsigned)a.H);
    sp.batch = (int)(bh / (unsigned)a.H);
    sp.first_q = sp.first_k = 0;
    sp.len_q = a.Sq;
    sp.len_k = a.Sk;
    sp.tile = a.causal ? tiles - 1 - (int)t : (int)t;                         // most keys first
  }
  const int kv_head = head / (a.H / a.Hk);
  const int row0 = sp.tile * 128, offset = sp.len_k - sp.len_q;
  const int last = row0 + 127 < sp.len_q - 1 ? row0 + 127 : sp.len_q - 1;
  const int keys_tile = !a.causal ? sp.len_k : (last + offset + 1 < sp.len_k ? last + offset + 1 : sp.len_k);
  const int n = keys_tile > 0 ? (keys_tile + 127) / 128 : 0;

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
      mbar_init(b.s + i, 1);
      mbar_init(b.ds_ready + i, 8);
    }
    mbar_init(&b.q, 1);
    mbar_init(&b.dp, 1);
    mbar_init(&b.dp_read, 8);
    mbar_init(&b.out, 1);
    mbar_init(&b.fix, 1);
    mbar_init(&b.drain, 1);
    b.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(&b.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = b.tmem;

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    bool ok = true;
    if (lane == 0 && n > 0) {
      mbar_expect_tx(&b.q, 2 * C::kTile);
      load_tile<DP>(smem, &map_q, head, sp.first_q + row0, sp.batch, &b.q);
      load_tile<DP>(smem + C::kTile, &map_do, head, sp.first_q + row0, sp.batch, &b.q);
    }
    int j = 0;
    for (; j < n && ok; ++j) {
      const uint32_t ks = (uint32_t)j % C::kK, kp = ((uint32_t)j / C::kK) & 1u;
      if (!(ok = wait_warp(b.k_empty + ks, kp ^ 1u, abort_flag))) break;
      unsigned char* dst = smem + C::kKRing + ks * C::kTile;
      const bool ragged = a.cu_q != nullptr && (j + 1) * 128 > sp.len_k;      // at most once: the last tile of the sequence
      uint64_t* bar = ragged ? &b.fix : b.k_full + ks;
      if (lane == 0) {
        mbar_expect_tx(bar, C::kTile);
        load_tile<DP>(dst, &map_k, kv_head, sp.first_k + j * 128, sp.batch, bar);
      }
      if (ragged) {
        if (!wait_warp(&b.fix, 0, abort_flag)) ok = false;
        clear_rows<DP>(dst, sp.len_k - j * 128);
        if (lane == 0) mbar_arrive(b.k_full + ks);
      }
      const uint32_t vs = (uint32_t)j % C::kV, vp = ((uint32_t)j / C::kV) & 1u;
      if (!(ok = wait_warp(b.v_empty + vs, vp ^ 1u, abort_flag))) break;
      if (lane == 0) {
        mbar_expect_tx(b.v_full + vs, C::kTile);
        load_tile<DP>(smem + C::kVRing + vs * C::kTile, &map_v, kv_head, sp.first_k + j * 128, sp.batch, b.v_full + vs);
      }
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.error, 0, kErrLoad);
        *abort_flag = 1;
      }
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else {
      for (int m = j > C::kK ? j - C::kK : 0; m < j; ++m) mbar_wait(b.k_full + m % C::kK, (m / C::kK) & 1u, kWaitNs);
      for (int m = j > C::kV ? j - C::kV : 0; m < j; ++m) mbar_wait(b.v_full + m % C::kV, (m / C::kV) & 1u, kWaitNs);
    }
    if (n > 0) mbar_wait(&b.q, 0, kWaitNs);
  } else if (warp == 9) {
    // ------------------------------------------------------------ products
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(BF16, 128, false), id_o = idesc(BF16, DP, true);
      const uint32_t q_addr = smem_u32(smem), do_addr = q_addr + C::kTile;
      const uint32_t k_ring = smem_u32(smem + C::kKRing), v_ring = smem_u32(smem + C::kVRing);
      bool ok = n == 0 || wait(&b.q, 0, abort_flag);
      auto scores = [&](int j) {
        if (!wait(b.k_full + j % C::kK, ((uint32_t)j / C::kK) & 1u, abort_flag)) return false;
        mma_columns<DP>(tmem + C::kS + (j & 1) * 128, q_addr, k_ring + ((uint32_t)j % C::kK) * C::kTile, id_s);
        commit(b.s + (j & 1));
        return true;
      };
      auto dprobs = [&](int j) {
        if (!wait(b.v_full + j % C::kV, ((uint32_t)j / C::kV) & 1u, abort_flag)) return false;
        mma_columns<DP>(tmem + C::kDp, do_addr, v_ring + ((uint32_t)j % C::kV) * C::kTile, id_s);
        commit(&b.dp);
        commit(b.v_empty + j % C::kV);
        return true;
      };
      if (ok && n > 0) ok = scores(0) && dprobs(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          if (!(ok = wait(&b.dp_read, j & 1u, abort_flag))) break;
          fence_after();
          if (!(ok = dprobs(j + 1))) break;
        }
        if (!(ok = wait(b.ds_ready + (j & 1), (j >> 1) & 1u, abort_flag))) break;
        fence_after();
        const uint32_t ds = tmem + C::kS + (j & 1) * 128;
        mma_rows<0, 8>(tmem + C::kDq, ds, ds + 64, k_ring + ((uint32_t)j % C::kK) * C::kTile, id_o, j > 0);
        commit(b.k_empty + j % C::kK);
        if (j + 2 < n) ok = scores(j + 2);
      }
      if (ok) commit(&b.out);
      else {
        atomicCAS(a.error, 0, kErrMma);
        *abort_flag = 1;
      }
      commit(&b.drain);
      mbar_wait(&b.drain, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ probabilities and score gradients: thread = query
    const int g = warp >> 2;
    const int row = row0 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_dp = tmem + C::kDp + g * 64 + lanes;
    const float sl2 = a.scale * kLog2e;
    const bool exists = row < sp.len_q;
    float lse2 = INFINITY, delta = 0.f;
    if (exists) {
      const int64_t at = stat_row(a, sp.batch, head) + sp.first_q + row;
      const float x = a.lse[at];
      lse2 = x == -INFINITY ? INFINITY : x * kLog2e;
      delta = a.delta[at];
    }
    const int keys = !a.causal ? sp.len_k : (row + offset + 1 < sp.len_k ? row + offset + 1 : sp.len_k);
    const int keys_all = __shfl_sync(0xffffffffu, keys, 0);
    const F2 scale2 = f2(sl2), base2 = f2(-lse2), delta2 = f2(-delta);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const bool masked = keys_all < j * 128 + g * 64 + 64;
      const int left = keys - j * 128 - g * 64;
      if (!(ok = wait_warp(b.s + (j & 1), (j >> 1) & 1u, abort_flag))) break;
      fence_after();
      const uint32_t t_s = tmem + C::kS + (j & 1) * 128 + g * 64 + lanes;
      F2 p[32];
      uint32_t s[2][32];
      tmem_ld32(t_s, s[0]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_wait_ld(s[c]);
        if (c == 0) tmem_ld32(t_s + 32, s[1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          split(fma2(f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, base2), x0, x1);
          p[c * 16 + e] = f2(ex2_hw(x0), ex2_hw(x1));
        }
      }
      if (!(ok = wait_warp(&b.dp, j & 1u, abort_flag))) break;
      fence_after();
      tmem_ld32(t_dp, s[0]);
      tmem_ld32(t_dp + 32, s[1]);
      tmem_wait_ld(s[0]);
      tmem_wait_ld(s[1]);
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.dp_read);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          split(p[c * 16 + e] * (f2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])) + delta2), x0, x1);
          if (masked) {
            x0 = c * 32 + 2 * e < left ? x0 : 0.f;
            x1 = c * 32 + 2 * e + 1 < left ? x1 : 0.f;
          }
          w[e] = pack2<BF16>(x0, x1);
        }
        tmem_st16(t_s + c * 16, w);
      }
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b.ds_ready + (j & 1));
    }
    if (ok && n > 0) {
      ok = wait_warp(&b.out, 0, abort_flag);
      fence_after();
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.error, 0, kErrCompute);
        *abort_flag = 1;
      }
    } else {
      // each warpgroup writes half of the columns
      uint16_t* out = row_ptr(a.dq, sp.batch, head, sp.first_q + row);
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const int col = g * (DP / 2) + c * 32;
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(tmem + C::kDq + lanes + col, o);
          tmem_wait_ld(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (exists) store32<BF16>(out, col, a.D, o, a.scale, rows_are_wide(a.dq));
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    tmem_free(tmem, 512);
  }
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

template <int DP, bool BF16>
cudaError_t launch(const AttnArgs& a, cudaStream_t stream) {
  const bool packed = a.cu_q != nullptr;
  CUtensorMap mq, mk, mv, mdo;
  if (a.Sq > 0 && (!make_map(&mq, a.q, BF16, a.D, a.H, a.Sq, a.B) || !make_map(&mdo, a.dout, BF16, a.D, a.H, a.Sq, a.B)))
    return cudaErrorInvalidValue;
  if (a.Sk > 0 && (!make_map(&mk, a.k, BF16, a.D, a.Hk, a.Sk, a.B) || !make_map(&mv, a.v, BF16, a.D, a.Hk, a.Sk, a.B)))
    return cudaErrorInvalidValue;
  if (a.Sq == 0) mq = mdo = mk;                              // nothing of what is missing is ever loaded
  if (a.Sk == 0) mk = mv = mq;
  if (a.Sq > 0) {
    const int64_t blocks = ((int64_t)a.B * a.Sq * a.H + 15) / 16;
    attention_delta_kernel<BF16><<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (a.Sk > 0) {
    cudaError_t e = allow_smem<attention_dkv_kernel<DP, BF16>>(Dkv<DP>::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t tiles = packed ? a.Sk / 128 + (int64_t)a.nseq + 1 : ((int64_t)a.Sk + 127) / 128;
    const int64_t ctas = tiles * a.Hk * a.B;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    attention_dkv_kernel<DP, BF16><<<(unsigned)ctas, kThreads, Dkv<DP>::kSmem, stream>>>(mq, mk, mv, mdo, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (a.Sq > 0) {
    cudaError_t e = allow_smem<attention_dq_kernel<DP, BF16>>(Dq<DP>::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t tiles = packed ? a.Sq / 128 + (int64_t)a.nseq + 1 : ((int64_t)a.Sq + 127) / 128;
    const int64_t ctas = tiles * a.H * a.B;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    attention_dq_kernel<DP, BF16><<<(unsigned)ctas, kThreads, Dq<DP>::kSmem, stream>>>(mq, mk, mv, mdo, a, (int)tiles);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream) {
  if (a.B <= 0 || a.H <= 0 || (a.Sq <= 0 && a.Sk <= 0)) return cudaSuccess;
  if (a.Hk <= 0 || a.H % a.Hk != 0 || a.D <= 0 || a.D % 8 != 0 || a.D > kAttnMaxDim || a.Sk < 0 || a.Sq < 0) return cudaErrorInvalidValue;
  if (a.D <= 64) return a.is_bf16 ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
  return a.is_bf16 ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
}

}  // namespace pccl
