// Attention, forward pass: one CTA per 256 queries of one head, a running maximum and sum per query, keys and values in one
// pass (attention.h has the formulas, attention.cuh the tiles).
//
//   warps 0-3   softmax of queries 0-127: one query per thread, its 128 scores of a key tile in registers
//   warps 4-7   the same for queries 128-255
//   warp 8      TMA: the query tiles once, then key and value tiles into a ring
//   warp 9      tensor memory; one thread issues the products
// The products of one half run while the other half is in its softmax:
//   S0(j)  S1(j) | P0(j) V -> O0, S0(j+1) | P1(j) V -> O1, S1(j+1) | ...
// Tensor memory: S0, S1 (128 columns each, P over the first 64 of them), O0, O1 (DP columns each).  Products of one CTA run in
// the order of issue, so S0(j+1) may be written over P0(j), and a finished S0(j+1) says that O0 holds the sum up to j.
//
// The running maximum only follows the true one when it has fallen behind by a factor of 2^8: sums and products are then at
// most 2^8 times larger than with the true maximum, far inside fp32 and inside the range of 16-bit probabilities, and O, which
// would have to be read and written to be rescaled, is left alone for all but the first few tiles.  Probabilities are rounded
// to 16 bits for the product (half a step of the inputs' own type); their sum is taken before that, in 32 bits.
#include "attention.cuh"

namespace pccl {

namespace {

using namespace attn;

constexpr int kThreads = 320;
constexpr float kBehind = 8.f;                  // binary orders of magnitude that the running maximum may fall behind

template <int DP>
struct Fwd {
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr uint32_t kTile = (DP / 64) * kBlockBytes;
  static constexpr uint32_t kRing = 2 * kTile;
  static constexpr uint32_t kBars = kRing + kStages * kTile;
  static constexpr uint32_t kSmem = kBars + 256 + 1024;     // barriers, slack for the alignment of the swizzled tiles
  static constexpr uint32_t kS = 0, kO = 256;               // tensor memory columns
  static constexpr uint32_t kCols = 512;
};

struct Bars {
  uint64_t full[8], empty[8], q[2], s[2], p[2], o[2], fix, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= 256, "the barriers' part of shared memory");

// Scores from place `left` on become -inf.
__device__ __forceinline__ void mask32(uint32_t* r, int left) {
#pragma unroll
  for (int e = 0; e < 32; ++e) r[e] = e < left ? r[e] : 0xff800000u;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a, int tiles) {
  using C = Fwd<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Bars& b = *reinterpret_cast<Bars*>(smem + C::kBars);
  volatile int* abort_flag = &b.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- this CTA's queries.  With a causal mask the last tiles have the most keys: they come first.
  Span sp;
  int head;
  if (a.cu_q != nullptr) {
    head = (int)(blockIdx.x % (unsigned)a.H);
    sp = find_span(a, (int)(blockIdx.x / (unsigned)a.H), 256, false);
    if (sp.tile < 0) {                                       // behind the last sequence
      if (a.zero_tail) {
        zero_rows(a.o, head, sp.first_q, 256, a.Sq, a.D);
        const int r = sp.first_q + (int)threadIdx.x;
        if (threadIdx.x < 256 && r < a.Sq) a.lse[stat_row(a, 0, head) + r] = -INFINITY;
      }
      return;
    }
  } else {
    const unsigned bh = blockIdx.x % (unsigned)(a.B * a.H), t = blockIdx.x / (unsigned)(a.B * a.H);
    head = (int)(bh % (unsigned)a.H);
    sp.batch = (int)(bh / (unsigned)a.H);
    sp.first_q = sp.first_k = 0;
    sp.len_q = a.Sq;
    sp.len_k = a.Sk;
    sp.tile = a.causal ? tiles - 1 - (int)t : (int)t;
  }
  const int kv_head = head / (a.H / a.Hk);
  const int row0 = sp.tile * 256, offset = sp.len_k - sp.len_q;
  int n[2];                                                  // key tiles that each half sees
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int first = row0 + h * 128;
    const int last = first + 127 < sp.len_q - 1 ? first + 127 : sp.len_q - 1;
    const int keys = !a.causal ? sp.len_k : (last + offset + 1 < sp.len_k ? last + offset + 1 : sp.len_k);
    n[h] = first < sp.len_q && keys > 0 ? (keys + 127) / 128 : 0;
  }
  const int nmax = n[0] > n[1] ? n[0] : n[1];

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(b.full + i, 1);
      mbar_init(b.empty + i, 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(b.q + h, 1);
      mbar_init(b.s + h, 1);
      mbar_init(b.p + h, 4);
      mbar_init(b.o + h, 1);
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

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    bool ok = true;
    if (lane == 0) {
      for (int h = 0; h < 2; ++h)
        if (n[h] > 0) {
          mbar_expect_tx(b.q + h, C::kTile);
          load_tile<DP>(smem + h * C::kTile, &map_q, head, sp.first_q + row0 + h * 128, sp.batch, b.q + h);
        }
    }
    uint32_t it = 0;
    for (; (int)it < 2 * nmax; ++it) {                       // K0, V0, K1, V1, ...
      const uint32_t st = it % C::kStages, ph = (it / C::kStages) & 1u;
      if (!wait_warp(b.empty + st, ph ^ 1u, abort_flag)) {
        ok = false;
        break;
      }
      const int j = (int)(it >> 1), row = j * 128;
      const bool value = (it & 1u) != 0;
      unsigned char* dst = smem + C::kRing + st * C::kTile;
      // the rows behind a packed sequence are its neighbour's
      const bool ragged = value && a.cu_q != nullptr && row + 128 > sp.len_k;
      uint64_t* bar = ragged ? &b.fix : b.full + st;
      if (lane == 0) {
        mbar_expect_tx(bar, C::kTile);
        load_tile<DP>(dst, value ? &map_v : &map_k, kv_head, sp.first_k + row, sp.batch, bar);
      }
      if (ragged) {                                          // at most once: the last tile of the sequence
        if (!wait_warp(&b.fix, 0, abort_flag)) ok = false;
        clear_rows<DP>(dst, sp.len_k - row);
        if (lane == 0) mbar_arrive(b.full + st);
      }
    }
    if (!ok && lane == 0) {
      atomicCAS(a.error, 0, kErrLoad);
      *abort_flag = 1;
    }
    // what was asked for has to land before the CTA leaves its shared memory
    for (uint32_t m = it > (uint32_t)C::kStages ? it - C::kStages : 0; m < it; ++m)
      mbar_wait(b.full + m % C::kStages, (m / C::kStages) & 1u, kWaitNs / C::kStages);
    for (int h = 0; h < 2; ++h)
      if (n[h] > 0) mbar_wait(b.q + h, 0, kWaitNs);
  } else if (warp == 9) {
    // ------------------------------------------------------------ products
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(BF16, 128, false), id_o = idesc(BF16, DP, true);
      const uint32_t q_addr = smem_u32(smem), ring = smem_u32(smem + C::kRing);
      bool ok = true;
      auto tile_at = [&](uint32_t it) { return ring + (it % C::kStages) * C::kTile; };
      auto loaded = [&](uint32_t it) { return wait(b.full + it % C::kStages, (it / C::kStages) & 1u, abort_flag); };
      auto scores = [&](int h, int j) {
        mma_columns<DP>(tmem + C::kS + h * 128, q_addr + h * C::kTile, tile_at(2 * j), id_s);
        commit(b.s + h);
      };
      if (nmax > 0) {
        ok = loaded(0);
        for (int h = 0; h < 2 && ok; ++h)
          if (n[h] > 0) {
            ok = wait(b.q + h, 0, abort_flag);
            if (ok) scores(h, 0);
          }
        if (ok) commit(b.empty + 0);
      }
      for (int j = 0; j < nmax && ok; ++j) {
        ok = loaded(2 * j + 1);
        for (int h = 0; h < 2 && ok; ++h) {
          if (j < n[h]) {
            if (!(ok = wait(b.p + h, j & 1u, abort_flag))) break;
            fence_after();
            const uint32_t p = tmem + C::kS + h * 128;
            mma_rows(tmem + C::kO + h * 128, p, p + 32, tile_at(2 * j + 1), id_o, j > 0);
            if (j + 1 == n[h]) commit(b.o + h);
          }
          if (h == 0 && j + 1 < nmax) ok = loaded(2 * j + 2);
          if (ok && j + 1 < n[h]) scores(h, j + 1);
        }
        if (!ok) break;
        commit(b.empty + (2 * j + 1) % C::kStages);
        if (j + 1 < nmax) commit(b.empty + (2 * j + 2) % C::kStages);
      }
      if (!ok) {
        atomicCAS(a.error, 0, kErrMma);
        *abort_flag = 1;
      }
      commit(&b.drain);
      mbar_wait(&b.drain, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax: thread = query
    const int h = warp >> 2;
    const int row = row0 + h * 128 + (warp & 3) * 32 + lane;          // within the sequence
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + C::kS + h * 128 + lanes, t_o = tmem + C::kO + h * 128 + lanes;
    const float sl2 = a.scale * kLog2e;
    const float behind = kBehind / sl2;
    const int keys = !a.causal ? sp.len_k : (row + offset + 1 < sp.len_k ? row + offset + 1 : sp.len_k);   // that this query sees
    const int keys_all = __shfl_sync(0xffffffffu, keys, 0);           // that every query of the warp sees
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n[h]; ++j) {
      if (!(ok = wait_warp(b.s + h, j & 1u, abort_flag))) break;
      fence_after();
      const bool masked = keys_all < (j + 1) * 128;
      const int left = keys - j * 128;                                // keys of this tile that this query sees
      uint32_t s[2][32];                                              // two quarters of the row, the next one on its way
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      tmem_ld32(t_s, s[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_wait_ld(s[c & 1]);
        tmem_ld32(t_s + ((c + 1) & 3) * 32, s[(c + 1) & 1]);          // behind the last quarter the first one again
        uint32_t* r = s[c & 1];
        if (masked) mask32(r, left - c * 32);
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = fmaxf(fmaxf(top[i], __uint_as_float(r[e + i])), __uint_as_float(r[e + 4 + i]));
      }
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
        tmem_wait_ld(s[c & 1]);
        if (c < 3) tmem_ld32(t_s + (c + 1) * 32, s[(c + 1) & 1]);
        uint32_t* r = s[c & 1];
        if (masked) mask32(r, left - c * 32);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const F2 x = fma2(f2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), scale2, base2);
          float x0, x1;
          split(x, x0, x1);
          x0 = ex2_hw(x0);
          x1 = ex2_hw(x1);
          sum2[e & 1] = sum2[e & 1] + f2(x0, x1);
          w[e] = pack2<BF16>(x0, x1);
        }
        tmem_st16(t_s + c * 16, w);
      }
      float a0, a1;
      split(sum2[0] + sum2[1], a0, a1);
      l += a0 + a1;
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b.p + h);
    }
    if (ok && n[h] > 0) {
      ok = wait_warp(b.o + h, 0, abort_flag);
      fence_after();
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.error, 0, kErrCompute);
        *abort_flag = 1;
      }
    } else {
      const bool exists = row < sp.len_q;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* out = row_ptr(a.o, sp.batch, head, sp.first_q + row);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (n[h] > 0) {
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (l == 0.f) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (exists) store32<BF16>(out, c * 32, a.D, o, inv);
      }
      if (exists) a.lse[stat_row(a, sp.batch, head) + sp.first_q + row] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    tmem_free(tmem, C::kCols);
  }
}

template <int DP, bool BF16>
cudaError_t launch(const AttnArgs& a, cudaStream_t stream) {
  using C = Fwd<DP>;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, a.q, BF16, a.D, a.H, a.Sq, a.B)) return cudaErrorInvalidValue;
  if (a.Sk == 0) mk = mv = mq;                               // no key is ever loaded
  else if (!make_map(&mk, a.k, BF16, a.D, a.Hk, a.Sk, a.B) || !make_map(&mv, a.v, BF16, a.D, a.Hk, a.Sk, a.B)) return cudaErrorInvalidValue;
  auto kernel = attention_fwd_kernel<DP, BF16>;
  static thread_local bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t tiles = a.cu_q != nullptr ? a.Sq / 256 + (int64_t)a.nseq + 1 : ((int64_t)a.Sq + 255) / 256;
  const int64_t ctas = tiles * a.H * (a.cu_q != nullptr ? 1 : a.B);
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  kernel<<<(unsigned)ctas, kThreads, C::kSmem, stream>>>(mq, mk, mv, a, (int)tiles);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_forward(const AttnArgs& a, cudaStream_t stream) {
  if (a.B <= 0 || a.H <= 0 || a.Sq <= 0) return cudaSuccess;
  if (a.Hk <= 0 || a.H % a.Hk != 0 || a.D <= 0 || a.D % 8 != 0 || a.D > kAttnMaxDim || a.Sk < 0) return cudaErrorInvalidValue;
  if (a.D <= 64) return a.is_bf16 ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
  return a.is_bf16 ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
}

}  // namespace pccl
