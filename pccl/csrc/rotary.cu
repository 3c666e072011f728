// Norms of queries and keys for each head with the rotation of positions, forward and backward (rotary.h has the formulas).
//
// A row of one head is held by a group of 8, 16 or 32 lanes.  A lane holds four pairs: columns 4l and half + 4l on (two loads
// of 8 bytes), or 8l on where the pairs are neighbours; lanes behind the rotated columns hold eight of the others.  So the
// rotation stays within a lane, and the sum over the row takes the only exchanges.  A group takes several heads of the same row
// one after the other, because they share the angles, with the loads of a few heads in flight.  One read and one write of the data.
//
// What bounds it.  8192 rows of 16 + 16 heads of 128, bf16: forward 26.9 us (5.0 TB/s: 0.76 of the measured copy rate), backward
// 48.1 (4.2 TB/s); 32 + 32 heads 48.3 (5.6 TB/s) and 85.2 (4.7 TB/s).  A call of this length is never far from its start and its end;
// behind that are, in the forward pass, the instructions: its issue slots are two thirds full, which is why the arithmetic is on
// pairs of 32-bit numbers.  In the backward pass neither they (52 %) nor DRAM (54 % of its nominal rate) are: four warps on a scheduler
// load four heads and then compute on them, and the largest share of their waiting, a third, is for those loads.
//
// The backward pass computes the norms again (its x is read for the gradient anyway).  A group sums its share of a weight's
// gradient in registers over all its rows, a block (of queries, or of keys) adds up its groups in order, and a second small
// kernel the blocks: no atomic addition, so the bits are the same from call to call.
//
// A position outside of the table makes its rows NaN; nothing is read there.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "act.cuh"
#include "pdl.cuh"
#include "rotary.h"

namespace pccl {

namespace {

constexpr int kForward = 128, kBackward = 256;               // threads of a block

// A lane's eight elements: the first and the second members of its four pairs, two and two for the packed arithmetic.
struct Pairs {
  F2 a[2], b[2];
};
template <bool BF16>
__device__ __forceinline__ void widen(uint32_t w, float& lo, float& hi) {
  if constexpr (BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = x.x;
    hi = x.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// From the elements in the order of the columns (c0 on, c1 on) and back.
template <bool NEIGHBOURS>
__device__ __forceinline__ void pair_up(const float* e, Pairs& p) {
  if constexpr (NEIGHBOURS) {
    p.a[0] = f2(e[0], e[2]), p.a[1] = f2(e[4], e[6]);
    p.b[0] = f2(e[1], e[3]), p.b[1] = f2(e[5], e[7]);
  } else {
    p.a[0] = f2(e[0], e[1]), p.a[1] = f2(e[2], e[3]);
    p.b[0] = f2(e[4], e[5]), p.b[1] = f2(e[6], e[7]);
  }
}
template <bool NEIGHBOURS>
__device__ __forceinline__ void take_apart(const Pairs& p, float* e) {
  if constexpr (NEIGHBOURS) {
    split(p.a[0], e[0], e[2]), split(p.a[1], e[4], e[6]);
    split(p.b[0], e[1], e[3]), split(p.b[1], e[5], e[7]);
  } else {
    split(p.a[0], e[0], e[1]), split(p.a[1], e[2], e[3]);
    split(p.b[0], e[4], e[5]), split(p.b[1], e[6], e[7]);
  }
}
template <bool BF16, bool NEIGHBOURS>
__device__ __forceinline__ void unpack(const uint2& x, const uint2& y, Pairs& p) {
  float e[8];
  widen<BF16>(x.x, e[0], e[1]);
  widen<BF16>(x.y, e[2], e[3]);
  widen<BF16>(y.x, e[4], e[5]);
  widen<BF16>(y.y, e[6], e[7]);
  pair_up<NEIGHBOURS>(e, p);
}
template <bool BF16, bool NEIGHBOURS>
__device__ __forceinline__ void store(uint16_t* x, uint16_t* y, const Pairs& p) {
  float e[8];
  take_apart<NEIGHBOURS>(p, e);
  *reinterpret_cast<uint2*>(x) = make_uint2(narrow<BF16>(e[0], e[1]), narrow<BF16>(e[2], e[3]));
  *reinterpret_cast<uint2*>(y) = make_uint2(narrow<BF16>(e[4], e[5]), narrow<BF16>(e[6], e[7]));
}
__device__ __forceinline__ float dot(const Pairs& x, const Pairs& y) {
  float lo, hi;
  split(fma2(x.a[0], y.a[0], fma2(x.a[1], y.a[1], fma2(x.b[0], y.b[0], x.b[1] * y.b[1]))), lo, hi);
  return lo + hi;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint16_t* row_at(const RotaryTensor& t, int b, int s, int h) {
  return static_cast<uint16_t*>(t.p) + (int64_t)b * t.sb + (int64_t)s * t.ss + (int64_t)h * t.sh;
}
// Four weights.
__device__ __forceinline__ void load_w4(const void* w, int type, int col, float* f) {
  if (type == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<const float*>(w)[col + i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t x = static_cast<const uint16_t*>(w)[col + i];
      f[i] = type == 0 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
    }
  }
}

// A lane's eight columns: four from c0 and four from c1.
struct Columns {
  int c0, c1, angle;               // angle: first of its four pairs
  bool on, turned;
};
template <bool NEIGHBOURS>
__device__ __forceinline__ Columns columns(int l, int half, int D) {
  Columns c;
  c.on = l * 8 < D;
  c.turned = l * 8 < 2 * half;
  c.angle = l * 4;
  const bool apart = !NEIGHBOURS && c.turned;
  c.c0 = apart ? l * 4 : l * 8;
  c.c1 = apart ? half + l * 4 : l * 8 + 4;
  return c;
}
template <bool NEIGHBOURS>
__device__ __forceinline__ void load_weights(const RotaryArgs& a, int which, const Columns& col, Pairs& w) {
  float e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col.on) {
    load_w4(a.w[which], a.w_type, col.c0, e);
    load_w4(a.w[which], a.w_type, col.c1, e + 4);
  }
  pair_up<NEIGHBOURS>(e, w);
}
struct Angles {
  F2 c[2], s[2];
};
__device__ __forceinline__ void load_angles(Angles& t, const RotaryArgs& a, int64_t pos, const Columns& col) {
  const bool known = pos >= 0 && pos < a.table;
  const float nan = __int_as_float(0x7fffffff);
  float4 c = make_float4(nan, nan, nan, nan), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (known) {
    c = make_float4(1.f, 1.f, 1.f, 1.f);
    if (col.turned) {
      c = *reinterpret_cast<const float4*>(a.cos + pos * a.half + col.angle);
      s = *reinterpret_cast<const float4*>(a.sin + pos * a.half + col.angle);
    }
  }
  t.c[0] = f2(c.x, c.y), t.c[1] = f2(c.z, c.w);
  t.s[0] = f2(s.x, s.y), t.s[1] = f2(s.z, s.w);
}
// A lane's pairs turned by its angles (forward), or back.  Where not all columns are turned, those that are not (cos 1, or NaN for
// an unknown position) keep clear of what their neighbours hold.
template <bool BACK>
__device__ __forceinline__ void rotate(Pairs& p, const Angles& t, bool all, bool turned) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 s = BACK ? t.s[i] : t.s[i] * f2(-1.f), n = BACK ? t.s[i] * f2(-1.f) : t.s[i];
    F2 x = p.b[i] * s, y = p.a[i] * n;
    if (!all && !turned) x = y = f2(0.f);
    p.a[i] = fma2(p.a[i], t.c[i], x);
    p.b[i] = fma2(p.b[i], t.c[i], y);
  }
}

struct Item {
  int b, s, h0, h1;                // heads [h0, h1) of one row
};
__device__ __forceinline__ Item item_at(const RotaryArgs& a, int which, uint32_t row, uint32_t chunk) {
  Item it;
  it.b = (int)(row / (uint32_t)a.S);
  it.s = (int)(row - (uint32_t)it.b * (uint32_t)a.S);
  it.h0 = (int)chunk * a.heads_per_item;
  it.h1 = it.h0 + a.heads_per_item < a.H[which] ? it.h0 + a.heads_per_item : a.H[which];
  return it;
}
__device__ __forceinline__ int64_t position(const RotaryArgs& a, const Item& it) {
  if (a.positions == nullptr) return it.s;
  const int64_t i = (int64_t)it.b * a.S + it.s;
  return a.positions64 ? static_cast<const int64_t*>(a.positions)[i] : (int64_t) static_cast<const int*>(a.positions)[i];
}
// Block b works on queries or on keys: its number among theirs, and how many they are.
__device__ __forceinline__ int share_of(const RotaryArgs& a, uint32_t& block, uint32_t& blocks) {
  const bool keys = (int)blockIdx.x >= a.q_blocks;
  block = keys ? blockIdx.x - (uint32_t)a.q_blocks : blockIdx.x;
  blocks = keys ? gridDim.x - (uint32_t)a.q_blocks : (uint32_t)a.q_blocks;
  return keys ? 1 : 0;
}

// ---------------------------------------------------------------- forward
template <bool BF16, bool NEIGHBOURS, int L>
__global__ void __launch_bounds__(kForward) rotary_forward_kernel(const __grid_constant__ RotaryArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = 4;
  constexpr uint32_t groups = kForward / L;
  const Columns col = columns<NEIGHBOURS>(threadIdx.x & (L - 1), a.half, a.D);
  const float inv_d = 1.f / (float)a.D;
  const bool all = 2 * a.half == a.D;
  uint32_t block, blocks;
  const int which = share_of(a, block, blocks);
  const RotaryTensor &tx = a.x[which], &ty = a.y[which];
  const uint32_t rows = (uint32_t)a.B * (uint32_t)a.S, chunks = (uint32_t)a.chunks[which];
  Pairs w;
  load_weights<NEIGHBOURS>(a, which, col, w);
  // a group: one chunk of heads in one row; groups without one go through the exchanges with the others
  const uint64_t items = (uint64_t)rows * chunks, i = (uint64_t)block * groups + threadIdx.x / L;
  const bool exists = i < items;
  const uint32_t row = exists ? (uint32_t)(chunks == 1 ? i : i / chunks) : 0, chunk = exists ? (uint32_t)(i - (uint64_t)row * chunks) : 0;
  const Item it = item_at(a, which, row, chunk);
  const int h1 = exists && col.on ? it.h1 : it.h0;
  Angles t;
  load_angles(t, a, position(a, it), col);
  for (int r = 0; r < a.heads_per_item; r += U) {
    uint2 q[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = it.h0 + r + u;
      const uint16_t* p = row_at(tx, it.b, it.s, h);
      q[u][0] = h < h1 ? *reinterpret_cast<const uint2*>(p + col.c0) : make_uint2(0, 0);
      q[u][1] = h < h1 ? *reinterpret_cast<const uint2*>(p + col.c1) : make_uint2(0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u >= a.heads_per_item) break;
      const int h = it.h0 + r + u;
      Pairs x;
      unpack<BF16, NEIGHBOURS>(q[u][0], q[u][1], x);
      const F2 rs = f2(rsqrtf(fmaf(group_sum<L>(dot(x, x)), inv_d, a.eps)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x.a[i] = x.a[i] * (rs * w.a[i]);
        x.b[i] = x.b[i] * (rs * w.b[i]);
      }
      rotate<false>(x, t, all, col.turned);
      if (h < h1) {
        uint16_t* p = row_at(ty, it.b, it.s, h);
        store<BF16, NEIGHBOURS>(p + col.c0, p + col.c1, x);
      }
    }
  }
}

// ---------------------------------------------------------------- backward
template <bool BF16, bool NEIGHBOURS, int L>
__global__ void __launch_bounds__(kBackward, 2) rotary_backward_kernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float sums[kBackward * 8];
  pdl_wait();
  pdl_trigger();
  constexpr int U = 4;
  constexpr uint32_t groups = kBackward / L;
  const Columns col = columns<NEIGHBOURS>(threadIdx.x & (L - 1), a.half, a.D);
  const float inv_d = 1.f / (float)a.D;
  const bool all = 2 * a.half == a.D;
  uint32_t block, blocks;
  const int which = share_of(a, block, blocks);
  const RotaryTensor &tx = a.x[which], &td = a.dy[which], &ty = a.y[which];
  const uint32_t rows = (uint32_t)a.B * (uint32_t)a.S, chunks = (uint32_t)a.chunks[which];
  Pairs w, dw;
  load_weights<NEIGHBOURS>(a, which, col, w);
#pragma unroll
  for (int i = 0; i < 2; ++i) dw.a[i] = dw.b[i] = f2(0.f);
  const uint64_t items = (uint64_t)rows * chunks;
  for (uint64_t i0 = (uint64_t)block * groups; i0 < items; i0 += (uint64_t)blocks * groups) {
    const uint64_t i = i0 + threadIdx.x / L;
    const bool exists = i < items;
    const uint32_t row = exists ? (uint32_t)(chunks == 1 ? i : i / chunks) : 0, chunk = exists ? (uint32_t)(i - (uint64_t)row * chunks) : 0;
    const Item it = item_at(a, which, row, chunk);
    const int h1 = exists && col.on ? it.h1 : it.h0;
    Angles t;
    load_angles(t, a, position(a, it), col);
    for (int r = 0; r < a.heads_per_item; r += U) {
      uint2 qx[U][2], qd[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = it.h0 + r + u;
        const uint16_t *px = row_at(tx, it.b, it.s, h), *pd = row_at(td, it.b, it.s, h);
        qx[u][0] = h < h1 ? *reinterpret_cast<const uint2*>(px + col.c0) : make_uint2(0, 0);
        qx[u][1] = h < h1 ? *reinterpret_cast<const uint2*>(px + col.c1) : make_uint2(0, 0);
        qd[u][0] = h < h1 ? *reinterpret_cast<const uint2*>(pd + col.c0) : make_uint2(0, 0);
        qd[u][1] = h < h1 ? *reinterpret_cast<const uint2*>(pd + col.c1) : make_uint2(0, 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u >= a.heads_per_item) break;
        const int h = it.h0 + r + u;
        Pairs x, g;
        unpack<BF16, NEIGHBOURS>(qx[u][0], qx[u][1], x);
        unpack<BF16, NEIGHBOURS>(qd[u][0], qd[u][1], g);
        rotate<true>(g, t, all, col.turned);                 // the gradient behind the weights
        const F2 rs = f2(rsqrtf(fmaf(group_sum<L>(dot(x, x)), inv_d, a.eps)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x.a[i] = x.a[i] * rs;
          x.b[i] = x.b[i] * rs;
          if (h < h1) {                                      // behind the last head an unknown position's NaN stands in g
            dw.a[i] = fma2(g.a[i], x.a[i], dw.a[i]);
            dw.b[i] = fma2(g.b[i], x.b[i], dw.b[i]);
          }
          g.a[i] = g.a[i] * w.a[i];
          g.b[i] = g.b[i] * w.b[i];
        }
        const F2 mean = f2(group_sum<L>(dot(g, x)) * -inv_d);
        if (h < h1) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            g.a[i] = rs * fma2(x.a[i], mean, g.a[i]);
            g.b[i] = rs * fma2(x.b[i], mean, g.b[i]);
          }
          uint16_t* p = row_at(ty, it.b, it.s, h);
          store<BF16, NEIGHBOURS>(p + col.c0, p + col.c1, g);
        }
      }
    }
  }
  // the block's groups in order
  const int at = (threadIdx.x / L) * (L * 8);
  if (col.on) {
    float e[8];
    take_apart<NEIGHBOURS>(dw, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[at + col.c0 + i] = e[i];
      sums[at + col.c1 + i] = e[4 + i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.D; c += kBackward) {
    float s = 0.f;
    for (int g = 0; g < (int)groups; ++g) s += sums[g * L * 8 + c];
    a.partial[(int64_t)blockIdx.x * a.D + c] = s;
  }
}

// dw[c] = sum of the blocks' shares: 32 columns per block, eight warps that each add up every eighth share.
__global__ void __launch_bounds__(kBackward) rotary_weights_kernel(const __grid_constant__ RotaryArgs a, int blocks) {
  __shared__ float sums[8][32];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  const int first = which ? a.q_blocks : 0, last = which ? blocks : a.q_blocks;
  float s = 0.f;
  if (c < a.D) {
    for (int b = first + warp; b < last; b += 64) {          // eight loads on their way at once
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = b + i * 8 < last ? a.partial[(int64_t)(b + i * 8) * a.D + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[i];
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < a.D) {
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
    if (a.w_type == 2) static_cast<float*>(a.dw[which])[c] = s;
    else if (a.w_type == 0) static_cast<__nv_bfloat16*>(a.dw[which])[c] = __float2bfloat16_rn(s);
    else static_cast<__half*>(a.dw[which])[c] = __float2half_rn(s);
  }
}

int lanes_of(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

template <bool BF16, bool NEIGHBOURS, int L>
cudaError_t launch(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  if (!backward) return launch_pdl(rotary_forward_kernel<BF16, NEIGHBOURS, L>, dim3(blocks), dim3(kForward), 0, s, a);
  const cudaError_t e = launch_pdl(rotary_backward_kernel<BF16, NEIGHBOURS, L>, dim3(blocks), dim3(kBackward), 0, s, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(rotary_weights_kernel, dim3((a.D + 31) / 32, 2), dim3(kBackward), 0, s, a, blocks);
}
template <bool BF16, bool NEIGHBOURS>
cudaError_t launch_lanes(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  switch (lanes_of(a.D)) {
    case 8: return launch<BF16, NEIGHBOURS, 8>(a, backward, blocks, s);
    case 16: return launch<BF16, NEIGHBOURS, 16>(a, backward, blocks, s);
    default: return launch<BF16, NEIGHBOURS, 32>(a, backward, blocks, s);
  }
}
cudaError_t launch_any(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  if (a.D <= 0 || a.D % 8 != 0 || a.D > kRotaryMaxDim || a.half % 4 != 0 || a.half <= 0 || 2 * a.half > a.D || blocks <= 0)
    return cudaErrorInvalidValue;
  if (a.is_bf16) return a.interleaved ? launch_lanes<true, true>(a, backward, blocks, s) : launch_lanes<true, false>(a, backward, blocks, s);
  return a.interleaved ? launch_lanes<false, true>(a, backward, blocks, s) : launch_lanes<false, false>(a, backward, blocks, s);
}

}  // namespace

int rotary_blocks(RotaryArgs& a, bool backward, int sm_count) {
  const int lanes = lanes_of(a.D), groups = (backward ? kBackward : kForward) / lanes;
  const int64_t rows = (int64_t)a.B * a.S;
  // Heads per item: as many of a row as possible share its angles, but every SM wants eight blocks (forward: one item per group), or
  // two blocks that walk over six items or more (backward).  8192 rows of 16 + 16 heads of 128, 16 / 8 / 4 heads per item: backward
  // 51.1 / 48.0 / 51.6 us, forward 26.9 / 27.7 / 29.8; of 32 + 32 heads 85.2 / 88.4 / 95.2 and 48.3 / 49.6 / 54.6.
  const int64_t most = backward ? (int64_t)sm_count * 2 : INT32_MAX, want = (int64_t)sm_count * groups * (backward ? 12 : 8);
  int hpi = 16;
  for (;; hpi /= 2) {
    a.heads_per_item = hpi;
    for (int i = 0; i < 2; ++i) a.chunks[i] = (a.H[i] + hpi - 1) / hpi;
    if (hpi == 1 || rows * (a.chunks[0] + a.chunks[1]) >= want) break;
  }
  int64_t need[2];
  for (int i = 0; i < 2; ++i) need[i] = (rows * a.chunks[i] + groups - 1) / groups;
  if (need[0] + need[1] > most) {                            // in proportion, one block at least for what is there
    const int64_t q = most * need[0] / (need[0] + need[1]);
    need[0] = need[0] > 0 && q == 0 ? 1 : q;
    need[1] = need[1] > 0 && most - need[0] == 0 ? 1 : most - need[0];
  }
  a.q_blocks = (int)need[0];
  return (int)(need[0] + need[1]);
}
cudaError_t launch_rotary_forward(const RotaryArgs& a, int blocks, cudaStream_t s) { return launch_any(a, false, blocks, s); }
cudaError_t launch_rotary_backward(const RotaryArgs& a, int blocks, cudaStream_t s) { return launch_any(a, true, blocks, s); }

}  // namespace pccl
