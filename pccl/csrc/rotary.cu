// Norms of queries and keys for each head with the rotation of positions, forward and backward (rotary.h has the formulas).
//
// A row of one head is held by a group of 8, 16 or 32 lanes, eight neighbouring columns (16 bytes) per lane: the sums over
// the row are a few exchanges within the group, and so is the partner of a column that lies half a head away.  A group takes
// several heads of the same row one after the other, because they share the angles (of two 32-bit numbers per pair, as many
// bytes as the row itself), with the loads of four heads in flight.  One read and one write of the data; bound by HBM.
//
// The backward pass computes the norms again (its x is read for the gradient anyway).  A group sums its share of the weights'
// gradients in registers over all its rows, a block adds up its groups in order, and a second small kernel the blocks:
// no atomic addition, so the bits are the same from call to call.
//
// A position outside of the table makes its rows NaN; nothing is read there.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "rotary.h"

namespace pccl {

namespace {

constexpr int kThreads = 256;
enum Pairing : int { kHalves = 0, kHalvesOdd = 1, kNeighbours = 2 };      // halves of a multiple of eight columns, of four more; (2i, 2i + 1)

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float load_w(const void* w, int type, int i) {
  if (type == 2) return static_cast<const float*>(w)[i];
  return type == 0 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : __half2float(static_cast<const __half*>(w)[i]);
}
__device__ __forceinline__ uint4* at(const RotaryTensor& t, int b, int s, int h, int col) {
  return reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.p) + (int64_t)b * t.sb + (int64_t)s * t.ss + (int64_t)h * t.sh + col);
}

// The angles of a lane's eight columns.  Columns that are not rotated: cos 1, sin 0.
struct Angles {
  float c[8], s[8];                // s: with the sign of the column's place in its pair
};
template <int PAIR>
__device__ __forceinline__ void load_angles(Angles& t, const RotaryArgs& a, int64_t pos, int col) {
  const int half = a.half;
  const bool known = pos >= 0 && pos < a.table;
  const float* cs = a.cos + (known ? pos : 0) * half;
  const float* sn = a.sin + (known ? pos : 0) * half;
#pragma unroll
  for (int v = 0; v < 2; ++v) {                              // four columns at a time
    const int e = col + v * 4;
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (e < 2 * half) {
      if constexpr (PAIR == kNeighbours) {
        const float2 x = *reinterpret_cast<const float2*>(cs + (e >> 1)), y = *reinterpret_cast<const float2*>(sn + (e >> 1));
        c[0] = c[1] = x.x;
        c[2] = c[3] = x.y;
        s[0] = -y.x;
        s[1] = y.x;
        s[2] = -y.y;
        s[3] = y.y;
      } else {
        const bool first = e < half;
        const float4 x = *reinterpret_cast<const float4*>(cs + (first ? e : e - half)), y = *reinterpret_cast<const float4*>(sn + (first ? e : e - half));
        c[0] = x.x, c[1] = x.y, c[2] = x.z, c[3] = x.w;
        s[0] = first ? -y.x : y.x, s[1] = first ? -y.y : y.y, s[2] = first ? -y.z : y.z, s[3] = first ? -y.w : y.w;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.c[v * 4 + i] = known ? c[i] : __int_as_float(0x7fffffff);
      t.s[v * 4 + i] = s[i];
    }
  }
}
// n rotated by the angles (forward), or back.  Whole warps.
template <int PAIR, int L, bool BACK>
__device__ __forceinline__ void rotate(const float* n, float* y, const Angles& t, int half, int col) {
  const int lane = threadIdx.x & 31, base = lane & ~(L - 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float other;                   // of columns that are not rotated: 0, whatever their neighbours hold
    if constexpr (PAIR == kNeighbours) {
      other = n[i ^ 1];
    } else {
      // the partner half a head away: four columns off within its lane where the half is not a multiple of eight
      const int e = col + i, p = e < half ? e + half : (e < 2 * half ? e - half : e);
      const int src = base + ((p >> 3) & (L - 1));
      other = __shfl_sync(0xffffffffu, n[PAIR == kHalvesOdd ? i ^ 4 : i], src);
    }
    other = col + i < 2 * half ? other : 0.f;
    y[i] = BACK ? fmaf(n[i], t.c[i], -other * t.s[i]) : fmaf(n[i], t.c[i], other * t.s[i]);
  }
}

struct Item {
  int b, s, which, h0, h1;         // heads [h0, h1) of queries (0) or keys (1) in one row
};
__device__ __forceinline__ Item item_at(const RotaryArgs& a, int64_t i) {
  const int chunks = a.chunks[0] + a.chunks[1];
  const int64_t row = i / chunks;
  int c = (int)(i - row * chunks);
  Item it;
  it.b = (int)(row / a.S);
  it.s = (int)(row - (int64_t)it.b * a.S);
  it.which = c >= a.chunks[0] ? 1 : 0;
  if (it.which) c -= a.chunks[0];
  it.h0 = c * a.heads_per_item;
  it.h1 = it.h0 + a.heads_per_item < a.H[it.which] ? it.h0 + a.heads_per_item : a.H[it.which];
  return it;
}
__device__ __forceinline__ int64_t position(const RotaryArgs& a, const Item& it) {
  if (a.positions == nullptr) return it.s;
  const int64_t i = (int64_t)it.b * a.S + it.s;
  return a.positions64 ? static_cast<const int64_t*>(a.positions)[i] : (int64_t) static_cast<const int*>(a.positions)[i];
}

// ---------------------------------------------------------------- forward
template <bool BF16, int PAIR, int L>
__global__ void __launch_bounds__(kThreads) rotary_forward_kernel(const __grid_constant__ RotaryArgs a, int64_t items) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = 4;
  const int col = (threadIdx.x & (L - 1)) * 8;
  const bool on = col < a.D;
  const float inv_d = 1.f / (float)a.D;
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const bool exists = i < items;                             // groups without an item go through the exchanges with the others
  Item it = item_at(a, exists ? i : 0);
  if (!exists) it.h1 = it.h0;
  float w[8];
  Angles t;
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = on ? load_w(a.w[it.which], a.w_type, col + e) : 0.f;
  load_angles<PAIR>(t, a, position(a, it), col);
  for (int r = 0; r < a.heads_per_item; r += U) {            // the same for all groups of a warp
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = it.h0 + r + u;
      q[u] = on && h < it.h1 ? *at(a.x[it.which], it.b, it.s, h, col) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u >= a.heads_per_item) break;
      const int h = it.h0 + r + u;
      float x[8], n[8], y[8];
      unpack8<BF16>(q[u], x);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
      const float rs = rsqrtf(fmaf(group_sum<L>(ss), inv_d, a.eps));
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = x[e] * rs * w[e];
      rotate<PAIR, L, false>(n, y, t, a.half, col);
      if (on && h < it.h1) *at(a.y[it.which], it.b, it.s, h, col) = pack8<BF16>(y);
    }
  }
}

// ---------------------------------------------------------------- backward
template <bool BF16, int PAIR, int L>
__global__ void __launch_bounds__(kThreads) rotary_backward_kernel(const __grid_constant__ RotaryArgs a, int64_t items) {
  __shared__ float sums[kThreads * 8];
  pdl_wait();
  pdl_trigger();
  constexpr int U = 2;
  const int col = (threadIdx.x & (L - 1)) * 8;
  const bool on = col < a.D;
  const float inv_d = 1.f / (float)a.D;
  constexpr int groups = kThreads / L;
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  // all groups of a block take equally many steps: the exchanges want whole warps
  for (int64_t i0 = (int64_t)blockIdx.x * groups; i0 < items; i0 += (int64_t)gridDim.x * groups) {
    const int64_t i = i0 + threadIdx.x / L;
    Item it = item_at(a, i < items ? i : 0);
    if (i >= items) it.h1 = it.h0;
    float w[8], acc[8];
    Angles t;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = on ? load_w(a.w[it.which], a.w_type, col + e) : 0.f;
      acc[e] = 0.f;
    }
    load_angles<PAIR>(t, a, position(a, it), col);
    for (int r = 0; r < a.heads_per_item; r += U) {
      uint4 qx[U], qd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = it.h0 + r + u;
        const bool here = on && h < it.h1;
        qx[u] = here ? *at(a.x[it.which], it.b, it.s, h, col) : make_uint4(0, 0, 0, 0);
        qd[u] = here ? *at(a.dy[it.which], it.b, it.s, h, col) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u >= a.heads_per_item) break;
        const int h = it.h0 + r + u;
        const bool here = on && h < it.h1;
        float x[8], d[8], g[8];
        unpack8<BF16>(qx[u], x);
        unpack8<BF16>(qd[u], d);
        rotate<PAIR, L, true>(d, g, t, a.half, col);         // g: the gradient behind the weights
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        const float rs = rsqrtf(fmaf(group_sum<L>(ss), inv_d, a.eps));
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= rs;
          if (here) acc[e] = fmaf(g[e], x[e], acc[e]);
          g[e] *= w[e];
          dot = fmaf(g[e], x[e], dot);
        }
        dot = group_sum<L>(dot) * inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = rs * fmaf(-x[e], dot, g[e]);
        if (here) *at(a.y[it.which], it.b, it.s, h, col) = pack8<BF16>(g);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (it.which == 0) dw[0][e] += acc[e];
      else dw[1][e] += acc[e];
    }
  }
  // the block's groups in order
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[threadIdx.x * 8 + e] = dw[which][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += kThreads) {
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += sums[g * L * 8 + c];
      a.partial[((int64_t)blockIdx.x * 2 + which) * a.D + c] = s;
    }
  }
}

// dw[c] = sum of the blocks' shares: 32 columns per block, eight warps that each add up every eighth share.
__global__ void __launch_bounds__(kThreads) rotary_weights_kernel(const __grid_constant__ RotaryArgs a, int blocks) {
  __shared__ float sums[8][32];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;       // c runs through queries, then keys
  float s = 0.f;
  if (c < 2 * a.D)
    for (int b = warp; b < blocks; b += 8) s += a.partial[(int64_t)b * 2 * a.D + c];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * a.D) {
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
    const int which = c >= a.D ? 1 : 0, i = c - which * a.D;
    if (a.w_type == 2) static_cast<float*>(a.dw[which])[i] = s;
    else if (a.w_type == 0) static_cast<__nv_bfloat16*>(a.dw[which])[i] = __float2bfloat16_rn(s);
    else static_cast<__half*>(a.dw[which])[i] = __float2half_rn(s);
  }
}

int lanes_of(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }
int64_t items_of(const RotaryArgs& a) { return (int64_t)a.B * a.S * (a.chunks[0] + a.chunks[1]); }

template <bool BF16, int PAIR, int L>
cudaError_t launch(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  if (!backward) return launch_pdl(rotary_forward_kernel<BF16, PAIR, L>, dim3(blocks), dim3(kThreads), 0, s, a, items_of(a));
  const cudaError_t e = launch_pdl(rotary_backward_kernel<BF16, PAIR, L>, dim3(blocks), dim3(kThreads), 0, s, a, items_of(a));
  if (e != cudaSuccess) return e;
  return launch_pdl(rotary_weights_kernel, dim3((2 * a.D + 31) / 32), dim3(kThreads), 0, s, a, blocks);
}
template <bool BF16, int PAIR>
cudaError_t launch_lanes(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  switch (lanes_of(a.D)) {
    case 8: return launch<BF16, PAIR, 8>(a, backward, blocks, s);
    case 16: return launch<BF16, PAIR, 16>(a, backward, blocks, s);
    default: return launch<BF16, PAIR, 32>(a, backward, blocks, s);
  }
}
template <bool BF16>
cudaError_t launch_pairing(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  if (a.interleaved) return launch_lanes<BF16, kNeighbours>(a, backward, blocks, s);
  return a.half % 8 == 0 ? launch_lanes<BF16, kHalves>(a, backward, blocks, s) : launch_lanes<BF16, kHalvesOdd>(a, backward, blocks, s);
}
cudaError_t launch_any(const RotaryArgs& a, bool backward, int blocks, cudaStream_t s) {
  if (a.D <= 0 || a.D % 8 != 0 || a.D > kRotaryMaxDim || a.half % 4 != 0 || a.half <= 0 || 2 * a.half > a.D || blocks <= 0)
    return cudaErrorInvalidValue;
  return a.is_bf16 ? launch_pairing<true>(a, backward, blocks, s) : launch_pairing<false>(a, backward, blocks, s);
}

}  // namespace

int rotary_blocks(RotaryArgs& a, bool backward, int sm_count) {
  const int lanes = lanes_of(a.D), groups = kThreads / lanes;
  const int64_t rows = (int64_t)a.B * a.S;
  // eight heads per item where that still gives every SM four blocks, else fewer: a short call wants many groups
  int hpi = 8;
  for (;; hpi /= 2) {
    a.heads_per_item = hpi;
    for (int i = 0; i < 2; ++i) a.chunks[i] = (a.H[i] + hpi - 1) / hpi;
    if (hpi == 1 || rows * (a.chunks[0] + a.chunks[1]) >= (int64_t)sm_count * 4 * groups) break;
  }
  const int64_t need = (rows * (a.chunks[0] + a.chunks[1]) + groups - 1) / groups;
  const int64_t most = backward ? (int64_t)sm_count * 4 : INT32_MAX;
  return need > most ? (int)most : (int)need;
}
cudaError_t launch_rotary_forward(const RotaryArgs& a, int blocks, cudaStream_t s) { return launch_any(a, false, blocks, s); }
cudaError_t launch_rotary_backward(const RotaryArgs& a, int blocks, cudaStream_t s) { return launch_any(a, true, blocks, s); }

}  // namespace pccl
