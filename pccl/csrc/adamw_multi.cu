// AdamW over a list of tensors in one launch, states in 32 or in 8 bits.
//
//   g = grad * clip,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// One warp takes a block of 256 elements of one tensor, eight neighbours per lane; which tensor it is, is looked up in
// the table that comes with the launch's arguments, so nothing is copied to the device first and a captured launch carries
// its own table.  Streaming: 28 bytes per parameter with states in 32 bits and a 16-bit gradient and parameter beside the 32-bit
// copy, 16 bytes with states in 8 bits.
//
// What bounds it.  308 million parameters: with states in 32 bits 1382 us, 6.24 TB/s (0.95 of the measured copy rate); tensors off
// vector boundaries 1402.  With three blocks on an SM, more loads on their way, 1404; with four 1590.  In 8 bits 955 us, 5.16 TB/s: the
// codes cost about 80 instructions for each element, and the issue slots are three quarters full; misaligned 1277: as full, DRAM at 42 %
// instead of 57 %, a third more instructions for accesses of one element and the exchange between lanes.  Reading the
// states back (adamw_dequantize) 458 us, 6.72 TB/s.
//
// 8-bit states.  A block keeps the size A of its largest value in 32 bits and a code c per element:
//   m = sign * A (c / 127)^2,  v = A (c / 255)^4
// Powers give small values finer steps than large ones: a v of 1e-9 of the largest still has a code of its own, which it needs,
// because its root divides.  A value between two codes becomes one of them by chance, in proportion to its distances, so that
// the mean is exact: rounding to the nearest code would stop an average whose change per step (1 - b2 of it) is below half a
// step of the code, which at b2 = 0.999 is nearly always.  The chance is a hash of the element's place in the state, the
// step and the seed: the same call gives the same bits.  A v that is not zero never gets code 0, and a block whose largest size is
// below 2^-80 is held as zeros.  A block that holds a value that is not finite reads back as NaN throughout: a broken step does not hide.
//
// What zeros for a small v cost.  At each step at most 2^-80 is dropped, which fades by b2 a step, so v lacks at most 2^-80 b2 / (1 - b2)
// in all, and so much over (1 - b2) / (1 - b2^t) of that, never more, after the correction of its bias: the root lacks at most
// r = 2^-40 / sqrt(1 - b2).  The quotient m / (root + eps) is then too large by r / eps of itself at most, whatever m is.  Where eps is
// below 32 r (1.3e-10 at b2 = 0.95, 9.2e-10 at 0.999) 8-bit states are refused: with eps = 1e-15, gradients of 2e-12 that
// stop would move a parameter by 1800 lr in one step.
// The parameter is updated from the 32-bit m and v, before they are rounded.
//
// The products and sums that lead to a code are rounded one by one (no fused multiply-add): what a code is does not hang on what
// a compiler makes of the expression.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "act.cuh"
#include "adamw_multi.h"
#include "pdl.cuh"

namespace pccl {

namespace {

constexpr int kThreads = 256;

template <int MAX>
struct Table {
  AdamTensor t[MAX];
  int count;
};

// Two rounds of multiply and xor-shift.  The multipliers are the leading bits of the fractional parts of the square roots
// of 2 and 3, both odd.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

// 8-bit pieces of the state and 16- or 32-bit elements, eight at a time.
struct Raw8 {
  uint4 a, b;                              // fp32: both; 16 bits: a
};
template <int TYPE>
__device__ __forceinline__ void widen(const Raw8& r, float* f) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if constexpr (TYPE == kAdamF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  } else if constexpr (TYPE == kAdamBf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
}
// 32 bytes in one access.
__device__ __forceinline__ void load32(const void* p, Raw8& r) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const float* f) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]),
               "f"(f[5]), "f"(f[6]), "f"(f[7])
               : "memory");
}
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, int64_t i, Raw8& r) {
  if constexpr (TYPE == kAdamF32) load32(static_cast<const float*>(base) + i, r);
  else r.a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i));
}
// One element as it lies in memory, and its value.
template <int TYPE>
__device__ __forceinline__ uint32_t load_bits(const void* base, int64_t i) {
  if constexpr (TYPE == kAdamF32) return static_cast<const uint32_t*>(base)[i];
  else return static_cast<const uint16_t*>(base)[i];
}
template <int TYPE>
__device__ __forceinline__ float from_bits(uint32_t w) {
  if constexpr (TYPE == kAdamF32) return __uint_as_float(w);
  else if constexpr (TYPE == kAdamBf16) return __uint_as_float(w << 16);
  else return __half2float(__ushort_as_half((unsigned short)w));
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (TYPE == kAdamBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <int TYPE>
__device__ __forceinline__ void store1(void* base, int64_t i, float x) {
  if constexpr (TYPE == kAdamF32) static_cast<float*>(base)[i] = x;
  else if constexpr (TYPE == kAdamBf16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(base)[i] = __float2half_rn(x);
}

__device__ __forceinline__ void unpair(const F2* a, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) split(a[i], f[2 * i], f[2 * i + 1]);
}

// A product that is rounded by itself.  The packed multiplication is no such thing: what adds its result up may become one fused
// operation with it (seen: a quarter of the moments one unit in the last place off).
__device__ __forceinline__ F2 times(const F2& a, const F2& b) {
  float a0, a1, b0, b1;
  split(a, a0, a1);
  split(b, b0, b1);
  return f2(__fmul_rn(a0, b0), __fmul_rn(a1, b1));
}

// ---- codes
constexpr float kSigned = 16129.f, kUnsigned = 4228250625.f;      // 127^2, 255^4 (rounded to 32 bits)
constexpr float kSignedUnit = (float)(1.0 / 16129.0), kUnsignedUnit = (float)(1.0 / 4228250625.0);
constexpr float kLeast = 8.271806125530277e-25f;                  // 2^-80

// Four codes as fp32, two and two: the byte becomes the last mantissa byte of 2^23 + c, which is exact (conversions between
// integers and floats run at a quarter of the rate of additions).
template <bool SIGNED>
__device__ __forceinline__ void codes4(uint32_t w, F2& a, F2& b) {
  if constexpr (SIGNED) w ^= 0x80808080u;                       // c + 128
  const F2 off = f2(SIGNED ? -8388736.f : -8388608.f);
  a = f2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7541))) + off;
  b = f2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7542)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7543))) + off;
}
template <bool SIGNED>
__device__ __forceinline__ F2 decode2(const F2& c, const F2& unit) {
  if constexpr (SIGNED) {
    float x, y;
    split(c, x, y);
    return unit * f2(fabsf(x) * x, fabsf(y) * y);
  } else {
    const F2 c2 = c * c;
    return unit * (c2 * c2);
  }
}
// Eight values.
template <bool SIGNED>
__device__ __forceinline__ void decode8(const uint2& w, float unit, F2* x) {
  codes4<SIGNED>(w.x, x[0], x[1]);
  codes4<SIGNED>(w.y, x[2], x[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = decode2<SIGNED>(x[i], f2(unit));
}
template <bool SIGNED>
__device__ __forceinline__ F2 power2(const F2& c) {
  const F2 c2 = c * c;
  return SIGNED ? c2 : c2 * c2;
}
__device__ __forceinline__ float root_hw(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Codes of two values, as floats 2^23 + c (unsigned) or 1.5 * 2^23 + c (signed), whose last byte is the code.  inv: 1 / A (0: the
// block holds zeros); u: noise in (0, 1).  c starts as the whole part of the hardware's root.  Where that is off by one, because
// the root lies within 2^-16 of a whole number, the comparison moves it to the right neighbour all the same, but for noise
// within 2^-16 of 0 or 1.
template <bool SIGNED>
__device__ __forceinline__ void encode2(const F2& x, const F2& inv, const F2& u, bool zeros, float& r0, float& r1) {
  constexpr float top = SIGNED ? 127.f : 255.f;
  float x0, x1, y0, y1;
  split(x, x0, x1);
  split((x * inv) * f2(SIGNED ? kSigned : kUnsigned), y0, y1);
  float c0 = root_hw(fabsf(y0)), c1 = root_hw(fabsf(y1));
  if constexpr (!SIGNED) {
    c0 = root_hw(c0);
    c1 = root_hw(c1);
  }
  const F2 c = f2(__fadd_rz(c0, 8388608.f), __fadd_rz(c1, 8388608.f)) + f2(-8388608.f);
  const F2 next = c + f2(1.f), lo = power2<SIGNED>(c);
  const F2 step = u * fma2(lo, f2(-1.f), power2<SIGNED>(next));           // times -1 is exact: a subtraction
  float l0, l1, s0, s1, a0, a1, b0, b1;
  split(lo, l0, l1);
  split(step, s0, s1);
  split(c, a0, a1);
  split(next, b0, b1);
  a0 = fminf(s0 < __fsub_rn(fabsf(y0), l0) ? b0 : a0, top);
  a1 = fminf(s1 < __fsub_rn(fabsf(y1), l1) ? b1 : a1, top);
  if constexpr (SIGNED) {
    r0 = copysignf(a0, x0) + 12582912.f;
    r1 = copysignf(a1, x1) + 12582912.f;
  } else {
    // not below 1 where x is not zero (its bits as a number, at most 1) and the block is not held as zeros
    const uint32_t most = zeros ? 0u : 1u;
    r0 = __uint_as_float(max(__float_as_uint(a0 + 8388608.f), 0x4B000000u + min(__float_as_uint(x0), most)));
    r1 = __uint_as_float(max(__float_as_uint(a1 + 8388608.f), 0x4B000000u + min(__float_as_uint(x1), most)));
  }
}
__device__ __forceinline__ uint32_t bytes4(float a, float b, float c, float d) {
  const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// 16 bits of noise n as (n + 1/2) / 2^16, exactly: the bits of 1 + that, less 1.
__device__ __forceinline__ float noise_hi(uint32_t h) { return __uint_as_float(((h >> 9) & 0x007fff80u) | 0x3f800040u); }
__device__ __forceinline__ float noise_lo(uint32_t h) { return __uint_as_float(((h << 7) & 0x007fff80u) | 0x3f800040u); }

// The block's largest size: sizes are not negative, so their bits are in the order of their values, infinities and NaN on top.
__device__ __forceinline__ float block_max(const F2* x) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    split(x[i], a, b);
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(a), "f"(b));
  }
  uint32_t m = __float_as_uint(fabsf(top));
  m = __reduce_max_sync(0xffffffffu, m);
  const float f = __uint_as_float(m);
  return m >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : (f < kLeast ? 0.f : f);
}

// Where a block lies, and what is read of it.  The loads of a warp's next block are on their way while it works on this one.
template <bool BITS8>
struct Block {
  int k;                                                       // tensor
  int64_t at;                                                  // place of the lane's first element within it
  uint64_t sblk;                                               // place within the state
  bool whole;                                                  // 256 elements on vector boundaries; the same for the whole warp
  Raw8 g, p;
  uint2 cm, cv;                                                // 8 bits
  float m_scale, v_scale;
};
template <int PT>
__device__ __forceinline__ void* weights_of(const AdamTensor& t) {
  return PT == kAdamF32 ? t.param : static_cast<void*>(t.master);
}
// Off vector boundaries, or at a tensor's end: neighbouring lanes read neighbouring elements.
template <int PT, int GT, bool BITS8>
__device__ __forceinline__ void fetch_ragged(const AdamTensor& t, Block<BITS8>& x) {
  uint32_t g[8], p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t e = x.at - (threadIdx.x & 31) * 7 + i * 32;
    g[i] = e < t.n ? load_bits<GT>(t.grad, e) : 0u;
    p[i] = e < t.n ? static_cast<const uint32_t*>(weights_of<PT>(t))[e] : 0u;
  }
  x.g = {make_uint4(g[0], g[1], g[2], g[3]), make_uint4(g[4], g[5], g[6], g[7])};
  x.p = {make_uint4(p[0], p[1], p[2], p[3]), make_uint4(p[4], p[5], p[6], p[7])};
}
template <int PT, int GT, bool BITS8, int MAX>
__device__ __forceinline__ void fetch(const AdamMultiArgs& a, const Table<MAX>& table, uint32_t blk, int k, Block<BITS8>& x) {
  // the last tensor that starts at or before this block: mostly the last block's, else one behind it
  if (k + 1 < table.count && table.t[k + 1].first <= blk) {
    int hi = table.count;
    while (hi - k > 1) {
      const int mid = (k + hi) >> 1;
      if (table.t[mid].first <= blk) k = mid;
      else hi = mid;
    }
  }
  const AdamTensor& t = table.t[k];
  const int lane = threadIdx.x & 31;
  x.k = k;
  x.at = (int64_t)(blk - t.first) * kAdamBlock + lane * 8;
  x.sblk = a.first_block + blk;
  const void* weights = weights_of<PT>(t);
  const uintptr_t bad = (reinterpret_cast<uintptr_t>(weights) & 31u) | (reinterpret_cast<uintptr_t>(t.grad) & (GT == kAdamF32 ? 31u : 15u)) |
                        (PT == kAdamF32 ? 0u : reinterpret_cast<uintptr_t>(t.param) & 15u);
  x.whole = bad == 0 && x.at - lane * 8 + kAdamBlock <= t.n;
  if (x.whole) {
    load8<GT>(t.grad, x.at, x.g);
    load8<kAdamF32>(weights, x.at, x.p);
  } else {
    fetch_ragged<PT, GT>(t, x);
  }
  if constexpr (BITS8) {                                       // the state's blocks are whole: behind a tensor's end they hold zeros
    const uint64_t si = x.sblk * kAdamBlock + (uint64_t)lane * 8;
    x.cm = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + si));
    x.cv = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + si));
    x.m_scale = a.m_scale[x.sblk];
    x.v_scale = a.v_scale[x.sblk];
  }
}

// A warp's 256 numbers: from those of neighbouring lanes in turn, one to a word, to eight neighbours of each lane.
template <int TYPE>
__device__ __forceinline__ void exchange(float* s, const Raw8& r, float* x) {
  const int lane = threadIdx.x & 31;
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i * 32 + lane] = from_bits<TYPE>(w[i]);
  __syncwarp();
  const float4 a = reinterpret_cast<const float4*>(s)[lane * 2], b = reinterpret_cast<const float4*>(s)[lane * 2 + 1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  __syncwarp();
}

template <int PT, int GT, bool BITS8, int MAX>
__global__ void __launch_bounds__(kThreads, BITS8 ? 4 : 2) adamw_multi_kernel(const __grid_constant__ AdamMultiArgs a,
                                                                              const __grid_constant__ Table<MAX> table) {
  __shared__ __align__(16) float stage[kThreads / 32][kAdamBlock];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  float gs = a.grad_scale;
  if (a.total_sq_norm != nullptr) {
    const float norm = sqrtf(*a.total_sq_norm) * a.grad_scale;
    const float clip = a.max_grad_norm / (norm + 1e-6f);
    gs = clip >= 1.f ? gs : gs * clip;                   // a norm that is NaN makes every gradient NaN
  }
  const uint32_t warps = gridDim.x * (kThreads / 32);
  uint32_t blk = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (blk >= a.blocks) return;
  Block<BITS8> x;
  fetch<PT, GT, BITS8, MAX>(a, table, blk, 0, x);
  for (;;) {
    const AdamTensor& t = table.t[x.k];
    void* weights = weights_of<PT>(t);
    const int64_t at = x.at;
    const uint64_t sblk = x.sblk, si = sblk * kAdamBlock + (uint64_t)lane * 8;
    const bool whole = x.whole;
    float g[8], p[8];
    F2 m[4], v[4];                                             // pairs of neighbours
    Raw8 rm, rv;
    if constexpr (!BITS8) {
      load8<kAdamF32>(a.m, (int64_t)si, rm);
      load8<kAdamF32>(a.v, (int64_t)si, rv);
    } else {
      decode8<true>(x.cm, __fmul_rn(x.m_scale, kSignedUnit), m);
      decode8<false>(x.cv, __fmul_rn(x.v_scale, kUnsignedUnit), v);
    }
    if (whole) {
      widen<GT>(x.g, g);
      widen<kAdamF32>(x.p, p);
    } else {
      exchange<GT>(stage[threadIdx.x >> 5], x.g, g);           // for eight in a row
      exchange<kAdamF32>(stage[threadIdx.x >> 5], x.p, p);
    }
    if constexpr (!BITS8) {
      float y[8], z[8];
      widen<kAdamF32>(rm, y);
      widen<kAdamF32>(rv, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = f2(y[2 * i], y[2 * i + 1]);
        v[i] = f2(z[2 * i], z[2 * i + 1]);
      }
    }
    blk += warps;
    const bool more = blk < a.blocks;
    if constexpr (!BITS8) {
      if (more) fetch<PT, GT, BITS8, MAX>(a, table, blk, x.k, x);
    }
    // ---- the step
    const F2 keep = f2(1.f - a.lr * t.decay), rate = f2(-a.lr * a.bias1);
    const bool tiny_eps = !BITS8 && a.eps < 1e-15f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F2 y = f2(g[2 * i], g[2 * i + 1]) * f2(gs);
      m[i] = times(f2(a.beta1), m[i]) + times(f2(a.one_minus_beta1), y);
      v[i] = times(f2(a.beta2), v[i]) + times(f2(a.one_minus_beta2), y * y);
      // the update's root and quotient are the hardware's (a few units in the last place of the update, not of the parameter)
      float a0, a1;
      split(v[i] * f2(a.bias2), a0, a1);
      if (tiny_eps) {                                          // a v below 2^-126 counts
        asm("sqrt.approx.f32 %0, %0;" : "+f"(a0));
        asm("sqrt.approx.f32 %0, %0;" : "+f"(a1));
      } else {
        a0 = root_hw(a0);
        a1 = root_hw(a1);
      }
      split(f2(a0, a1) + f2(a.eps), a0, a1);
      split(fma2(f2(p[2 * i], p[2 * i + 1]), keep, m[i] * rate * f2(rcp_hw(a0), rcp_hw(a1))), p[2 * i], p[2 * i + 1]);
    }
    // ---- states
    uint32_t cm[2] = {0u, 0u}, cv[2] = {0u, 0u};
    if constexpr (BITS8) {
      const float am = block_max(m), av = block_max(v);
      const float im = am > 0.f ? __fdiv_rn(1.f, am) : 0.f, iv = av > 0.f ? __fdiv_rn(1.f, av) : 0.f;
      const uint32_t base = (uint32_t)si + (uint32_t)(si >> 32) * 0x9E3779B1u + a.key;    // blocks do not straddle 2^32
      float km[8], kv[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t n0 = mix(base + 2 * i), n1 = mix(base + 2 * i + 1);
        encode2<true>(m[i], f2(im), f2(noise_hi(n0), noise_hi(n1)) + f2(-1.f), false, km[2 * i], km[2 * i + 1]);
        encode2<false>(v[i], f2(iv), f2(noise_lo(n0), noise_lo(n1)) + f2(-1.f), !(iv > 0.f), kv[2 * i], kv[2 * i + 1]);
      }
      for (int i = 0; i < 2; ++i) {
        cm[i] = bytes4(km[4 * i], km[4 * i + 1], km[4 * i + 2], km[4 * i + 3]);
        cv[i] = bytes4(kv[4 * i], kv[4 * i + 1], kv[4 * i + 2], kv[4 * i + 3]);
      }
      if (lane == 0) {
        a.m_scale[sblk] = am;
        a.v_scale[sblk] = av;
      }
      // padding is in the state's last block of a tensor too: its codes are 0
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + si), make_uint2(cm[0], cm[1]));
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + si), make_uint2(cv[0], cv[1]));
    }
    // ---- stores
    if constexpr (!BITS8) {                                    // behind a tensor's end: zeros, as they were
      float y[8], z[8];
      unpair(m, y);
      unpair(v, z);
      store32(static_cast<float*>(a.m) + si, y);
      store32(static_cast<float*>(a.v) + si, z);
    }
    if (whole) {
      store32(static_cast<float*>(weights) + at, p);
      if constexpr (PT != kAdamF32)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.param) + at) =
            make_uint4(narrow2<PT>(p[0], p[1]), narrow2<PT>(p[2], p[3]), narrow2<PT>(p[4], p[5]), narrow2<PT>(p[6], p[7]));
    } else {
      const int64_t first = at - lane * 8;
      float* s = stage[threadIdx.x >> 5];
      reinterpret_cast<float4*>(s)[lane * 2] = make_float4(p[0], p[1], p[2], p[3]);
      reinterpret_cast<float4*>(s)[lane * 2 + 1] = make_float4(p[4], p[5], p[6], p[7]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t e = first + i * 32 + lane;
        if (e < t.n) {
          const float y = s[i * 32 + lane];
          static_cast<float*>(weights)[e] = y;
          if constexpr (PT != kAdamF32) store1<PT>(t.param, e, y);
        }
      }
      __syncwarp();
    }
    if (!more) break;
    if constexpr (BITS8) fetch<PT, GT, BITS8, MAX>(a, table, blk, x.k, x);
  }
}

// 2 bytes in, 8 out per element; a lane takes eight neighbours of one block.
__global__ void __launch_bounds__(kThreads) adamw_dequantize_kernel(const uint8_t* m, const float* m_scale, const uint8_t* v,
                                                                    const float* v_scale, float* m_out, float* v_out, int64_t n) {
  pdl_wait();
  pdl_trigger();
  const int64_t stride = (int64_t)gridDim.x * kThreads * 8;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8; i < n; i += stride) {
    const uint2 cm = *reinterpret_cast<const uint2*>(m + i), cv = *reinterpret_cast<const uint2*>(v + i);
    const float um = __fmul_rn(m_scale[i / kAdamBlock], kSignedUnit), uv = __fmul_rn(v_scale[i / kAdamBlock], kUnsignedUnit);
    F2 p[4], q[4];
    float x[8], y[8];
    decode8<true>(cm, um, p);
    decode8<false>(cv, uv, q);
    unpair(p, x);
    unpair(q, y);
    store32(m_out + i, x);
    store32(v_out + i, y);
  }
}

template <int PT, int GT, bool BITS8, int MAX>
cudaError_t launch(const AdamMultiArgs& a, const AdamTensor* tensors, int count, int sm_count, cudaStream_t s) {
  Table<MAX> table;
  memcpy(table.t, tensors, sizeof(AdamTensor) * (size_t)count);
  table.count = count;
  const uint32_t need = (a.blocks + kThreads / 32 - 1) / (kThreads / 32), most = (uint32_t)sm_count * (BITS8 ? 4 : 2);
  return launch_pdl(adamw_multi_kernel<PT, GT, BITS8, MAX>, dim3(need < most ? need : most), dim3(kThreads), 0, s, a, table);
}
template <int PT, int GT>
cudaError_t launch_bits(const AdamMultiArgs& a, const AdamTensor* tensors, int count, bool bits8, int sm_count, cudaStream_t s) {
  // a short list does not carry the long table with it
  if (count <= 64)
    return bits8 ? launch<PT, GT, true, 64>(a, tensors, count, sm_count, s) : launch<PT, GT, false, 64>(a, tensors, count, sm_count, s);
  return bits8 ? launch<PT, GT, true, kAdamTensors>(a, tensors, count, sm_count, s)
               : launch<PT, GT, false, kAdamTensors>(a, tensors, count, sm_count, s);
}
template <int PT>
cudaError_t launch_grad(const AdamMultiArgs& a, const AdamTensor* t, int count, int gt, bool bits8, int sm_count, cudaStream_t s) {
  if (gt == kAdamBf16) return launch_bits<PT, kAdamBf16>(a, t, count, bits8, sm_count, s);
  if (gt == kAdamF16) return launch_bits<PT, kAdamF16>(a, t, count, bits8, sm_count, s);
  return launch_bits<PT, kAdamF32>(a, t, count, bits8, sm_count, s);
}

}  // namespace

double adamw_least_eps(double beta2) { return ldexp(1.0, -35) / sqrt(1.0 - beta2); }

uint32_t adamw_noise_key(uint64_t seed, int64_t step) { return mix(mix((uint32_t)seed ^ mix((uint32_t)(seed >> 32))) + (uint32_t)step); }

cudaError_t launch_adamw_multi(const AdamMultiArgs& a, const AdamTensor* tensors, int count, int pt, int gt, bool bits8, int sm_count,
                               cudaStream_t s) {
  if (count <= 0 || a.blocks == 0) return cudaSuccess;
  if (count > kAdamTensors) return cudaErrorInvalidValue;
  if (pt == kAdamBf16) return launch_grad<kAdamBf16>(a, tensors, count, gt, bits8, sm_count, s);
  if (pt == kAdamF16) return launch_grad<kAdamF16>(a, tensors, count, gt, bits8, sm_count, s);
  return launch_grad<kAdamF32>(a, tensors, count, gt, bits8, sm_count, s);
}

cudaError_t launch_adamw_dequantize(const int8_t* m, const float* m_scale, const uint8_t* v, const float* v_scale, float* m_out,
                                    float* v_out, int64_t n, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  const int64_t blocks = (n / 8 + kThreads - 1) / kThreads;
  return launch_pdl(adamw_dequantize_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(kThreads), 0, s,
                    reinterpret_cast<const uint8_t*>(m), m_scale, v, v_scale, m_out, v_out, n);
}

}  // namespace pccl
