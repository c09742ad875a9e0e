// The AdamW step over many tensors at once, with the gradients' norm clipped, and its C
// ABI (include/cugo_b200.h).
//
//   c = min(1, max_norm / (|g| + 1e-6)), g = c g           (one norm over all tensors)
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// One launch takes up to kMostTensors tensors: their pointers travel as the kernel's
// parameters (nothing of a call is kept on the device, and a captured graph holds them
// by value).  A warp takes 256 elements at a time, a thread 8 of them; a tile of 8 or 32
// such blocks finds its tensor by a search over the tensors' first tiles.
//
// States in 8 bits: e4m3 codes with one scale per 256 elements of a tensor, the warp's.
// The scale is a power of two (an e8m0 byte), the smallest that keeps the block's largest
// value at or below 448 (e4m3's largest).  Codes are rounded up or down by random bits.
// Both belong together: m and v move by little per step (v by a thousandth), far less
// than e4m3's steps of 1/8 to 1/16, and rounding to nearest would leave them where they
// are; and with a scale that follows the largest value exactly, every code would be
// re-rounded at every step, where a power of two leaves the grid in place, so that a
// value that moved by the share f of a step is off its grid by f only, and the noise of
// the moving average stays at about sqrt(f) steps.  A second moment above 0 never rounds
// to 0: a step is then too short instead of unbounded.  The step itself uses m and v
// before rounding.
//
// bf16 parameters are rounded by random bits too: lr times the update is mostly below
// half of bf16's 2^-8, and to nearest nothing would move.
//
// The random bits of element number e (counted over the call's tensors in blocks of 256,
// so that no two elements share one) are a 32-bit mix of e, the step and the seed: one
// per element, 16 bits for m, 16 for v, and a product of them for p.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/cugo_b200.h"

namespace {

using i64 = int64_t;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlock = 256;              // elements of a scale
constexpr int kThreads = 256, kPer = 8;  // 8 warps, a scale's block at a time each
constexpr int kWarps = kThreads / 32;
constexpr int kSms = 148;
constexpr int kBlocks = 4;  // of a scale, that a warp takes of many
constexpr int kNormBlocks = 8 * kSms;
constexpr int kFewTensors = 40, kMostTensors = 400;

struct Tensor {
  void* p;
  const void* g;
  void *m, *v;
  uint8_t *ms, *vs;  // the scales (8-bit states)
  i64 n;
  int wide;          // every pointer is a multiple of 16 bytes
  int first_tile;    // of the launch
  i64 first_block;   // blocks of 256 elements before this tensor in the call
};

// A tile is kWarps x per_warp blocks of 256 elements, per_warp consecutive ones a warp.
template <int kMost>
struct Tensors {
  int count, tiles, per_warp;
  Tensor t[kMost];
};

// What the step's scalars come to, written by prepare_kernel.
struct Scalars {
  float clip;       // c
  float step_size;  // lr / (1 - b1^t)
  float keep;       // 1 - lr wd
  float root;       // 1 / sqrt(1 - b2^t)
  uint32_t key;     // of the random bits
};

struct Options {
  double lr, beta1, beta2, decay;
  const float* lr_dev;  // or null
  float b1, c1, b2, c2, eps, max_norm;
  uint32_t seed;
};

// A 32-bit mixer: xor-shifts and odd products (constants found by C. Wellons' search for
// low bias, 2018).
__device__ __forceinline__ uint32_t mix_middle(uint32_t x) {  // between its first and last shift
  x *= 0x7feb352du;
  x ^= x >> 15;
  return x * 0x846ca68bu;
}
// A parameter's 16 bits, from the mix before its last shift.
__device__ __forceinline__ uint32_t random_p(uint32_t x) { return ((x ^ (x >> 16)) * 0x2c1b3c6du) >> 16; }
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = mix_middle(x ^ (x >> 16));
  return x ^ (x >> 16);
}

__device__ __forceinline__ double sum_warp(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// The tensor that holds a tile: the last whose first tile is not behind it.
template <int kMost>
__device__ __forceinline__ int find(const Tensors<kMost>& a, int tile) {
  int low = 0, high = a.count;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (a.t[mid].first_tile <= tile) low = mid;
    else high = mid;
  }
  return low;
}

// A thread's 8 consecutive values, aligned and all there where kWide is set, else the first
// n of them, and zeros.
template <bool kWide>
__device__ __forceinline__ void load8(const float* p, int n, float (&f)[8]) {
  if constexpr (kWide) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? p[e] : 0.0f;
  }
}

template <bool kWide>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int n, float (&f)[8]) {
  if constexpr (kWide) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? __bfloat162float(p[e]) : 0.0f;
  }
}

template <bool kWide>
__device__ __forceinline__ void store8(float* p, int n, const float (&f)[8]) {
  if constexpr (kWide) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = f[e];
  }
}

// The upper halves of f (rounded there already) as bf16.
template <bool kWide>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int n, const float (&f)[8]) {
  if constexpr (kWide) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __byte_perm(__float_as_uint(f[2 * e]), __float_as_uint(f[2 * e + 1]), 0x7632);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(__float_as_uint(f[e]) >> 16);
  }
}

// 8 codes as floats, not scaled.
__device__ __forceinline__ void decode(uint32_t a, uint32_t b, float (&f)[8]) {
  const uint32_t w[2] = {a, b};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(w[e / 2] >> (16 * (e % 2)));
    const float2 t = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    f[2 * e] = t.x;
    f[2 * e + 1] = t.y;
  }
}

template <bool kWide>
__device__ __forceinline__ void load_codes(const uint8_t* p, int n, float (&f)[8]) {
  uint32_t w[2] = {0, 0};
  if constexpr (kWide) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    w[0] = q.x, w[1] = q.y;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) w[e / 4] |= static_cast<uint32_t>(p[e]) << (8 * (e % 4));
  }
  decode(w[0], w[1], f);
}

template <bool kWide>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * e], f[4 * e + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * e + 2], f[4 * e + 3]), __NV_SATFINITE, __NV_E4M3);
    w[e] = __byte_perm(a, b, 0x5410);
  }
  if constexpr (kWide) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = static_cast<uint8_t>(w[e / 4] >> (8 * (e % 4)));
  }
}

// 2^(byte - 127) and its inverse, for the scale bytes 27 .. 247 that this file writes
// (byte 0, an untouched state, counts as the smallest float that is no denormal).
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((byte > 0 ? byte : 1) << 23); }
__device__ __forceinline__ float inverse_of(int byte) { return __uint_as_float((254 - byte) << 23); }

// The scale of a block whose largest finite magnitude is `largest`: 448 = 1.75 x 2^8.
__device__ __forceinline__ int scale_byte(float largest) {
  const int bits = __float_as_int(largest);
  const int e = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return e < 27 ? 27 : e > 247 ? 247 : e;
}

// The magnitude a (at most 448) rounded to e4m3's grid, up where the random number r says
// so: 16 bits, as a share of a step, from bit 4 on, and half of the last.  Below 2^-6 the
// steps are 2^-9, which 2^-6 more brings to the same place; above they are 1/8 of the
// power of two.
__device__ __forceinline__ float round_e4m3(float a, uint32_t r) {
  float small;  // 1 below 2^-6, else 0
  asm("set.lt.f32.f32 %0, %1, %2;" : "=f"(small) : "f"(a), "f"(0.015625f));
  const uint32_t bits = (__float_as_uint(fmaf(small, 0.015625f, a)) + r) & 0xfff00000u;
  return fmaf(small, -0.015625f, __uint_as_float(bits));
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A warp's largest magnitude; infinite or NaN where one is.  kSigned: some may be negative.
template <bool kSigned>
__device__ __forceinline__ float warp_largest(const float (&f)[8]) {
  float top = 0.0f, r;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    if constexpr (kSigned) top = max_nan(top, fabsf(f[e]), fabsf(f[e + 1]));
    else top = max_nan(top, f[e], f[e + 1]);
  }
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(top));
  return r;
}

// The same over the finite magnitudes only (as bits they order as the values do).
__device__ __forceinline__ float warp_largest_finite(const float (&f)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(f[e]) & 0x7fffffffu;
    top = b < 0x7f800000u && b > top ? b : top;
  }
  return __uint_as_float(__reduce_max_sync(kFull, top));
}

__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two floats in one instruction each.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(Two t, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v));
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// a + b, the products before them already rounded.  Where both stay packed the results are
// those of one operation without the rounding between (codes differed from the formula's), so
// the sum is taken apart.
__device__ __forceinline__ void sum(Two a, Two b, float& x, float& y) {
  float ax, ay, bx, by;
  split(a, ax, ay);
  split(b, bx, by);
  x = __fadd_rn(ax, bx);
  y = __fadd_rn(ay, by);
}

// Where a thread's 8 elements and its warp's scales are, and the first element's number.
template <typename P>
struct Place {
  P* p;
  void *m, *v;
  uint8_t *ms, *vs;
  i64 number;
  int n;  // of the 8, how many are the tensor's
};

template <typename P, bool kEight>
__device__ __forceinline__ Place<P> place_of(const Tensor& t, i64 block, int lane) {
  const i64 i = block * kBlock + lane * kPer, left = t.n - i;
  constexpr int kSize = kEight ? 1 : 4;
  return {static_cast<P*>(t.p) + i, static_cast<char*>(t.m) + i * kSize, static_cast<char*>(t.v) + i * kSize,
          t.ms + block, t.vs + block, t.first_block * kBlock + i, left < 0 ? 0 : left < 8 ? static_cast<int>(left) : 8};
}

// The step of a thread's 8 elements: their values, with the states' codes not scaled yet
// (scales ms, vs).
template <typename P, bool kEight, bool kWide>
__device__ __forceinline__ void step8(const Place<P>& at, const Options& o, const Scalars& s, int ms, int vs,
                                      float (&p)[8], const float (&g)[8], float (&m)[8], float (&v)[8]) {
  constexpr bool kRandom = kEight || sizeof(P) == 2;
  float b1 = o.b1, b2 = o.b2;
  if constexpr (kEight) {  // the scale is a power of two: exact in the factor
    b1 *= scale_of(ms);
    b2 *= scale_of(vs);
  }
  const Two c1 = two(o.c1, o.c1), clip = two(s.clip, s.clip), c2 = two(o.c2, o.c2), d1 = two(b1, b1), d2 = two(b2, b2),
            keep = two(s.keep, s.keep);
  float nan = 0.0f;  // NaN where a parameter is after the step
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const Two q = mul(two(g[e], g[e + 1]), clip), mm = two(m[e], m[e + 1]), vv = two(v[e], v[e + 1]);
    if constexpr (kEight) {
      // Every product rounded, as the formula is written: which way a state's code goes is
      // then a matter of the formula, and not of how it was compiled.
      sum(mul(mm, d1), mul(q, c1), m[e], m[e + 1]);
      sum(mul(vv, d2), mul(mul(q, q), c2), v[e], v[e + 1]);
    } else {
      split(fma2(mm, d1, mul(q, c1)), m[e], m[e + 1]);
      split(fma2(vv, d2, mul(mul(q, q), c2)), v[e], v[e + 1]);
    }
    split(mul(two(p[e], p[e + 1]), keep), p[e], p[e + 1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float u = __fdividef(m[e + h], fmaf(sqrt_fast(v[e + h]), s.root, o.eps));
      p[e + h] = fmaf(-s.step_size, u, p[e + h]);
    }
    if constexpr (sizeof(P) == 2) nan = max_nan(nan, p[e], p[e + 1]);
  }
  uint32_t x[8];  // the mix before its last shift, x ^= x >> 16
  if constexpr (kRandom) {
    // The number is a multiple of 8, so element e's differs in the last three bits only: the
    // mix's first shift is the same for all eight.
    uint32_t n = static_cast<uint32_t>(at.number) ^ (s.key + static_cast<uint32_t>(at.number >> 32) * 0x9e3779b9u);
    n ^= n >> 16;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = mix_middle(n ^ e);
  }
  if constexpr (sizeof(P) == 2) {
    if (__any_sync(kFull, isnan(nan))) {  // NaN stays what it is, as infinities do below
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!isnan(p[e])) p[e] = __uint_as_float(__float_as_uint(p[e]) + random_p(x[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = __uint_as_float(__float_as_uint(p[e]) + random_p(x[e]));
    }
  }
  store8<kWide>(at.p, at.n, p);
  if constexpr (kEight) {
    float top_m = warp_largest<true>(m), top_v = warp_largest<false>(v);
    const bool rare = !(top_m < INFINITY && top_v < INFINITY);
    if (rare) {
      top_m = warp_largest_finite(m);
      top_v = warp_largest_finite(v);
    }
    const int mb = scale_byte(top_m), vb = scale_byte(top_v);
    const float mi = inverse_of(mb), vi = inverse_of(vb);
    const Two mi2 = two(mi, mi), vi2 = two(vi, vi);
    float cm[8], cv[8], low = 448.0f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      split(mul(two(m[e], m[e + 1]), mi2), cm[e], cm[e + 1]);
      split(mul(two(v[e], v[e + 1]), vi2), cv[e], cv[e + 1]);
      low = min3(low, cv[e], cv[e + 1]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t high = x[e] >> 16;
      const float q = round_e4m3(fabsf(cm[e]), ((x[e] ^ high) & 0xffffu) * 16u + 8u);
      cm[e] = __uint_as_float(__float_as_uint(q) | (__float_as_uint(cm[e]) & 0x80000000u));
      cv[e] = round_e4m3(cv[e], ((x[e] >> 12) & 0xffff0u) | 8u);
    }
    if (low < 0.001953125f) {  // 2^-9: a second moment above 0 does not become 0
#pragma unroll
      for (int e = 0; e < 8; ++e) cv[e] = v[e] > 0.0f ? fmaxf(cv[e], 0.001953125f) : cv[e];
    }
    if (rare) {  // infinities and NaN become NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(fabsf(m[e]) < INFINITY)) cm[e] = __uint_as_float(0x7fc00000u);
        if (!(v[e] < INFINITY)) cv[e] = __uint_as_float(0x7fc00000u);
      }
    }
    store_codes<kWide>(static_cast<uint8_t*>(at.m), at.n, cm);
    store_codes<kWide>(static_cast<uint8_t*>(at.v), at.n, cv);
    if ((threadIdx.x & 31) == 0) {
      *at.ms = static_cast<uint8_t>(mb);
      *at.vs = static_cast<uint8_t>(vb);
    }
  } else {
    store8<kWide>(static_cast<float*>(at.m), at.n, m);
    store8<kWide>(static_cast<float*>(at.v), at.n, v);
  }
}

// States in 32 bits: 8 elements of everything straight into registers.
template <typename P, typename G, int kMost>
__global__ void __launch_bounds__(kThreads)
    adamw_kernel(const __grid_constant__ Tensors<kMost> a, const __grid_constant__ Options o, const Scalars* scalars) {
  const Scalars s = *scalars;
  for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const Tensor& t = a.t[find(a, tile)];
    const i64 first = (static_cast<i64>(tile - t.first_tile) * kWarps + (threadIdx.x >> 5)) * a.per_warp;
    for (int u = 0; u < a.per_warp; ++u) {
      const i64 block = first + u;
      if (block * kBlock >= t.n) break;  // the whole warp
      const Place<P> at = place_of<P, false>(t, block, threadIdx.x & 31);
      const G* const grad = static_cast<const G*>(t.g) + (at.p - static_cast<const P*>(t.p));
      float p[8], g[8], m[8], v[8];
      if (t.wide && (block + 1) * kBlock <= t.n) {
        load8<true>(at.p, 8, p);
        load8<true>(grad, 8, g);
        load8<true>(static_cast<const float*>(at.m), 8, m);
        load8<true>(static_cast<const float*>(at.v), 8, v);
        step8<P, false, true>(at, o, s, 0, 0, p, g, m, v);
      } else {
        load8<false>(at.p, at.n, p);
        load8<false>(grad, at.n, g);
        load8<false>(static_cast<const float*>(at.m), at.n, m);
        load8<false>(static_cast<const float*>(at.v), at.n, v);
        step8<P, false, false>(at, o, s, 0, 0, p, g, m, v);
      }
    }
  }
}

// A block that is not whole, or of a tensor that is not aligned; a call of its own, so that
// its registers are no one else's.
template <typename P, typename G>
__device__ __noinline__ void step8_direct(const Tensor& t, const Options& o, const Scalars* scalars, i64 block, int ms,
                                          int vs) {
  const Scalars s = *scalars;
  const Place<P> at = place_of<P, true>(t, block, threadIdx.x & 31);
  float p[8], g[8], m[8], v[8];
  load8<false>(at.p, at.n, p);
  load8<false>(static_cast<const G*>(t.g) + (at.p - static_cast<const P*>(t.p)), at.n, g);
  load_codes<false>(static_cast<const uint8_t*>(at.m), at.n, m);
  load_codes<false>(static_cast<const uint8_t*>(at.v), at.n, v);
  step8<P, true, false>(at, o, s, ms, vs, p, g, m, v);
}

// States in 8 bits: some 70 instructions an element leave few registers for loads in flight,
// so a warp's blocks are copied to shared memory ahead of the arithmetic, kDepth of them
// (20 to 32 bytes a thread are spilled all the same).
// bf16 parameters and gradients are bound by the instructions (a step of 276 million of
// them 659 us, 4.2 TB/s); fp32 ones by memory (71 million, with the norm's reading 233 us,
// 6.0 TB/s).  Two, three and four blocks an SM: 661, 625 and 707 us (bf16, before the
// products were rounded each).
template <typename P, typename G>
struct Stage {
  static constexpr int kP = kBlock * sizeof(P), kG = kBlock * sizeof(G), kBytes = kP + kG + 2 * kBlock;
  static constexpr int kDepth = kBytes <= 1536 ? 3 : 2;
};

__device__ __forceinline__ void copy16(char* to, const void* from) {
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
}

template <typename P, typename G, int kMost>
__global__ void __launch_bounds__(kThreads, 3)
    adamw8_kernel(const __grid_constant__ Tensors<kMost> a, const __grid_constant__ Options o, const Scalars* scalars) {
  using S = Stage<P, G>;
  __shared__ __align__(16) char shared[kWarps][S::kDepth][S::kBytes];
  const Scalars s = *scalars;
  const int lane = threadIdx.x & 31;
  char(*const own)[S::kBytes] = shared[threadIdx.x >> 5];
  for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const Tensor& t = a.t[find(a, tile)];
    const i64 first = (static_cast<i64>(tile - t.first_tile) * kWarps + (threadIdx.x >> 5)) * a.per_warp;
    const i64 blocks = (t.n + kBlock - 1) / kBlock;
    const int count = blocks <= first ? 0 : blocks - first < a.per_warp ? static_cast<int>(blocks - first) : a.per_warp;
    // Blocks that are whole and aligned, from the first on.
    const i64 whole = t.wide ? t.n / kBlock - first : 0;
    const int staged = whole <= 0 ? 0 : whole < count ? static_cast<int>(whole) : count;
    int ms = 0, vs = 0;  // lane u: block u's scales
    if (lane < count) {
      ms = t.ms[first + lane];
      vs = t.vs[first + lane];
    }
    const char* const p0 = static_cast<const char*>(t.p) + first * S::kP + 16 * lane;
    const char* const g0 = static_cast<const char*>(t.g) + first * S::kG + 16 * lane;
    // The lower half of the warp copies m's codes, the upper v's.
    const char* const c0 = static_cast<const char*>(lane < 16 ? t.m : t.v) + first * kBlock + 16 * (lane & 15);
    const auto fetch = [&](int u, char* to) {
      if (u < staged) {
#pragma unroll
        for (int k = 0; k < S::kP; k += 512) copy16(to + k + 16 * lane, p0 + u * S::kP + k);
#pragma unroll
        for (int k = 0; k < S::kG; k += 512) copy16(to + S::kP + k + 16 * lane, g0 + u * S::kG + k);
        copy16(to + S::kP + S::kG + 16 * lane, c0 + u * kBlock);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int u = 0; u < S::kDepth; ++u) fetch(u, own[u]);
    Place<P> at = place_of<P, true>(t, first, lane);
    int slot = 0;
    for (int u = 0; u < count; ++u) {
      const int bm = __shfl_sync(kFull, ms, u), bv = __shfl_sync(kFull, vs, u);
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kDepth - 1) : "memory");
      __syncwarp();
      if (u < staged) {
        float p[8], g[8], m[8], v[8];
        const char* const from = own[slot];
        load8<true>(reinterpret_cast<const P*>(from) + lane * kPer, 8, p);
        load8<true>(reinterpret_cast<const G*>(from + S::kP) + lane * kPer, 8, g);
        const uint2 cm = *reinterpret_cast<const uint2*>(from + S::kP + S::kG + 8 * lane);
        const uint2 cv = *reinterpret_cast<const uint2*>(from + S::kP + S::kG + kBlock + 8 * lane);
        decode(cm.x, cm.y, m);
        decode(cv.x, cv.y, v);
        __syncwarp();  // the slot is read
        fetch(u + S::kDepth, own[slot]);
        step8<P, true, true>(at, o, s, bm, bv, p, g, m, v);
      } else {
        fetch(u + S::kDepth, own[slot]);
        step8_direct<P, G>(t, o, scalars, first + u, bm, bv);
      }
      at.p += kBlock;
      at.m = static_cast<char*>(at.m) + kBlock;
      at.v = static_cast<char*>(at.v) + kBlock;
      ++at.ms;
      ++at.vs;
      at.number += kBlock;
      slot = slot + 1 == S::kDepth ? 0 : slot + 1;
    }
  }
}

// Sums of the gradients' squares, in 64 bits from the squares on (exact there), so that the
// norm, and with it every rounding of a clipped step, does not hang on the order.  71 million
// fp32 gradients 57 us, 5.0 TB/s (44 us in 32 bits).
template <typename G, int kMost>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Tensors<kMost> a, double* partial) {
  __shared__ double part[kThreads / 32];
  double sum = 0.0;
  for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const Tensor& t = a.t[find(a, tile)];
    const i64 first = (static_cast<i64>(tile - t.first_tile) * kWarps + (threadIdx.x >> 5)) * a.per_warp;
    const G* const at = static_cast<const G*>(t.g);
    const auto add = [&](const float (&g)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fma(static_cast<double>(g[e]), static_cast<double>(g[e]), sum);
    };
    const int lane = threadIdx.x & 31;
    if (t.wide && a.per_warp == kBlocks && (first + kBlocks) * kBlock <= t.n) {  // all loads at once
      float g[kBlocks][8];
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) load8<true>(at + (first + u) * kBlock + lane * kPer, 8, g[u]);
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) add(g[u]);
    } else {
      for (int u = 0; u < a.per_warp; ++u) {
        const i64 i = (first + u) * kBlock + lane * kPer;
        float g[8];
        if (t.wide && i + kPer <= t.n) load8<true>(at + i, 8, g);
        else load8<false>(at + i, t.n - i < 8 ? static_cast<int>(t.n - i) : 8, g);
        add(g);
      }
    }
  }
  sum = sum_warp(sum);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int k = 0; k < kThreads / 32; ++k) sum += part[k];
    partial[blockIdx.x] = sum;
  }
}

// Counts the step and writes its scalars; the partial sums are added in order.
__global__ void __launch_bounds__(kThreads) prepare_kernel(const Options o, const double* partial, int partials,
                                                           i64* step, Scalars* scalars, float* norm) {
  __shared__ double part[kThreads / 32];
  double sum = 0.0;
  for (int b = threadIdx.x; b < partials; b += kThreads) sum += partial[b];
  sum = sum_warp(sum);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  Scalars s;
  s.clip = 1.0f;
  if (partials > 0) {
    sum = 0.0;
    for (int k = 0; k < kThreads / 32; ++k) sum += part[k];
    const float n = static_cast<float>(sqrt(sum));
    const float c = o.max_norm / (n + 1e-6f);
    s.clip = c > 1.0f ? 1.0f : c;  // NaN stays NaN
    *norm = n;
  }
  const i64 t = *step + 1;
  *step = t;
  const double lr = o.lr_dev ? static_cast<double>(*o.lr_dev) : o.lr;
  s.step_size = static_cast<float>(lr / (1.0 - pow(o.beta1, static_cast<double>(t))));
  s.keep = static_cast<float>(1.0 - lr * o.decay);
  s.root = static_cast<float>(1.0 / sqrt(1.0 - pow(o.beta2, static_cast<double>(t))));
  s.key = mix(o.seed + static_cast<uint32_t>(t) * 0x9e3779b9u);
  *scalars = s;
}

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? CUGO_B200_OK : CUGO_B200_ERR_LAUNCH;
}

// The status of a call that returns its error.  The runtime keeps that until it is asked for
// the last one: taken here, it is not the next call's.
inline int status(cudaError_t rc) {
  if (rc == cudaSuccess) return CUGO_B200_OK;
  cudaGetLastError();
  return CUGO_B200_ERR_LAUNCH;
}

// The call's tensors, host arrays of `count`.
struct Lists {
  void* const* p;
  const void* const* g;
  void* const *m, *const *v, *const *ms, *const *vs;
  const int64_t* n;
  i64 count;
};

// Tensors first .. of the lists that fit one launch, empty ones left out; returns the
// number of the first one that did not, or -1 where they have too many tiles.
template <int kMost>
i64 fill(const Lists& l, i64 first, int per_warp, i64& blocks_before, Tensors<kMost>& a) {
  a.count = 0;
  a.per_warp = per_warp;
  i64 tiles = 0, k = first;
  for (; k < l.count && a.count < kMost; ++k) {
    if (l.n[k] == 0) continue;
    const i64 blocks = (l.n[k] - 1) / kBlock + 1, more = (blocks - 1) / (kWarps * per_warp) + 1;
    if (tiles + more > INT32_MAX) return -1;
    Tensor& t = a.t[a.count++];
    const bool wide = aligned(l.p[k], 16) && aligned(l.g[k], 16) && aligned(l.m[k], 16) && aligned(l.v[k], 16);
    t = {l.p[k], l.g[k], l.m[k], l.v[k], l.ms ? static_cast<uint8_t*>(l.ms[k]) : nullptr,
         l.vs ? static_cast<uint8_t*>(l.vs[k]) : nullptr, l.n[k], wide, static_cast<int>(tiles), blocks_before};
    tiles += more;
    blocks_before += blocks;
  }
  a.tiles = static_cast<int>(tiles);
  return k;
}

template <typename P, typename G, int kMost>
int launch_sized(const Lists& l, bool eight, const Options& o, double* partial, int64_t* step, Scalars* scalars,
                 float* norm, cudaStream_t stream) {
  // Four blocks a warp share the search for their tensor and keep copies in flight; where
  // that leaves an SM less than two rounds of tiles, one, for balance.
  i64 total = 0;
  for (i64 k = 0; k < l.count; ++k) total += l.n[k] / kBlock;
  const int per_warp = total >= static_cast<i64>(kSms) * 4 * kWarps * kBlocks * 2 ? kBlocks : 1;
  Tensors<kMost> a;
  int partials = 0;
  if (norm) {
    i64 before = 0;
    for (i64 k = 0; k < l.count;) {
      k = fill<kMost>(l, k, per_warp, before, a);
      if (k < 0) return CUGO_B200_ERR_CAPACITY;
      if (a.tiles == 0) break;
      const int blocks = a.tiles < kNormBlocks ? a.tiles : kNormBlocks;
      norm_kernel<G, kMost><<<blocks, kThreads, 0, stream>>>(a, partial + partials);
      partials += blocks;
    }
    if (partials == 0) {  // no elements at all: a norm of 0
      if (int rc = status(cudaMemsetAsync(partial, 0, sizeof(double), stream))) return rc;
      partials = 1;
    }
  }
  prepare_kernel<<<1, kThreads, 0, stream>>>(o, partial, partials, step, scalars, norm);
  i64 before = 0;
  for (i64 k = 0; k < l.count;) {
    k = fill<kMost>(l, k, per_warp, before, a);
    if (k < 0) return CUGO_B200_ERR_CAPACITY;
    if (a.tiles == 0) break;
    const int blocks = a.tiles < kSms * 64 ? a.tiles : kSms * 64;
    if (eight) adamw8_kernel<P, G, kMost><<<blocks, kThreads, 0, stream>>>(a, o, scalars);
    else adamw_kernel<P, G, kMost><<<blocks, kThreads, 0, stream>>>(a, o, scalars);
  }
  return launch_status();
}

template <typename P, typename G>
int launch(const Lists& l, bool eight, const Options& o, double* partial, int64_t* step, Scalars* scalars,
           float* norm, cudaStream_t stream) {
  // The parameters of a launch are copied to the device with it: few tensors, few bytes.
  return l.count <= kFewTensors ? launch_sized<P, G, kFewTensors>(l, eight, o, partial, step, scalars, norm, stream)
                                : launch_sized<P, G, kMostTensors>(l, eight, o, partial, step, scalars, norm, stream);
}

// Launches that `count` tensors may take.
inline i64 launches_of(i64 count) { return count <= kFewTensors ? 1 : (count + kMostTensors - 1) / kMostTensors; }

}  // namespace

extern "C" {

int64_t cugo_b200_adamw_scratch_bytes(int64_t count) {
  if (count < 0) return 0;
  return 64 + launches_of(count) * kNormBlocks * static_cast<int64_t>(sizeof(double));
}

int cugo_b200_adamw(int64_t count, void* const* params, const void* const* grads, void* const* exp_avgs,
                    void* const* exp_avg_sqs, void* const* exp_avg_scales, void* const* exp_avg_sq_scales,
                    const int64_t* sizes, int32_t param_dtype, int32_t grad_dtype, int32_t state_bits, double lr,
                    const float* lr_dev, double beta1, double beta2, double eps, double weight_decay,
                    double max_norm, uint32_t seed, int64_t* step, float* norm, void* scratch,
                    int64_t scratch_bytes, cudaStream_t stream) {
  if (count < 0 || (param_dtype != 0 && param_dtype != 1) || (grad_dtype != 0 && grad_dtype != 1) ||
      (state_bits != 32 && state_bits != 8) || !step)
    return CUGO_B200_ERR_ARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) ||
      (!lr_dev && !(lr >= 0.0)) || (norm && !(max_norm >= 0.0)))
    return CUGO_B200_ERR_ARG;
  if (count > 0 && (!params || !grads || !exp_avgs || !exp_avg_sqs || !sizes)) return CUGO_B200_ERR_ARG;
  const bool eight = state_bits == 8;
  if (eight && count > 0 && (!exp_avg_scales || !exp_avg_sq_scales)) return CUGO_B200_ERR_ARG;
  const int p_bytes = param_dtype == 0 ? 4 : 2, g_bytes = grad_dtype == 0 ? 4 : 2;
  for (int64_t k = 0; k < count; ++k) {
    if (sizes[k] < 0) return CUGO_B200_ERR_ARG;
    if (sizes[k] == 0) continue;
    if (!params[k] || !grads[k] || !exp_avgs[k] || !exp_avg_sqs[k] ||
        (eight && (!exp_avg_scales[k] || !exp_avg_sq_scales[k])))
      return CUGO_B200_ERR_ARG;
    if (!aligned(params[k], p_bytes) || !aligned(grads[k], g_bytes) ||
        (!eight && (!aligned(exp_avgs[k], 4) || !aligned(exp_avg_sqs[k], 4))))
      return CUGO_B200_ERR_ALIGN;
  }
  if (!aligned(step, 8) || !aligned(scratch, 8)) return CUGO_B200_ERR_ALIGN;
  if (!scratch || scratch_bytes < cugo_b200_adamw_scratch_bytes(count)) return CUGO_B200_ERR_CAPACITY;
  Options o{};
  o.lr = lr;
  o.lr_dev = lr_dev;
  o.beta1 = beta1;
  o.beta2 = beta2;
  o.decay = weight_decay;
  o.b1 = static_cast<float>(beta1);
  o.c1 = static_cast<float>(1.0 - beta1);
  o.b2 = static_cast<float>(beta2);
  o.c2 = static_cast<float>(1.0 - beta2);
  o.eps = static_cast<float>(eps);
  o.max_norm = static_cast<float>(max_norm);
  o.seed = seed;
  const Lists l{params, grads, exp_avgs, exp_avg_sqs, eight ? exp_avg_scales : nullptr,
                eight ? exp_avg_sq_scales : nullptr, sizes, count};
  Scalars* scalars = static_cast<Scalars*>(scratch);
  double* partial = reinterpret_cast<double*>(static_cast<char*>(scratch) + 64);
  if (param_dtype == 0)
    return grad_dtype == 0 ? launch<float, float>(l, eight, o, partial, step, scalars, norm, stream)
                           : launch<float, __nv_bfloat16>(l, eight, o, partial, step, scalars, norm, stream);
  return grad_dtype == 0 ? launch<__nv_bfloat16, float>(l, eight, o, partial, step, scalars, norm, stream)
                         : launch<__nv_bfloat16, __nv_bfloat16>(l, eight, o, partial, step, scalars, norm, stream);
}

}  // extern "C"
