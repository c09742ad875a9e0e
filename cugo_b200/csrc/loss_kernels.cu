// Losses over rows of logits, forward and backward, and their C ABI
// (include/cugo_b200.h): the log-probability of a given action and the entropy of its
// masked categorical (action_logp), the clipped policy loss with an entropy bonus and a
// KL term (policy_loss), and the preference loss over pairs of sequences
// (preference_pairs, on action_logp's rows).
//
// Mathematics of one row.  With x the logits, all sums run in base 2 and relative to
// M = ceil(max x log2(e)), a whole number:
//   y_j = x_j log2(e) - M   (one FMA; its rounding is the only one, so p_j keeps fp32's
//                            relative accuracy however large x is)
//   s = sum 2^y_j,  t = sum 2^y_j y_j,  log2 p_j = y_j - log2 s,  H = ln 2 (log2 s - t/s)
// Parts of a row that have other maxima are brought together by powers of two, without a
// rounding.
// A reference row z_j (M', s') adds u = sum 2^y_j (y_j - z_j):
//   KL(p|q) = ln 2 (u/s - log2 s + log2 s'),
// which is infinite where the reference masks an entry that the row does not: such an entry
// is looked for, its p may be 0 in 32 bits.
// Every gradient wanted here is, with 1 at the taken action a,
//   d_j = hot [j = a] + 2^y_j (c_0 + c_1 y_j + c_2 (y_j - z_j)),
// so a row needs its sums, four coefficients and one more look at its entries.
//
// An illegal entry counts as -2^30, and so does every entry below that (-inf, -1e30, a mask
// of the type's lowest value): its 2^y is 0 beside any other entry and every product
// stays finite, so no entry needs a branch.  (M, as a float, is off by at most 2^-24 of
// itself, the same for the whole row: below 2^31 that shifts y by less than 128, which the
// sums bear.  The bound is a power of two, so that its own product is exact.)  What
// stands in an illegal place (NaN, infinities) is never used; NaN in a legal place stays
// NaN.  Sums over rows are taken in 64 bits, per warp or block, and
// added over the blocks in order: the same result on every run.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/cugo_b200.h"

namespace {

namespace cg = cooperative_groups;
using i64 = int64_t;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMasked = -1073741824.0f;  // -2^30
constexpr float kMasked2 = kMasked * kLog2e;  // a maximum of masked entries only
constexpr int kSms = 148;
constexpr int kSums = 6;   // policy, entropy, KL, KL to the old policy, clipped, used
constexpr int kStats = 7;  // the loss, then the means of the six

enum Type : int { kFp32 = 0, kBf16 = 1, kFp16 = 2 };

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A maximum in base-2 units, up to a whole number.
__device__ __forceinline__ float base2(float x) { return ceilf(x * kLog2e); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

// Two floats in one register pair, an instruction for both.
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
__device__ __forceinline__ Two add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float both(Two t) {
  float a, b;
  split(t, a, b);
  return a + b;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <int kType>
using Stored = std::conditional_t<kType == kFp32, float, std::conditional_t<kType == kBf16, __nv_bfloat16, __half>>;

template <int kType>
__device__ __forceinline__ void store_one(void* base, i64 at, float g) {
  if constexpr (kType == kFp32) static_cast<float*>(base)[at] = g;
  else if constexpr (kType == kBf16) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(g);
  else static_cast<__half*>(base)[at] = __float2half_rn(g);
}

// N values at element `at`, not read again soon; `wide`: that address is a multiple of the
// N values' bytes, or of 16.
template <int kType, int N>
__device__ __forceinline__ void store_grad(void* base, i64 at, const float (&g)[N], bool wide) {
  if (!wide) {
#pragma unroll
    for (int e = 0; e < N; ++e) store_one<kType>(base, at + e, g[e]);
    return;
  }
  if constexpr (kType == kFp32) {
    float* d = static_cast<float*>(base) + at;
#pragma unroll
    for (int e = 0; e < N; e += 4)
      __stcs(reinterpret_cast<float4*>(d + e), make_float4(g[e], g[e + 1], g[e + 2], g[e + 3]));
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      if constexpr (kType == kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(g[e], g[e + 1]);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(g[e], g[e + 1]);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    uint16_t* d = static_cast<uint16_t*>(base) + at;
    if constexpr (N == 8) __stcs(reinterpret_cast<uint4*>(d), make_uint4(w[0], w[1], w[2], w[3]));
    else __stcs(reinterpret_cast<uint2*>(d), make_uint2(w[0], w[1]));
  }
}

// f with the type as a constant: one branch around a loop instead of one inside.
template <typename F>
__device__ __forceinline__ void with_type(int type, F f) {
  if (type == kFp32) f(std::integral_constant<int, kFp32>{});
  else if (type == kBf16) f(std::integral_constant<int, kBf16>{});
  else f(std::integral_constant<int, kFp16>{});
}

__host__ __device__ __forceinline__ int type_bytes(int type) { return type == kFp32 ? 4 : 2; }

// What a row's gradient is made of (d_j above; the scale and 1 / s are in it).
struct Coefs {
  float hot, c0, c1, c2;
};

// The sums of a row, or of a part of one.
struct Sums {
  float m, s, t;    // M, sum 2^y, sum 2^y y
  // The reference's, and sum 2^y (y - z).  sr's sign is set where the reference masks an entry
  // that the row does not.
  float mr, sr, u;
};

__device__ __forceinline__ bool infinite(float sr) { return __float_as_int(sr) < 0; }
__device__ __forceinline__ float marked(float sr, bool infinite) { return infinite ? -sr : sr; }

__device__ __forceinline__ Sums no_sums() { return {kMasked2, 0.0f, 0.0f, kMasked2, 0.0f, 0.0f}; }

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float sum_warp(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;  // the same bits in every lane: each addition has the same two operands in both
}

// A warp's 32 parts joined: every part is brought to the warp's maximum once.
template <bool kRef>
__device__ __forceinline__ Sums join_warp(Sums v) {
  Sums r;
  r.m = warp_max_nan(v.m);
  const float d = v.m - r.m, f = exp2_fast(d);
  r.t = sum_warp(f * (v.t + d * v.s));
  r.s = sum_warp(f * v.s);
  r.mr = kMasked2;
  r.sr = r.u = 0.0f;
  if constexpr (kRef) {
    r.mr = warp_max_nan(v.mr);
    const float dr = v.mr - r.mr;
    r.sr = marked(sum_warp(fabsf(v.sr) * exp2_fast(dr)), __any_sync(kFull, infinite(v.sr)));
    r.u = sum_warp(f * (v.u + (d - dr) * v.s));
  }
  return r;
}

__device__ __forceinline__ double sum_warp(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Over the kLanes lanes that share a row (all lanes of the warp take part).
template <int kLanes>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

template <int kLanes>
__device__ __forceinline__ float max_lanes(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

struct Rows {
  const void* logits;
  i64 ld;
  const void* ref;    // or null
  i64 ldr;
  const bool* legal;  // or null
  i64 ldm;
  const i64* actions;
  const float* weight;  // or null
  i64 rows;
  int vocab;
};

// action_logp's outputs (any may be null).
struct Score {
  float* logp;
  float* entropy;
  float2* lse;   // {maximum, log2 of the sum}, in base-2 units; {0, +inf}: the row does not count
  float* zeros;  // [rows] written as 0 (the coefficients that preference_pairs fills in)
};

struct Policy {
  const float* logp_old;
  const float* adv;
  const float* ref_logp;  // or null
  float low, high, kl_coef, entropy_coef;
  const float *kl_coef_dev, *entropy_coef_dev;  // or null; multiply the two
  float denominator;            // not 0: given; 0: *denominator_dev, the sum of the weights, or the rows
  const float* denominator_dev;
  const double* weight_sums;    // partial sums of the weights, or null (sum them here)
  int n_weight_sums;
  float grad_scale;
  const float* grad_scale_dev;  // or null; multiplies grad_scale
  void* dlogits;                // or null
  i64 ldd;
  int dtype, width;             // columns vocab .. width - 1 are written as 0
  float* logp;                  // or null
  double* partial;              // [blocks][kSums], or null: no means wanted
};

// What policy_loss reads of a row beside its logits.
struct RowInputs {
  i64 action;
  float weight, logp_old, adv, ref_logp;
};

template <bool kPolicy>
__device__ __forceinline__ RowInputs row_inputs(const Rows& r, const Policy& a, i64 row) {
  RowInputs in;
  in.action = r.actions[row];
  in.weight = r.weight ? r.weight[row] : 1.0f;
  in.logp_old = in.adv = in.ref_logp = 0.0f;
  if constexpr (kPolicy) {
    in.logp_old = a.logp_old[row];
    in.adv = a.adv[row];
    if (a.ref_logp) in.ref_logp = a.ref_logp[row];
  }
  return in;
}

// log2(s) of a positive s as a whole number and the logarithm of what lies in [3/4, 3/2):
// each is exact to its own size, which their sum is not.
struct Log2 {
  float whole, part;
};

__device__ __forceinline__ Log2 split_log2(float s) {
  const int bits = __float_as_int(s), k = (bits - 0x3f400000) >> 23;
  return {static_cast<float>(k), log2f(__int_as_float(bits - (k << 23)))};
}

// Whether a row's whole weight is at its entry x_a: in 32 bits (all), and of the only open
// entry, whose products are then the row's sums (only).
struct Certain {
  bool all, only;
};

__device__ __forceinline__ Certain certain(float x_a, const Sums& v) {
  const float y = fmaf(x_a, kLog2e, -v.m), e = exp2_fast(y);
  return {e >= v.s, e >= v.s && v.t == e * y};
}

// log p of an entry x_a: x_a - ln 2 (M + log2 s), the large terms in 64 bits and one rounding
// at the end (log p of long sequences are added up, so what is alike in every row counts).
// For the same reason two small things that are known come out again: kLog2e is log2(e)
// (1 - kLow), which makes log Z less by that share of the mean logit, and 2^y as the
// hardware has it is 3.0e-8 of itself too small in the mean (over [-24, 0), by value).  Never
// above 0, and 0 where nothing else has weight, which no mean knows about.
__device__ __forceinline__ float log_prob(float x_a, const Sums& v, const Log2& log_s, float mean_y, bool all) {
  constexpr double kLn2d = 0.693147180559945309, kLow = 1.0 - kLn2d * kLog2e, kHardware = 3.0e-8;
  const double m = v.m;
  const double log_z = kLn2d * (m + log_s.whole + log_s.part + kLow * (m + mean_y)) + kHardware;
  const float log_p = static_cast<float>(x_a - log_z);
  return all || log_p > 0.0f ? 0.0f : log_p;
}

__device__ __forceinline__ float entropy_of(const Log2& log_s, float mean_y, bool only) {
  const float h = kLn2 * (log_s.whole + (log_s.part - mean_y));
  return only || h < 0.0f ? 0.0f : h;
}

// A row's outputs in action_logp.
__device__ __forceinline__ void store_score(const Score& o, i64 row, bool used, const Sums& v, float x_a) {
  const Log2 log_s = split_log2(v.s);
  const float mean_y = __fdividef(v.t, v.s);
  const Certain sure = certain(x_a, v);
  if (o.logp) o.logp[row] = used ? log_prob(x_a, v, log_s, mean_y, sure.all) : 0.0f;
  if (o.entropy) o.entropy[row] = used ? entropy_of(log_s, mean_y, sure.only) : 0.0f;
  if (o.lse) o.lse[row] = used ? make_float2(v.m, log_s.whole + log_s.part) : make_float2(0.0f, INFINITY);
  if (o.zeros) o.zeros[row] = 0.0f;
}

// What a row adds to the means, before its weight.
struct Terms {
  float v[kSums];
  __device__ __forceinline__ void add_to(double* acc, float w) const {
#pragma unroll
    for (int k = 0; k < kSums; ++k) acc[k] += static_cast<double>(w) * v[k];
  }
};

// A row's loss terms and its gradient's coefficients, from its sums and its action's entry.
template <bool kRef>
__device__ __forceinline__ Coefs policy_row(const Policy& a, const RowInputs& in, const Sums& v, float x_a,
                                            float scale, Terms& terms, float& logp) {
  const Log2 log_s = split_log2(v.s);
  const float inv_s = 1.0f / v.s, mean_y = v.t * inv_s, w = in.weight;
  const Certain sure = certain(x_a, v);
  logp = log_prob(x_a, v, log_s, mean_y, sure.all);
  const float entropy = entropy_of(log_s, mean_y, sure.only);
  const float log_ratio = logp - in.logp_old;
  const float ratio = expf(log_ratio), adv = in.adv;
  const float bounded = ratio < a.low ? a.low : ratio > a.high ? a.high : ratio;
  // min(r A, clamp(r) A); where the two are equal the ratio still moves the loss.
  const bool moves = !(ratio * adv > bounded * adv);
  const float gain = moves ? ratio * adv : bounded * adv;
  float g = moves ? -ratio * adv : 0.0f;
  float kl = 0.0f, mean_d = 0.0f, c2 = 0.0f;
  if constexpr (kRef) {
    mean_d = v.u * inv_s;
    kl = kLn2 * (mean_d - (log_s.whole + log_s.part) + log2f(v.sr));
    c2 = a.kl_coef * kLn2;
    if (c2 == 0.0f) mean_d = 0.0f;  // which may be infinite
  } else if (a.ref_logp) {
    const float d = in.ref_logp - logp, e = expm1f(d);
    kl = e - d;
    g -= a.kl_coef * e;
  }
  // lp + H = ln 2 (y - mean y), lp - lq - KL = ln 2 ((y - z) - mean (y - z)).
  const float c1 = a.entropy_coef * kLn2, k = scale * w, ks = k * inv_s;
  Coefs c;
  c.hot = k * g;
  c.c0 = ks * (-g - c1 * mean_y - c2 * mean_d);
  c.c1 = ks * c1;
  c.c2 = ks * c2;
  terms = {{-gain, entropy, kl, expm1f(log_ratio) - log_ratio, ratio < a.low || ratio > a.high ? 1.0f : 0.0f, 1.0f}};
  return c;
}

// The same with its device-resident coefficients read (a captured graph keeps their
// addresses).
__device__ __forceinline__ Policy resolved(Policy a) {
  if (a.kl_coef_dev) a.kl_coef *= *a.kl_coef_dev;
  if (a.entropy_coef_dev) a.entropy_coef *= *a.entropy_coef_dev;
  return a;
}

// The denominator of the means: given, the sum of the weights, or the rows.  Every block
// adds the same numbers in the same order.  Uses and synchronises the whole block.
__device__ double block_denominator(const Policy& a, const float* weight, i64 rows) {
  if (a.denominator != 0.0f) return a.denominator;
  if (a.denominator_dev) return *a.denominator_dev;
  if (!weight) return static_cast<double>(rows);
  __shared__ double part[32];
  __shared__ double total;
  double t = 0.0;
  if (a.weight_sums)
    for (int i = threadIdx.x; i < a.n_weight_sums; i += blockDim.x) t += a.weight_sums[i];
  else
    for (i64 i = threadIdx.x; i < rows; i += 8 * blockDim.x) {  // eight loads in flight
      float w[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = i + q * blockDim.x < rows ? weight[i + q * blockDim.x] : 0.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) t += w[q];
    }
  t = sum_warp(t);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (unsigned k = 0; k < blockDim.x / 32; ++k) t += part[k];
    total = t;
  }
  __syncthreads();
  return total;
}

// The scale of every gradient: a batch without weight has no mean, and no gradient.
__device__ __forceinline__ float grad_scale_of(const Policy& a, double denominator) {
  const float g = a.grad_scale * (a.grad_scale_dev ? *a.grad_scale_dev : 1.0f);
  return denominator == 0.0 ? 0.0f : static_cast<float>(g / denominator);
}

// The warps' sums of a block, added in order, into partial[block].
__device__ void store_partial(const Policy& a, const double (&acc)[kSums]) {
  if (!a.partial) return;
  __shared__ double part[32][kSums];
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < kSums; ++k) part[warp][k] = acc[k];
  __syncthreads();
  if (threadIdx.x < kSums) {
    double t = 0.0;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) t += part[w][threadIdx.x];
    a.partial[(i64)blockIdx.x * kSums + threadIdx.x] = t;
  }
}

// ---- short rows: 8, 16 or 32 lanes per row, the row in registers ------------------------
//
// Lane l of a row's kLanes holds entries l, l + kLanes, ..., kPer of them.  A warp takes
// 32 / kLanes consecutive rows: few entries per lane would leave the row's reductions and
// its one logarithm to most of the time.  Rows are copied by 16-byte vectors into the
// warp's own shared memory, the next rows' while these are computed, so the loads are wide
// and in flight however the rows are aligned (a row of 179 fp32 starts at any multiple of 4
// bytes): as one run where they lie one after another (a stride of little more than the
// entries), else each by itself.  A gradient whose rows lie one after another leaves the
// same way.
//
// Bound by instructions, most of them per entry (the mask, two exponentials with a
// reference, the sums, the gradient), the rest a row's reductions and its loss terms.
// 262,144 rows of 179 fp32 with masks: 56 us, 4.3 TB/s (a warp per row that reads in place:
// 267 us); policy loss of 32,768 such rows with the full KL and a bf16 gradient: 23 us,
// 2.9 TB/s, and 3 us for the means.  That one is held at 12 warps an SM by shared memory
// (14.7 KB a warp).  Rows of 385 to 1,024 entries with a reference and a gradient spill 212
// bytes a thread (16,384 rows of 1,000 bf16: 54 us, 1.8 TB/s).

constexpr int kShortWarps = 4;

__device__ __forceinline__ void copy16(void* to, const void* from, int bytes = 16) {
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
}

// Copies a run of rows: the 16-byte granules that hold it, from its first byte's granule
// on (an allocation starts at a granule, so that lies inside); what lies behind its last
// byte is not read.  The run's first byte stands at to + (its address mod 16).  kMost: the
// run's largest number of bytes.
template <int kMost>
__device__ __forceinline__ void copy_run(char* to, const char* from, int bytes, int lane) {
  const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(from)) & 15, total = skip + bytes;
  const int behind = 16 * lane - (total & ~15);  // of whole granules
  from += 16 * lane - skip;
  to += 16 * lane;
#pragma unroll
  for (int k = 0; k < kMost + 15; k += 512)
    if (behind < -k) copy16(to + k, from + k);
  if (total & 15) {  // the last granule, in part: after the whole ones, at the same stride
    const int k = total >> 4 << 4;
    if ((k >> 4 & 31) == lane) copy16(to + k - 16 * lane, from + k - 16 * lane, total & 15);
  }
}

// The warp's shared memory: two stages, one gradient.  Sizes in bytes, multiples of 16.
struct Layout {
  int logits, ref, legal, grad;
  // Row q of a stage stands q pitches behind the first: of a run, at the first row's address
  // mod 16; of rows `apart`, at its own.
  bool apart;
  int pitch, pitch_ref, pitch_legal;
  __host__ __device__ int stage() const { return logits + ref + legal; }
  __host__ __device__ int warp() const { return 2 * stage() + grad; }
};

template <typename V>
__device__ __forceinline__ int skip16(const V* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p)) & 15; }

template <typename T, int kLanes, int kPer, bool kRef, bool kPolicy>
__global__ void __launch_bounds__(32 * kShortWarps, kPolicy ? 4 : 6)
    short_rows_kernel(const Rows r, const Score o, const Policy given, const Layout lay) {
  const Policy a = kPolicy ? resolved(given) : given;
  constexpr int kRows = 32 / kLanes;
  extern __shared__ __align__(16) char shared[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, sub = lane / kLanes;
  const int own = warp * lay.warp(), out = own + 2 * lay.stage();  // offsets in `shared`
  const int vocab = r.vocab;
  float scale = 0.0f;
  double acc[kSums] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  if constexpr (kPolicy) scale = grad_scale_of(a, block_denominator(a, r.weight, r.rows));
  const i64 stride = (i64)gridDim.x * kShortWarps * kRows;
  i64 first = ((i64)blockIdx.x * kShortWarps + warp) * kRows;

  // One mask for all rows stays where the first two turns put it.
  const bool own_masks = r.legal && r.ldm != 0, one_mask = r.legal && r.ldm == 0;

  // Where the rows of this warp's turn begin, and how far its next turn is.
  const T* x_first = static_cast<const T*>(r.logits) + first * r.ld;
  const T* z_first = kRef ? static_cast<const T*>(r.ref) + first * r.ldr : nullptr;
  const bool* m_first = r.legal + first * r.ldm;
  const i64 x_step = stride * r.ld, z_step = kRef ? stride * r.ldr : 0, m_step = stride * r.ldm;
  const auto fetch = [&](i64 row, const T* x, const T* z, const bool* m, int at) {
    constexpr int kGap = kRows > 1 ? 64 : 0, kRow = kLanes * kPer, kSize = sizeof(T);
    constexpr int kRun = kRows * (kRow * kSize + kGap);
    const int n = r.rows - row < kRows ? static_cast<int>(r.rows - row) - 1 : kRows - 1;
    char* const to = shared + own + at * lay.stage();
    const auto from = [](const auto* p) { return reinterpret_cast<const char*>(p); };
    if (!lay.apart) {
      copy_run<kRun>(to, from(x), n * lay.pitch + vocab * kSize, lane);
      if constexpr (kRef) copy_run<kRun>(to + lay.logits, from(z), n * lay.pitch_ref + vocab * kSize, lane);
      if (own_masks)
        copy_run<kRows * (kRow + kGap)>(to + lay.logits + lay.ref, from(m), n * lay.pitch_legal + vocab, lane);
    } else {
#pragma unroll 1
      for (int q = 0; q <= n; ++q) {
        copy_run<kRow * kSize>(to + q * lay.pitch, from(x + q * r.ld), vocab * kSize, lane);
        if constexpr (kRef)
          copy_run<kRow * kSize>(to + lay.logits + q * lay.pitch_ref, from(z + q * r.ldr), vocab * kSize, lane);
        if (own_masks)
          copy_run<kRow>(to + lay.logits + lay.ref + q * lay.pitch_legal, from(m + q * r.ldm), vocab, lane);
      }
    }
    if (one_mask && row < 2 * stride) copy_run<kRow>(to + lay.logits + lay.ref, from(m), vocab, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  RowInputs next;
  if (first < r.rows) {
    fetch(first, x_first, z_first, m_first, 0);
    next = row_inputs<kPolicy>(r, a, first + sub < r.rows ? first + sub : r.rows - 1);
  }
  int at = 0;
  for (; first < r.rows; first += stride, at ^= 1, x_first += x_step, z_first += z_step, m_first += m_step) {
    const RowInputs in = next;
    if (first + stride < r.rows) {
      fetch(first + stride, x_first + x_step, z_first + z_step, m_first + m_step, at ^ 1);
      next = row_inputs<kPolicy>(r, a, first + stride + sub < r.rows ? first + stride + sub : r.rows - 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    const bool real = first + sub < r.rows;
    const int back = real ? sub : static_cast<int>(r.rows - 1 - first);  // the row's place in the run
    const i64 row = first + back;
    const int stage = own + at * lay.stage(), place = lay.apart ? back : 0;
    const T* const x =
        reinterpret_cast<const T*>(shared + stage + back * lay.pitch + skip16(x_first + place * r.ld));
    const T* z_row = nullptr;
    if constexpr (kRef)
      z_row = reinterpret_cast<const T*>(shared + stage + lay.logits + back * lay.pitch_ref +
                                         skip16(z_first + place * r.ldr));
    const bool* const lm = reinterpret_cast<const bool*>(shared + stage + lay.logits + lay.ref + back * lay.pitch_legal +
                                                         skip16(m_first + place * r.ldm));
    bool used = real && in.weight != 0.0f && in.action >= 0 && in.action < vocab;
    const int action = used ? static_cast<int>(in.action) : 0;
    float x_a = max_nan(to_float(x[action]), kMasked);
    if (r.legal && !lm[action]) x_a = kMasked;
    used = used && !(x_a <= kMasked);

    float y[kPer], z[kPer], e[kPer], low = 0.0f, one = 0.0f;  // low: the reference's, past the row's end too
    // Entry l + kLanes k lies in the row where behind < -kLanes k.  A row may be read past
    // its end (the stage is that long); what stands there is not used.
    const int behind = l - vocab;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool in_row = behind < -kLanes * k;
      const int c = l + kLanes * k;
      y[k] = in_row ? max_nan(to_float(x[c]), kMasked) : kMasked;
      if constexpr (kRef) {
        const float raw = to_float(z_row[c]);
        if (k % 2) low = min3(low, one, raw);
        else one = raw;
        z[k] = in_row ? max_nan(raw, kMasked) : kMasked;
      }
    }
    if (r.legal) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const bool open = lm[l + kLanes * k];
        y[k] = open ? y[k] : kMasked;
        if constexpr (kRef) z[k] = open ? z[k] : kMasked;
      }
    }
    bool infinite = false;  // the reference masks an entry that the row does not
    if (kRef && low <= kMasked)
#pragma unroll
      for (int k = 0; k < kPer; ++k) infinite = infinite || (z[k] <= kMasked && y[k] > kMasked);
    float top = kMasked, top_r = kMasked;
#pragma unroll
    for (int k = 0; k < kPer; k += 2) {
      top = max_nan(top, y[k], y[k + 1]);
      if constexpr (kRef) top_r = max_nan(top_r, z[k], z[k + 1]);
    }
    Sums v;
    v.m = base2(max_lanes<kLanes>(top));
    v.mr = kRef ? base2(max_lanes<kLanes>(top_r)) : 0.0f;
    const Two unit = two(kLog2e, kLog2e), from = two(-v.m, -v.m), from_r = two(-v.mr, -v.mr);
    Two s2 = two(0.0f, 0.0f), t2 = s2, sr2 = s2, u2 = s2;
#pragma unroll
    for (int k = 0; k < kPer; k += 2) {
      const Two yy = fma(two(y[k], y[k + 1]), unit, from);
      split(yy, y[k], y[k + 1]);
      e[k] = exp2_fast(y[k]);
      e[k + 1] = exp2_fast(y[k + 1]);
      const Two ee = two(e[k], e[k + 1]);
      s2 = add(s2, ee);
      t2 = fma(ee, yy, t2);
      if constexpr (kRef) {
        const Two zz = fma(two(z[k], z[k + 1]), unit, from_r);
        split(zz, z[k], z[k + 1]);
        sr2 = add(sr2, two(exp2_fast(z[k]), exp2_fast(z[k + 1])));
        const Two d = fma(zz, two(-1.0f, -1.0f), yy);
        split(d, z[k], z[k + 1]);
        u2 = fma(ee, d, u2);
      }
    }
    v.s = sum_lanes<kLanes>(both(s2));
    v.t = sum_lanes<kLanes>(both(t2));
    v.sr = v.u = 0.0f;
    if constexpr (kRef) {
      v.sr = sum_lanes<kLanes>(both(sr2));
      v.u = sum_lanes<kLanes>(both(u2) + (infinite ? INFINITY : 0.0f));
    }
    if constexpr (!kPolicy) {
      if (l == 0 && real) store_score(o, row, used, v, x_a);
    } else {
      Coefs c{0.0f, 0.0f, 0.0f, 0.0f};
      float logp = 0.0f;
      if (used) {
        Terms terms;
        c = policy_row<kRef>(a, in, v, x_a, scale, terms, logp);
        if (l == 0) terms.add_to(acc, in.weight);
      }
      if (a.logp && l == 0 && real) a.logp[row] = logp;
      if (a.dlogits) {
        const Two c0 = two(c.c0, c.c0), c1 = two(c.c1, c.c1), c2 = two(c.c2, c.c2);
#pragma unroll
        for (int k = 0; k < kPer; k += 2) {
          Two g = fma(c1, two(y[k], y[k + 1]), c0);
          if constexpr (kRef) g = fma(c2, two(z[k], z[k + 1]), g);
          g = mul(g, two(e[k], e[k + 1]));
          split(g, y[k], y[k + 1]);
        }
        if (!used)  // the row may hold anything: its zeros are written as such
#pragma unroll
          for (int k = 0; k < kPer; ++k) y[k] = 0.0f;
        // The action's entry once more, with the hot term, by the lane that holds it.
        float hot = 0.0f;
        const bool mine = used && l == action % kLanes;
        if (mine) {
          const float y_a = fmaf(x_a, kLog2e, -v.m);
          hot = fmaf(c.c1, y_a, c.c0);
          if constexpr (kRef) {
            const float z_a = fmaf(max_nan(to_float(z_row[action]), kMasked), kLog2e, -v.mr);
            hot = fmaf(c.c2, y_a - z_a, hot);
          }
          hot = fmaf(hot, exp2_fast(y_a), c.hot);
        }
        with_type(a.dtype, [&](auto type) {
          constexpr int kType = decltype(type)::value, kBytes = sizeof(Stored<kType>);
          const auto write = [&](void* base) {  // the lane's entries of a row
#pragma unroll
            for (int k = 0; k < kPer; ++k)
              if (behind < -kLanes * k) store_one<kType>(base, l + kLanes * k, y[k]);
            for (int j = vocab + l; j < a.width; j += kLanes) store_one<kType>(base, j, 0.0f);
            if (mine) store_one<kType>(base, action, hot);
          };
          if (lay.grad) {
            const uintptr_t to = reinterpret_cast<uintptr_t>(a.dlogits) + first * a.ldd * kBytes;
            const int lead = static_cast<int>(to & 15);
            if (real) write(shared + out + lead + sub * static_cast<int>(a.ldd) * kBytes);
            __syncwarp();
            const int n = static_cast<int>(r.rows - first < kRows ? r.rows - first : kRows);
            const int end = lead + ((n - 1) * static_cast<int>(a.ldd) + a.width) * kBytes;
            char* const global = reinterpret_cast<char*>(to - lead);
            for (int k = 16 * lane; k < end; k += 512) {
              if (k >= lead && k + 16 <= end) {
                __stcs(reinterpret_cast<uint4*>(global + k), *reinterpret_cast<const uint4*>(shared + out + k));
              } else {  // the run's ends: its own bytes only
                for (int b = k < lead ? lead : k; b < k + 16 && b < end; b += 2)
                  *reinterpret_cast<uint16_t*>(global + b) = *reinterpret_cast<const uint16_t*>(shared + out + b);
              }
            }
          } else if (real) {
            write(static_cast<char*>(a.dlogits) + row * a.ldd * kBytes);
          }
        });
      }
    }
    __syncwarp();  // the stage and the gradient's place are free again
  }
  if constexpr (kPolicy) {
#pragma unroll
    for (int k = 0; k < kSums; ++k) acc[k] = sum_warp(acc[k]);
    store_partial(a, acc);
  }
}

// ---- long rows: a block, or a cluster of blocks, per row -----------------------------------
//
// A row is cut into 16-byte vectors (a head of up to one vector to its first 16-byte
// boundary, and a tail, entry by entry), and over the blocks of a cluster where it is much
// longer than a block's shared memory, or where there are few rows.  A thread looks at
// its vectors once for its sums, with a maximum of its own that rescales them when it
// grows, and where a gradient is wanted once more for that.  Between the two the warps' sums
// are joined through shared memory, and the blocks' of a cluster through distributed shared
// memory.
//
// A thread's vectors come through its own slots of shared memory; a slot that has been
// looked at for the last time is filled at once, with the same row's vector further on or
// with the next row's, so the copies run on under the second look, its stores and the
// next row's reductions.  They are waited for in two chunks of the slots.  For a gradient
// the slots keep the row, so that it crosses the memory bus once; vectors of it that no
// slot holds are read from memory both times.
//
// Sums alone are bound by the exponentials (their pipe 61% at 16,384 entries) and by each
// row's joins and barriers (some 400 instructions a warp): 2,048 rows of 131,072 bf16 in
// 96 us, 5.6 TB/s; 8,192 of 16,384 in 60 us, 4.5 TB/s.  With a gradient no pipe is full
// (exponentials 50%, memory 43%, 2.0 instructions a cycle): a block's warps go through the
// first look, the joins and the second look in step.  2,048 of 131,072 in 254 us, 4.2 TB/s
// (233 us where a fifth of them has weight 0 and is not read), with the full KL 417 us; its
// kernels spill 4 to 38 bytes a thread.  What may be masked costs a bound per entry: 8,192
// of 16,384 with flags 106 us for the sums, 195 us with the gradient (120 us without).

constexpr int kLongThreads = 256, kWideThreads = 512;
constexpr int kGroup = 4;   // vectors of a thread looked at together
constexpr int kChunks = 2;  // of a row's slots, waited for one after another

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ void unpack(const uint4 raw, float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(raw.x), f[1] = __uint_as_float(raw.y);
    f[2] = __uint_as_float(raw.z), f[3] = __uint_as_float(raw.w);
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        f[2 * e] = t.x;
        f[2 * e + 1] = t.y;
      }
    }
  }
}

// The largest (kMost; NaN stays) or smallest entry of vectors, in the entries' own type:
// two at once where it has 16 bits.
template <typename T, bool kMost, int kCount>
__device__ __forceinline__ float extreme(const uint4 (&x)[kCount]) {
  if constexpr (sizeof(T) == 4) {
    float r = __uint_as_float(x[0].x);
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const float a = __uint_as_float(x[k].x), b = __uint_as_float(x[k].y), c = __uint_as_float(x[k].z),
                  d = __uint_as_float(x[k].w);
      if constexpr (kMost) r = max_nan(max_nan(r, a, b), c, d);
      else r = min3(min3(r, a, b), c, d);
    }
    return r;
  } else {
    using Pair = std::conditional_t<std::is_same_v<T, __nv_bfloat16>, __nv_bfloat162, __half2>;
    const auto pair = [](uint32_t w) { return *reinterpret_cast<const Pair*>(&w); };
    Pair r = pair(x[0].x);
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) r = kMost ? __hmax2_nan(r, pair(w[e])) : __hmin2(r, pair(w[e]));
    }
    return kMost ? max_nan(to_float(r.x), to_float(r.y)) : fminf(to_float(r.x), to_float(r.y));
  }
}

// The flags of a vector's entries, a byte each; read by words, which lie in the flags' own
// 16-byte granules wherever the flags begin.
template <int kN>
struct Flags {
  uint32_t w[kN / 4];

  __device__ __forceinline__ static Flags load(const bool* lm) {
    const auto at = reinterpret_cast<uintptr_t>(lm);
    const int off = static_cast<int>(at & 3);
    Flags f;
    if ((at & (kN - 1)) == 0) {
      if constexpr (kN == 8) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(lm));
        f.w[0] = q.x;
        f.w[1] = q.y;
      } else {
        f.w[0] = __ldg(reinterpret_cast<const uint32_t*>(lm));
      }
    } else {
      const uint32_t* const q = reinterpret_cast<const uint32_t*>(at - off);
      uint32_t low = __ldg(q);
#pragma unroll
      for (int k = 0; k < kN / 4; ++k) {
        const uint32_t high = off || k + 1 < kN / 4 ? __ldg(q + k + 1) : 0u;
        f.w[k] = __funnelshift_r(low, high, 8 * off);
        low = high;
      }
    }
    return f;
  }

  // The entries whose flag is 0 as -inf.
  template <typename T>
  __device__ __forceinline__ uint4 apply(const uint4 raw) const {
    uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // Each flag's byte over its entry's bytes, as all ones or zeros.
      constexpr bool kSmall = sizeof(T) == 2;
      const uint32_t open = kSmall ? __byte_perm(w[e / 2 % (kN / 4)], 0, e % 2 ? 0x3322 : 0x1100) * 0xffu
                                   : __byte_perm(w[0], 0, 0x1111 * e) * 0xffu;
      constexpr uint32_t kLow = !kSmall ? 0xff800000u : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u : 0xfc00fc00u;
      x[e] = (x[e] & open) | (kLow & ~open);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
  }
};

// The row's part that a block takes, and its vectors.
template <typename T>
struct Part {
  const T* x;         // the row
  const T* z;         // the reference's row, or null
  const bool* lm;     // the row's flags, or null
  int head, vectors;  // entries before the first whole vector; whole vectors
  int first, last;    // the vectors to look at
  int vocab;
  bool z_wide;        // the reference's vectors are aligned as the row's are

  // `entries` entries of a row from entry c0 on; of their vectors, the share of block
  // `rank` of 2^log_parts.
  __device__ __forceinline__ Part() : x(nullptr), z(nullptr), lm(nullptr), head(0), vectors(0), first(0), last(0),
                                      vocab(0), z_wide(false) {}
  __device__ __forceinline__ Part(const Rows& r, i64 row, int c0, int entries, int log_parts, int rank) {
    x = static_cast<const T*>(r.logits) + row * r.ld + c0;
    z = r.ref ? static_cast<const T*>(r.ref) + row * r.ldr + c0 : nullptr;
    lm = r.legal ? r.legal + row * r.ldm + c0 : nullptr;
    vocab = entries;
    head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
    if (head > entries) head = entries;
    vectors = (entries - head) / kVec<T>;
    z_wide = (reinterpret_cast<uintptr_t>(z + head) & 15) == 0;
    const int each = (vectors + (1 << log_parts) - 1) >> log_parts;
    first = each * rank < vectors ? each * rank : vectors;
    last = first + each < vectors ? first + each : vectors;
  }

  __device__ __forceinline__ const uint4* vector(int v) const {
    return reinterpret_cast<const uint4*>(x + head) + v;
  }
  // The reference's entries beside vector v.
  __device__ __forceinline__ uint4 ref_vector(int v) const {
    const T* at = z + head + v * kVec<T>;
    if (z_wide) return __ldg(reinterpret_cast<const uint4*>(at));
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) w[e] = reinterpret_cast<const uint32_t*>(at)[e];
      else w[e] = reinterpret_cast<const uint16_t*>(at)[2 * e] |
                  static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[2 * e + 1]) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ Flags<kVec<T>> flags(int v) const { return Flags<kVec<T>>::load(lm + head + v * kVec<T>); }
  // Entry number i of those outside the vectors, or -1: rank 0 takes them all.
  __device__ __forceinline__ int loose(int i) const {
    const int tail = head + vectors * kVec<T>;
    const int c = i < head ? i : tail + i - head;
    return c < vocab ? c : -1;
  }
  __device__ __forceinline__ float one(const T* p, int c) const {
    return lm && !lm[c] ? kMasked : max_nan(to_float(p[c]), kMasked);
  }
};

// A thread's running sums, the odd and the even entries' side by side.
struct Running {
  float m, mr;
  Two s, t, sr, u;
  bool infinite;  // the reference masks an entry that the row does not
};

__device__ __forceinline__ Running nothing_yet() {
  const Two zero = two(0.0f, 0.0f);
  return {kMasked2, kMasked2, zero, zero, zero, zero, false};
}

// New maxima (in base-2 units) where they are larger, also for NaN.
template <bool kRef>
__device__ __forceinline__ void raise(Running& v, float m, float mr) {
  if (!(m <= v.m)) {
    const float d = v.m - m, f = exp2_fast(d);
    const Two dd = two(d, d), ff = two(f, f);
    v.t = mul(ff, fma(dd, v.s, v.t));
    if constexpr (kRef) v.u = mul(ff, fma(dd, v.s, v.u));
    v.s = mul(v.s, ff);
    v.m = m;
  }
  if constexpr (kRef) {
    if (!(mr <= v.mr)) {
      const float d = v.mr - mr, f = exp2_fast(d);
      v.u = fma(two(-d, -d), v.s, v.u);
      v.sr = mul(v.sr, two(f, f));
      v.mr = mr;
    }
  }
}

// Adds kN entries, none above the maxima.
template <bool kRef, int kN>
__device__ __forceinline__ void accumulate(Running& v, const float (&x)[kN], const float (&z)[kN]) {
  const Two unit = two(kLog2e, kLog2e), from = two(-v.m, -v.m), from_r = two(-v.mr, -v.mr);
#pragma unroll
  for (int e = 0; e < kN; e += 2) {
    const Two y = fma(two(x[e], x[e + 1]), unit, from);
    float y0, y1;
    split(y, y0, y1);
    const Two p = two(exp2_fast(y0), exp2_fast(y1));
    v.s = add(v.s, p);
    v.t = fma(p, y, v.t);
    if constexpr (kRef) {
      const Two q = fma(two(z[e], z[e + 1]), unit, from_r);
      float q0, q1;
      split(q, q0, q1);
      v.sr = add(v.sr, two(exp2_fast(q0), exp2_fast(q1)));
      v.u = fma(p, fma(q, two(-1.0f, -1.0f), y), v.u);
    }
  }
}

// Adds whole vectors as they are: one look at their largest entry for all.  An entry of
// -inf makes the sums NaN (0 times -inf), and so does a masked entry of the reference (whose
// fp16 knows no other than -inf); the row is then taken again with care.
template <typename T, bool kRef, int kCount>
__device__ __forceinline__ void add_vectors(Running& v, const uint4 (&x)[kCount], const uint4 (&z)[kCount]) {
  constexpr int kN = kVec<T>;
  raise<kRef>(v, base2(extreme<T, true>(x)), kRef ? base2(extreme<T, true>(z)) : kMasked2);
  if constexpr (kRef && !std::is_same_v<T, __half>)
    if (extreme<T, false>(z) <= kMasked) v.u = two(NAN, NAN);
#pragma unroll
  for (int k = 0; k < kCount; ++k) {
    float f[kN], q[kN];
    unpack<T>(x[k], f);
    if constexpr (kRef) unpack<T>(z[k], q);
    accumulate<kRef>(v, f, q);
  }
}

// A vector's entries, none below kMasked.
template <typename T>
__device__ __forceinline__ void bounded(const uint4 raw, float (&f)[kVec<T>]) {
  unpack<T>(raw, f);
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e) f[e] = max_nan(f[e], kMasked);
}

template <int kN>
__device__ __forceinline__ float largest(const float (&x)[kN]) {
  const float top = max_nan(max_nan(x[0], x[1], x[2]), x[3]);
  if constexpr (kN == 8) return max_nan(max_nan(top, x[4], x[5]), x[6], x[7]);
  else return top;
}

// Adds vectors of which entries may be masked.
template <typename T, bool kRef, int kCount>
__device__ __forceinline__ void add_bounded(Running& v, const uint4 (&x)[kCount], const uint4 (&z)[kCount]) {
  constexpr int kN = kVec<T>;
#pragma unroll
  for (int h = 0; h < kCount; ++h) {
    float f[kN], q[kN];
    bounded<T>(x[h], f);
    if constexpr (kRef) {
      bounded<T>(z[h], q);
#pragma unroll
      for (int e = 0; e < kN; ++e) v.infinite = v.infinite || (q[e] <= kMasked && f[e] > kMasked);
    }
    raise<kRef>(v, base2(largest(f)), kRef ? base2(largest(q)) : kMasked2);
    accumulate<kRef>(v, f, q);
  }
}

// d_j of a vector's entries, without the action's own term.
template <bool kRef, int kN>
__device__ __forceinline__ void gradient(const Coefs& c, float m, float mr, const float (&x)[kN],
                                         const float (&z)[kN], float (&g)[kN]) {
  const Two unit = two(kLog2e, kLog2e), from = two(-m, -m), from_r = two(-mr, -mr);
  const Two c0 = two(c.c0, c.c0), c1 = two(c.c1, c.c1), c2 = two(c.c2, c.c2);
#pragma unroll
  for (int e = 0; e < kN; e += 2) {
    const Two y = fma(two(x[e], x[e + 1]), unit, from);
    Two d = fma(c1, y, c0);
    if constexpr (kRef) {
      const Two q = fma(two(z[e], z[e + 1]), unit, from_r);
      d = fma(c2, fma(q, two(-1.0f, -1.0f), y), d);
    }
    float y0, y1;
    split(y, y0, y1);
    split(mul(d, two(exp2_fast(y0), exp2_fast(y1))), g[e], g[e + 1]);
  }
}

// Entry j's, with the action's term where it is the action.
template <typename T, bool kRef>
__device__ __forceinline__ float gradient_of(const Part<T>& p, const Coefs& c, float m, float mr, int j, bool hot) {
  const float y = fmaf(p.one(p.x, j), kLog2e, -m);
  float g = fmaf(c.c1, y, c.c0);
  if constexpr (kRef) g = fmaf(c.c2, y - fmaf(p.one(p.z, j), kLog2e, -mr), g);
  return fmaf(g, exp2_fast(y), hot ? c.hot : 0.0f);
}

// The action's entry once more, by the thread that wrote its vector: so no entry has to be
// compared with it.
template <typename T, bool kRef, int kType>
__device__ __forceinline__ void write_hot(const Part<T>& p, const Coefs& c, float m, float mr, int action, void* row,
                                          int tid, int step) {  // step: a power of two
  const int v = (action - p.head) / kVec<T>;
  if (action >= p.head && v >= p.first && v < p.last && ((v - p.first) & (step - 1)) == tid)
    store_one<kType>(row, action, gradient_of<T, kRef>(p, c, m, mr, action, true));
}

template <typename T, int kType>
__device__ __forceinline__ void write_zeros(const Part<T>& p, void* row, bool wide, int tid, int step) {
  float g[kVec<T>] = {};
  for (int i = p.first + tid; i < p.last; i += step) store_grad<kType>(row, p.head + i * kVec<T>, g, wide);
}

// The gradient of whole vectors, `apart` entries from one to the next.  kMasks: entries may
// be masked.
template <typename T, bool kRef, int kType, bool kMasks, int kCount>
__device__ __forceinline__ void write_vectors(const Coefs& c, float m, float mr, Stored<kType>* to, int apart, bool wide,
                                              const uint4 (&x)[kCount], const uint4 (&z)[kCount]) {
  constexpr int kN = kVec<T>;
#pragma unroll
  for (int k = 0; k < kCount; ++k) {
    float f[kN], q[kN], g[kN];
    if constexpr (kMasks) bounded<T>(x[k], f);
    else unpack<T>(x[k], f);
    if constexpr (kRef && kMasks) bounded<T>(z[k], q);
    else if constexpr (kRef) unpack<T>(z[k], q);
    gradient<kRef>(c, m, mr, f, q, g);
    store_grad<kType>(to, k * apart, g, wide);
  }
}

// Whether a row's vectors are aligned in the gradient.
template <typename T, int kType>
__device__ __forceinline__ bool grad_wide(const void* row, int head) {
  constexpr int kBytes = kVec<T> * static_cast<int>(sizeof(Stored<kType>));
  const uintptr_t to = reinterpret_cast<uintptr_t>(row) + head * sizeof(Stored<kType>);
  return to % (kBytes < 16 ? kBytes : 16) == 0;
}

// What one thread works out of a row for all.
struct RowResult {
  Coefs c;
  float m, mr;
  bool used, again;
};

template <int kLeft>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// What the threads of a block of long rows share beside their slots.
struct LongShared {
  Sums warp_sums[kWideThreads / 32];
  Sums block_sums[2];
  RowInputs row_in;  // thread 32's, for thread 0
  float row_x;       // the action's entry
  RowResult result;  // thread 0's, for all
  double acc[kSums];
};

// A block's rows from `row` on.  kMasks false: entries are taken as they are, until a row's
// sums are not numbers; that row is returned (the number of rows, if there is none).
// true: with legal, and entries of -inf and the like.  slots: vectors of a thread that shared
// memory holds; buffer: whose turn it is of block_sums.
template <typename T, bool kRef, bool kPolicy, bool kMasks>
__device__ __forceinline__ i64 long_rows(const Rows& r, const Score& o, const Policy& a, const float scale,
                                         const int slots, LongShared& sh, i64 row0, int& buffer) {
  constexpr int kN = kVec<T>, kLook = kRef || kMasks ? 2 : kGroup;  // vectors looked at together
  extern __shared__ __align__(16) uint4 slot[];  // [slots][threads], then the reference's
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x / 32, step = blockDim.x;
  const int log_parts = __ffs(parts) - 1, log_step = __ffs(step) - 1;  // both are powers of two
  const int chunk = (slots + kChunks * kGroup - 1) / (kChunks * kGroup) * kGroup;
  uint4* const mine = slot + tid;
  uint4* const mine_r = mine + slots * step;
  const i64 rows_step = gridDim.x / parts;

  // A row that may count (its action's own entry is still to be seen), or none; the same in
  // the whole cluster.
  struct Candidate {
    i64 row;
    int action;  // -1: it does not count
  };
  const auto candidate = [&](i64 row) {
    Candidate c{row, -1};
    if (row < r.rows) {
      const i64 action = r.actions[row];
      const float w = r.weight ? r.weight[row] : 1.0f;
      if (action >= 0 && action < r.vocab && w != 0.0f) c.action = static_cast<int>(action);
    }
    return c;
  };
  // Of a part's vectors, how many are this thread's and in slots.
  const auto slotted = [&](const Part<T>& p) {
    const int n = (p.last - p.first - tid + step - 1) >> log_step;
    return p.last - p.first <= tid ? 0 : n < slots ? n : slots;
  };
  // Starts the copies of a chunk of a part's slots, n of which are this thread's; always a
  // group of its own.
  const auto fetch = [&](const uint4* x, const uint4* z, int n, int c) {
    const int end = (c + 1) * chunk < n ? (c + 1) * chunk : n;
    int k = c * chunk, at = k * step;
    for (; k + kGroup <= end; k += kGroup, at += kGroup * step)
#pragma unroll
      for (int h = 0; h < kGroup; ++h) {
        copy16(mine + at + h * step, x + at + h * step);
        if constexpr (kRef) copy16(mine_r + at + h * step, z + at + h * step);
      }
    for (; k < end; ++k, at += step) {
      copy16(mine + at, x + at);
      if constexpr (kRef) copy16(mine_r + at, z + at);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // This thread's first vector of a part in memory, and the reference's.
  const auto first_x = [&](const Part<T>& p) { return p.vector(p.first + tid); };
  const auto first_z = [&](const Part<T>& p) {
    return kRef ? reinterpret_cast<const uint4*>(p.z + p.head) + p.first + tid : nullptr;
  };

  // The next row from `c` on that may count; those before it get their zeros here, so that
  // copies are always under way for the row that comes next.
  const auto skip = [&](Candidate c) {
    for (; c.row < r.rows && c.action < 0; c = candidate(c.row + rows_step)) {
      const i64 row = c.row;
      if (tid == 0 && rank == 0) {
        if constexpr (!kPolicy) store_score(o, row, false, no_sums(), 0.0f);
        else if (a.logp) a.logp[row] = 0.0f;
      }
      if constexpr (kPolicy)
        if (a.dlogits)
          with_type(a.dtype, [&](auto type) {
            constexpr int kType = decltype(type)::value;
            const Part<T> p(r, row, 0, r.vocab, log_parts, rank);
            Stored<kType>* const to = static_cast<Stored<kType>*>(a.dlogits) + row * a.ldd;
            write_zeros<T, kType>(p, to, grad_wide<T, kType>(to, p.head), tid, step);
            if (rank == 0) {
              if (tid < r.vocab - p.vectors * kN) store_one<kType>(to, p.loose(tid), 0.0f);
              for (int j = r.vocab + tid; j < a.width; j += step) store_one<kType>(to, j, 0.0f);
            }
          });
    }
    return c;
  };

  Candidate now = skip(candidate(row0)), next = now, after = now;
  const bool write = kPolicy && a.dlogits;  // a second look
  Part<T> p;
  int n_slotted = 0;
  if (now.row < r.rows) {
    p = Part<T>(r, now.row, 0, r.vocab, log_parts, rank);
    n_slotted = slotted(p);
    next = skip(candidate(now.row + rows_step));
  }
#pragma unroll
  for (int c = 0; c < kChunks; ++c) fetch(first_x(p), first_z(p), n_slotted, c);
  for (; now.row < r.rows; now = next, next = after) {
    Part<T> p_next = p;
    int n_next = 0;
    if (next.row < r.rows) {
      p_next = Part<T>(r, next.row, 0, r.vocab, log_parts, rank);
      n_next = slotted(p_next);
    }
    after = candidate(next.row + rows_step);  // looked at when this row is done
    const uint4 *const x_next = first_x(p_next), *const z_next = first_z(p_next);
    const i64 row = now.row;
    const int action = now.action, i0 = p.first + tid;
    const int n_loose = rank == 0 ? r.vocab - p.vectors * kN : 0;
    if (tid == (step > 32 ? 32 : 0)) {
      sh.row_in = row_inputs<kPolicy>(r, a, row);
      sh.row_x = p.one(p.x, action);
    }
    // Some vectors of the row, `step` apart, from slot k on or from vector i on in memory.
    const auto masked = [&](int i, auto& x, auto& z) {
      if constexpr (kMasks) {
        constexpr int kCount = std::extent_v<std::remove_reference_t<decltype(x)>>;
        if (p.lm) {
          Flags<kN> f[kCount];
#pragma unroll
          for (int h = 0; h < kCount; ++h) f[h] = p.flags(i + h * step);
#pragma unroll
          for (int h = 0; h < kCount; ++h) {
            x[h] = f[h].template apply<T>(x[h]);
            if constexpr (kRef) z[h] = f[h].template apply<T>(z[h]);
          }
        }
      }
    };
    const auto from_slots = [&](const uint4* at, const uint4* at_r, int k, auto& x, auto& z) {
      constexpr int kCount = std::extent_v<std::remove_reference_t<decltype(x)>>;
#pragma unroll
      for (int h = 0; h < kCount; ++h) {
        x[h] = at[h * step];
        if constexpr (kRef) z[h] = at_r[h * step];
      }
      masked(i0 + k * step, x, z);
    };
    const auto from_memory = [&](int i, auto& x, auto& z) {
      constexpr int kCount = std::extent_v<std::remove_reference_t<decltype(x)>>;
#pragma unroll
      for (int h = 0; h < kCount; ++h) {
        x[h] = __ldg(p.vector(i + h * step));
        if constexpr (kRef) z[h] = p.ref_vector(i + h * step);
      }
      masked(i, x, z);
    };
    Running run = nothing_yet();
    const auto add = [&](const auto& x, const auto& z) {
      if constexpr (kMasks) add_bounded<T, kRef>(run, x, z);
      else add_vectors<T, kRef>(run, x, z);
    };
    // The row by as many vectors as the slots hold; slots that need not be kept for a second
    // look are filled again at once, with the row's vectors further on or the next row's.
    const int in_part = p.last - p.first, n_all = in_part <= tid ? 0 : (in_part - tid + step - 1) >> log_step;
    int base = 0;  // vectors before those in the slots
    for (;; base += slots) {
      const int n = n_all - base < slots ? n_all - base : slots;
      const bool more = !write && slots > 0 && (base + slots) * step < in_part;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (write && c > 0) wait_copies<0>();
        else wait_copies<kChunks - 1>();
        static_assert(kChunks == 2, "the waits are for two");
        const int end = (c + 1) * chunk < n ? (c + 1) * chunk : n;
        const uint4 *at = mine + c * chunk * step, *at_r = mine_r + c * chunk * step;
        int k = c * chunk;
#pragma unroll 1
        for (; k + kLook <= end; k += kLook, at += kLook * step, at_r += kLook * step) {
          uint4 x[kLook], z[kLook];
          from_slots(at, at_r, base + k, x, z);
          add(x, z);
        }
#pragma unroll 1
        for (; k < end; ++k, at += step, at_r += step) {
          uint4 x[1], z[1];
          from_slots(at, at_r, base + k, x, z);
          add(x, z);
        }
        if (more) {
          const int behind = base + slots, left = n_all - behind;
          fetch(first_x(p) + behind * step, kRef ? first_z(p) + behind * step : nullptr, left < slots ? left : slots, c);
        } else if (!write) {
          fetch(x_next, z_next, n_next, c);
        }
      }
      if (!more) break;
    }
    if (write || slots == 0) {  // what no slot holds
      int i = i0 + slots * step;
#pragma unroll 1
      for (; i + step < p.last; i += 2 * step) {
        uint4 x[2], z[2];
        from_memory(i, x, z);
        add(x, z);
      }
      if (i < p.last) {
        uint4 x[1], z[1];
        from_memory(i, x, z);
        add(x, z);
      }
    }
    if (tid < n_loose) {
      // One entry, and one that adds nothing beside it: were there nothing else, it would
      // weigh as much as a masked entry, and a row of such does not count.
      const int c = p.loose(tid);
      const float f[2] = {p.one(p.x, c), kMasked};
      float q[2] = {kMasked, kMasked};
      if constexpr (kRef) {
        q[0] = p.one(p.z, c);
        run.infinite = run.infinite || (q[0] <= kMasked && f[0] > kMasked);
      }
      raise<kRef>(run, base2(f[0]), base2(q[0]));
      accumulate<kRef>(run, f, q);
    }
    Sums v = no_sums();
    v.m = run.m;
    v.s = both(run.s);
    v.t = both(run.t);
    if constexpr (kRef) {
      v.mr = run.mr;
      v.sr = marked(both(run.sr), run.infinite);
      v.u = both(run.u);
    }
    v = join_warp<kRef>(v);
    if (lane == 0) sh.warp_sums[tid >> 5] = v;
    __syncthreads();
    if (tid < 32) v = join_warp<kRef>(lane < warps ? sh.warp_sums[lane] : no_sums());
    if (parts > 1) {
      if (tid == 0) sh.block_sums[buffer] = v;
      cluster.sync();
      // Every block adds the blocks' sums in the same order.
      if (tid < 32)
        v = join_warp<kRef>(lane < parts ? *cluster.map_shared_rank(&sh.block_sums[buffer], lane) : no_sums());
      buffer ^= 1;
    }
    if (tid == 0) {
      // Not a number: for an entry that is one, or for one of -inf.
      const float sum = v.s + v.t + (kRef ? v.sr + v.u : 0.0f);
      sh.result.again = !kMasks && !(fabsf(sum) < INFINITY);
      if (kRef && infinite(v.sr)) {
        v.sr = -v.sr;
        v.u += INFINITY;
      }
      const float row_x = sh.row_x;
      const bool used = !(row_x <= kMasked);
      if (!sh.result.again) {
        if constexpr (!kPolicy) {
          if (rank == 0) store_score(o, row, used, v, row_x);
        } else {
          const RowInputs in = sh.row_in;
          float logp = 0.0f;
          if (used) {
            Terms terms;
            sh.result.c = policy_row<kRef>(a, in, v, row_x, scale, terms, logp);
            if (rank == 0) terms.add_to(sh.acc, in.weight);
          }
          if (a.logp && rank == 0) a.logp[row] = logp;
          sh.result.m = v.m;
          sh.result.mr = v.mr;
          sh.result.used = used;
        }
      }
    }
    __syncthreads();  // the result is there; row_in and warp_sums are free again
    if (!kMasks && sh.result.again) {
      wait_copies<0>();
      return row;
    }
    if constexpr (kPolicy) {
      if (write) {
        const Coefs c = sh.result.c;  // of a row that counts; not used for another
        const float m = sh.result.m, mr = sh.result.mr;
        const bool used = sh.result.used;
        with_type(a.dtype, [&](auto type) {
          constexpr int kType = decltype(type)::value;
          using S = Stored<kType>;
          S* const to = static_cast<S*>(a.dlogits) + row * a.ldd;
          const bool wide = grad_wide<T, kType>(to, p.head);
          const auto put = [&](S* place, const auto& x, const auto& z) {
            write_vectors<T, kRef, kType, kMasks>(c, m, mr, place, step * kN, wide, x, z);
          };
          if (!used) write_zeros<T, kType>(p, to, wide, tid, step);
          for (int q = 0; q < kChunks; ++q) {
            if (used) {
              const int end = (q + 1) * chunk < n_slotted ? (q + 1) * chunk : n_slotted;
              const uint4 *at = mine + q * chunk * step, *at_r = mine_r + q * chunk * step;
              int k = q * chunk;
              S* place = to + p.head + (i0 + k * step) * kN;
#pragma unroll 1
              for (; k + kLook <= end; k += kLook, at += kLook * step, at_r += kLook * step) {
                uint4 x[kLook], z[kLook];
                from_slots(at, at_r, k, x, z);
                put(place, x, z);
                place += kLook * step * kN;
              }
#pragma unroll 1
              for (; k < end; ++k, at += step, at_r += step) {
                uint4 x[1], z[1];
                from_slots(at, at_r, k, x, z);
                put(place, x, z);
                place += step * kN;
              }
            }
            fetch(x_next, z_next, n_next, q);
          }
          if (used)
#pragma unroll 1
            for (int i = i0 + slots * step; i < p.last; i += step) {
              uint4 x[1], z[1];
              from_memory(i, x, z);
              put(to + p.head + i * kN, x, z);
            }
          if (used) write_hot<T, kRef, kType>(p, c, m, mr, action, to, tid, step);
          if (tid < n_loose) {
            const int j = p.loose(tid);
            store_one<kType>(to, j, used ? gradient_of<T, kRef>(p, c, m, mr, j, j == action) : 0.0f);
          }
          if (rank == 0)
            for (int j = r.vocab + tid; j < a.width; j += step) store_one<kType>(to, j, 0.0f);
        });
      }
    }
    after = skip(after);
    p = p_next;
    n_slotted = n_next;
  }
  return r.rows;
}

template <typename T, bool kRef, bool kPolicy, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kWideThreads ? 2 : 3)
    long_rows_kernel(const Rows r, const Score o, const Policy given, const int slots) {
  const Policy a = kPolicy ? resolved(given) : given;
  __shared__ LongShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  float scale = 0.0f;
  if (threadIdx.x == 0)
#pragma unroll
    for (int k = 0; k < kSums; ++k) sh.acc[k] = 0.0;
  if constexpr (kPolicy) scale = grad_scale_of(a, block_denominator(a, r.weight, r.rows));
  int buffer = 0;
  i64 row = blockIdx.x / cluster.num_blocks();
  // Rows as they are cost less than rows whose entries may be masked; the first one that
  // turns out to have such, and all behind it, go the second way.
  if (!r.legal) row = long_rows<T, kRef, kPolicy, false>(r, o, a, scale, slots, sh, row, buffer);
  if (row < r.rows) long_rows<T, kRef, kPolicy, true>(r, o, a, scale, slots, sh, row, buffer);
  if (cluster.num_blocks() > 1) cluster.sync();  // no block leaves while another may read its sums
  if constexpr (kPolicy)
    if (threadIdx.x == 0 && a.partial)
#pragma unroll
      for (int k = 0; k < kSums; ++k) a.partial[(i64)blockIdx.x * kSums + k] = sh.acc[k];
}

// ---- the means of policy_loss ---------------------------------------------------------------

constexpr int kWeightBlock = 4096;  // weights a block adds up

__global__ void __launch_bounds__(512) weight_sums_kernel(const float* weight, i64 rows, i64 per_block,
                                                          double* sums) {
  __shared__ double part[16];
  const i64 first = blockIdx.x * per_block;
  const i64 last = first + per_block < rows ? first + per_block : rows;
  double t = 0.0;
  for (i64 i = first + threadIdx.x; i < last; i += blockDim.x) t += weight[i];
  t = sum_warp(t);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (int k = 0; k < 16; ++k) t += part[k];
    sums[blockIdx.x] = t;
  }
}

constexpr int kMeansGroups = 4;  // warps, at most, that add a kind of partial sums

__global__ void __launch_bounds__(32 * kSums * kMeansGroups)
    policy_means_kernel(const Policy given, const float* weight, i64 rows, int blocks, float* stats, float* loss) {
  const Policy a = resolved(given);
  __shared__ double part[kSums][kMeansGroups], means[kSums];
  const double d = block_denominator(a, weight, rows);
  const int groups = blockDim.x / (32 * kSums), step = 32 * groups;
  const int warp = threadIdx.x >> 5, k = warp / groups, group = warp % groups;
  double t = 0.0;
  for (int b = 32 * group + (threadIdx.x & 31); b < blocks; b += 8 * step) {  // eight loads in flight
    double x[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = b + q * step < blocks ? a.partial[(b + q * step) * kSums + k] : 0.0;
#pragma unroll
    for (int q = 0; q < 8; ++q) t += x[q];
  }
  t = sum_warp(t);
  if ((threadIdx.x & 31) == 0) part[k][group] = t;
  __syncthreads();
  if (threadIdx.x < kSums) {
    t = part[threadIdx.x][0];
    for (int g = 1; g < groups; ++g) t += part[threadIdx.x][g];
    t = d == 0.0 ? 0.0 : t / d;
    means[threadIdx.x] = t;
    stats[threadIdx.x + 1] = static_cast<float>(t);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    // A KL that may be infinite takes no part in the loss where its coefficient is 0.
    const double kl = a.kl_coef == 0.0f ? 0.0 : a.kl_coef * means[2];
    stats[0] = static_cast<float>(means[0] - a.entropy_coef * means[1] + kl);
    if (loss) *loss = stats[0];
    stats[kStats] = static_cast<float>(d);
  }
}

// ---- action_logp's backward --------------------------------------------------------------------
//
// With a row's maximum and sum kept by the forward nothing is left to reduce: a warp
// takes kSpan entries of a row (or a whole shorter row) and writes their gradients
//   d_j = d_logp ([j = a] - p_j) - d_entropy p_j (log p_j + H),  times *scale.
// Four vectors of a lane are in flight at once, and the last rows come first, of which the
// forward may have left some in L2 (79 against 77 us).  Bound by memory: 8,192 rows of 16,384
// bf16 77 us, 7.0 TB/s.

constexpr int kSpan = 4096;
constexpr int kBackWarps = 8;

struct Back {
  const float2* lse;
  const float* entropy;    // or null (no d_entropy)
  const float* d_logp;     // or null: 0
  const float* d_entropy;  // or null: 0
  const float* scale;      // device scalar, or null
  void* dlogits;
  i64 ldd;
  int dtype;
};

template <typename T>
__global__ void __launch_bounds__(32 * kBackWarps, 4) logp_backward_kernel(const Rows r, const Back b, int spans) {
  const int lane = threadIdx.x & 31;
  const i64 unit = r.rows * spans - 1 - ((i64)blockIdx.x * kBackWarps + (threadIdx.x >> 5));
  if (unit < 0) return;
  const i64 row = unit / spans;
  const int c0 = static_cast<int>(unit - row * spans) * kSpan;
  const float2 lse = b.lse[row];
  const float scale = b.scale ? *b.scale : 1.0f;
  const float g1 = b.d_logp ? b.d_logp[row] * scale : 0.0f;
  const float g2 = b.d_entropy ? b.d_entropy[row] * scale : 0.0f;
  // A row that does not count, and one whose gradient is 0, is not read.
  const bool used = lse.y != INFINITY && !(g1 == 0.0f && g2 == 0.0f);
  const float inv_s = exp2_fast(-lse.y);
  Coefs k;
  k.hot = g1;
  k.c0 = inv_s * (-g1 - g2 * ((b.d_entropy ? b.entropy[row] : 0.0f) - kLn2 * lse.y));
  k.c1 = inv_s * (-g2 * kLn2);
  k.c2 = 0.0f;
  const Part<T> p(r, row, c0, r.vocab - c0 < kSpan ? r.vocab - c0 : kSpan, 0, 0);
  const int hot = used ? static_cast<int>(r.actions[row]) - c0 : -1;
  with_type(b.dtype, [&](auto type) {
    constexpr int kType = decltype(type)::value;
    using S = Stored<kType>;
    S* const to = static_cast<S*>(b.dlogits) + row * b.ldd + c0;
    const bool wide = grad_wide<T, kType>(to, p.head);
    if (!used) {
      write_zeros<T, kType>(p, to, wide, lane, 32);
    } else {
      const auto write = [&](int i, auto count) {
        constexpr int kCount = decltype(count)::value;
        uint4 x[kCount];
#pragma unroll
        for (int h = 0; h < kCount; ++h) x[h] = __ldcs(p.vector(i + 32 * h));
        if (p.lm) {
          Flags<kVec<T>> f[kCount];
#pragma unroll
          for (int h = 0; h < kCount; ++h) f[h] = p.flags(i + 32 * h);
#pragma unroll
          for (int h = 0; h < kCount; ++h) x[h] = f[h].template apply<T>(x[h]);
        }
        S* const at = to + p.head + i * kVec<T>;
        const int apart = 32 * kVec<T>;
        if (!p.lm && extreme<T, false>(x) > kMasked)
          write_vectors<T, false, kType, false>(k, lse.x, 0.0f, at, apart, wide, x, x);
        else
          write_vectors<T, false, kType, true>(k, lse.x, 0.0f, at, apart, wide, x, x);
      };
      int i = lane;
      for (; i + (kGroup - 1) * 32 < p.last; i += kGroup * 32) write(i, std::integral_constant<int, kGroup>{});
      for (; i < p.last; i += 32) write(i, std::integral_constant<int, 1>{});
      write_hot<T, false, kType>(p, k, lse.x, 0.0f, hot, to, lane, 32);
    }
    for (int i = lane; i < p.vocab - p.vectors * kVec<T>; i += 32) {
      const int c = p.loose(i);
      store_one<kType>(to, c, used ? gradient_of<T, false>(p, k, lse.x, 0.0f, c, c == hot) : 0.0f);
    }
  });
}

// ---- the preference loss over pairs --------------------------------------------------------------
//
// Sequence j holds rows offsets[j] .. offsets[j + 1] - 1 (bounds outside the rows are
// brought inside); pair i prefers sequence 2 i to 2 i + 1.  kLanes threads take a pair:
// the two scores in 64 bits, the margin, then the rows' d loss / d logp.  A few hundred bytes
// a sequence: latency only (128 pairs 7 us, 16 pairs of up to 1,024 rows 12 us).

struct Pairs {
  const float* logp;
  const float* ref_logp;
  const float* weight;  // or null
  const float2* lse;    // which rows count
  const i64* offsets;
  i64 pairs, rows;
  float beta, smoothing;
  bool average;
  float* margin;    // [pairs]
  float* seq_logp;  // [2 pairs]
  float* d_logp;    // [rows], or null
  double* partial;  // [blocks][2]: their sums, of a launch of more
  float* means[2];  // the loss and the share of margins above 0, written here by a launch of one block
};

constexpr int kPairThreads = 1024;

template <int kLanes>
__global__ void __launch_bounds__(kPairThreads) pairs_kernel(const Pairs a) {
  constexpr int kWarps = kLanes / 32, kGroups = kPairThreads / kLanes;
  __shared__ double part[kPairThreads / 32][3];
  __shared__ double block_sums[kPairThreads / 32][2];
  const int tid = threadIdx.x, lane = tid % kLanes, group = tid / kLanes;
  double loss = 0.0, above = 0.0;
  const i64 stride = (i64)gridDim.x * kGroups;
  // Every group goes round as often as the block's first one, so that the barriers meet.
  for (i64 base = (i64)blockIdx.x * kGroups; base < a.pairs; base += stride) {
    const i64 pair = base + group;
    const bool real = pair < a.pairs;
    i64 from[2] = {0, 0}, to[2] = {0, 0};
    double score[2], total[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (real) {
        from[h] = a.offsets[2 * pair + h];
        to[h] = a.offsets[2 * pair + h + 1];
        from[h] = from[h] < 0 ? 0 : from[h];
        to[h] = to[h] > a.rows ? a.rows : to[h];
      }
      double sums[3] = {0.0, 0.0, 0.0};  // w (logp - ref), w logp, w
      for (i64 t = from[h] + lane; t < to[h]; t += kLanes) {
        if (a.lse[t].y == INFINITY) continue;
        const double w = a.weight ? a.weight[t] : 1.0f;
        sums[0] += w * (static_cast<double>(a.logp[t]) - a.ref_logp[t]);
        sums[1] += w * a.logp[t];
        sums[2] += w;
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) sums[k] = sum_warp(sums[k]);
      if constexpr (kWarps > 1) {
        __syncthreads();
        if ((tid & 31) == 0)
#pragma unroll
          for (int k = 0; k < 3; ++k) part[tid >> 5][k] = sums[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          sums[k] = 0.0;
          for (int q = 0; q < kWarps; ++q) sums[k] += part[group * kWarps + q][k];
        }
      }
      const double n = a.average && sums[2] != 0.0 ? 1.0 / sums[2] : 1.0;
      score[h] = sums[0] * n;
      total[h] = n;
      if (real && lane == 0) a.seq_logp[2 * pair + h] = static_cast<float>(sums[1] * n);
    }
    if (!real) continue;
    const float m = static_cast<float>(a.beta * (score[0] - score[1]));
    // -log sigmoid(m), -log sigmoid(-m) and the two sigmoids from one exponential.
    const float e = expf(-fabsf(m)), soft = log1pf(e);
    const float lose = soft + fmaxf(-m, 0.0f), win = soft + fmaxf(m, 0.0f);
    if (lane == 0) {
      a.margin[pair] = m;
      loss += (1.0f - a.smoothing) * lose + a.smoothing * win;
      above += m > 0.0f ? 1.0 : 0.0;
    }
    if (a.d_logp) {
      const float large = 1.0f / (1.0f + e), small = e * large;
      const float up = m > 0.0f ? large : small, down = m > 0.0f ? small : large;
      const float slope = a.beta * (a.smoothing * up - (1.0f - a.smoothing) * down) / static_cast<float>(a.pairs);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float d = static_cast<float>((h ? -slope : slope) * total[h]);
        for (i64 t = from[h] + lane; t < to[h]; t += kLanes) a.d_logp[t] = a.weight ? d * a.weight[t] : d;
      }
    }
  }
  // The groups' sums are in lane 0 of their first warps.
  if ((tid & 31) == 0) {
    block_sums[tid >> 5][0] = loss;
    block_sums[tid >> 5][1] = above;
  }
  __syncthreads();
  if (tid < 2) {
    double t = 0.0;
    for (int q = 0; q < kPairThreads / 32; ++q) t += block_sums[q][tid];
    if (gridDim.x == 1) *a.means[tid] = static_cast<float>(t / a.pairs);
    else a.partial[(i64)blockIdx.x * 2 + tid] = t;
  }
}

__global__ void pair_means_kernel(const double* partial, int blocks, i64 pairs, float* loss, float* above) {
  const int k = threadIdx.x >> 5;
  double t = 0.0;
  for (int b = threadIdx.x & 31; b < blocks; b += 32) t += partial[2 * b + k];
  t = sum_warp(t);
  if ((threadIdx.x & 31) == 0) *(k ? above : loss) = static_cast<float>(t / pairs);
}

// ---- host ------------------------------------------------------------------------------------

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

inline bool type_ok(int t) { return t == kFp32 || t == kBf16 || t == kFp16; }

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// A matrix of `rows` rows of `cols` entries: pointer, stride and alignment.
inline int check_matrix(const void* p, i64 ld, i64 rows, i64 cols, int bytes) {
  if (rows > 0 && !p) return CUGO_B200_ERR_ARG;
  if (ld < cols && rows > 1) return CUGO_B200_ERR_ARG;
  return aligned(p, bytes) ? CUGO_B200_OK : CUGO_B200_ERR_ALIGN;
}

int check_rows(const Rows& r, int dtype) {
  if (r.rows < 0 || r.vocab < 1 || !type_ok(dtype)) return CUGO_B200_ERR_ARG;
  if (r.rows > 0 && !r.actions) return CUGO_B200_ERR_ARG;
  if (int rc = check_matrix(r.logits, r.ld, r.rows, r.vocab, type_bytes(dtype))) return rc;
  if (r.ref)
    if (int rc = check_matrix(r.ref, r.ldr, r.rows, r.vocab, type_bytes(dtype))) return rc;
  if (r.legal && r.ldm != 0)  // 0: one mask for all rows
    if (int rc = check_matrix(r.legal, r.ldm, r.rows, r.vocab, 1)) return rc;
  return CUGO_B200_OK;
}

constexpr int kShortShared = 222 << 10;  // bytes of shared memory that a block of short rows may have

// An SM's shared memory for long rows, a block's other part, and the bytes of slots that a
// block of `per_sm` may have.
constexpr int kLongShared = 224 << 10, kLongStatic = 2 << 10;
constexpr int long_slots(int per_sm) { return kLongShared / per_sm - kLongStatic; }

// How a launch goes over long rows.
struct Plan {
  int threads, blocks, parts, slots, shared;
};

// A block per row; few rows get up to 8, each with at least 4,096 entries, and none less
// than 128 threads (300 rows of 4,000 bf16, sums only: four warps 4.3 us, one 5.4 us; 900
// rows 6.6 and 5.8 us).
//
// Sums only: the slots pass the row through, and small blocks spread the rows' reductions
// best: 24 of one warp an SM up to 1,024 vectors (65,536 rows of 2,000 bf16: 97 us, six of
// 128 threads 185 us; 20,000 of 8,192: 68 and 86 us), six of 128 threads above (8,192 rows of
// 16,384 with the loss's terms 68 us, of one warp 72 us; 2,048 of 131,072 96 and 111 us).
//
// With a gradient the slots keep the row for the second look, and what they do not hold is
// read twice.  One warp up to 512 vectors (65,536 rows of 2,000 bf16: 198 us, 128 threads
// 317 us), two up to 1,024 (20,000 rows of 5,000: 116, one warp 122, 128 threads 137 us),
// four up to 2,048; then 256 threads, three blocks an SM; rows above a third of an SM's
// shared memory take 512 threads, two blocks, which hold half as much again each (4,096
// rows of 49,152 bf16: 176 against 188 us); above three quarters of it, two such blocks a
// row (2,048 rows of 131,072: 256 us, one block 268 us, four of 256 threads that hold it all
// 335 us; of 65,536: 270, one block 243 us).  A cluster's barriers cost more than what is
// read again, so no row takes more.
Plan long_plan(i64 rows, int vocab, int size, bool ref, bool stage, bool write) {
  Plan p{};
  const int copies = ref ? 2 : 1;
  const i64 bytes = static_cast<i64>(vocab) * size;
  p.parts = 1;
  p.threads = kLongThreads;
  int per_sm = 3;
  if (write && bytes > kLongShared / 3) {
    p.threads = kWideThreads;
    per_sm = 2;
    if (bytes > kLongShared * 3 / 4) p.parts = 2;
  }
  while (p.parts < 8 && rows * p.parts < kSms && vocab / (2 * p.parts) >= 4096) p.parts *= 2;
  const i64 each = (bytes / 16 + p.parts - 1) / p.parts;  // vectors
  if (!write || each <= 16 * 128) {
    p.threads = 128;
    if (rows > 6 * kSms) {
      if (each <= (write ? 512 : 1024)) p.threads = 32;
      else if (write && each * copies <= 1536) p.threads = 64;
    }
    per_sm = 768 / p.threads;
  }
  if (stage) {
    const i64 want = (each + p.threads - 1) / p.threads, room = long_slots(per_sm) / (p.threads * 16 * copies);
    p.slots = static_cast<int>(want < room ? want : room);
  }
  p.shared = p.slots * p.threads * 16 * copies;
  const i64 most = static_cast<i64>(kSms) * per_sm / p.parts;
  p.blocks = static_cast<int>(rows < most ? rows : most) * p.parts;
  return p;
}

inline i64 round16(i64 n) { return (n + 15) / 16 * 16; }

// Bytes of a run of n rows in shared memory, its last row `width` entries long, with a
// granule for its alignment.
inline i64 run_bytes(i64 n, i64 ld, i64 width, int size) { return round16(((n - 1) * ld + width) * size + 15); }

template <typename T, bool kRef, bool kPolicy, int kThreads>
int launch_planned(const Plan& p, const Rows& r, const Score& o, const Policy& a, cudaStream_t stream) {
  const auto kernel = long_rows_kernel<T, kRef, kPolicy, kThreads>;
  // The most that any plan asks of this kernel, whatever this one does: the attribute is the
  // process's, and another thread may be between its setting and its launch.
  constexpr int kMost = long_slots(kThreads == kWideThreads ? 2 : 3);
  if (p.shared > (40 << 10))
    if (int rc = status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost)))
      return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.blocks);
  cfg.blockDim = dim3(p.threads);
  cfg.dynamicSmemBytes = p.shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts > 1;  // of clusters, even of one block, at most eight blocks share an SM
  return status(cudaLaunchKernelEx(&cfg, kernel, r, o, a, p.slots));
}

template <typename T, bool kRef, bool kPolicy>
int launch_long(const Rows& r, const Score& o, const Policy& a, cudaStream_t stream, int& blocks) {
  // The reference's vectors are copied beside the logits' where both are aligned alike.
  constexpr int kSize = sizeof(T);
  const auto apart = reinterpret_cast<uintptr_t>(r.ref) - reinterpret_cast<uintptr_t>(r.logits);
  const bool alike = apart % 16 == 0 && (r.rows <= 1 || (r.ldr - r.ld) * kSize % 16 == 0);
  const bool stage = !kRef || alike;
  const Plan p = long_plan(r.rows, r.vocab, kSize, kRef, stage, a.dlogits != nullptr);
  blocks = p.blocks;
  if constexpr (kPolicy)
    if (p.threads == kWideThreads) return launch_planned<T, kRef, kPolicy, kWideThreads>(p, r, o, a, stream);
  return launch_planned<T, kRef, kPolicy, kLongThreads>(p, r, o, a, stream);
}

template <typename T, int kLanes, int kPer, bool kRef, bool kPolicy>
int launch_short(const Rows& r, const Score& o, const Policy& a, const Layout& lay, cudaStream_t stream, int& blocks) {
  const auto kernel = short_rows_kernel<T, kLanes, kPer, kRef, kPolicy>;
  const int shared = lay.warp() * kShortWarps;
  if (shared > (44 << 10))  // with the static part, past what needs no opt-in
    if (int rc = status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShortShared)))
      return rc;
  constexpr int kRows = kShortWarps * 32 / kLanes;
  const i64 want = (r.rows + kRows - 1) / kRows;
  int per_sm = (226 << 10) / (shared + (3 << 10));
  if (per_sm > (kPolicy ? 4 : 6)) per_sm = kPolicy ? 4 : 6;  // by registers
  blocks = static_cast<int>(want < per_sm * kSms ? want : per_sm * kSms);
  kernel<<<blocks, 32 * kShortWarps, shared, stream>>>(r, o, a, lay);
  return launch_status();
}

template <typename T, int kLanes, int kPer, bool kRef, bool kPolicy>
Layout short_layout(const Rows& r, const Policy& a) {
  constexpr int kRows = 32 / kLanes, kLong = kLanes * kPer;  // entries that a row is read to
  Layout lay = {};
  // Rows lie one after another: up to 64 bytes between them are copied along (262,144 rows of
  // 179 fp32, 64 bytes apart: 56 us, each by itself 78 us; 400,000 of 60: 54 and 90 us).
  const auto run = [&](i64 ld, int size) { return ld >= r.vocab && (ld - r.vocab) * size <= 64; };
  const bool masks_run = !r.legal || r.ldm == 0 || run(r.ldm, 1);
  lay.apart = kRows > 1 && !(run(r.ld, sizeof(T)) && (!kRef || run(r.ldr, sizeof(T))) && masks_run);
  const auto place = [&](i64 ld, int size, int& pitch) {
    pitch = static_cast<int>(lay.apart ? run_bytes(1, 0, kLong, size) : kRows > 1 ? ld * size : 0);
    return lay.apart ? kRows * pitch : static_cast<int>(run_bytes(kRows, kRows > 1 ? ld : 0, kLong, size));
  };
  lay.logits = place(r.ld, sizeof(T), lay.pitch);
  if (kRef) lay.ref = place(r.ldr, sizeof(T), lay.pitch_ref);
  if (r.legal) lay.legal = place(r.ldm, 1, lay.pitch_legal);
  if (r.ldm == 0) lay.pitch_legal = 0;
  // Between the rows of a wider gradient stands what is not this call's to write.
  if (a.dlogits && (kRows == 1 || a.ldd == a.width)) {
    const i64 grad = run_bytes(kRows, kRows > 1 ? a.ldd : 0, a.width, type_bytes(a.dtype));
    if ((lay.warp() + grad) * kShortWarps <= kShortShared) lay.grad = static_cast<int>(grad);
  }
  return lay;
}

template <typename T, bool kRef, bool kPolicy>
int launch_rows(const Rows& r, const Score& o, const Policy& a, cudaStream_t stream, int& blocks) {
#define CUGO_SHORT(lanes, per)                                                              \
  if (r.vocab <= (lanes) * (per)) {                                                         \
    const Layout lay = short_layout<T, lanes, per, kRef, kPolicy>(r, a);                    \
    return launch_short<T, lanes, per, kRef, kPolicy>(r, o, a, lay, stream, blocks);        \
  }
  CUGO_SHORT(8, 4)
  CUGO_SHORT(8, 8)
  CUGO_SHORT(8, 24)
  CUGO_SHORT(16, 24)
  CUGO_SHORT(32, 32)
#undef CUGO_SHORT
  return launch_long<T, kRef, kPolicy>(r, o, a, stream, blocks);
}

// blocks: how many ran, each with a partial sum.
template <bool kRef, bool kPolicy>
int launch_typed(int dtype, const Rows& r, const Score& o, const Policy& a, cudaStream_t stream, int& blocks) {
  if (dtype == kFp32) return launch_rows<float, kRef, kPolicy>(r, o, a, stream, blocks);
  if (dtype == kBf16) return launch_rows<__nv_bfloat16, kRef, kPolicy>(r, o, a, stream, blocks);
  return launch_rows<__half, kRef, kPolicy>(r, o, a, stream, blocks);
}

inline i64 weight_blocks(i64 rows) {
  const i64 b = (rows + kWeightBlock - 1) / kWeightBlock;
  return b < kSms ? b : kSms;
}

constexpr int kMostBlocks = 24 * kSms;  // of any launch over rows
constexpr i64 kMostEntries = 1 << 30;  // of a row, its zeros behind included: loops over them count in 32 bits

}  // namespace

extern "C" {

int cugo_b200_action_logp(const void* logits, int64_t ld, int32_t dtype, const bool* legal, int64_t ldm,
                          const int64_t* actions, const float* weight, int64_t rows, int64_t vocab,
                          float* logp, float* entropy, float* lse, float* zeros, cudaStream_t stream) {
  if (vocab < 1 || vocab > kMostEntries) return CUGO_B200_ERR_ARG;
  const Rows r{logits, ld, nullptr, 0, legal, ldm, actions, weight, rows, static_cast<int>(vocab)};
  if (int rc = check_rows(r, dtype)) return rc;
  if (rows > 0 && !logp && !entropy && !lse) return CUGO_B200_ERR_ARG;
  if (!aligned(lse, 8)) return CUGO_B200_ERR_ALIGN;
  if (rows == 0) return CUGO_B200_OK;
  const Score o{logp, entropy, reinterpret_cast<float2*>(lse), zeros};
  int blocks;
  return launch_typed<false, false>(dtype, r, o, Policy{}, stream, blocks);
}

int cugo_b200_action_logp_backward(const void* logits, int64_t ld, int32_t dtype, const bool* legal,
                                   int64_t ldm, const int64_t* actions, const float* lse,
                                   const float* entropy, const float* d_logp, const float* d_entropy,
                                   const float* scale, int64_t rows, int64_t vocab, void* dlogits,
                                   int64_t ldd, int32_t grad_dtype, cudaStream_t stream) {
  if (vocab < 1 || vocab > kMostEntries) return CUGO_B200_ERR_ARG;
  const Rows r{logits, ld, nullptr, 0, legal, ldm, actions, nullptr, rows, static_cast<int>(vocab)};
  if (int rc = check_rows(r, dtype)) return rc;
  if (!type_ok(grad_dtype) || (rows > 0 && (!lse || (d_entropy && !entropy)))) return CUGO_B200_ERR_ARG;
  if (int rc = check_matrix(dlogits, ldd, rows, vocab, type_bytes(grad_dtype))) return rc;
  if (!aligned(lse, 8)) return CUGO_B200_ERR_ALIGN;
  if (rows == 0) return CUGO_B200_OK;
  const Back b{reinterpret_cast<const float2*>(lse), entropy, d_logp, d_entropy, scale, dlogits, ldd, grad_dtype};
  const int spans = static_cast<int>((vocab + kSpan - 1) / kSpan);
  const i64 blocks = (rows * spans + kBackWarps - 1) / kBackWarps;
  if (blocks > INT32_MAX) return CUGO_B200_ERR_CAPACITY;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == kFp32) logp_backward_kernel<float><<<grid, 32 * kBackWarps, 0, stream>>>(r, b, spans);
  else if (dtype == kBf16) logp_backward_kernel<__nv_bfloat16><<<grid, 32 * kBackWarps, 0, stream>>>(r, b, spans);
  else logp_backward_kernel<__half><<<grid, 32 * kBackWarps, 0, stream>>>(r, b, spans);
  return launch_status();
}

int64_t cugo_b200_policy_loss_scratch_bytes(int64_t rows) {
  if (rows <= 0) return 0;
  const int64_t blocks = rows < kMostBlocks ? rows * 8 : kMostBlocks;
  return (kSms + (blocks < kMostBlocks ? blocks : kMostBlocks) * kSums) * static_cast<int64_t>(sizeof(double));
}

int cugo_b200_policy_loss(const void* logits, int64_t ld, int32_t dtype, const void* ref_logits, int64_t ldr,
                          const bool* legal, int64_t ldm, const int64_t* actions, const float* logp_old,
                          const float* adv, const float* weight, const float* ref_logp, int64_t rows,
                          int64_t vocab, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                          const float* kl_coef_dev, const float* entropy_coef_dev, float denominator,
                          const float* denominator_dev, float grad_scale, const float* grad_scale_dev, void* dlogits,
                          int64_t ldd, int32_t grad_dtype, int64_t width, float* logp, float* stats, float* loss,
                          void* scratch, int64_t scratch_bytes, cudaStream_t stream) {
  if (vocab < 1 || vocab > kMostEntries || width > kMostEntries) return CUGO_B200_ERR_ARG;
  const Rows r{logits, ld, ref_logits, ldr, legal, ldm, actions, weight, rows, static_cast<int>(vocab)};
  if (int rc = check_rows(r, dtype)) return rc;
  if ((!stats && !dlogits) || (loss && !stats) || (rows > 0 && (!logp_old || !adv)) || (ref_logits && ref_logp))
    return CUGO_B200_ERR_ARG;
  if (!(clip_low >= 0.0f) || !(clip_high >= 0.0f)) return CUGO_B200_ERR_ARG;
  if (dlogits) {
    if (!type_ok(grad_dtype) || width < vocab) return CUGO_B200_ERR_ARG;
    if (int rc = check_matrix(dlogits, ldd, rows, width, type_bytes(grad_dtype))) return rc;
  }
  if (!aligned(scratch, 8)) return CUGO_B200_ERR_ALIGN;
  if (rows == 0) {
    if (stats)
      if (int rc = status(cudaMemsetAsync(stats, 0, (kStats + 1) * sizeof(float), stream))) return rc;
    return loss ? status(cudaMemsetAsync(loss, 0, sizeof(float), stream)) : CUGO_B200_OK;
  }
  if (!scratch || scratch_bytes < cugo_b200_policy_loss_scratch_bytes(rows)) return CUGO_B200_ERR_CAPACITY;
  double* sums = static_cast<double*>(scratch);
  Policy a{};
  a.logp_old = logp_old;
  a.adv = adv;
  a.ref_logp = ref_logp;
  a.low = 1.0f - clip_low;
  a.high = 1.0f + clip_high;
  a.kl_coef = kl_coef;
  a.entropy_coef = entropy_coef;
  a.kl_coef_dev = kl_coef_dev;
  a.entropy_coef_dev = entropy_coef_dev;
  a.denominator = denominator;
  a.denominator_dev = denominator_dev;
  a.grad_scale = grad_scale;
  a.grad_scale_dev = grad_scale_dev;
  a.dlogits = dlogits;
  a.ldd = ldd;
  a.dtype = grad_dtype;
  a.width = static_cast<int>(width);
  a.logp = logp;
  a.partial = stats ? sums + kSms : nullptr;
  if (weight && denominator == 0.0f && !denominator_dev && rows > kWeightBlock) {
    const i64 blocks = weight_blocks(rows);
    weight_sums_kernel<<<static_cast<unsigned>(blocks), 512, 0, stream>>>(weight, rows, (rows + blocks - 1) / blocks,
                                                                         sums);
    if (int rc = launch_status()) return rc;
    a.weight_sums = sums;
    a.n_weight_sums = static_cast<int>(blocks);
  }
  int blocks = 0;
  const int rc = ref_logits ? launch_typed<true, true>(dtype, r, Score{}, a, stream, blocks)
                            : launch_typed<false, true>(dtype, r, Score{}, a, stream, blocks);
  if (rc || !stats) return rc;
  const int groups = blocks > 4 * kSms ? kMeansGroups : 1;
  policy_means_kernel<<<1, 32 * kSums * groups, 0, stream>>>(a, weight, rows, blocks, stats, loss);
  return launch_status();
}

int64_t cugo_b200_preference_pairs_scratch_bytes(int64_t pairs) {
  return pairs > 0 ? 2 * kSms * static_cast<int64_t>(sizeof(double)) : 0;
}

int cugo_b200_preference_pairs(const float* logp, const float* ref_logp, const float* weight, const float* lse,
                               const int64_t* offsets, int64_t pairs, int64_t rows, float beta, float smoothing,
                               int32_t average, float* margin, float* seq_logp, float* d_logp, float* loss,
                               float* accuracy, void* scratch, int64_t scratch_bytes, cudaStream_t stream) {
  if (pairs < 0 || rows < 0 || !loss || !accuracy || !(smoothing >= 0.0f && smoothing <= 1.0f)) return CUGO_B200_ERR_ARG;
  if (pairs > 0 && (!offsets || !margin || !seq_logp)) return CUGO_B200_ERR_ARG;
  if (rows > 0 && (!logp || !ref_logp || !lse)) return CUGO_B200_ERR_ARG;
  if (!aligned(scratch, 8) || !aligned(lse, 8)) return CUGO_B200_ERR_ALIGN;
  if (pairs == 0) {
    if (int rc = status(cudaMemsetAsync(loss, 0, sizeof(float), stream))) return rc;
    return status(cudaMemsetAsync(accuracy, 0, sizeof(float), stream));
  }
  if (!scratch || scratch_bytes < cugo_b200_preference_pairs_scratch_bytes(pairs)) return CUGO_B200_ERR_CAPACITY;
  const Pairs a{logp, ref_logp, weight, reinterpret_cast<const float2*>(lse), offsets, pairs, rows, beta, smoothing,
                average != 0, margin, seq_logp, d_logp, static_cast<double*>(scratch), {loss, accuracy}};
  // Short sequences: a warp per pair; long ones: a block per pair.  By the mean, which the
  // host knows: 256 rows a pair, 16 pairs: warp 10.5 us, block 14.7; 148 pairs: 12.6 and 16.3;
  // 1,000: 15 and 50.  2,048 rows a pair: 35 and 15, 45 and 17, 45 and 52.  One long pair among
  // many short ones is one warp's.
  int blocks;
  if (rows / pairs <= 256) {
    const i64 want = (pairs + kPairThreads / 32 - 1) / (kPairThreads / 32);
    blocks = static_cast<int>(want < kSms ? want : kSms);
    pairs_kernel<32><<<blocks, kPairThreads, 0, stream>>>(a);
  } else {
    blocks = static_cast<int>(pairs < kSms ? pairs : kSms);
    pairs_kernel<kPairThreads><<<blocks, kPairThreads, 0, stream>>>(a);
  }
  if (int rc = launch_status()) return rc;
  if (blocks > 1) pair_means_kernel<<<1, 64, 0, stream>>>(a.partial, blocks, pairs, loss, accuracy);
  return launch_status();
}

}  // extern "C"
