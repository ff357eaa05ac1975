// Head + softmax cross entropy over many classes: shared definitions of the wide (matrix-product) and narrow (one-pass) forms.
//
//   z[p,v] = sum_c w[v,c] h[p,c] + b[v]      p = (n, hw): a pixel or row, P = N HW of them; V classes
//   lse[p] = log sum_v exp z;  nll[p] = lse[p] - z[p,y_p] (0 where y_p is outside [0,V): the row takes no part)
//   G[p,v] = g_p (exp(z - lse) - [v = y_p]);  dh[p,:] = sum_v G w[v,:];  dw[v,:] = sum_p G h[p,:];  db[v] = sum_p G
//
// Numbers on the matrix cores.  Products run on v_mfma_f32_16x16x32_f16 with fp32 accumulation.  Every row of h and of w is scaled by a power of two of its own
// (ex[p], ew[v]: exact, put back in the epilogue) so that its largest element lies in [2^13, 2^14), then split into fp16 planes: an fp32 value into two
// (11 + 11 bits, x = hi + lo to 2^-22 relative or 2^-39 of the row's largest; where lo is kept 2^12 times as large, 2^-51), a bf16 value (8 bits) into one, exactly down to
// 2^-37 of the row's largest.
// A product of two-plane operands is hi hi + hi lo + lo hi (lo lo is below 2^-22): three matrix instructions for fp32 x fp32, two for bf16 x fp32, one for
// bf16 x bf16; G has two planes unless h and w are both bf16.  fp32's own matrix instruction does 1/16 of the fp16 rate, so three of these are 5 times its speed at its accuracy.
#pragma once
#include "ms_common.h"

namespace ms {

typedef _Float16 ms_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 ms_h4 __attribute__((ext_vector_type(4)));
typedef short ms_s4 __attribute__((ext_vector_type(4)));
typedef float ms_f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kCeTopExp = 13;         // scaled rows: largest magnitude in [2^13, 2^14)
constexpr int kCePad = 256;           // rows of the packed operands are padded to whole tiles

// the exponent of the power of two that `amax` is divided by to lie in [2^13, 2^14); 0 for a row of zeros or one with an infinity / NaN (it stays one), no smaller than 2^-100
__device__ __forceinline__ int ce_exponent(float amax) {
  const unsigned b = __float_as_uint(amax);
  if (b >= 0x7F800000u || b == 0u) return 0;
  const int e = (int)(b >> 23) - 127;                 // (a subnormal reads as -127: the clamp below)
  return max(e - kCeTopExp, -100);
}
__device__ __forceinline__ float ce_pow2(int e) { return __uint_as_float((unsigned)(min(max(e, -126), 127) + 127) << 23); }

// log2(x) - less, x >= 0 (less: a whole number): the exponent apart from the logarithm of the mantissa in [1, 2).  The log instruction cuts its result off: of x = 2^9 .. 2^13 it would lie half a step of 8 .. 16
// (4.8e-7) too low on average, and the gradients of a few thousand rows add such a bias up (db 1.2e-6 instead of 1e-7 off).
__device__ __forceinline__ float ce_log2(float x, float less = 0.f) {
  const int e = __builtin_amdgcn_frexp_expf(x) - 1;
  return ((float)e - less) + __builtin_amdgcn_logf(__builtin_amdgcn_ldexpf(x, -e));
}

// A log-sum L (in log2) is subtracted from logits as the fp32 value next to it; with what that leaves over, d = L - fp32(L) and c = 2^d, exp2(z - L) = exp2(z - fp32(L)) / c and
// G = g (exp2(z - L) - hot) = g / c (exp2(z - fp32(L)) - c hot): the rounding of a log-sum of 40 (2^-19) costs nothing, and a row that is sure of its label keeps what is left of 1 - p.
__device__ __forceinline__ float ce_rest(float m, float lg, float rounded) { return (m - rounded) + lg; }      // L = m + lg
__device__ __forceinline__ float ce_rest_nat(float lse, float rounded) {                                       // L = lse log2(e)
  const float d = __builtin_fmaf(lse, kLog2e, -rounded) + lse * 1.92596299112661746e-8f;
  return fminf(fmaxf(d, -1.f), 1.f);                  // (beyond 2^24 the fp32 log-sum itself is whole units off)
}
__device__ __forceinline__ float ce_lse_nat(float m, float lg) { return (float)(((double)m + (double)lg) * 0.69314718055994530942); }

// A product as fp32 holds it, for what is split: left to itself the compiler rounds the product to fp16 straight (v_fma_mixlo) where it forms hi and by way of fp32 (v_cvt) where it
// forms lo, and for one element in some thousands the two planes then belong to different hi (2^-11 off).
__device__ __forceinline__ float ce_rounded(float x) {
  asm("" : "+v"(x));
  return x;
}

// {hi, lo} planes of a scaled value
__device__ __forceinline__ void ce_split(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// {hi, 2^12 lo}: the low plane keeps its 11 bits far below the high plane's lowest step (values to 2^-37 instead of 2^-25).  A product's low pairs are summed first and that sum
// brought back by 2^-12 before the high pair is added.
constexpr int kCeLoExp = 12;
__device__ __forceinline__ void ce_split_far(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)((x - (float)hi) * (float)(1 << kCeLoExp));
}

// ... {hi, lo} of eight at once: conversions in pairs, and x - hi as one multiply-add that reads the half-precision operand as it is (the factor -1 is hidden from the compiler, which
// would make a conversion and a subtraction of it; 104 classes x 16 channels x 1 M pixels 168 -> 163 us)
typedef _Float16 ms_h2 __attribute__((ext_vector_type(2)));
typedef float ms_f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void ce_split8(ms_f4 a, ms_f4 b, ms_h8& hi, ms_h8& lo) {
  union { ms_h2 p[4]; ms_h8 h; } H, L;
  float neg1 = -1.f;
  asm("" : "+s"(neg1));
  const ms_f2 v[4] = {{a[0], a[1]}, {a[2], a[3]}, {b[0], b[1]}, {b[2], b[3]}};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    H.p[i] = __builtin_convertvector(v[i], ms_h2);
    const ms_f2 r = {__builtin_fmaf((float)H.p[i][0], neg1, v[i][0]), __builtin_fmaf((float)H.p[i][1], neg1, v[i][1])};
    L.p[i] = __builtin_convertvector(r, ms_h2);
  }
  hi = H.h; lo = L.h;
}

// ... {hi, 2^12 lo} of eight at once: 2^12 (x - hi) as a multiply-add of the half-precision operand and 2^12 x
__device__ __forceinline__ void ce_split8_far(ms_f4 a, ms_f4 b, ms_h8& hi, ms_h8& lo) {
  union { ms_h2 p[4]; ms_h8 h; } H, L;
  float neg = -(float)(1 << kCeLoExp);
  asm("" : "+s"(neg));
  const ms_f2 v[4] = {{a[0], a[1]}, {a[2], a[3]}, {b[0], b[1]}, {b[2], b[3]}};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    H.p[i] = __builtin_convertvector(v[i], ms_h2);
    const ms_f2 r = {__builtin_fmaf((float)H.p[i][0], neg, v[i][0] * (float)(1 << kCeLoExp)), __builtin_fmaf((float)H.p[i][1], neg, v[i][1] * (float)(1 << kCeLoExp))};
    L.p[i] = __builtin_convertvector(r, ms_h2);
  }
  hi = H.h; lo = L.h;
}

}  // namespace ms
