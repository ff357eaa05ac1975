// Activation checkpoints in 8 bits, and the backward of BatchNorm + LeakyReLU that reads them.
//
// A plane (n, c) of HW elements is cut into blocks of kA8Block = 256 (the last one may be shorter).  With centre_c below, d = x - centre_c in 64 bits:
//   s = fp32(fp32(max |d|) / 127) with the quotient in 64 bits,  q = rint(d / s) in [-127, 127], and where that is 0 although d is not, q = sign(d):  x' = centre_c + q s.
// |x' - x| <= s/2, or < s where the sign was kept.  A sign is never lost, so the activation's mask needs no rounded value:
//   centre_c = the zero of the BatchNorm's output, -shift/scale, where it lies within 4 standard deviations of the mean (else the mean; 0 without a record):
//   there sign(scale x' + shift) = sign(scale) sign(q) = sign(scale x + shift) exactly.  Taking the centre out also spends no step on a channel's offset.
// A block whose max is below 2^-120 is kept as zeros (s = 0); one with an infinity or a NaN gets s = NaN, and everything read from it is NaN.
//
// The arithmetic per element is 64-bit where a step's border is decided (one subtraction, product and rint: on this chip a double operation costs what two float
// ones do, and the kernels wait for memory): the same value falls on the same side of a border whatever form computes it.
//
// All of these kernels are bound by HBM; the notes at each say what it moves.
#include <algorithm>
#include "ms_common.h"
#include "maxstyle_hip.h"

namespace ms {

constexpr int kA8Block = 256;        // elements per scale: one wave's 64 lanes x 4; 8.125 bits an element (64 would cost 8.5 and gain 0.2 bit of step on normal data)
constexpr int kA8Threads = 256;

struct A8Centre { double c; bool zero; };
__device__ __forceinline__ A8Centre a8_centre(const float4* __restrict__ coef, int c) {
  if (coef == nullptr) return A8Centre{0.0, false};
  const float4 f = coef[c];            // {scale, shift, mean, invstd}
  const double t = -(double)f.y / (double)f.x, m = (double)f.z;
  const bool z = fabs(t - m) * (double)f.w <= 4.0;      // (false for a NaN: scale = 0)
  return A8Centre{z ? t : m, z};
}

__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 64));
  return v;
}

// s and 1/s of a block from the bits of max |d| (a NaN's bits are above an infinity's, and both above every number)
__device__ __forceinline__ float a8_scale(unsigned amax_bits, double& rinv) {
  if (amax_bits >= 0x7F800000u) { rinv = 0.0; return __uint_as_float(0x7FC00000u); }
  const float s = (float)((double)__uint_as_float(amax_bits) / 127.0);
  if (s < 7.52316385e-37f) { rinv = 0.0; return 0.f; }      // 2^-120
  rinv = 1.0 / (double)s;
  return s;
}
__device__ __forceinline__ int a8_quant(double d, double rinv, float s) {
  const double t = d * rinv;
  double r = rint(t);
  if (fabs(fabs(t - r) - 0.5) < 1e-9 && rinv != 0.0) r = rint(d / (double)s);      // next to a border: the quotient itself decides (rare)
  int q = (int)r;
  if (q == 0 && rinv != 0.0) q = d > 0.0 ? 1 : (d < 0.0 ? -1 : 0);
  return q;
}

// One wave takes kPackBlocks consecutive blocks of a plane (all their loads in flight before the first reduction).  Moves 4 (2) + 1 bytes an element.
constexpr int kPackBlocks = 4;
template <typename AT, bool VEC>
__global__ __launch_bounds__(kA8Threads) void act8_pack_kernel(const void* __restrict__ x, const float4* __restrict__ coef, int8_t* __restrict__ q, float* __restrict__ s,
                                                               int C, int HW, int nb, int items, int total) {
  using IO = ActIO<AT>;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int item = blockIdx.x * (kA8Threads / 64) + wave;
  if (item >= total) return;
  const int plane = item / items, b0 = (item - plane * items) * kPackBlocks;
  const double ctr = a8_centre(coef, plane % C).c;
  const size_t base = (size_t)plane * HW;
  float v[kPackBlocks][4];
#pragma unroll
  for (int b = 0; b < kPackBlocks; ++b) {
    const int e0 = (b0 + b) * kA8Block;
    if (VEC) {
      const int e = e0 + lane * 4;
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if (e < HW) t = IO::ld4(x, base + e);
      v[b][0] = t.x; v[b][1] = t.y; v[b][2] = t.z; v[b][3] = t.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) { const int e = e0 + j * 64 + lane; v[b][j] = e < HW ? IO::ld1(x, base + e) : 0.f; }
    }
  }
#pragma unroll
  for (int b = 0; b < kPackBlocks; ++b) {
    if (b0 + b >= nb) break;
    const int e0 = (b0 + b) * kA8Block;
    unsigned am = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = VEC ? e0 + lane * 4 + j : e0 + j * 64 + lane;
      const unsigned bits = __float_as_uint((float)fabs((double)v[b][j] - ctr));
      am = max(am, e < HW ? bits : 0u);
    }
    am = wave_max_u(am);
    double rinv;
    const float sc = a8_scale(am, rinv);
    if (lane == 0) s[(size_t)plane * nb + b0 + b] = sc;
    int k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = a8_quant((double)v[b][j] - ctr, rinv, sc);
    if (VEC) {
      const int e = e0 + lane * 4;
      if (e < HW) *reinterpret_cast<unsigned*>(q + base + e) = (k[0] & 255) | ((k[1] & 255) << 8) | ((k[2] & 255) << 16) | ((unsigned)(k[3] & 255) << 24);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) { const int e = e0 + j * 64 + lane; if (e < HW) q[base + e] = (int8_t)k[j]; }
    }
  }
}

// x' = centre + q s, rounded once.  Moves 1 + 4 (2) bytes an element.
template <typename AT, bool VEC>
__global__ __launch_bounds__(kA8Threads) void act8_unpack_kernel(const int8_t* __restrict__ q, const float* __restrict__ s, const float4* __restrict__ coef,
                                                                 void* __restrict__ x, int C, int HW, int nb, int items, int total) {
  using IO = ActIO<AT>;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int item = blockIdx.x * (kA8Threads / 64) + wave;
  if (item >= total) return;
  const int plane = item / items, b0 = (item - plane * items) * kPackBlocks;
  const double ctr = a8_centre(coef, plane % C).c;
  const size_t base = (size_t)plane * HW;
#pragma unroll
  for (int b = 0; b < kPackBlocks; ++b) {
    if (b0 + b >= nb) break;
    const double sc = (double)s[(size_t)plane * nb + b0 + b];
    const int e0 = (b0 + b) * kA8Block;
    if (VEC) {
      const int e = e0 + lane * 4;
      if (e < HW) {
        const int w = *reinterpret_cast<const int*>(q + base + e);
        IO::st4(x, base + e, make_float4((float)(ctr + (double)(int8_t)w * sc), (float)(ctr + (double)(int8_t)(w >> 8) * sc),
                                         (float)(ctr + (double)(int8_t)(w >> 16) * sc), (float)(ctr + (double)(w >> 24) * sc)));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) { const int e = e0 + j * 64 + lane; if (e < HW) IO::st1(x, base + e, (float)(ctr + (double)q[base + e] * sc)); }
    }
  }
}

// What the backward needs of a channel: the mask rule and the offset of x' - mean = off + q s
struct A8Chan { double ctr, sc, zc; float off; int mode; };      // mode 0: mask from ref_q | +1 / -1 / 2: sign(q), sign(-q), never (scale = 0 cannot be centred) | 3: sc * (q s) + zc > 0
__device__ __forceinline__ A8Chan a8_chan(const float4* __restrict__ coef, int c, bool has_ref) {
  const A8Centre t = a8_centre(coef, c);
  const float4 f = coef[c];
  A8Chan a;
  a.ctr = t.c; a.sc = (double)f.x; a.zc = (double)f.x * t.c + (double)f.y;
  a.off = (float)(t.c - (double)f.z);
  a.mode = has_ref ? 0 : (t.zero ? (f.x > 0.f ? 1 : -1) : 3);
  return a;
}
__device__ __forceinline__ bool a8_on(const A8Chan& a, int q, int ref, float s) {
  if (a.mode == 0) return ref > 0;
  if (a.mode == 1) return q > 0;
  if (a.mode == -1) return q < 0;
  return a.sc * ((double)q * (double)s) + a.zc > 0.0;
}

// 4 consecutive elements (VEC) or 1: g' = g * (on ? 1 : slope), x' - mean
template <typename AT, bool VEC> struct A8Vec;
template <typename AT> struct A8Vec<AT, true> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void ldg(const void* g, size_t e, float* o) { const float4 t = ActIO<AT>::ld4(g, e); o[0] = t.x; o[1] = t.y; o[2] = t.z; o[3] = t.w; }
  static __device__ __forceinline__ void stg(void* g, size_t e, const float* o) { ActIO<AT>::st4(g, e, make_float4(o[0], o[1], o[2], o[3])); }
  static __device__ __forceinline__ int ldq(const int8_t* q, size_t e) { return *reinterpret_cast<const int*>(q + e); }
  static __device__ __forceinline__ int get(int w, int j) { return (int)(int8_t)(w >> (8 * j)); }
};
template <typename AT> struct A8Vec<AT, false> {
  static constexpr int n = 1;
  static __device__ __forceinline__ void ldg(const void* g, size_t e, float* o) { o[0] = ActIO<AT>::ld1(g, e); }
  static __device__ __forceinline__ void stg(void* g, size_t e, const float* o) { ActIO<AT>::st1(g, e, o[0]); }
  static __device__ __forceinline__ int ldq(const int8_t* q, size_t e) { return q[e]; }
  static __device__ __forceinline__ int get(int w, int) { return w; }
};

// First pass: partial sums of g' and g' (x' - mean) of each (plane, segment) -> part[c][n S + s], the layout ms_bn_bwd_full reads; with OUT optionally g' and x'
// themselves (the training engine's convolutions read both).
template <typename AT, bool VEC, bool OUT>
__global__ __launch_bounds__(kA8Threads) void act8_bwd_reduce_kernel(const void* __restrict__ gin, const int8_t* __restrict__ ref, const int8_t* __restrict__ q,
                                                                     const float* __restrict__ s, const float4* __restrict__ coef, void* __restrict__ gout, void* __restrict__ uout,
                                                                     float2* __restrict__ part, int C, int HW, int nb, int seg, int S, int N, float slope) {
  using V = A8Vec<AT, VEC>;
  __shared__ double redd[16];
  const int si = blockIdx.x % S, pl = blockIdx.x / S;
  const int n = pl / C, c = pl - n * C;
  const size_t plane = (size_t)pl, base = plane * HW;
  const A8Chan a = a8_chan(coef, c, ref != nullptr);
  const int beg = si * seg, end = min(HW, beg + seg);
  double d1 = 0.0, d2 = 0.0;            // (in fp32 a thread's 64 terms left dgamma and dbeta 1.6e-7 off; the additions are hidden behind the loads)
#pragma unroll 4
  for (int i = beg + (int)threadIdx.x * V::n; i < end; i += kA8Threads * V::n) {
    float g[4], s1 = 0.f, s2 = 0.f;
    V::ldg(gin, base + i, g);
    const int w = V::ldq(q, base + i), rw = ref != nullptr ? V::ldq(ref, base + i) : 0;
    const float sc = s[plane * nb + (i >> 8)];
    float o[4], u[4];
#pragma unroll
    for (int j = 0; j < V::n; ++j) {
      const int k = V::get(w, j);
      o[j] = a8_on(a, k, V::get(rw, j), sc) ? g[j] : g[j] * slope;
      s1 += o[j];
      s2 += o[j] * (a.off + (float)k * sc);
      if (OUT && uout != nullptr) u[j] = (float)(a.ctr + (double)k * (double)sc);
    }
    d1 += (double)s1; d2 += (double)s2;
    if (OUT && gout != nullptr) V::stg(gout, base + i, o);
    if (OUT && uout != nullptr) V::stg(uout, base + i, u);
  }
  d1 = block_sum_d(d1, redd);
  d2 = block_sum_d(d2, redd);
  if (threadIdx.x == 0) part[(size_t)c * ((size_t)N * S) + (size_t)n * S + si] = make_float2((float)d1, (float)d2);
}

// du = scale (g' - S1/M - (x' - mean) invstd^2 S2/M)
struct A8Coef { float sc, k1, k2; };
__device__ __forceinline__ A8Coef a8_coef(const float4 f, double s1, double s2, double count) {
  return A8Coef{f.x, (float)(s1 / count), (float)(s2 * (double)f.w * (double)f.w / count)};
}

// Second pass: every workgroup sums its channel's partials again (N S of them, fixed order, 64 bits), then writes its segment of du.  Channels in groups whose data stays
// in the last-level cache between the passes were slower at every group size (24 .. 160 MB: 567 .. 224 us against 194 in one group).
template <typename AT, bool VEC>
__global__ __launch_bounds__(kA8Threads) void act8_bwd_apply_kernel(const void* __restrict__ gin, const int8_t* __restrict__ ref, const int8_t* __restrict__ q,
                                                                    const float* __restrict__ s, const float4* __restrict__ coef, const float2* __restrict__ part,
                                                                    void* __restrict__ du, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                    int C, int HW, int nb, int seg, int S, int N, float slope) {
  using V = A8Vec<AT, VEC>;
  __shared__ double redd[16];
  const int id = gridDim.x - 1 - blockIdx.x;        // from the end: what the first pass read last is still in the last-level cache (193 -> 188 us at 16x64x256x256)
  const int si = id % S, pl = id / S;
  const int n = pl / C, c = pl - n * C;
  const size_t plane = (size_t)pl, base = plane * HW;
  const A8Chan a = a8_chan(coef, c, ref != nullptr);
  const float4 f = coef[c];
  double d1 = 0.0, d2 = 0.0;
  const int np = N * S;
  const float2* row = part + (size_t)c * np;
  for (int i = threadIdx.x; i < np; i += kA8Threads) { const float2 t = row[i]; d1 += (double)t.x; d2 += (double)t.y; }
  d1 = block_sum_d(d1, redd);
  d2 = block_sum_d(d2, redd);
  if (n == 0 && si == 0 && threadIdx.x == 0) { dgamma[c] = (float)(d2 * (double)f.w); dbeta[c] = (float)d1; }
  const A8Coef k = a8_coef(f, d1, d2, (double)N * HW);
  const int beg = si * seg, end = min(HW, beg + seg);
#pragma unroll 4
  for (int i = beg + (int)threadIdx.x * V::n; i < end; i += kA8Threads * V::n) {
    float g[4];
    V::ldg(gin, base + i, g);
    const int w = V::ldq(q, base + i), rw = ref != nullptr ? V::ldq(ref, base + i) : 0;
    const float sc = s[plane * nb + (i >> 8)];
#pragma unroll
    for (int j = 0; j < V::n; ++j) {
      const int kq = V::get(w, j);
      const float o = a8_on(a, kq, V::get(rw, j), sc) ? g[j] : g[j] * slope;
      g[j] = k.sc * ((o - k.k1) - (a.off + (float)kq * sc) * k.k2);
    }
    V::stg(du, base + i, g);
  }
}

// Both passes in one for channels of up to kA8One elements: a workgroup holds its channel in registers - g and the checkpoint are read once, and it is one launch
// (the deep levels: 4x128x12x12 4.3 us against 8.4 in two launches, and 3 us of host time less).
constexpr int kA8One = 16384, kA8Per = 16;       // elements of a channel; of a thread (1024 threads, or 256 up to 4096 elements)
template <typename AT, bool VEC>
__global__ __launch_bounds__(1024) void act8_bwd_one_kernel(const void* __restrict__ gin, const int8_t* __restrict__ ref, const int8_t* __restrict__ q, const float* __restrict__ s,
                                                            const float4* __restrict__ coef, void* __restrict__ du, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                            int C, int HW, int nb, int N, float slope) {
  using V = A8Vec<AT, VEC>;
  constexpr int R = kA8Per / V::n;
  __shared__ double redd[16];
  const int c = blockIdx.x, total = N * HW / V::n;
  const A8Chan a = a8_chan(coef, c, ref != nullptr);
  float g[R][V::n], sc[R];
  int w[R], rw[R];
  size_t at[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int i = min(k * (int)blockDim.x + (int)threadIdx.x, total - 1) * V::n, n = i / HW, e = i - n * HW;        // (clamped: the loads need no branch)
    const size_t plane = (size_t)n * C + c;
    at[k] = plane * HW + e;
    float t[4];
    V::ldg(gin, at[k], t);
#pragma unroll
    for (int j = 0; j < V::n; ++j) g[k][j] = t[j];
    w[k] = V::ldq(q, at[k]);
    rw[k] = ref != nullptr ? V::ldq(ref, at[k]) : 0;
    sc[k] = s[plane * nb + (e >> 8)];
  }
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    if (k * (int)blockDim.x + (int)threadIdx.x >= total) continue;
#pragma unroll
    for (int j = 0; j < V::n; ++j) {
      const int kq = V::get(w[k], j);
      g[k][j] = a8_on(a, kq, V::get(rw[k], j), sc[k]) ? g[k][j] : g[k][j] * slope;
      s1 += g[k][j];
      s2 += g[k][j] * (a.off + (float)kq * sc[k]);
    }
  }
  const double d1 = block_sum_d((double)s1, redd), d2 = block_sum_d((double)s2, redd);
  const float4 f = coef[c];
  if (threadIdx.x == 0) { dgamma[c] = (float)(d2 * (double)f.w); dbeta[c] = (float)d1; }
  const A8Coef k2 = a8_coef(f, d1, d2, (double)N * HW);
#pragma unroll
  for (int k = 0; k < R; ++k) {
    if (k * (int)blockDim.x + (int)threadIdx.x >= total) continue;
    float t[4];
#pragma unroll
    for (int j = 0; j < V::n; ++j) t[j] = k2.sc * ((g[k][j] - k2.k1) - (a.off + (float)V::get(w[k], j) * sc[k]) * k2.k2);
    V::stg(du, at[k], t);
  }
}

struct A8Split { int seg, S; };
static A8Split a8_split(long planes, int HW) {
  // segments of 1024 elements (256 threads x 4) up to 16384: long ones amortise the second pass's prologue, short ones fill the chip from few planes
  int seg = 1024;
  while (seg < 16384 && planes * cdiv(HW, seg) > 4096) seg <<= 1;
  return A8Split{seg, cdiv(HW, seg)};
}

static int a8_check(int N, int C, int HW, const char* who) {
  if (N < 1 || C < 1 || HW < 1) { set_error("%s: invalid shape", who); return MS_ERR_INVALID; }
  if ((long long)N * C * cdiv(HW, 1024) >= (1LL << 31) - 8 || HW > 0x7FFFFFFF - 32768) { set_error("%s: more than 2^31 segments of 1024 elements", who); return MS_ERR_INVALID; }
  return MS_OK;
}
// A launch holds less than 2^32 threads: 2^24 segments of 256 threads, 2^26 items of one wave.  (Planes of a few elements reach it first.)
static int a8_launchable(long long groups, long long most, const char* who) {
  if (groups < most) return MS_OK;
  set_error("%s: more than 2^24 segments (or 2^26 runs of 1024 elements) of the planes", who);
  return MS_ERR_INVALID;
}
static int a8_aligned(const float* coef4, const void* part, const char* who) {
  if (!aligned16(coef4) || (reinterpret_cast<uintptr_t>(part) & 7u)) { set_error("%s: coef4 must be 16-byte aligned, partial sums 8-byte", who); return MS_ERR_ALIGN; }
  return MS_OK;
}
static bool a8_al(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename AT>
static int act8_pack_impl(const void* x, const float* coef4, int8_t* q, float* s, int N, int C, int HW, void* stream) {
  if (int e = a8_check(N, C, HW, "ms_act8_pack")) return e;
  if (int e = a8_launchable((long long)N * C * cdiv(cdiv(HW, kA8Block), kPackBlocks), 1LL << 26, "ms_act8_pack")) return e;
  if (x == nullptr || q == nullptr || s == nullptr) { set_error("ms_act8_pack: null pointer"); return MS_ERR_INVALID; }
  if (int e = a8_aligned(coef4, nullptr, "ms_act8_pack")) return e;
  const int nb = cdiv(HW, kA8Block), items = cdiv(nb, kPackBlocks), total = N * C * items;
  const bool vec = HW % 4 == 0 && a8_al(x, 4 * ActIO<AT>::kBytes) && a8_al(q, 4);      // rows of whole 4-element words; otherwise element by element
  dim3 grid(cdiv(total, kA8Threads / 64)), block(kA8Threads);
  if (vec) MS_LAUNCH((act8_pack_kernel<AT, true>), grid, block, 0, (hipStream_t)stream, x, (const float4*)coef4, q, s, C, HW, nb, items, total);
  else MS_LAUNCH((act8_pack_kernel<AT, false>), grid, block, 0, (hipStream_t)stream, x, (const float4*)coef4, q, s, C, HW, nb, items, total);
  return check_launch("act8_pack");
}
template <typename AT>
static int act8_unpack_impl(const int8_t* q, const float* s, const float* coef4, void* x, int N, int C, int HW, void* stream) {
  if (int e = a8_check(N, C, HW, "ms_act8_unpack")) return e;
  if (int e = a8_launchable((long long)N * C * cdiv(cdiv(HW, kA8Block), kPackBlocks), 1LL << 26, "ms_act8_unpack")) return e;
  if (x == nullptr || q == nullptr || s == nullptr) { set_error("ms_act8_unpack: null pointer"); return MS_ERR_INVALID; }
  if (int e = a8_aligned(coef4, nullptr, "ms_act8_unpack")) return e;
  const int nb = cdiv(HW, kA8Block), items = cdiv(nb, kPackBlocks), total = N * C * items;
  const bool vec = HW % 4 == 0 && a8_al(x, 4 * ActIO<AT>::kBytes) && a8_al(q, 4);
  dim3 grid(cdiv(total, kA8Threads / 64)), block(kA8Threads);
  if (vec) MS_LAUNCH((act8_unpack_kernel<AT, true>), grid, block, 0, (hipStream_t)stream, q, s, (const float4*)coef4, x, C, HW, nb, items, total);
  else MS_LAUNCH((act8_unpack_kernel<AT, false>), grid, block, 0, (hipStream_t)stream, q, s, (const float4*)coef4, x, C, HW, nb, items, total);
  return check_launch("act8_unpack");
}

template <typename AT>
static bool a8_bwd_vec(const void* g, const int8_t* ref, const int8_t* q, const void* o1, const void* o2, int HW) {
  const unsigned b = 4 * ActIO<AT>::kBytes;
  return HW % 4 == 0 && a8_al(g, b) && a8_al(o1, b) && a8_al(o2, b) && a8_al(q, 4) && a8_al(ref, 4);
}
template <typename AT>
static int act8_bwd_reduce_impl(const void* gin, const int8_t* ref, const int8_t* q, const float* s, const float* coef4, void* gout, void* uout, float* part2,
                                int N, int C, int HW, float slope, void* stream) {
  if (int e = a8_check(N, C, HW, "ms_act8_bwd_reduce")) return e;
  if (gin == nullptr || q == nullptr || s == nullptr || coef4 == nullptr || part2 == nullptr) { set_error("ms_act8_bwd_reduce: null pointer"); return MS_ERR_INVALID; }
  if (int e = a8_aligned(coef4, part2, "ms_act8_bwd_reduce")) return e;
  const A8Split sp = a8_split((long)N * C, HW);
  if (int e = a8_launchable((long long)N * C * sp.S, 1LL << 24, "ms_act8_bwd_reduce")) return e;
  dim3 grid(N * C * sp.S), block(kA8Threads);
  const int nb = cdiv(HW, kA8Block);
  hipStream_t st = (hipStream_t)stream;
  if (a8_bwd_vec<AT>(gin, ref, q, gout, uout, HW))
    MS_LAUNCH((act8_bwd_reduce_kernel<AT, true, true>), grid, block, 0, st, gin, ref, q, s, (const float4*)coef4, gout, uout, (float2*)part2, C, HW, nb, sp.seg, sp.S, N, slope);
  else
    MS_LAUNCH((act8_bwd_reduce_kernel<AT, false, true>), grid, block, 0, st, gin, ref, q, s, (const float4*)coef4, gout, uout, (float2*)part2, C, HW, nb, sp.seg, sp.S, N, slope);
  return check_launch("act8_bwd_reduce");
}

template <typename AT>
static int act8_bn_act_bwd_impl(const void* g, const int8_t* ref, const int8_t* q, const float* s, const float* coef4, void* du, float* dgamma, float* dbeta,
                                int N, int C, int HW, float slope, void* ws, size_t ws_bytes, void* stream) {
  if (int e = a8_check(N, C, HW, "ms_act8_bn_act_bwd")) return e;
  if (g == nullptr || q == nullptr || s == nullptr || coef4 == nullptr || du == nullptr || dgamma == nullptr || dbeta == nullptr) {
    set_error("ms_act8_bn_act_bwd: null pointer"); return MS_ERR_INVALID;
  }
  if (ws == nullptr || ws_bytes < ms_act8_bwd_ws_bytes(N, C, HW)) { set_error("ms_act8_bn_act_bwd: workspace too small"); return MS_ERR_WORKSPACE; }
  if (int e = a8_aligned(coef4, ws, "ms_act8_bn_act_bwd")) return e;
  const A8Split sp = a8_split((long)N * C, HW);
  const int nb = cdiv(HW, kA8Block);
  hipStream_t st = (hipStream_t)stream;
  const bool vec = a8_bwd_vec<AT>(g, ref, q, du, nullptr, HW);
  if ((long long)N * HW <= kA8One) {
    const dim3 b1(N * HW <= kA8One / 4 ? 256 : 1024);
    if (vec) MS_LAUNCH((act8_bwd_one_kernel<AT, true>), dim3(C), b1, 0, st, g, ref, q, s, (const float4*)coef4, du, dgamma, dbeta, C, HW, nb, N, slope);
    else MS_LAUNCH((act8_bwd_one_kernel<AT, false>), dim3(C), b1, 0, st, g, ref, q, s, (const float4*)coef4, du, dgamma, dbeta, C, HW, nb, N, slope);
    return check_launch("act8_bwd_one");
  }
  if (int e = a8_launchable((long long)N * C * sp.S, 1LL << 24, "ms_act8_bn_act_bwd")) return e;
  const dim3 block(kA8Threads), grid(N * C * sp.S);
#define A8_ARGS(PART) st, g, ref, q, s, (const float4*)coef4, PART
  if (vec) MS_LAUNCH((act8_bwd_reduce_kernel<AT, true, false>), grid, block, 0, A8_ARGS(nullptr), nullptr, (float2*)ws, C, HW, nb, sp.seg, sp.S, N, slope);
  else MS_LAUNCH((act8_bwd_reduce_kernel<AT, false, false>), grid, block, 0, A8_ARGS(nullptr), nullptr, (float2*)ws, C, HW, nb, sp.seg, sp.S, N, slope);
  if (int e = check_launch("act8_bwd_reduce")) return e;
  if (vec) MS_LAUNCH((act8_bwd_apply_kernel<AT, true>), grid, block, 0, A8_ARGS((const float2*)ws), du, dgamma, dbeta, C, HW, nb, sp.seg, sp.S, N, slope);
  else MS_LAUNCH((act8_bwd_apply_kernel<AT, false>), grid, block, 0, A8_ARGS((const float2*)ws), du, dgamma, dbeta, C, HW, nb, sp.seg, sp.S, N, slope);
#undef A8_ARGS
  return check_launch("act8_bwd_apply");
}
}  // namespace ms

extern "C" int ms_act8_block(void) { return ms::kA8Block; }
extern "C" int ms_act8_pack(const float* x, const float* coef4, int8_t* q, float* s, int N, int C, int HW, void* stream) {
  return ms::act8_pack_impl<float>(x, coef4, q, s, N, C, HW, stream);
}
extern "C" int ms_act8_pack_bf16(const uint16_t* x, const float* coef4, int8_t* q, float* s, int N, int C, int HW, void* stream) {
  return ms::act8_pack_impl<ms::ms_bf16>(x, coef4, q, s, N, C, HW, stream);
}
extern "C" int ms_act8_unpack(const int8_t* q, const float* s, const float* coef4, float* x, int N, int C, int HW, void* stream) {
  return ms::act8_unpack_impl<float>(q, s, coef4, x, N, C, HW, stream);
}
extern "C" int ms_act8_unpack_bf16(const int8_t* q, const float* s, const float* coef4, uint16_t* x, int N, int C, int HW, void* stream) {
  return ms::act8_unpack_impl<ms::ms_bf16>(q, s, coef4, x, N, C, HW, stream);
}
extern "C" int ms_act8_bwd_parts(int N, int C, int HW) { return N * ms::a8_split((long)N * C, HW).S; }
extern "C" int ms_act8_bwd_reduce(const float* gin, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, float* gout, float* uout, float* part2,
                                  int N, int C, int HW, float slope, void* stream) {
  return ms::act8_bwd_reduce_impl<float>(gin, ref_q, q, s, coef4, gout, uout, part2, N, C, HW, slope, stream);
}
extern "C" int ms_act8_bwd_reduce_bf16(const uint16_t* gin, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, uint16_t* gout, uint16_t* uout, float* part2,
                                       int N, int C, int HW, float slope, void* stream) {
  return ms::act8_bwd_reduce_impl<ms::ms_bf16>(gin, ref_q, q, s, coef4, gout, uout, part2, N, C, HW, slope, stream);
}
extern "C" size_t ms_act8_bwd_ws_bytes(int N, int C, int HW) { return (size_t)C * ms_act8_bwd_parts(N, C, HW) * sizeof(float2); }
extern "C" int ms_act8_bn_act_bwd(const float* g, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, float* du, float* dgamma, float* dbeta,
                                  int N, int C, int HW, float slope, void* ws, size_t ws_bytes, void* stream) {
  return ms::act8_bn_act_bwd_impl<float>(g, ref_q, q, s, coef4, du, dgamma, dbeta, N, C, HW, slope, ws, ws_bytes, stream);
}
extern "C" int ms_act8_bn_act_bwd_bf16(const uint16_t* g, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, uint16_t* du, float* dgamma, float* dbeta,
                                       int N, int C, int HW, float slope, void* ws, size_t ws_bytes, void* stream) {
  return ms::act8_bn_act_bwd_impl<ms::ms_bf16>(g, ref_q, q, s, coef4, du, dgamma, dbeta, N, C, HW, slope, ws, ws_bytes, stream);
}
