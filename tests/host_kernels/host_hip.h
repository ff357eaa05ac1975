// The part of the HIP language that the kernels of ms_class_ce*.hip, ms_act8.hip and ms_logit_ce.hip use, for the CPU: every lane of a workgroup is a fiber, a workgroup's
// fibers run one collective operation each in turn (shuffles, matrix instructions, barriers), workgroups run one behind the other.  The kernels' own source is
// compiled against it (build.py): what is executed is each load, store and DMA as the code makes it, at the address the code computes.
//
// Not modelled: timing, counted waits (a DMA has landed when it is issued), the order of lanes between two collectives.
#pragma once
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <algorithm>
#include <cmath>
#include <functional>
#include <type_traits>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __shared__ static
#define __launch_bounds__(...)

struct dim3 { unsigned x, y, z; dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {} };
struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
struct alignas(16) int4 { int x, y, z, w; };
struct alignas(8) uint2 { unsigned x, y; };
inline float2 make_float2(float a, float b) { return {a, b}; }
inline float4 make_float4(float a, float b, float c, float d) { return {a, b, c, d}; }
inline uint2 make_uint2(unsigned a, unsigned b) { return {a, b}; }
inline float __uint_as_float(unsigned u) { float f; memcpy(&f, &u, 4); return f; }
inline unsigned __float_as_uint(float f) { unsigned u; memcpy(&u, &f, 4); return u; }
inline int min(int a, int b) { return a < b ? a : b; }
inline int max(int a, int b) { return a > b ? a : b; }
inline long min(long a, long b) { return a < b ? a : b; }
inline long max(long a, long b) { return a > b ? a : b; }
inline unsigned min(unsigned a, unsigned b) { return a < b ? a : b; }
inline unsigned max(unsigned a, unsigned b) { return a > b ? a : b; }

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return 0; }
inline const char* hipGetErrorString(hipError_t) { return ""; }

namespace host {
constexpr int kLanes = 64, kMaxThreads = 1024, kStack = 96 * 1024;
struct Slot { unsigned char b[40]; };
struct Wave { int count, alive, gen; Slot in[2][kLanes]; float out[2][kLanes][4]; };
struct Fiber { void* sp; dim3 tid; int wave, lane; bool done; };
extern Fiber fibers[kMaxThreads];
extern Wave waves[kMaxThreads / kLanes];
extern int cur, nthreads, bar_count, bar_gen, bar_alive;
extern dim3 block_idx, block_dim, grid_dim;
extern char lds_anchor;
void yield();
void launch(dim3 grid, dim3 block, const std::function<void()>& f);

// All live lanes of a wave put a value; returns the buffer that holds them.  `last` runs once, when the last has arrived.
template <typename T, typename F>
inline int exchange(const T& v, F last) {
  static_assert(sizeof(T) <= sizeof(Slot), "");
  Fiber& f = fibers[cur];
  Wave& w = waves[f.wave];
  const int g = w.gen, k = g & 1;
  memcpy(w.in[k][f.lane].b, &v, sizeof(T));
  if (++w.count == w.alive) { w.count = 0; last(w, k); ++w.gen; }
  else while (w.gen == g) yield();
  return k;
}
template <typename T> inline int exchange(const T& v) { return exchange(v, [](Wave&, int) {}); }
template <typename T> inline T of(int k, int lane) { T v; memcpy(&v, waves[fibers[cur].wave].in[k][lane].b, sizeof(T)); return v; }
template <typename T> inline T at(Wave& w, int k, int lane) { T v; memcpy(&v, w.in[k][lane].b, sizeof(T)); return v; }

template <typename V, int KL>      // KL: elements of a lane's fragment
inline void mfma(Wave& w, int k) {
  struct P { V a, b; };
  static float A[16][4 * KL], B[4 * KL][16];
  for (int l = 0; l < kLanes; ++l) {
    const P p = at<P>(w, k, l);
    for (int e = 0; e < KL; ++e) { A[l & 15][(l >> 4) * KL + e] = (float)p.a[e]; B[(l >> 4) * KL + e][l & 15] = (float)p.b[e]; }
  }
  for (int m = 0; m < 16; ++m) {
    float s[16] = {};
    for (int kk = 0; kk < 4 * KL; ++kk)
      for (int n = 0; n < 16; ++n) s[n] += A[m][kk] * B[kk][n];
    for (int n = 0; n < 16; ++n) w.out[k][n + 16 * (m >> 2)][m & 3] = s[n];
  }
}
template <typename V, int KL, typename C>
inline C mfma16(V a, V b, C c) {
  struct P { V a, b; } p{a, b};
  const int k = exchange(p, [](Wave& w, int kk) { mfma<V, KL>(w, kk); });
  const Fiber& f = fibers[cur];
  for (int r = 0; r < 4; ++r) c[r] += waves[f.wave].out[k][f.lane][r];
  return c;
}
template <typename S> inline S read_tr16(const S* p) {      // 16 lanes hold 4 rows x 16 columns; lane i gets column i
  const S own = *p;
  const int k = exchange(own), l = fibers[cur].lane, base = l & ~15, i = l & 15;
  S r;
  for (int e = 0; e < 4; ++e) r[e] = of<S>(k, base + 4 * e + (i >> 2))[i & 3];
  return r;
}
template <typename R> inline void dma16(R rsrc, unsigned lds, int voff, int soff) {
  const unsigned off = (unsigned)voff + (unsigned)soff;
  char* dst = &lds_anchor + (int)lds + 16 * fibers[cur].lane;
  if (off >= (unsigned)rsrc[2]) { memset(dst, 0, 16); return; }
  memcpy(dst, (const char*)(((uint64_t)((unsigned)rsrc[1] & 0xFFFFu) << 32) | (unsigned)rsrc[0]) + off, 16);
}
inline unsigned lds_addr(const void* p) { return (unsigned)(int)((const char*)p - &lds_anchor); }
}  // namespace host

#define threadIdx (host::fibers[host::cur].tid)
#define blockIdx host::block_idx
#define blockDim host::block_dim
#define gridDim host::grid_dim

inline void __syncthreads() {
  const int g = host::bar_gen;
  if (++host::bar_count == host::bar_alive) { host::bar_count = 0; ++host::bar_gen; }
  else while (host::bar_gen == g) host::yield();
}
template <typename T> inline T __shfl_xor(T v, int off, int) { const int k = host::exchange(v); return host::of<T>(k, host::fibers[host::cur].lane ^ off); }
template <typename T> inline T __shfl(T v, int lane, int) { const int k = host::exchange(v); return host::of<T>(k, lane); }
inline unsigned long long __ballot(bool p) {
  const int k = host::exchange((int)p), base = host::fibers[host::cur].wave * host::kLanes;
  unsigned long long r = 0;
  for (int l = 0; l < host::kLanes; ++l) if (base + l < host::nthreads && !host::fibers[base + l].done && host::of<int>(k, l) != 0) r |= 1ull << l;
  return r;
}
inline bool __any(bool p) { return __ballot(p) != 0; }
inline int atomicMax(int* p, int v) { const int o = *p; if (v > o) *p = v; return o; }
template <typename... P, typename... A>
inline void hipLaunchKernelGGL(void (*f)(P...), dim3 grid, dim3 block, unsigned, hipStream_t, A... a) { host::launch(grid, block, [=]() { f(a...); }); }

#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_logf(x) log2f(x)
#define __builtin_amdgcn_ldexpf(x, e) ldexpf(x, e)
inline int host_frexp_exp(float x) { int e = 0; if (x != 0.f && std::isfinite(x)) (void)frexpf(x, &e); return e; }
#define __builtin_amdgcn_frexp_expf(x) host_frexp_exp(x)
#define __builtin_amdgcn_s_setprio(x) ((void)0)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) host::mfma16<std::decay_t<decltype(a)>, 8>(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, x, y, z) host::mfma16<std::decay_t<decltype(a)>, 4>(a, b, c)
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(p) host::read_tr16(p)
