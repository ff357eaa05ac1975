// Head + softmax cross entropy over many classes, wide form: three matrix products (logits, dh, dw) over pieces of (rows x classes); see ms_class_ce.h.
//
// Passes of one training call (all on the caller's stream, nothing allocated, no atomics on floats):
//   pack w, pack h      fp16 planes [rows][channels], power-of-two scales, padded to whole tiles
//   logits -> stats     tile of z stays in registers: (max, sum exp) of each row and class tile, and the label's own z
//   join                lse and nll of every row, loss in 64 bits
//   level               the scales that G is formed with; rows and classes far smaller than the largest are moved towards its scale
//   per piece           G (logits again, written as fp16 planes), dh += G w, dw += G^T h; db from G's epilogue
// The logits are never written; G exists for one piece at a time (kCePieceBytes: it
// stays in the 256 MB last-level cache between its writer and its two readers).
#include <algorithm>
#include "ms_class_ce.h"
#include "ms_class_ce_narrow.h"
#include "maxstyle_hip.h"

namespace ms {

constexpr size_t kCePieceBytes = (size_t)224 << 20, kCeStatsBytes = (size_t)256 << 20;

// ------------------------------------------------------------------------------------------------------------------------------ small passes
// Rows [rows][C] -> planes [rows_pad][Cp] and each row's 2^e.  One wave a row; 8 channels a lane where the rows are made of whole vectors.
//   weights: bpad[v] = b log2(e), or -inf behind the last class; features (labels != nullptr): a row that takes no part is packed as zeros when `drop` is set (it may hold anything)
struct CePack {
  const void* src; const float* b; const int64_t* labels; int classes, drop;
  _Float16* out; size_t plane; float *f, *bpad; int* lab32; int rows, rows_pad, C, Cp;
};
template <typename T, bool VEC>
__device__ __forceinline__ void ce_pack_row(const CePack& a, int r) {
  using IO = ActIO<T>;
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  if (r >= a.rows_pad) return;
  bool live = r < a.rows;
  if (a.labels != nullptr) {
    int y = -1;
    if (live) { const int64_t l = a.labels[r]; y = (l >= 0 && l < a.classes) ? (int)l : -1; }
    live = live && (!a.drop || y >= 0);
    if (lane == 0) a.lab32[r] = y;
  }
  const size_t base = (size_t)r * a.C;
  unsigned am = 0;
  auto see = [&](float v) { am = max(am, __float_as_uint(v) & 0x7FFFFFFFu); };
  if (live) {
    if (VEC) {
      for (int c = lane * 8; c < a.C; c += 512) {
        const float4 u = IO::ld4(a.src, base + c), v = IO::ld4(a.src, base + c + 4);
        see(u.x); see(u.y); see(u.z); see(u.w); see(v.x); see(v.y); see(v.z); see(v.w);
      }
    } else {
      for (int c = lane; c < a.C; c += 64) see(IO::ld1(a.src, base + c));
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) am = max(am, (unsigned)__shfl_xor((int)am, off, 64));
  const int e = ce_exponent(__uint_as_float(am));
  const float inv = ce_pow2(-e);
  if (lane == 0) {
    a.f[r] = am == 0u ? 0.f : ce_pow2(e);                // 0: a row of zeros (ce_level_kernel)
    if (a.bpad != nullptr) a.bpad[r] = r < a.rows ? (a.b != nullptr ? a.b[r] * kLog2e : 0.f) : -__builtin_inff();
  }
  for (int c = lane * 8; c < a.Cp; c += 512) {
    float v[8];
    if (VEC) {
      float4 p = make_float4(0.f, 0.f, 0.f, 0.f), d = p;
      if (live && c < a.C) { p = IO::ld4(a.src, base + c); d = IO::ld4(a.src, base + c + 4); }
      v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = d.x; v[5] = d.y; v[6] = d.z; v[7] = d.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (live && c + k < a.C) ? IO::ld1(a.src, base + c + k) : 0.f;
    }
    ms_h8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) { _Float16 x, y; ce_split_far(v[k] * inv, x, y); hi[k] = x; lo[k] = y; }
    *reinterpret_cast<ms_h8*>(a.out + (size_t)r * a.Cp + c) = hi;
    if (PL == 2) *reinterpret_cast<ms_h8*>(a.out + a.plane + (size_t)r * a.Cp + c) = lo;
  }
}
// the first wblocks workgroups: weights; the others: feature rows (there are none when the features come as planes)
template <typename HT, typename WT, bool VEC>
__global__ __launch_bounds__(256) void ce_pack_rows_kernel(CePack w, CePack h, int wblocks) {
  const int wave = threadIdx.x >> 6;
  const int id = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  if (id < wblocks) ce_pack_row<WT, VEC>(w, id * 4 + wave);
  else ce_pack_row<HT, VEC>(h, (id - wblocks) * 4 + wave);
}

// h [N][C][HW], HW > 1 -> the same packed rows.  A workgroup takes 64 pixels: a wave reads 64 neighbouring pixels of a channel at a time and writes 8 channels of each.
template <typename HT, int PL>
__global__ __launch_bounds__(1024) void ce_pack_planes_kernel(const void* __restrict__ h, const int64_t* __restrict__ labels, int classes, int drop, _Float16* __restrict__ out,
                                                              size_t plane, float* __restrict__ fx, int* __restrict__ lab32, long P, long Pp, int C, int Cp, int HW) {
  using IO = ActIO<HT>;
  __shared__ unsigned smax[16][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long p = ((long)blockIdx.y * gridDim.x + blockIdx.x) * 64 + lane;
  if (p >= Pp) return;                 // (whole workgroups: Pp is a multiple of 256)
  int y = -1;
  if (p < P) { const int64_t l = labels[p]; y = (l >= 0 && l < classes) ? (int)l : -1; }
  if (wave == 0) lab32[p] = y;
  const bool live = p < P && (!drop || y >= 0);
  const int n = (int)p / HW;
  const size_t base = (size_t)n * C * HW + (size_t)((int)p - n * HW);
  unsigned am = 0;
  for (int c0 = wave * 8; c0 < C; c0 += 128) {
#pragma unroll
    for (int k = 0; k < 8; ++k) if (live && c0 + k < C) am = max(am, __float_as_uint(IO::ld1(h, base + (size_t)(c0 + k) * HW)) & 0x7FFFFFFFu);
  }
  smax[wave][lane] = am;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; ++k) am = max(am, smax[k][lane]);
  const int e = ce_exponent(__uint_as_float(am));
  const float inv = ce_pow2(-e);
  if (wave == 0) fx[p] = am == 0u ? 0.f : ce_pow2(e);
  for (int c0 = wave * 8; c0 < Cp; c0 += 128) {
    ms_h8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      _Float16 x, z;
      ce_split_far((live && c0 + k < C) ? IO::ld1(h, base + (size_t)(c0 + k) * HW) * inv : 0.f, x, z);
      hi[k] = x; lo[k] = z;
    }
    *reinterpret_cast<ms_h8*>(out + (size_t)p * Cp + c0) = hi;
    if (PL == 2) *reinterpret_cast<ms_h8*>(out + plane + (size_t)p * Cp + c0) = lo;
  }
}

// rows that take part (for the mean over them): slots[workgroup]
constexpr int kCeSlots = 256, kCeRowBlocks = 1024;
__global__ __launch_bounds__(256) void ce_count_kernel(const int64_t* __restrict__ labels, long P, int classes, int* __restrict__ slots) {
  __shared__ int red[4];
  int k = 0;
  for (long p = (long)blockIdx.x * 256 + threadIdx.x; p < P; p += (long)gridDim.x * 256) { const int64_t l = labels[p]; k += (l >= 0 && l < classes) ? 1 : 0; }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) k += __shfl_xor(k, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = k;
  __syncthreads();
  if (threadIdx.x == 0) slots[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ int ce_count(const int* __restrict__ slots, int n, int* red /* 4 */) {       // by the first 256 threads of a workgroup; all get the sum
  int s = threadIdx.x < (unsigned)n ? slots[threadIdx.x] : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (threadIdx.x < 256 && (threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

constexpr int kCeNone = -100000;
// exponent of g_p 2^ex[p]; none for a row without a gradient or of zeros
__device__ __forceinline__ int ce_grad_exponent(float g) {
  const unsigned b = __float_as_uint(g) & 0x7FFFFFFFu;
  return (b != 0u && b < 0x7F800000u) ? (int)(b >> 23) - 126 : kCeNone;
}
__device__ __forceinline__ int ce_scale_exponent(float f) { return f > 0.f ? (int)(__float_as_uint(f) >> 23) - 127 : kCeNone; }
__device__ __forceinline__ int ce_row_exponent(float g, float fx) {
  const int a = ce_grad_exponent(g), b = ce_scale_exponent(fx);
  return (a == kCeNone || b == kCeNone) ? kCeNone : a + b;
}
// The upstream gradient of every row: grad[p], 0 where the label is not a class.  A row without one gets a log-sum of infinity: exp(z - inf) = 0 whatever its logits are.
// rowmax[workgroup]: the largest exponent of g_p 2^ex[p].
__global__ __launch_bounds__(256) void ce_rowgrad_kernel(const float* __restrict__ grad, const int* __restrict__ lab32, const float* __restrict__ fx, float* __restrict__ gp,
                                                         const float* __restrict__ lse_in, float* __restrict__ lse2, float* __restrict__ hot, int* __restrict__ rowmax, long P, long Pp) {
  __shared__ int red[4];
  int e = kCeNone;
  for (long p = (long)blockIdx.x * 256 + threadIdx.x; p < Pp; p += (long)gridDim.x * 256) {
    const float g = (p < P && lab32[p] >= 0) ? grad[p] : 0.f;
    e = max(e, ce_row_exponent(g, fx[p]));
    float ls = __builtin_inff(), d = 0.f;
    if (g != 0.f) {
      ls = lse_in[p] * kLog2e;
      d = ce_rest_nat(lse_in[p], ls);
    }
    gp[p] = g * __builtin_amdgcn_exp2f(-d);
    lse2[p] = ls; hot[p] = __builtin_amdgcn_exp2f(d);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) e = max(e, __shfl_xor(e, off, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = e;
  __syncthreads();
  if (threadIdx.x == 0) rowmax[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// The loss (first workgroup), and the scales that G is formed with.
//
// One G serves both products: G'[p,v] = G[p,v] 2^(r[p] + c[v] + scal), dh[p] = 2^-(r[p] + scal) sum_v G' w/2^c[v], dw[v] = 2^-(c[v] + scal) sum_p G' h/2^r[p].  With the rows' own
// exponents, r = ex, a row (class) far smaller than the largest would have its G' far below the largest although neither dh of the row nor dw of the class depends on its size, and a row
// of zeros has no exponent at all.  So every row's exponent of g_p 2^r[p], and every c[v], is brought to at least the largest less kCeWindow - rows of zeros for nothing, others by
// dividing their planes by that much, as long as these keep 24 bits of the row's largest (kCeMove1 / 2: one / two planes).  Within 2^30 of the largest, G' is held to 2^-22 of itself
// (one plane: 2^-11) or 2^-41 (2^-29) g_p, whatever the row's and the class's size are.  Rows within the window, the ordinary case, are not touched.
// A class that is switched off (b = -inf) may hold anything finite and sets no scale; where it holds more than 4 times the largest of the others its planes are cleared (its G is 0, but
// for a row with this very label, whose loss is infinite).
constexpr int kCeWindow = 4, kCeMove1 = 16, kCeMove2 = 26, kCeClear = 1000;
struct CeLevel {
  const double* lsum; int n; float sign; int mean_valid; const int* slots; int nslots; long P; float* loss;
  const int* rowmax; int nrow; const float *fx, *gp, *fw, *bpad; float *fx2, *fw2; _Float16 *x, *w; size_t xpl, wpl; int xp, wp, V, Vp, Cp; long Pp; int* scal;
};
__device__ __forceinline__ void ce_move(_Float16* row, size_t plane, int planes, int Cp, int lane, int by) {
  const float f = ce_pow2(-by);
  for (int c = lane * 8; c < Cp; c += 512) {
    ms_h8 hi = *reinterpret_cast<const ms_h8*>(row + c), lo;
    if (planes == 2) lo = *reinterpret_cast<const ms_h8*>(row + plane + c);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float v = planes == 2 ? (float)hi[k] + (float)lo[k] * (1.f / (float)(1 << kCeLoExp)) : (float)hi[k];
      _Float16 a, b;
      ce_split_far(by == kCeClear ? 0.f : v * f, a, b);
      hi[k] = a; lo[k] = b;
    }
    *reinterpret_cast<ms_h8*>(row + c) = hi;
    if (planes == 2) *reinterpret_cast<ms_h8*>(row + plane + c) = lo;
  }
}
__global__ __launch_bounds__(1024) void ce_level_kernel(CeLevel a) {
  __shared__ double redd[16];
  __shared__ int redi[32];
  if (a.loss != nullptr && blockIdx.x == 0) {
    const int cnt = a.mean_valid ? ce_count(a.slots, a.nslots, redi) : 0;
    double s = 0.0;
    for (int i = threadIdx.x; i < a.n; i += 1024) s += a.lsum[i];
    s = block_sum_d(s, redd);
    if (threadIdx.x == 0) a.loss[0] = (float)((double)a.sign * s / (double)(a.mean_valid ? max(cnt, 1) : a.P));
  }
  if (a.rowmax == nullptr) return;
  int er = kCeNone, ew = kCeNone;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.nrow; i += 1024) er = max(er, a.rowmax[i]);
#pragma unroll 4
  for (int v = threadIdx.x * 4; v < a.V; v += 4096) {        // (padded to whole tiles)
    const float4 f = *reinterpret_cast<const float4*>(a.fw + v), b = *reinterpret_cast<const float4*>(a.bpad + v);
    const float ff[4] = {f.x, f.y, f.z, f.w}, bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) if (bb[k] != -__builtin_inff()) ew = max(ew, ce_scale_exponent(ff[k]));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { er = max(er, __shfl_xor(er, off, 64)); ew = max(ew, __shfl_xor(ew, off, 64)); }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0) { redi[wave] = er; redi[16 + wave] = ew; }
  __syncthreads();
  for (int k = 0; k < 16; ++k) { er = max(er, redi[k]); ew = max(ew, redi[16 + k]); }
  if (er == kCeNone) er = 0;
  if (ew == kCeNone) ew = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.scal[0] = min(max(kCeTopExp - (er + ew), -120), 120);
  // a wave takes 16 classes or rows: one lane each finds the new exponent, the whole wave moves those that need it
  for (long i0 = ((long)blockIdx.x * 16 + wave) * 16; i0 < a.Vp + a.Pp; i0 += (long)gridDim.x * 256) {
    const bool cls = i0 < a.Vp;
    const long r0 = cls ? i0 : i0 - a.Vp;
    const int planes = cls ? a.wp : a.xp;
    int by = 0;
    if (lane < 16) {
      const int e = ce_scale_exponent((cls ? a.fw : a.fx)[r0 + lane]), g = cls ? 0 : ce_grad_exponent(a.gp[r0 + lane]), top = (cls ? ew : er) - kCeWindow - g;
      int to = e == kCeNone ? 0 : e;
      if (g != kCeNone) {
        if (e == kCeNone) to = min(max(top, -126), 126);
        else to = min(max(e, min(top, e + (planes == 2 ? kCeMove2 : kCeMove1))), max(e, 120));
      }
      if (cls && e > ew + 2 && e != kCeNone) {          // (switched off)
        to = ew;
        by = kCeClear;
      } else {
        by = e == kCeNone ? 0 : to - e;
      }
      (cls ? a.fw2 : a.fx2)[r0 + lane] = ce_pow2(to);
    }
    for (unsigned long long m = __ballot(by != 0); m != 0; m &= m - 1) {
      const int k = __builtin_ctzll(m);
      ce_move((cls ? a.w : a.x) + (size_t)(r0 + k) * a.Cp, cls ? a.wpl : a.xpl, planes, a.Cp, lane, __shfl(by, k, 64));
    }
  }
}

struct CeRowGrad { float *gp, *hot; const float* fx; float sign; int mean_valid; const float* scale_dev; const int* slots; int nslots; int* rowmax; };

// part[t][p] = {max, sum exp} over one class range -> lse, nll; loss partials in 64 bits; with r.gp the rows' upstream gradients (ce_rowgrad_kernel's work).  64 rows a workgroup, 16 threads each over the class ranges.  All in units of log2.
__device__ __forceinline__ void ce_merge(float& m, float& l, float mo, float lo) {
  const float mn = fmaxf(m, mo), mm = mn == -__builtin_inff() ? 0.f : mn;
  l = l * __builtin_amdgcn_exp2f(m - mm) + lo * __builtin_amdgcn_exp2f(mo - mm);
  m = mn;
}
__global__ __launch_bounds__(1024) void ce_join_kernel(const float2* __restrict__ part, int nparts, size_t stride, const float* __restrict__ zlab, const int* __restrict__ lab32,
                                                       float* __restrict__ lse2, float* __restrict__ lse_out, float* __restrict__ nll_out, double* __restrict__ lsum, long p0, long P, CeRowGrad rg) {
  __shared__ float2 sh[16][64];
  __shared__ int redi[16];
  const int cnt = (rg.gp != nullptr && rg.mean_valid) ? ce_count(rg.slots, rg.nslots, redi) : 0;
  const int el = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const long pr = (long)blockIdx.x * 64 + el, p = p0 + pr;          // (padded)
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll 4
  for (int t = grp; t < nparts; t += 16) { const float2 o = part[(size_t)t * stride + pr]; ce_merge(m, l, o.x, o.y); }
  sh[grp][el] = make_float2(m, l);
  __syncthreads();
  if (grp != 0) return;
  for (int k = 1; k < 16; ++k) ce_merge(m, l, sh[k][el].x, sh[k][el].y);
  const float lg = ce_log2(l), ln2 = 0.693147180559945309f;      // (log2)
  float ls = m + lg;
  double acc = 0.0;
  if (rg.gp != nullptr) {
    const float g = (p < P && lab32[p] >= 0) ? rg.sign / (float)(rg.mean_valid ? max(cnt, 1) : P) * (rg.scale_dev != nullptr ? *rg.scale_dev : 1.f) : 0.f;
    const float d = g == 0.f ? 0.f : ce_rest(m, lg, ls);
    rg.gp[p] = g * __builtin_amdgcn_exp2f(-d); rg.hot[p] = __builtin_amdgcn_exp2f(d);
    if (g == 0.f) ls = __builtin_inff();
    int e = ce_row_exponent(g, rg.fx[p]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) e = max(e, __shfl_xor(e, off, 64));
    if (el == 0) rg.rowmax[p0 / 64 + blockIdx.x] = e;
  }
  lse2[p] = ls;
  if (p < P) {
    if (lse_out != nullptr) lse_out[p] = ce_lse_nat(m, lg);
    const float v = lab32[p] >= 0 ? ((m - zlab[p]) + lg) * ln2 : 0.f;        // (max - z) + log sum: nothing cancels where the label has the maximum
    if (nll_out != nullptr) nll_out[p] = v;
    acc = (double)v;
  }
  acc = wave_sum_d(acc);
  if (el == 0) lsum[p0 / 64 + blockIdx.x] = acc;
}

// ------------------------------------------------------------------------------------------------------------------------------ matrix products
struct CeOperand { const _Float16* p; size_t plane; int ld; int cols; };      // ROW: [mn][k], ld = row stride; COL: [k][mn], cols = valid columns
struct CeGemm {
  CeOperand a, b;
  int nseg, pa[3], pb[3];         // plane pairs summed into one accumulator: the low ones, then the high one
  int ksteps;                     // K / 64 of one pair
  int mt, nt, split;
  // logits epilogues
  const float *fw, *bpad, *fx; const int* lab; const float *lse, *gp, *hot; const int* scal;
  float2* part; size_t part_stride; float* zlab;
  _Float16* g; size_t g_plane; int g_ld; float* dbpart; size_t db_stride;
  int v0; long p0;                // first class / row of this piece
  // plain epilogue
  float* out; size_t out_split; int out_ld;
};
enum { CE_STATS = 0, CE_GRAD = 1, CE_GRAD2 = 2, CE_OUT = 3 };

constexpr int kCeBK = 64;
// Slabs of a K-split: shorter ones cost more in the sums behind than they save (16 rows x 512 channels x 5000 classes, fp32: 88, 79, 81 us at 6, 12, 24; bf16 73, 62, 60 at 2, 4, 8).
constexpr int kCeDeep = 12;

// Stage one 64-deep slab of an operand tile into LDS by DMA: 1 KB an instruction, the source address permuted so that the fragment reads below are free of bank conflicts.
//   ROW: [T rows][64 k]: 16-byte chunk j of row r lies at chunk j ^ (r & 7)
//   COL: [64 k][T columns]: 32-byte unit u of row k lies at unit u ^ f(k), f = (k & 3) | ((k >> 3) & 1) << 2 (T = 64 has four units: f = k & 3)
template <int T, bool COL, int NW>
__device__ __forceinline__ void ce_stage(const CeOperand& o, const _Float16* base, int mn0, int wave, int lane, unsigned lds) {
  constexpr int kInstr = T * kCeBK * 2 / 1024;
  const ms_i32x4 rs = ms_dma_rsrc(base);
#pragma unroll
  for (int t = 0; t < kInstr / NW; ++t) {
    const int ins = t * NW + wave;
    int voff;
    if (!COL) {
      const int row = ins * 8 + (lane >> 3), ch = (lane & 7) ^ (row & 7);
      voff = (int)(((unsigned)row * (unsigned)o.ld + ch * 8) * 2u);
    } else {
      constexpr int kRows = 1024 / (T * 2), kCh = T / 8;
      const int k = ins * kRows + lane / kCh, ch = lane % kCh;
      const int unit = (ch >> 1) ^ ((k & 3) | (T > 64 ? ((k >> 3) & 1) << 2 : 0));
      const int col = min(mn0 + unit * 16 + (ch & 1) * 8, o.cols - 8);        // columns behind the operand's last are read twice and never used
      voff = (int)(((unsigned)k * (unsigned)o.ld + (unsigned)col) * 2u);
    }
    ms_lds_dma16(rs, __builtin_amdgcn_readfirstlane(lds + ins * 1024), voff, 0);
  }
}
template <int T, bool COL>
__device__ __forceinline__ ms_h8 ce_frag(const _Float16* tile, int mn, int ks, int lane) {      // mn: first of 16, inside the tile
  const int q = lane >> 4, i = lane & 15;
  if (!COL) {
    return *reinterpret_cast<const ms_h8*>(tile + (mn + i) * kCeBK + (((ks * 4 + q) ^ (i & 7)) * 8));
  } else {
    const int f = (i >> 2) | (T > 64 ? (q & 1) << 2 : 0);
    const int k = ks * 32 + q * 8 + (i >> 2);
    const _Float16* a = tile + k * T + (((mn >> 4) ^ f) * 16) + (i & 3) * 4;
    typedef __attribute__((address_space(3))) ms_s4* lp;
    union { ms_s4 s[2]; ms_h8 h; } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)a);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(a + 4 * T));
    return u.h;
  }
}

// One BM x BN tile, (BM / WM) x (BN / WN) per wave, LDS double-buffered: slab t + 1 is on its way while slab t is multiplied; one barrier a slab.
template <int BM, int BN, int WM, int WN, int ST, bool ACOL, bool BCOL, int EPI>
__device__ __forceinline__ void ce_gemm_tile(CeGemm g, int id, _Float16 (*sm)[(BM + BN) * kCeBK]) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 16, NJ = TN / 16;
  static_assert((ST & (ST - 1)) == 0, "slab t lies in buffer t mod ST");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const int wm = wave / WN, wn = wave % WN;
  // Tiles of one XCD (workgroups are dealt to the 8 of them in turn) are neighbours: they share operand panels in that XCD's L2.
  const int tiles = g.mt * g.nt * g.split, per = tiles >> 3;
  if (id < per * 8) id = (id & 7) * per + (id >> 3);
  const int sp = id / (g.mt * g.nt);
  id -= sp * g.mt * g.nt;
  // groups of 8 class tiles wide: 8 x (up to 8) tiles in a row use 16 panels
  constexpr int GRP = 8;
  const int gsz = GRP * g.nt, gi = id / gsz, gm = min(GRP, g.mt - gi * GRP), gr = id - gi * gsz;
  const int mt = gi * GRP + gr % gm, nt = gr / gm;
  const int m0 = mt * BM, n0 = nt * BN;
  const int steps = g.ksteps * g.nseg;
  const int k0 = (int)((long)steps * sp / g.split), k1 = (int)((long)steps * (sp + 1) / g.split), klow = g.ksteps * (g.nseg - 1);      // steps below klow: low pairs

  ms_f4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = ms_f4{0.f, 0.f, 0.f, 0.f};

  const unsigned lds0 = ms_lds_addr(&sm[0][0]);
  auto stage = [&](int t) {
    const int seg = t / g.ksteps, kk = t - seg * g.ksteps;
    const unsigned buf = lds0 + (unsigned)(t & (ST - 1)) * (unsigned)((BM + BN) * kCeBK * 2);
    const _Float16* a = g.a.p + (size_t)g.pa[seg] * g.a.plane + (ACOL ? (size_t)kk * kCeBK * g.a.ld : (size_t)m0 * g.a.ld + (size_t)kk * kCeBK);
    const _Float16* b = g.b.p + (size_t)g.pb[seg] * g.b.plane + (BCOL ? (size_t)kk * kCeBK * g.b.ld : (size_t)n0 * g.b.ld + (size_t)kk * kCeBK);
    ce_stage<BM, ACOL, NW>(g.a, a, m0, wave, lane, buf);
    ce_stage<BN, BCOL, NW>(g.b, b, n0, wave, lane, buf + BM * kCeBK * 2);
  };
  constexpr int kLoads = (BM + BN) * kCeBK * 2 / 1024 / NW;         // DMA instructions of a slab and wave
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) if (k0 + s < k1) stage(k0 + s);
  int t = k0;
#pragma unroll 1
  for (int high = 0; high < 2; ++high) {      // low pairs, then the high one (a test of t inside one loop cost the 128 x 128 products 10 - 12 %)
    const int te = high ? k1 : min(klow, k1);
    for (; t < te; ++t) {
      if (ST > 2 && t + ST - 2 < k1) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kLoads * (ST - 2)) : "memory");      // the ST - 2 slabs behind t may be on their way
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();                    // slab t has landed for every wave, and nobody reads the buffer that slab t + ST - 1 goes to
      if (t + ST - 1 < k1) stage(t + ST - 1);
      const _Float16* sa = &sm[t & (ST - 1)][0];
      const _Float16* sb = sa + BM * kCeBK;
      // All fragments of the slab first, then its products in one run at raised priority: the other workgroup's (wave's) reads and DMA fill the gaps (1163 -> 1115 us for
      // 6400 rows x 512 channels x 32768 classes).  A ring of four slabs of 32 with counted waits was slower (1298: a barrier per 32).
      ms_h8 fa[2][MI], fb[2][NJ];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[ks][i] = ce_frag<BM, ACOL>(sa, wm * TM + i * 16, ks, lane);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[ks][j] = ce_frag<BN, BCOL>(sb, wn * TN + j * 16, ks, lane);
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[ks][i], fb[ks][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_s_setprio(0);
    }
    if (!high && te > k0) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] *= 1.f / (float)(1 << kCeLoExp);
    }
  }

  // Fragment layout of the result: column n = lane & 15, rows m = 4 (lane >> 4) + 0..3.
  if (EPI == CE_OUT) {
    float* o = g.out + (size_t)sp * g.out_split;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + wm * TM + i * 16 + q * 4 + r;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[(size_t)m * g.out_ld + n0 + wn * TN + j * 16 + li] = acc[i][j][r];
      }
    return;
  }

  const int vbase = m0 + wm * TM + q * 4;           // class inside the piece
  float fs[NJ];                                     // 2^ex log2(e)
  int lab[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const size_t p = (size_t)g.p0 + n0 + wn * TN + j * 16 + li;
    fs[j] = g.fx[p] * kLog2e;
    const int y = g.lab[p];
    lab[j] = y < 0 ? -1000000000 : y - g.v0 - vbase;             // label relative to this lane's first class
  }
  if (EPI == CE_STATS) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(g.fw + g.v0 + vbase + i * 16), b = *reinterpret_cast<const float4*>(g.bpad + g.v0 + vbase + i * 16);
      const float ff[4] = {f.x, f.y, f.z, f.w}, bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(acc[i][j][r] * ff[r], fs[j], bb[r]);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const size_t p = (size_t)g.p0 + n0 + wn * TN + j * 16 + li;
      if (__any((unsigned)lab[j] < (unsigned)(MI * 16))) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) if (lab[j] == i * 16 + r) g.zlab[p] = acc[i][j][r];
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mm = mx == -__builtin_inff() ? 0.f : mx;
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) l += __builtin_amdgcn_exp2f(acc[i][j][r] - mm);
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      if (q == 0) g.part[(size_t)(mt * WM + wm) * g.part_stride + (p - (size_t)g.p0)] = make_float2(mx, l);
    }
    return;
  }
  if (EPI == CE_GRAD || EPI == CE_GRAD2) {
    const float gn = ce_pow2(g.scal[0]);
    float gp[NJ], ls[NJ], rj[NJ], hot[NJ];
    bool here = false;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const size_t p = (size_t)g.p0 + n0 + wn * TN + j * 16 + li;
      gp[j] = g.gp[p]; ls[j] = g.lse[p]; hot[j] = g.hot[p];
      rj[j] = gp[j] * g.fx[p] * gn;
      here |= (unsigned)lab[j] < (unsigned)(MI * 16);
    }
    here = __any(here);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(g.fw + g.v0 + vbase + i * 16), b = *reinterpret_cast<const float4*>(g.bpad + g.v0 + vbase + i * 16);
      const float ff[4] = {f.x, f.y, f.z, f.w}, bb[4] = {b.x, b.y, b.z, b.w};
      float db[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r] * ff[r], fs[j], bb[r]) - ls[j]);
        if (here) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] -= lab[j] == i * 16 + r ? hot[j] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          db[r] = __builtin_fmaf(acc[i][j][r], gp[j], db[r]);
          acc[i][j][r] = ce_rounded(acc[i][j][r] * (rj[j] * ff[r]));
        }
      }
      if (g.dbpart != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int off = 1; off < 16; off <<= 1) db[r] += __shfl_xor(db[r], off, 64);
        }
        if (li == 0) *reinterpret_cast<float4*>(g.dbpart + (size_t)(nt * WN + wn) * g.db_stride + vbase + i * 16) = make_float4(db[0], db[1], db[2], db[3]);
      }
    }
    // G goes out through LDS as [row][class], 16 bytes a lane in whole rows
    _Float16* tile = &sm[0][0];
    constexpr int kCh = BM / 8, kSwz = kCh < 16 ? kCh - 1 : 15;
#pragma unroll
    for (int pl = 0; pl < (EPI == CE_GRAD2 ? 2 : 1); ++pl) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          ms_h4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const _Float16 hi = (_Float16)acc[i][j][r];
            v[r] = pl == 0 ? hi : (_Float16)((acc[i][j][r] - (float)hi) * (float)(1 << kCeLoExp));
          }
          const int row = wn * TN + j * 16 + li, col = wm * TM + i * 16 + q * 4;
          *reinterpret_cast<ms_h4*>(tile + row * BM + (((col >> 3) ^ (row & kSwz)) * 8) + (col & 7)) = v;
        }
      __syncthreads();
      _Float16* out = g.g + pl * g.g_plane + (size_t)n0 * g.g_ld + m0;
#pragma unroll
      for (int k = 0; k < BN * kCh / (NW * 64); ++k) {
        const int i = k * (NW * 64) + threadIdx.x, row = i / kCh, ch = i % kCh;
        *reinterpret_cast<ms_h8*>(out + (size_t)row * g.g_ld + ch * 8) = *reinterpret_cast<const ms_h8*>(tile + row * BM + ((ch ^ (row & kSwz)) * 8));
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int ST, bool ACOL, bool BCOL, int EPI>
__global__ __launch_bounds__(WM * WN * 64) void ce_gemm_kernel(CeGemm g) {
  __shared__ __attribute__((aligned(1024))) _Float16 sm[ST][(BM + BN) * kCeBK];
  ce_gemm_tile<BM, BN, WM, WN, ST, ACOL, BCOL, EPI>(g, blockIdx.x, sm);
}
// dh and dw of a piece in one launch, where both take tiles of T: the first nh workgroups dh (its operands as HROWS says), the others dw.
template <int T, int ST, bool HROWS>
__global__ __launch_bounds__(256) void ce_grads_kernel(CeGemm h, CeGemm w, int nh) {
  __shared__ __attribute__((aligned(1024))) _Float16 sm[ST][2 * T * kCeBK];
  if ((int)blockIdx.x < nh) ce_gemm_tile<T, T, 2, 2, ST, !HROWS, HROWS, CE_OUT>(h, blockIdx.x, sm);
  else ce_gemm_tile<T, T, 2, 2, ST, true, true, CE_OUT>(w, (int)blockIdx.x - nh, sm);
}

// The sums behind a piece's products, one launch: db from G's epilogue, dh and dw from their K-splits (each a range of workgroups; any may be empty).
// A product's partials [split][rows][ld] ->
//   planes  rows = channels, columns = pixels of this piece, written as [n][channel][hw];  f = 2^ex of the column
//   else    rows = classes (dw) or feature rows (dh with HW = 1) of this piece, columns = channels, written as [row][channel];  f = 2^ew / 2^ex of the row
//   first: nothing is there yet, else the fp32 running sum `acc` is added;  last: written to `out` in its type, else back to `acc`.
struct CeSum { const float* part; size_t out_split; int ld, split; const float* f; float* acc; void* out; int first, last, rows, cols; long r0; int HW, C, blocks, rblocks; };
struct CeSums { CeSum h, w; const float* dbpart; int dbn; size_t dbstride; float* db; int dbfirst, dbV, dbv0, dbblocks; const int* scal; };
template <typename OT>
__device__ __forceinline__ void ce_sum(const CeSum& a, int id, const int* scal, bool planes) {
  const float gi = ce_pow2(-scal[0]);
  const int row = (id % a.rblocks) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, ny = a.blocks / a.rblocks;
  if (row >= a.rows) return;
  for (int c = (id / a.rblocks) * 64 + lane; c < a.cols; c += ny * 64) {
    const float* src = a.part + (size_t)row * a.ld + c;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.split; ++k) s += src[k * a.out_split];
    size_t dst;
    if (planes) {
      const int p = (int)a.r0 + c, n = p / a.HW;
      dst = ((size_t)n * a.C + row) * a.HW + (p - n * a.HW);
      s *= gi / a.f[p];
    } else {
      dst = (size_t)(a.r0 + row) * a.C + c;
      s *= gi / a.f[a.r0 + row];
    }
    if (!a.first) s += a.acc[dst];
    if (a.last) ActIO<OT>::st1(a.out, dst, s); else a.acc[dst] = s;
  }
}
template <typename HT, typename WT>
__global__ __launch_bounds__(256) void ce_sums_kernel(CeSums a) {
  __shared__ double sh[4][64];
  int id = blockIdx.x;
  if (id < a.dbblocks) {
    const int el = threadIdx.x & 63, grp = threadIdx.x >> 6, v = id * 64 + el;
    double s = 0.0;
#pragma unroll 8
    for (int i = grp; i < a.dbn; i += 4) s += (double)a.dbpart[(size_t)i * a.dbstride + v];      // (columns padded to whole tiles)
    sh[grp][el] = s;
    __syncthreads();
    if (grp != 0 || v >= a.dbV) return;
    s += sh[1][el] + sh[2][el] + sh[3][el];
    a.db[a.dbv0 + v] = (float)(a.dbfirst ? s : s + (double)a.db[a.dbv0 + v]);
    return;
  }
  id -= a.dbblocks;
  if (id < a.h.blocks) { ce_sum<HT>(a.h, id, a.scal, a.h.HW > 1); return; }
  ce_sum<WT>(a.w, id - a.h.blocks, a.scal, false);
}

// ------------------------------------------------------------------------------------------------------------------------------ host
struct CePlan {
  long P, Pp; int Vp, Cp, HW;
  int xp, wp, gpl;               // planes of h, w, G
  int pb, vb;                    // rows / classes of a piece
  int nparts, sb;                // partial statistics of a row, rows whose statistics are formed at a time
  int split_x, split_w;
  size_t o_x, o_w, o_fx, o_fw, o_fx2, o_fw2, o_hot, o_b, o_lab, o_lse, o_zl, o_gp, o_part, o_scal, o_slots, o_rowmax, o_lsum, o_g, o_db, o_px, o_pw, o_ax, o_aw, total;
};
static size_t ce_al(size_t n) { return (n + 255) & ~(size_t)255; }
static long ce_up(long a, long b) { return (a + b - 1) / b * b; }

static CePlan ce_plan(int N, int C, int V, int HW, int types, bool grad) {
  CePlan k{};
  k.P = (long)N * HW; k.HW = HW;
  k.Pp = ce_up(k.P, kCePad); k.Vp = (int)ce_up(V, kCePad); k.Cp = (int)ce_up(C, kCeBK);
  k.xp = (types & 1) ? 1 : 2; k.wp = (types & 2) ? 1 : 2;
  k.gpl = (k.xp == 2 || k.wp == 2) ? 2 : 1;
  // Pieces of G: up to 16384 classes, and as many rows as kCePieceBytes holds, both cut evenly (6 pieces of 90 % fill the chip better than 5 whole ones and a scrap).
  // Half of both was 4 % slower (shorter sums, more partial results).
  auto even = [](long n, long most) { return ce_up((n + (n + most - 1) / most - 1) / ((n + most - 1) / most), kCePad); };
  k.vb = (int)even(k.Vp, 16384);
  k.pb = (int)even(k.Pp, std::max<long>(kCePad, (long)(kCePieceBytes / ((size_t)k.vb * 2 * k.gpl)) / kCePad * kCePad));
  k.nparts = k.Vp / 128 * 2;
  k.sb = (int)even(k.Pp, std::max<long>(kCePad, (long)(kCeStatsBytes / ((size_t)k.nparts * 8)) / kCePad * kCePad));
  size_t o = 0;
  auto take = [&](size_t n) { const size_t at = o; o += ce_al(n); return at; };
  k.o_x = take((size_t)k.xp * k.Pp * k.Cp * 2);
  k.o_w = take((size_t)k.wp * k.Vp * k.Cp * 2);
  k.o_fx = take(k.Pp * 4); k.o_fw = take((size_t)k.Vp * 4); k.o_b = take((size_t)k.Vp * 4);
  k.o_lab = take(k.Pp * 4); k.o_lse = take(k.Pp * 4); k.o_zl = take(k.Pp * 4); k.o_gp = take(k.Pp * 4);
  k.o_scal = take(64); k.o_slots = take(kCeSlots * 4); k.o_rowmax = take((size_t)(k.Pp / 64) * 4);
  k.o_lsum = take((size_t)(k.Pp / 64) * 8);
  // (two of a tile; 64-wide tiles, twice as many, are taken for less than 128 tiles of 128 x 128: 512 x 254 pairs at most)
  const size_t stats = std::max((size_t)k.nparts * k.sb * 8, (size_t)2 << 20);
  if (!grad) { k.o_part = take(stats); k.total = o; return k; }
  k.o_fx2 = take(k.Pp * 4); k.o_fw2 = take((size_t)k.Vp * 4); k.o_hot = take(k.Pp * 4);
  // The statistics are read before the first piece of G is written: they share its memory.
  k.o_part = o;
  k.o_g = take(std::max((size_t)k.gpl * k.pb * k.vb * 2, stats));
  k.o_db = take((size_t)(k.pb / 64 * 2) * k.vb * 4);
  // K-splits: enough tiles for the chip (256 CUs, two workgroups each at 128 x 128), each at least kCeDeep slabs (three pairs of planes at most)
  const long cp = ce_up(k.Cp, 128), rt = std::min<long>(k.pb, ce_up(k.P, 128)), vt = std::min<long>(k.vb, ce_up(V, 128));
  auto split = [&](long tiles, long ksteps) { return (int)std::max<long>(1, std::min<long>(std::min<long>(512 / std::max<long>(tiles, 1), ksteps * 3 / kCeDeep), 64)); };
  k.split_x = split(cp / 128 * (rt / 128), vt / 64);
  k.split_w = split(cp / 128 * (vt / 128), rt / 64);
  k.o_px = take((size_t)k.split_x * cp * k.pb * 4);
  k.o_pw = take((size_t)k.split_w * k.vb * cp * 4);
  k.o_ax = take((k.vb < k.Vp && (types & 1)) ? (size_t)k.P * C * 4 : 0);
  k.o_aw = take((k.pb < k.Pp && (types & 2)) ? (size_t)V * C * 4 : 0);
  k.total = o;
  return k;
}

// n workgroups over two axes: more than 2^32 threads of one axis cannot be launched (2^26 rows, one wave each)
static dim3 ce_grid(long n) { return n <= (1 << 20) ? dim3((unsigned)n) : dim3(1 << 20, (unsigned)((n + (1 << 20) - 1) >> 20)); }

static int ce_check(int N, int C, int V, int HW, int types, const char* who) {
  if (N < 1 || C < 1 || V < 1 || HW < 1 || types < 0 || types > 3) { set_error("%s: invalid shape", who); return MS_ERR_INVALID; }
  if (C > 8192 || V > (1 << 20) || (long long)N * HW > (1LL << 30)) { set_error("%s: supported up to 8192 channels, 2^20 classes, 2^30 rows", who); return MS_ERR_INVALID; }
  return MS_OK;
}

// Tile of a product of M x N (real sizes; the operands and results hold capM x capN, multiples of 128).
//   256: one workgroup a CU, half the LDS traffic a product: where there are enough of them for the chip.  G's kernel does without: its epilogue is as long as its product
//        at 512 channels, and only a second workgroup on the CU overlaps the two (381 against 428 us)
//   64:  few rows or classes: a quarter of the work a slab on four times the CUs (1 row x 512 channels x 1000 classes, fp32: 92 -> 59 us)
struct CeTile { int t, mt, nt; };
template <int EPI> static CeTile ce_tile(long M, long N, int split, long capM, long capN) {
  auto n = [](long x, long t) { return (x + t - 1) / t; };
  int t = 64;
  if ((EPI == CE_STATS || EPI == CE_OUT) && n(M, 256) * 256 <= capM && n(N, 256) * 256 <= capN && n(M, 256) * n(N, 256) * split >= 200) t = 256;
  else if (n(M, 128) * n(N, 128) * split >= 128) t = 128;
  return CeTile{t, (int)n(M, t), (int)n(N, t)};
}
template <int EPI, bool ACOL, bool BCOL>
static int ce_gemm(CeGemm g, const CeTile& c, hipStream_t st, const char* what) {
  g.mt = c.mt; g.nt = c.nt;
  const dim3 grid((unsigned)((long)g.mt * g.nt * g.split));
  if constexpr (EPI == CE_STATS || EPI == CE_OUT) {
    if (c.t == 256) {
      MS_LAUNCH((ce_gemm_kernel<256, 256, 2, 4, 2, ACOL, BCOL, EPI>), grid, dim3(512), 0, st, g);
      return check_launch(what);
    }
  }
  if (c.t == 128) MS_LAUNCH((ce_gemm_kernel<128, 128, 2, 2, 2, ACOL, BCOL, EPI>), grid, dim3(256), 0, st, g);
  else MS_LAUNCH((ce_gemm_kernel<64, 64, 2, 2, 4, ACOL, BCOL, EPI>), grid, dim3(256), 0, st, g);
  return check_launch(what);
}
static void ce_pairs(CeGemm& g, int a, int b) {       // planes of the two operands -> products
  g.nseg = 0;
  if (b == 2) { g.pa[g.nseg] = 0; g.pb[g.nseg++] = 1; }
  if (a == 2) { g.pa[g.nseg] = 1; g.pb[g.nseg++] = 0; }
  g.pa[g.nseg] = g.pb[g.nseg] = 0; ++g.nseg;
}

static int ce_run(const CeArgs& a, const char* who) {
  if (int e = ce_check(a.N, a.C, a.V, a.HW, a.types, who)) return e;
  if (a.h == nullptr || a.w == nullptr || a.labels == nullptr) { set_error("%s: null pointer", who); return MS_ERR_INVALID; }
  const bool need_grad = a.dh != nullptr || a.dw != nullptr || a.db != nullptr;
  if (ce_narrow_ok(a.N, a.C, a.V, a.HW)) return ce_narrow_run(a, need_grad, who);
  const CePlan k = ce_plan(a.N, a.C, a.V, a.HW, a.types, need_grad);
  if (a.ws == nullptr || a.ws_bytes < k.total) { set_error("%s: workspace too small", who); return MS_ERR_WORKSPACE; }
  if (!aligned16(a.ws)) { set_error("%s: workspace not 16-byte aligned", who); return MS_ERR_ALIGN; }
  char* ws = (char*)a.ws;
  auto f32 = [&](size_t o) { return (float*)(ws + o); };
  _Float16 *x = (_Float16*)(ws + k.o_x), *w = (_Float16*)(ws + k.o_w);
  const size_t xpl = (size_t)k.Pp * k.Cp, wpl = (size_t)k.Vp * k.Cp;
  int *lab = (int*)(ws + k.o_lab), *scal = (int*)(ws + k.o_scal), *slots = (int*)(ws + k.o_slots), *rowmax = (int*)(ws + k.o_rowmax);
  float *fx = f32(k.o_fx), *fw = f32(k.o_fw), *bp = f32(k.o_b), *lse = f32(k.o_lse), *zl = f32(k.o_zl), *gp = f32(k.o_gp);
  hipStream_t st = a.st;
  const bool rows_form = a.HW == 1, hb = (a.types & 1) != 0, wb = (a.types & 2) != 0;
  const int drop = need_grad ? 1 : 0;
  {
    const CePack pw{a.w, a.b, nullptr, 0, 0, w, wpl, fw, bp, nullptr, a.V, k.Vp, a.C, k.Cp};
    const CePack ph{a.h, nullptr, a.labels, a.V, drop, x, xpl, fx, nullptr, lab, a.N, (int)k.Pp, a.C, k.Cp};
    const bool vec = a.C % 8 == 0 && aligned16(a.w) && (!rows_form || aligned16(a.h));
    const int wblocks = k.Vp / 4;
    const dim3 grid = ce_grid(wblocks + (rows_form ? k.Pp / 4 : 0)), block(256);
    if (hb && wb && vec) MS_LAUNCH((ce_pack_rows_kernel<ms_bf16, ms_bf16, true>), grid, block, 0, st, pw, ph, wblocks);
    else if (hb && wb) MS_LAUNCH((ce_pack_rows_kernel<ms_bf16, ms_bf16, false>), grid, block, 0, st, pw, ph, wblocks);
    else if (hb && vec) MS_LAUNCH((ce_pack_rows_kernel<ms_bf16, float, true>), grid, block, 0, st, pw, ph, wblocks);
    else if (hb) MS_LAUNCH((ce_pack_rows_kernel<ms_bf16, float, false>), grid, block, 0, st, pw, ph, wblocks);
    else if (wb && vec) MS_LAUNCH((ce_pack_rows_kernel<float, ms_bf16, true>), grid, block, 0, st, pw, ph, wblocks);
    else if (wb) MS_LAUNCH((ce_pack_rows_kernel<float, ms_bf16, false>), grid, block, 0, st, pw, ph, wblocks);
    else if (vec) MS_LAUNCH((ce_pack_rows_kernel<float, float, true>), grid, block, 0, st, pw, ph, wblocks);
    else MS_LAUNCH((ce_pack_rows_kernel<float, float, false>), grid, block, 0, st, pw, ph, wblocks);
    if (int e = check_launch("class_ce_pack")) return e;
  }
  if (!rows_form) {
    const dim3 gx = ce_grid(k.Pp / 64);
    if (hb) MS_LAUNCH((ce_pack_planes_kernel<ms_bf16, 1>), gx, dim3(1024), 0, st, a.h, a.labels, a.V, drop, x, xpl, fx, lab, k.P, k.Pp, a.C, k.Cp, a.HW);
    else MS_LAUNCH((ce_pack_planes_kernel<float, 2>), gx, dim3(1024), 0, st, a.h, a.labels, a.V, drop, x, xpl, fx, lab, k.P, k.Pp, a.C, k.Cp, a.HW);
    if (int e = check_launch("class_ce_pack")) return e;
  }
  const int nslots = (int)std::min<long>(kCeSlots, k.P / 1024 + 1);
  if (a.mean_valid) {
    MS_LAUNCH(ce_count_kernel, dim3(nslots), dim3(256), 0, st, a.labels, k.P, a.V, slots);
    if (int e = check_launch("class_ce_count")) return e;
  }
  float* hot = need_grad ? f32(k.o_hot) : nullptr;
  const CeRowGrad rg{gp, hot, fx, a.sign, a.mean_valid, a.scale_dev, slots, nslots, rowmax};
  CeGemm g{};
  g.fw = fw; g.bpad = bp; g.fx = fx; g.lab = lab; g.lse = lse; g.gp = gp; g.hot = hot; g.scal = scal; g.zlab = zl;
  if (a.lse_in == nullptr) {
    // logits -> statistics: M = classes, N = rows
    for (long p0 = 0; p0 < k.Pp; p0 += k.sb) {
      const int pn = (int)std::min<long>(k.sb, k.Pp - p0);
      CeGemm d = g;
      d.a = CeOperand{w, wpl, k.Cp, 0}; d.b = CeOperand{x + (size_t)p0 * k.Cp, xpl, k.Cp, 0};
      ce_pairs(d, k.wp, k.xp);
      d.ksteps = k.Cp / kCeBK; d.split = 1; d.v0 = 0; d.p0 = p0;
      d.part = (float2*)(ws + k.o_part); d.part_stride = (size_t)pn;
      const CeTile tile = ce_tile<CE_STATS>(a.V, std::min<long>(pn, k.P - p0), 1, k.Vp, pn);
      if (int e = ce_gemm<CE_STATS, false, false>(d, tile, st, "class_ce_stats")) return e;
      MS_LAUNCH(ce_join_kernel, dim3((unsigned)(pn / 64)), dim3(1024), 0, st, (const float2*)d.part, tile.mt * 2, d.part_stride, zl, lab, lse, a.lse, a.nll,
                (double*)(ws + k.o_lsum), p0, k.P, need_grad ? rg : CeRowGrad{});
      if (int e = check_launch("class_ce_join")) return e;
    }
  }
  const int nrow = a.lse_in != nullptr ? (int)std::min<long>(k.Pp / 256, kCeRowBlocks) : (int)(k.Pp / 64);
  if (a.lse_in != nullptr) {
    MS_LAUNCH(ce_rowgrad_kernel, dim3(nrow), dim3(256), 0, st, a.grad, lab, fx, gp, a.lse_in, lse, hot, rowmax, k.P, k.Pp);
    if (int e = check_launch("class_ce_rowgrad")) return e;
  }
  if (need_grad || a.loss != nullptr) {
    CeLevel l{};
    l.lsum = (const double*)(ws + k.o_lsum); l.n = (int)(k.Pp / 64); l.sign = a.sign; l.mean_valid = a.mean_valid; l.slots = slots; l.nslots = nslots; l.P = k.P; l.loss = a.loss;
    if (need_grad) {
      l.rowmax = rowmax; l.nrow = nrow; l.fx = fx; l.gp = gp; l.fw = fw; l.bpad = bp; l.fx2 = f32(k.o_fx2); l.fw2 = f32(k.o_fw2); l.x = x; l.w = w; l.xpl = xpl; l.wpl = wpl;
      l.xp = k.xp; l.wp = k.wp; l.V = a.V; l.Vp = k.Vp; l.Cp = k.Cp; l.Pp = k.Pp; l.scal = scal;
    }
    const int blocks = need_grad ? (int)std::min<long>(kNumCU, (k.Vp + k.Pp) / 256) : 1;        // (every workgroup finds the largest exponents for itself)
    MS_LAUNCH(ce_level_kernel, dim3(blocks), dim3(1024), 0, st, l);
    if (int e = check_launch("class_ce_level")) return e;
  }
  if (need_grad) { fx = f32(k.o_fx2); fw = f32(k.o_fw2); g.fx = fx; g.fw = fw; }
  if (!need_grad) return MS_OK;
  const long cp = ce_up(k.Cp, 128);
  for (long p0 = 0; p0 < k.Pp; p0 += k.pb) {
    const int pn = (int)std::min<long>(k.pb, k.Pp - p0);
    for (int v0 = 0; v0 < k.Vp; v0 += k.vb) {
      const int vn = std::min(k.vb, k.Vp - v0);
      CeGemm d = g;
      d.a = CeOperand{w + (size_t)v0 * k.Cp, wpl, k.Cp, 0}; d.b = CeOperand{x + (size_t)p0 * k.Cp, xpl, k.Cp, 0};
      ce_pairs(d, k.wp, k.xp);
      d.ksteps = k.Cp / kCeBK; d.split = 1; d.v0 = v0; d.p0 = p0;
      _Float16* G = (_Float16*)(ws + k.o_g);
      const size_t gpl = (size_t)k.pb * k.vb;
      d.g = G; d.g_plane = gpl; d.g_ld = k.vb;
      d.dbpart = a.db != nullptr ? f32(k.o_db) : nullptr; d.db_stride = k.vb;
      const int rows = (int)std::min<long>(pn, k.P - p0), vr = std::min(vn, a.V - v0);      // (never empty: the padding is less than a piece's granule)
      const CeTile tile = ce_tile<CE_GRAD>(vr, rows, 1, vn, pn);
      if (k.gpl == 2) { if (int e = ce_gemm<CE_GRAD2, false, false>(d, tile, st, "class_ce_grad")) return e; }
      else { if (int e = ce_gemm<CE_GRAD, false, false>(d, tile, st, "class_ce_grad")) return e; }
      CeSums sums{};
      sums.scal = scal;
      if (a.db != nullptr) {
        sums.dbpart = f32(k.o_db); sums.dbn = tile.nt * 2; sums.dbstride = (size_t)k.vb; sums.db = a.db; sums.dbfirst = p0 == 0; sums.dbV = vr; sums.dbv0 = v0;
        sums.dbblocks = cdiv(vr, 64);
      }
      CeGemm gh{}, gw{};
      CeTile th{}, tw{};
      if (a.dh != nullptr) {        // dh^T [channels][pixels] = w^T G^T, or dh [rows][channels] = G w where the channels are neighbours
        CeGemm& o = gh;
        const CeOperand ow{w + (size_t)v0 * k.Cp, wpl, k.Cp, k.Cp}, og{G, gpl, k.vb, 0};
        if (rows_form) ce_pairs(o, k.gpl, k.wp); else ce_pairs(o, k.wp, k.gpl);
        o.ksteps = cdiv(vr, kCeBK); o.split = std::min(k.split_x, std::max(1, o.ksteps * o.nseg / kCeDeep));
        o.out = f32(k.o_px); o.out_split = (size_t)cp * k.pb;
        if (rows_form) {
          o.a = og; o.b = ow; o.out_ld = (int)cp;
          th = ce_tile<CE_OUT>(rows, a.C, o.split, pn, cp);
        } else {
          o.a = ow; o.b = og; o.out_ld = k.pb;
          th = ce_tile<CE_OUT>(a.C, rows, o.split, cp, pn);
        }
        CeSum& q = sums.h;
        q = CeSum{o.out, o.out_split, o.out_ld, o.split, fx, hb ? f32(k.o_ax) : (float*)a.dh, a.dh, v0 == 0, v0 + vn >= k.Vp, rows_form ? rows : a.C, rows_form ? a.C : rows, p0, a.HW, a.C, 0, 0};
        q.rblocks = cdiv(q.rows, 4); q.blocks = q.rblocks * std::min(cdiv(q.cols, 64), rows_form ? 4 : 64);
      }
      if (a.dw != nullptr) {        // dw [classes][channels] = G^T h
        CeGemm& o = gw;
        o.a = CeOperand{G, gpl, k.vb, k.vb}; o.b = CeOperand{x + (size_t)p0 * k.Cp, xpl, k.Cp, k.Cp};
        ce_pairs(o, k.gpl, k.xp);
        o.ksteps = cdiv(rows, kCeBK); o.split = std::min(k.split_w, std::max(1, o.ksteps * o.nseg / kCeDeep));
        o.out = f32(k.o_pw); o.out_ld = (int)cp; o.out_split = (size_t)k.vb * cp;
        tw = ce_tile<CE_OUT>(vr, a.C, o.split, vn, cp);
        CeSum& q = sums.w;
        q = CeSum{o.out, o.out_split, o.out_ld, o.split, fw, wb ? f32(k.o_aw) : (float*)a.dw, a.dw, p0 == 0, p0 + pn >= k.Pp, vr, a.C, (long)v0, 1, a.C, 0, 0};
        q.rblocks = cdiv(q.rows, 4); q.blocks = q.rblocks * std::min(cdiv(q.cols, 64), 4);
      }
      if (th.t == tw.t && th.t < 256) {
        gh.mt = th.mt; gh.nt = th.nt; gw.mt = tw.mt; gw.nt = tw.nt;
        const int nh = th.mt * th.nt * gh.split, n = nh + tw.mt * tw.nt * gw.split;
        if (n > 0) {
          if (th.t == 128 && rows_form) MS_LAUNCH((ce_grads_kernel<128, 2, true>), dim3(n), dim3(256), 0, st, gh, gw, nh);
          else if (th.t == 128) MS_LAUNCH((ce_grads_kernel<128, 2, false>), dim3(n), dim3(256), 0, st, gh, gw, nh);
          else if (rows_form) MS_LAUNCH((ce_grads_kernel<64, 4, true>), dim3(n), dim3(256), 0, st, gh, gw, nh);
          else MS_LAUNCH((ce_grads_kernel<64, 4, false>), dim3(n), dim3(256), 0, st, gh, gw, nh);
          if (int e = check_launch("class_ce_grads")) return e;
        }
      } else {
        if (a.dh != nullptr) {
          if (rows_form) { if (int e = ce_gemm<CE_OUT, false, true>(gh, th, st, "class_ce_dh")) return e; }
          else { if (int e = ce_gemm<CE_OUT, true, false>(gh, th, st, "class_ce_dh")) return e; }
        }
        if (a.dw != nullptr) { if (int e = ce_gemm<CE_OUT, true, true>(gw, tw, st, "class_ce_dw")) return e; }
      }
      const int blocks = sums.dbblocks + sums.h.blocks + sums.w.blocks;
      if (blocks > 0) {
        if (hb && wb) MS_LAUNCH((ce_sums_kernel<ms_bf16, ms_bf16>), dim3(blocks), dim3(256), 0, st, sums);
        else if (hb) MS_LAUNCH((ce_sums_kernel<ms_bf16, float>), dim3(blocks), dim3(256), 0, st, sums);
        else if (wb) MS_LAUNCH((ce_sums_kernel<float, ms_bf16>), dim3(blocks), dim3(256), 0, st, sums);
        else MS_LAUNCH((ce_sums_kernel<float, float>), dim3(blocks), dim3(256), 0, st, sums);
        if (int e = check_launch("class_ce_sums")) return e;
      }
    }
  }
  return MS_OK;
}
}  // namespace ms

extern "C" size_t ms_class_ce_ws_bytes(int N, int C, int V, int HW, int types, int need_grad) {
  if (ms::ce_check(N, C, V, HW, types, "ms_class_ce_ws_bytes")) return 0;
  if (ms::ce_narrow_ok(N, C, V, HW)) return ms::ce_narrow_ws_bytes(N, C, V, HW, types, need_grad != 0);
  return ms::ce_plan(N, C, V, HW, types, need_grad != 0).total;
}
extern "C" int ms_class_ce(const void* h, const void* w, const float* b, const int64_t* labels, float* loss_out, void* dh, void* dw, float* db, int N, int C, int V, int HW,
                           int types, float loss_sign, int mean_valid, const float* grad_scale_dev, void* ws, size_t ws_bytes, void* stream) {
  if (loss_out == nullptr) { ms::set_error("ms_class_ce: loss_out is NULL"); return MS_ERR_INVALID; }
  ms::CeArgs a{};
  a.h = h; a.w = w; a.b = b; a.labels = labels; a.loss = loss_out; a.dh = dh; a.dw = dw; a.db = db;
  a.sign = loss_sign; a.mean_valid = mean_valid ? 1 : 0; a.scale_dev = grad_scale_dev;
  a.N = N; a.C = C; a.V = V; a.HW = HW; a.types = types; a.ws = ws; a.ws_bytes = ws_bytes; a.st = (hipStream_t)stream;
  return ms::ce_run(a, "ms_class_ce");
}
extern "C" int ms_class_ce_fwd(const void* h, const void* w, const float* b, const int64_t* labels, float* nll, float* lse, int N, int C, int V, int HW, int types,
                               void* ws, size_t ws_bytes, void* stream) {
  if (nll == nullptr || lse == nullptr) { ms::set_error("ms_class_ce_fwd: null pointer"); return MS_ERR_INVALID; }
  ms::CeArgs a{};
  a.h = h; a.w = w; a.b = b; a.labels = labels; a.nll = nll; a.lse = lse; a.sign = 1.f;
  a.N = N; a.C = C; a.V = V; a.HW = HW; a.types = types; a.ws = ws; a.ws_bytes = ws_bytes; a.st = (hipStream_t)stream;
  return ms::ce_run(a, "ms_class_ce_fwd");
}
extern "C" int ms_class_ce_bwd(const void* h, const void* w, const float* b, const int64_t* labels, const float* lse, const float* grad, void* dh, void* dw, float* db,
                               int N, int C, int V, int HW, int types, void* ws, size_t ws_bytes, void* stream) {
  if (lse == nullptr || grad == nullptr || (dh == nullptr && dw == nullptr && db == nullptr)) { ms::set_error("ms_class_ce_bwd: null pointer"); return MS_ERR_INVALID; }
  ms::CeArgs a{};
  a.h = h; a.w = w; a.b = b; a.labels = labels; a.lse_in = lse; a.grad = grad; a.dh = dh; a.dw = dw; a.db = db; a.sign = 1.f;
  a.N = N; a.C = C; a.V = V; a.HW = HW; a.types = types; a.ws = ws; a.ws_bytes = ws_bytes; a.st = (hipStream_t)stream;
  return ms::ce_run(a, "ms_class_ce_bwd");
}
