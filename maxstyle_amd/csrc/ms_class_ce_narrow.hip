// Head + softmax cross entropy over many classes, narrow form (C <= 128, unless there are many classes for few rows): no operand and no product ever leaves the chip; see ms_class_ce.h.
//
//   prep    w -> fp16 planes in the order the LDS wants them, 64 classes a chunk with one power-of-two scale (an "image": the next kernel's DMA copies it as it
//           lies); rows that take part counted
//   pixels  a wave keeps NJ x 16 pixels' features in registers (one read of h) and runs over the classes once: e = exp(z - m) against a running maximum m is already
//           in the register layout the second product wants, o += w^T e, l += e; at the end dh = g (o / l - w[label]).  One read of h, one write of dh, w from L2.
//   classes roles exchanged: a wave keeps NJ x 16 classes' weights in registers and runs over pixels: z again, G, dw += h G^T, db += G.  Pixels are split over
//           workgroups; the partial dw are summed by
//   join    in a fixed order, with the loss.
// 8 P V C products, and nothing of size P V is stored.  What a training call waits for is the vector unit: counted over whole kernels, a logit (the padding's included) costs 18 vector
// instructions in the pixel pass and 15 - 16 in the class pass, 9 where the value alone is asked for, an exp2 among them.  Of the pixel pass's, 5.6 are the loop's exponent, sum and split into
// planes; the others scale the logit, keep the maximum and pick the label's logit (more of it where labels do not come in regions), or belong to the pixels' load and dh.
// 1M pixels, 104 classes, 16 channels: pixel pass 81 us, every cycle of the vector unit taken; class pass 85, 75 % of them.  256 classes, 64 channels (bf16): 231 and 225 us, 71 % and 60 %,
// the matrix cores 33 % and 25 %.  The value alone, 295k x 1000 classes x 64: 133 us, 83 % and 43 %.
#include <algorithm>
#include <type_traits>
#include "ms_class_ce.h"
#include "ms_class_ce_narrow.h"
#include "maxstyle_hip.h"

namespace ms {

constexpr int kCnClasses = 64;        // classes of one image chunk
constexpr int kCnPrep = 256;          // most workgroups that count
// 16-column groups a wave keeps.  Pixels: 2 - 4 halve the LDS reads a product, but leave two waves a SIMD for 3 to 4 (400k pixels x 64 channels, 151 classes: 144 -> 113 us).
// Classes: 4 where the registers hold them and there are that many (one pixel tile then serves 256 classes: 1M pixels x 64, 256 classes: 301 -> 227 us), else 2.
constexpr int kCnNJ = 2;

// Widths: KS steps of 32 channels; KS = 0 is 16 channels (the narrow networks' head) on the 16-deep matrix instruction, half the registers and loads of a padded step.
template <int KS> struct CnW {
  static constexpr int kW = KS == 0 ? 16 : KS * 32;              // channels of a packed row
  static constexpr int kN = KS == 0 ? 1 : KS;                    // k-steps
  static constexpr int kF = KS == 0 ? 4 : 8;                     // channels of a lane's fragment: ks * 32 + q * kF + k
  static constexpr int kCT = kW / 16;
  typedef typename std::conditional<KS == 0, ms_h4, ms_h8>::type Frag;
};
__device__ __forceinline__ ms_f4 cn_mfma(ms_h8 a, ms_h8 b, ms_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ ms_f4 cn_mfma(ms_h4 a, ms_h4 b, ms_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }

// 16-byte chunk j of row r of a tile of kW columns lies at chunk j ^ cn_swz(r): both the row reads and the transposing reads below are then free of bank conflicts
template <int KS> __device__ __forceinline__ int cn_swz(int r) { return KS == 0 ? 0 : KS == 1 ? (r >> 1) & 3 : (KS == 3 ? (r >> 2) & 3 : r & 7); }
template <int KS, int WP> struct CnImage {
  static constexpr int kPlane = kCnClasses * CnW<KS>::kW;                    // halves of one plane
  static constexpr int kBytes = WP * kPlane * 2 + 1024;                  // + 64 x {b log2(e)}, 2^e log2(e), 2^e of the chunk
};

// transposing read: lane (q, i) gets column mn + i of rows k .. k + 3, k = k0 + 4 q (swizzled tile of kW columns)
template <int KS>
__device__ __forceinline__ ms_h8 cn_tr2(const _Float16* tile, int k0, int k1, int mn, int lane) {
  const int q = lane >> 4, i = lane & 15;
  typedef __attribute__((address_space(3))) ms_s4* lp;
  union { ms_s4 s[2]; ms_h8 h; } u;
  const int ra = k0 + q * 4 + (i >> 2), rb = k1 + q * 4 + (i >> 2), ch = (mn >> 3) + ((i & 3) >> 1), off = (i & 1) * 4;
  u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(tile + ra * CnW<KS>::kW + ((ch ^ cn_swz<KS>(ra)) * 8) + off));
  u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(tile + rb * CnW<KS>::kW + ((ch ^ cn_swz<KS>(rb)) * 8) + off));
  return u.h;
}

// One workgroup a chunk of classes (the first nch), and all of them count: slots[block] = rows that take part.
// One scale for 64 classes: a weight is held to 2^-22, or 2^-39 of the chunk's largest - an absolute error that no logit notices.
template <typename WT, int WP, int KS>
__global__ __launch_bounds__(256) void cn_prep_kernel(const void* __restrict__ w, const float* __restrict__ b, const int64_t* __restrict__ labels, long P, int count,
                                                      char* __restrict__ img, int* __restrict__ slots, int nslots, int V, int nch, int C) {
  using IO = ActIO<WT>;
  using IM = CnImage<KS, WP>;
  __shared__ int red[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if ((int)blockIdx.x < nch) {
    const int v0 = blockIdx.x * 64;
    constexpr int kW = CnW<KS>::kW, kPer = 64 * kW / 256;
    float x[kPer], bv[kPer];
    // (clamped addresses: no load waits for another)
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = k * 256 + threadIdx.x;
      x[k] = IO::ld1(w, (size_t)min(v0 + i / kW, V - 1) * C + min(i % kW, C - 1));
      bv[k] = 0.f;
    }
    if (b != nullptr) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) bv[k] = b[min(v0 + (k * 256 + (int)threadIdx.x) / kW, V - 1)];
    }
    unsigned am = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = k * 256 + threadIdx.x, r = i / kW, c = i % kW;
      // a class that is switched off (b = -inf) may hold anything finite: its logit is -inf, and it sets no scale
      if (v0 + r >= V || c >= C || bv[k] == -__builtin_inff()) x[k] = 0.f;
      const unsigned bits = __float_as_uint(x[k]) & 0x7FFFFFFFu;
      am = max(am, bits < 0x7F800000u ? bits : 0u);          // (an infinity or NaN spoils its own class only)
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) am = max(am, (unsigned)__shfl_xor((int)am, off, 64));
    if (lane == 0) red[wave] = (int)am;
    __syncthreads();
    am = max(max((unsigned)red[0], (unsigned)red[1]), max((unsigned)red[2], (unsigned)red[3]));
    __syncthreads();
    const int e = ce_exponent(__uint_as_float(am));
    const float inv = ce_pow2(-e);
    char* im = img + (size_t)blockIdx.x * IM::kBytes;
    _Float16* pl = (_Float16*)im;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = k * 256 + threadIdx.x, r = i / kW, c = i % kW;
      _Float16 hi, lo;
      ce_split(x[k] * inv, hi, lo);
      const int at = r * kW + (((c >> 3) ^ cn_swz<KS>(r)) * 8) + (c & 7);
      pl[at] = hi;
      if (WP == 2) pl[IM::kPlane + at] = lo;
    }
    float* t = (float*)(im + WP * IM::kPlane * 2);
    if (threadIdx.x < 64) t[threadIdx.x] = v0 + (int)threadIdx.x < V ? (b != nullptr ? b[v0 + threadIdx.x] * kLog2e : 0.f) : -__builtin_inff();
    if (threadIdx.x == 64) { t[64] = ce_pow2(e) * kLog2e; t[65] = ce_pow2(e); }
  }
  if (!count || (int)blockIdx.x >= nslots) return;
  int k = 0;
  for (long p = (long)blockIdx.x * 256 + threadIdx.x; p < P; p += (long)nslots * 256) { const int64_t l = labels[p]; k += (l >= 0 && l < V) ? 1 : 0; }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) k += __shfl_xor(k, off, 64);
  if (lane == 0) red[wave] = k;
  __syncthreads();
  if (threadIdx.x == 0) slots[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// rows that take part, from the prep pass's slots (at most 256: one a thread of the first four waves)
__device__ __forceinline__ int cn_count(const int* __restrict__ slots, int n, int* red /* a word a wave */) {
  int s = threadIdx.x < (unsigned)n ? slots[threadIdx.x] : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

template <int WP, int KS>
__device__ __forceinline__ void cn_stage(const char* img, int chunk, unsigned lds, int wave, int lane) {
  constexpr int kN = CnImage<KS, WP>::kBytes / 1024;
  const ms_i32x4 rs = ms_dma_rsrc(img + (size_t)chunk * CnImage<KS, WP>::kBytes);
  for (int i = wave; i < kN; i += 4) ms_lds_dma16(rs, __builtin_amdgcn_readfirstlane(lds + i * 1024), i * 1024 + lane * 16, 0);
}

struct CnArgs {
  const void *h, *w; const int64_t* labels; const char* img; const int* slots; int nslots;
  float *nll, *lse_out; const float *lse_in, *grad, *scale_dev; float sign; int mean_valid, drop;
  void* dh; double* lsum;
  float *fx, *lse2, *gp, *hot; int* lab;    // what the class pass needs of every row (NULL: it does not run)
  long P; int C, HW, V, nch, w_vec;
  int full;                                 // C is the kernel's full width and h spans less than 4 GB: addresses are a scalar base and a 32-bit offset
};

// The running maximum m is moved only when a logit exceeds it by more than kCnSlack (in log2), for a whole wave at once: e = 2^(kCnTop + z - m) then stays below 2^15 in
// fp16 (and is held to 2^-34 of e at m: the lowest step of its low plane), and classes after the first few cost no rescaling - with a slack of 1 some pixel of 64 still
// had it done for most of 256 classes.  With the log-sum given (lse_in) m is that, and never moves.
constexpr float kCnSlack = 6.f, kCnTop = 9.f;
template <typename HT, typename WT, int KS, int NJ, bool DH>
__global__ __launch_bounds__(256, 2) void cn_pixels_kernel(CnArgs a) {
  using IO = ActIO<HT>;
  constexpr int HP = sizeof(HT) == 4 ? 2 : 1, WP = sizeof(WT) == 4 ? 2 : 1, CT = CnW<KS>::kCT, KN = CnW<KS>::kN, KF = CnW<KS>::kF, kW = CnW<KS>::kW;
  typedef typename CnW<KS>::Frag Frag;
  using IM = CnImage<KS, WP>;
  __shared__ __attribute__((aligned(1024))) char sm[2][IM::kBytes];
  __shared__ int redi[4];
  __shared__ double redd[16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const unsigned lds0 = ms_lds_addr(&sm[0][0]);
  const bool online = a.lse_in == nullptr;
  const int nch = (online || DH) ? a.nch : 0;
  if (nch > 0) cn_stage<WP, KS>(a.img, 0, lds0, wave, lane);

  // ---- this wave's pixels: scaled fp16 planes in the layout of a matrix operand (column = pixel li, 8 channels 32 ks + 8 q + k)
  Frag x[HP][KN][NJ];
  float fx[NJ];
  int lab[NJ];
  const int pw = (int)blockIdx.x * (4 * NJ * 16) + wave * (NJ * 16) + li;      // (at most 2^30 rows)
  const int P = (int)a.P;
  // every load unconditional, at a clamped address, and all of them in flight together (loads behind branches wait for one another: 20 us more at 400k pixels x 64 channels)
  float v[NJ][KN][KF];
  unsigned off[NJ];                    // of the pixel's first channel, in bytes (`full`)
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int p = min(pw + j * 16, P - 1), n = p / a.HW;
    const int64_t lb = a.labels[p];
    lab[j] = (lb >= 0 && lb < a.V && pw + j * 16 < P) ? (int)lb : -1;
    off[j] = ((unsigned)n * (unsigned)a.C * (unsigned)a.HW + (unsigned)(p - n * a.HW)) * (unsigned)sizeof(HT);
    if (a.full) {
      const unsigned at = off[j] + (unsigned)(q * KF) * (unsigned)a.HW * (unsigned)sizeof(HT);
#pragma unroll
      for (int ks = 0; ks < KN; ++ks)
#pragma unroll
        for (int k = 0; k < KF; ++k) v[j][ks][k] = IO::ld1((const char*)a.h + (size_t)(ks * 32 + k) * a.HW * sizeof(HT) + at, 0);
    } else {
      const size_t base = (size_t)n * a.C * a.HW + (size_t)(p - n * a.HW);
#pragma unroll
      for (int ks = 0; ks < KN; ++ks)
#pragma unroll
        for (int k = 0; k < KF; ++k) v[j][ks][k] = IO::ld1(a.h, base + (size_t)min(ks * 32 + q * KF + k, a.C - 1) * a.HW);
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const bool live = pw + j * 16 < P && (!a.drop || lab[j] >= 0);
    unsigned am = 0;
#pragma unroll
    for (int ks = 0; ks < KN; ++ks)
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        if (!live || ks * 32 + q * KF + k >= a.C) v[j][ks][k] = 0.f;
        am = max(am, __float_as_uint(v[j][ks][k]) & 0x7FFFFFFFu);
      }
    am = max(am, (unsigned)__shfl_xor((int)am, 16, 64));
    am = max(am, (unsigned)__shfl_xor((int)am, 32, 64));
    const int e = ce_exponent(__uint_as_float(am));
    const float inv = ce_pow2(-e);
    fx[j] = am == 0u ? 0.f : ce_pow2(e);          // 0: a pixel of zeros, which sets no scale in the class pass
#pragma unroll
    for (int ks = 0; ks < KN; ++ks)
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        _Float16 hi, lo;
        ce_split(v[j][ks][k] * inv, hi, lo);
        x[0][ks][j][k] = hi;
        if (HP == 2) x[HP - 1][ks][j][k] = lo;
      }
  }

  int key[NJ];                         // the 32 classes that the label lies in, for the lane of the four that has it
  float m[NJ], l[NJ], zl[NJ];          // in units of log2; m is the same in the four lanes of a pixel, l and zl are each lane's part
  ms_f4 o[CT][NJ];
  float scale = 1.f;                   // 2^e of the chunk that o is measured in
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    key[j] = lab[j] >= 0 && ((lab[j] >> 2) & 3) == q ? lab[j] >> 5 : -1;
    m[j] = -__builtin_inff(); l[j] = 0.f; zl[j] = 0.f;
    if (!online) {
      m[j] = pw + j * 16 < P ? a.lse_in[pw + j * 16] * kLog2e : 0.f;
      if (m[j] == -__builtin_inff()) m[j] = __builtin_nanf("");          // every class is switched off: there is no softmax
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
  }
  for (int t = 0; t < nch; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                   // chunk t has landed for every wave, and nobody reads the buffer that chunk t + 1 goes to
    if (t + 1 < nch) cn_stage<WP, KS>(a.img, t + 1, lds0 + (unsigned)((t + 1) & 1) * (unsigned)IM::kBytes, wave, lane);
    const _Float16* wp = (const _Float16*)sm[t & 1];
    const float* tb = (const float*)(sm[t & 1] + WP * IM::kPlane * 2);
    const float wl2 = tb[64];
    if (DH) {
      const float sc = tb[65];
      if (sc != scale) {               // (chunks of like weights share a scale)
        const float f = scale / sc;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[c][j] *= f;
        scale = sc;
      }
    }
    float fs[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) fs[j] = fx[j] * wl2;
#pragma unroll 1
    for (int h2 = 0; h2 < 2; ++h2) {
      if (t * kCnClasses + h2 * 32 >= a.V) break;
      // z of two tiles of 16 classes: 4 q + r of each
      ms_f4 s[2][NJ];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) s[tt][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
        const int r = h2 * 32 + tt * 16 + li;
#pragma unroll
        for (int ks = 0; ks < KN; ++ks) {
          const int at = r * kW + (KS == 0 ? q * 4 : ((ks * 4 + q) ^ cn_swz<KS>(r)) * 8);
          const Frag hi = *reinterpret_cast<const Frag*>(wp + at);
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[tt][j] = cn_mfma(hi, x[0][ks][j], s[tt][j]);
          if (HP == 2) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[tt][j] = cn_mfma(hi, x[HP - 1][ks][j], s[tt][j]);
          }
          if (WP == 2) {
            const Frag lo = *reinterpret_cast<const Frag*>(wp + IM::kPlane + at);
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[tt][j] = cn_mfma(lo, x[0][ks][j], s[tt][j]);
          }
        }
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const float4 b = *reinterpret_cast<const float4*>(tb + h2 * 32 + tt * 16 + q * 4);
        const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[tt][j][r] = __builtin_fmaf(s[tt][j][r], fs[j], bb[r]);
      }
      if (online) {
        bool grow = false, here = false;
        float mx[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          mx[j] = fmaxf(fmaxf(fmaxf(s[0][j][0], s[0][j][1]), fmaxf(s[0][j][2], s[0][j][3])), fmaxf(fmaxf(s[1][j][0], s[1][j][1]), fmaxf(s[1][j][2], s[1][j][3])));
          grow |= mx[j] > m[j] + kCnSlack;
          here |= key[j] == t * 2 + h2;
        }
        if (__any(here)) {             // some pixel's label is among these 32 classes (seldom so in a label map): chosen by its bits 0, 1 and 4
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            float z[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
              const float z0 = (lab[j] & 1) != 0 ? s[tt][j][1] : s[tt][j][0], z1 = (lab[j] & 1) != 0 ? s[tt][j][3] : s[tt][j][2];
              z[tt] = (lab[j] & 2) != 0 ? z1 : z0;
            }
            const float zz = (lab[j] & 16) != 0 ? z[1] : z[0];
            zl[j] = key[j] == t * 2 + h2 ? zz : zl[j];
          }
        }
        if (__any(grow)) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            float mn = fmaxf(m[j], mx[j]);
            mn = fmaxf(mn, __shfl_xor(mn, 16, 64));
            mn = fmaxf(mn, __shfl_xor(mn, 32, 64));
            const float f = m[j] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[j] - mn);
            m[j] = mn;
            l[j] *= f;
            if (DH) {
#pragma unroll
              for (int c = 0; c < CT; ++c) o[c][j] *= f;
            }
          }
        }
      }
      ms_h8 gh[NJ], gl[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float mm = (m[j] == -__builtin_inff() ? 0.f : m[j]) - kCnTop;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[tt][j][r] = __builtin_amdgcn_exp2f(s[tt][j][r] - mm);
            l[j] += s[tt][j][r];
          }
        if (DH) ce_split8(s[0][j], s[1][j], gh[j], gl[j]);
      }
      if (DH) {
        // Two planes of e also for a bf16 dh: o / l - w[label] nearly cancels where the network is sure, and has to be right to more than e's 11 bits there.
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const ms_h8 wh = cn_tr2<KS>(wp, h2 * 32, h2 * 32 + 16, c * 16, lane);
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, gh[j], o[c][j], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, gl[j], o[c][j], 0, 0, 0);
          if (WP == 2) {                    // (also for a bf16 dh: where the classes' weights are nearly equal dh is their difference)
            const ms_h8 wl = cn_tr2<KS>(wp + IM::kPlane, h2 * 32, h2 * 32 + 16, c * 16, lane);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl, gh[j], o[c][j], 0, 0, 0);
          }
        }
      }
    }
  }
  // ---- rows: loss, what the class pass needs, dh
  const float cnt = (float)(a.mean_valid ? max(cn_count(a.slots, a.nslots, redi), 1) : P);
  double acc_l = 0.0;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int p = pw + j * 16;
    float lse2 = m[j], fac = 1.f, rest = 0.f;
    const float top = m[j] == -__builtin_inff() ? kCnTop : m[j] - (m[j] - kCnTop);          // what the exponentials were raised by (kCnTop where m holds it)
    if (!online) {
      rest = ce_rest_nat(a.lse_in[min(p, P - 1)], lse2);
      fac = __builtin_amdgcn_exp2f(-top) * __builtin_amdgcn_exp2f(-rest);
    } else {
      l[j] += __shfl_xor(l[j], 16, 64);
      l[j] += __shfl_xor(l[j], 32, 64);
      zl[j] += __shfl_xor(zl[j], 16, 64);             // (one lane of the four holds it, the others 0)
      zl[j] += __shfl_xor(zl[j], 32, 64);
      fac = 1.f / l[j];
      const float lg = ce_log2(l[j], top);
      lse2 = m[j] + lg;
      rest = ce_rest(m[j], lg, lse2);
      const float ln2 = 0.693147180559945309f, nll = lab[j] >= 0 ? ((m[j] - zl[j]) + lg) * ln2 : 0.f;
      if (q == 0 && p < P) {
        if (a.nll != nullptr) { a.nll[p] = nll; a.lse_out[p] = ce_lse_nat(m[j], lg); }
        acc_l += (double)nll;
      }
    }
    float gp = 0.f;
    if (lab[j] >= 0) gp = a.grad != nullptr ? a.grad[p] : a.sign / cnt * (a.scale_dev != nullptr ? *a.scale_dev : 1.f);
    if (a.fx != nullptr) {
      if (q == 0) {                                   // (arrays padded to whole workgroups)
        const float d = gp == 0.f ? 0.f : rest;
        a.fx[p] = fx[j]; a.gp[p] = gp * __builtin_amdgcn_exp2f(-d); a.hot[p] = __builtin_amdgcn_exp2f(d); a.lab[p] = lab[j];
        a.lse2[p] = gp == 0.f ? __builtin_inff() : lse2;        // a row that takes no part: exp2(z - inf) = 0 whatever z is
      }
    }
    if (DH) {
      const size_t wrow = (size_t)max(lab[j], 0) * a.C;
      const float f = scale * fac;
      float wl[CT][4];                    // the label's weights (16 bytes a lane: 4-byte loads from 64 rows at once cost 100 us a million pixels)
      if (a.w_vec) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const float4 t = ActIO<WT>::ld4(a.w, wrow + min(c * 16 + q * 4, a.C - 4));
          wl[c][0] = t.x; wl[c][1] = t.y; wl[c][2] = t.z; wl[c][3] = t.w;
        }
      } else {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) wl[c][r] = ActIO<WT>::ld1(a.w, wrow + min(c * 16 + q * 4 + r, a.C - 1));
      }
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) wl[c][r] = gp == 0.f ? 0.f : gp * (o[c][j][r] * f - wl[c][r]);
      if (a.full) {
        const unsigned at = off[j] + (unsigned)(q * 4) * (unsigned)a.HW * (unsigned)sizeof(HT);
        if (p < P) {
#pragma unroll
          for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) IO::st1((char*)a.dh + (size_t)(c * 16 + r) * a.HW * sizeof(HT) + at, 0, wl[c][r]);
        }
      } else {
        const int pc = min(p, P - 1), n = pc / a.HW;
        const size_t base = (size_t)n * a.C * a.HW + (size_t)(pc - n * a.HW);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int cc = c * 16 + q * 4 + r;
            if (cc < a.C && p < P) IO::st1(a.dh, base + (size_t)cc * a.HW, wl[c][r]);
          }
      }
    }
  }
  if (a.lsum != nullptr) {
    acc_l = block_sum_d(acc_l, redd);
    if (threadIdx.x == 0) a.lsum[blockIdx.x] = acc_l;
  }
}

// ------------------------------------------------------------------------------------------------------------------------------ dw, db
struct CnwArgs {
  const void* h; const char* img; const float *fx, *lse2, *gp, *hot; const int* lab;
  float *dwp, *dbp; size_t dw_split; int db_split;
  long P; int C, HW, V, units, wpx, splits, tiles;
};

// Pixel tile in LDS: [plane][channel][TP pixels], 16-byte chunk j of row c at j ^ (c & 7).
template <typename HT, typename WT, int KS, int NJ, int TP, bool VEC>
__global__ __launch_bounds__(256, 2) void cn_classes_kernel(CnwArgs a) {
  using IO = ActIO<HT>;
  typedef typename CnW<KS>::Frag Frag;
  constexpr int HP = sizeof(HT) == 4 ? 2 : 1, WP = sizeof(WT) == 4 ? 2 : 1;
  using IM = CnImage<KS, WP>;
  constexpr int CT = CnW<KS>::kCT, KN = CnW<KS>::kN, KF = CnW<KS>::kF, kC = CnW<KS>::kW, kTasks = kC * (TP / 8) / 256;
  __shared__ __attribute__((aligned(1024))) _Float16 xs[HP * kC * TP];
  __shared__ __attribute__((aligned(16))) float rows[5][TP];       // 2^ex, lse, g_p 2^ex, g_p, the label's 1 in units of exp2(z - lse)
  __shared__ __attribute__((aligned(16))) int labs[TP];
  __shared__ int tmax[2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const int wv = 4 / a.wpx, unit = blockIdx.y * wv + wave % wv, wp_ = wave / wv;
  const bool busy = unit < a.units;
  const int v0 = unit * (NJ * 16);
  // this wave's classes
  Frag w[WP][KN][NJ];
  float bw[NJ], db[NJ];
  const float wl2 = busy ? ((const float*)(a.img + (size_t)(v0 >> 6) * IM::kBytes + WP * IM::kPlane * 2))[64] : 0.f;      // (the classes of a wave lie in one chunk)
  ms_f4 o[CT][NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int v = min(v0 + j * 16 + li, ((a.V + 63) & ~63) - 1), r = v & 63;      // (a class behind the last chunk repeats its last row and is not stored)
    const char* im = a.img + (size_t)(v >> 6) * IM::kBytes;
    const float* tb = (const float*)(im + WP * IM::kPlane * 2);
    bw[j] = tb[r]; db[j] = 0.f;
#pragma unroll
    for (int pl = 0; pl < WP; ++pl)
#pragma unroll
      for (int ks = 0; ks < KN; ++ks) w[pl][ks][j] = *reinterpret_cast<const Frag*>((const _Float16*)im + pl * IM::kPlane + r * kC + (KS == 0 ? q * 4 : ((ks * 4 + q) ^ cn_swz<KS>(r)) * 8));
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
  }
  const int t0 = (int)((long)a.tiles * blockIdx.x / a.splits), t1 = (int)((long)a.tiles * (blockIdx.x + 1) / a.splits);

  // G 2^ex is scaled so that the largest |g_p| 2^ex met so far lies below 2^kCeTopExp: the partial sums are moved along when a tile brings a larger one.  A pixel of zeros takes no part
  // in that: its G is not needed for dw.  The low plane of G is kept 2^12 times as large, against the pixels' high plane divided by 2^12: G holds its bits to 2^-37, so that one pixel of
  // large features (2^10 and more of the others) does not push the others' G into fp16's lowest steps.
  int kmax = -100000;
  float gn = 0.f;
  if (threadIdx.x < 2) tmax[threadIdx.x] = -100000;

  float pre[kTasks][8];
  float prow[4];
  int plab;
  auto load = [&](int t) {
    const long p0 = (long)t * TP;
#pragma unroll
    for (int k = 0; k < kTasks; ++k) {
      const int task = k * 256 + threadIdx.x, c = task / (TP / 8), pc = (task % (TP / 8)) * 8;
      const long p = p0 + pc;
      if (VEC) {           // whole 8-pixel groups lie in one image
        const int n = (int)p / a.HW;
        const size_t at = (size_t)n * a.C * a.HW + (size_t)c * a.HW + (size_t)((int)p - n * a.HW);
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
        if (c < a.C && p < a.P) { u = IO::ld4(a.h, at); v = IO::ld4(a.h, at + 4); }
        pre[k][0] = u.x; pre[k][1] = u.y; pre[k][2] = u.z; pre[k][3] = u.w; pre[k][4] = v.x; pre[k][5] = v.y; pre[k][6] = v.z; pre[k][7] = v.w;
      } else {
        int n = (int)p / a.HW, hw = (int)p - n * a.HW;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pre[k][e] = (c < a.C && p + e < a.P) ? IO::ld1(a.h, (size_t)n * a.C * a.HW + (size_t)c * a.HW + (size_t)hw) : 0.f;
          if (++hw == a.HW) { hw = 0; ++n; }
        }
      }
    }
    if (threadIdx.x < TP) {
      const long p = p0 + threadIdx.x;        // (the row arrays are padded)
      prow[0] = a.fx[p]; prow[1] = a.lse2[p]; prow[2] = a.gp[p]; prow[3] = a.hot[p]; plab = a.lab[p];
    }
  };
  if (t0 < t1) load(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();                           // nobody reads the tile before this one
    if (threadIdx.x < TP) {
      rows[0][threadIdx.x] = prow[0]; rows[1][threadIdx.x] = prow[1]; rows[2][threadIdx.x] = prow[2] * prow[0]; rows[3][threadIdx.x] = prow[2]; rows[4][threadIdx.x] = prow[3];
      labs[threadIdx.x] = plab;
      const unsigned gb = __float_as_uint(prow[2]) & 0x7FFFFFFFu;
      int e = (gb != 0u && gb < 0x7F800000u && prow[0] > 0.f) ? (int)(gb >> 23) - 126 + (int)(__float_as_uint(prow[0]) >> 23) - 127 : -100000;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) e = max(e, __shfl_xor(e, off, 64));
      if (lane == 0) atomicMax(&tmax[t & 1], e);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTasks; ++k) {
      const int task = k * 256 + threadIdx.x, c = task / (TP / 8), ch = task % (TP / 8);
      ms_h8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // 1 / 2^ex by exponent arithmetic; a row that takes no part is all zeros, whatever it holds
        const float inv = __uint_as_float((254u << 23) - __float_as_uint(rows[0][ch * 8 + e]));
        const float v = rows[3][ch * 8 + e] == 0.f ? 0.f : pre[k][e] * inv;
        _Float16 x, y;
        ce_split(v, x, y);
        hi[e] = x; lo[e] = y;
      }
      const int at = c * TP + ((ch ^ (c & 7)) * 8);
      *reinterpret_cast<ms_h8*>(xs + at) = hi;
      if (HP == 2) *reinterpret_cast<ms_h8*>(xs + kC * TP + at) = lo;
    }
    if (t + 1 < t1) load(t + 1);
    const int tm = tmax[t & 1];
    __syncthreads();
    if (threadIdx.x == 0) tmax[t & 1] = -100000;          // (next used by tile t + 2)
    if (tm > kmax) {
      const float f = kmax < -50000 ? 0.f : ce_pow2(kmax - tm);
      kmax = tm;
      gn = ce_pow2(min(max(kCeTopExp - kmax, -120), 120));
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[c][j] *= f;
    }
    if (busy) {
#pragma unroll 1
      for (int sub = wp_; sub < TP / 32; sub += a.wpx) {
        const int p0 = sub * 32;
        ms_f4 s[2][NJ];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[tt][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KN; ++ks)
#pragma unroll
            for (int pl = 0; pl < HP; ++pl) {
              // rows of the operand = pixels, channels 32 ks + KF q + k: transposing reads of 4 channel rows at a time
              typedef __attribute__((address_space(3))) ms_s4* lp;
              union { ms_s4 s[KF / 4]; Frag h; } u;
              const int c = ks * 32 + q * KF + (li >> 2), chn = ((p0 + tt * 16) >> 3) + ((li & 3) >> 1), off = (li & 1) * 4;
              const _Float16* b = xs + pl * kC * TP;
              u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(b + c * TP + ((chn ^ (c & 7)) * 8) + off));
              if constexpr (KS > 0) u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(b + (c + 4) * TP + ((chn ^ ((c + 4) & 7)) * 8) + off));
#pragma unroll
              for (int j = 0; j < NJ; ++j) s[tt][j] = cn_mfma(u.h, w[0][ks][j], s[tt][j]);
              if (WP == 2 && pl == 0) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) s[tt][j] = cn_mfma(u.h, w[WP - 1][ks][j], s[tt][j]);
              }
            }
        }
        ms_h8 gh[NJ], gl[NJ];
        constexpr bool kG2 = HP == 2 || WP == 2;          // planes of G: one where nothing is fp32
        bool here = false;
        int y4[2][4];
        float h4[2][4];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int pr = p0 + tt * 16 + q * 4;
          const float4 f = *reinterpret_cast<const float4*>(&rows[0][pr]), ls = *reinterpret_cast<const float4*>(&rows[1][pr]);
          const int4 yy = *reinterpret_cast<const int4*>(&labs[pr]);
          const float4 hh = *reinterpret_cast<const float4*>(&rows[4][pr]);
          h4[tt][0] = hh.x; h4[tt][1] = hh.y; h4[tt][2] = hh.z; h4[tt][3] = hh.w;
          const float ff[4] = {f.x * wl2, f.y * wl2, f.z * wl2, f.w * wl2}, l4[4] = {ls.x, ls.y, ls.z, ls.w};
          y4[tt][0] = yy.x - v0; y4[tt][1] = yy.y - v0; y4[tt][2] = yy.z - v0; y4[tt][3] = yy.w - v0;
#pragma unroll
          for (int r = 0; r < 4; ++r) here |= (unsigned)y4[tt][r] < (unsigned)(NJ * 16);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[tt][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][j][r], ff[r], bw[j]) - l4[r]);
        }
        if (__any(here)) {             // some pixel's label is among this wave's classes
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r) s[tt][j][r] -= y4[tt][r] - li == j * 16 ? h4[tt][r] : 0.f;
          }
        }
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int pr = p0 + tt * 16 + q * 4;
          const float4 rr = *reinterpret_cast<const float4*>(&rows[2][pr]), gg = *reinterpret_cast<const float4*>(&rows[3][pr]);
          const float r4[4] = {rr.x * gn, rr.y * gn, rr.z * gn, rr.w * gn}, g4[4] = {gg.x, gg.y, gg.z, gg.w};
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              db[j] = __builtin_fmaf(s[tt][j][r], g4[r], db[j]);
              s[tt][j][r] *= r4[r];
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) ce_split8_far(s[0][j], s[1][j], gh[j], gl[j]);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const int row = c * 16 + li;
          union { ms_h4 p[2]; ms_h8 h; } xh, xl;
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const int px = p0 + tt * 16 + q * 4, at = row * TP + (((px >> 3) ^ (row & 7)) * 8) + (px & 7);
            xh.p[tt] = *reinterpret_cast<const ms_h4*>(xs + at);
            if (HP == 2 && kG2) xl.p[tt] = *reinterpret_cast<const ms_h4*>(xs + kC * TP + at);
          }
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh.h, gh[j], o[c][j], 0, 0, 0);
          if (kG2) {
            const ms_h8 xd = xh.h * (_Float16)(1.f / (float)(1 << kCeLoExp));
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xd, gl[j], o[c][j], 0, 0, 0);
            if (HP == 2) {
#pragma unroll
              for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl.h, gh[j], o[c][j], 0, 0, 0);
            }
          }
        }
      }
    }
  }
  if (!busy) return;
  const float back = kmax < -50000 ? 0.f : ce_pow2(-min(max(kCeTopExp - kmax, -120), 120));
  const int split = blockIdx.x * a.wpx + wp_;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int v = v0 + j * 16 + li;
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) db[j] += __shfl_xor(db[j], off, 64);
    if (v >= a.V) continue;
    if (q == 0) a.dbp[(size_t)split * a.db_split + v] = db[j];
#pragma unroll
    for (int c = 0; c < CT; ++c)
      *reinterpret_cast<float4*>(a.dwp + split * a.dw_split + (size_t)v * kC + c * 16 + q * 4) = make_float4(o[c][j][0] * back, o[c][j][1] * back, o[c][j][2] * back, o[c][j][3] * back);
  }
}

// dw, db: sums of the splits in a fixed order; the loss (last workgroup).  A workgroup sums 64 elements, 16 threads each.
template <typename WT>
__global__ __launch_bounds__(1024) void cn_join_kernel(const float* __restrict__ dwp, const float* __restrict__ dbp, size_t dw_split, int db_split, int splits, void* __restrict__ dw,
                                                       float* __restrict__ db, int V, int C, int kC, int dw_blocks, const double* __restrict__ lsum, int nl, const int* __restrict__ slots,
                                                       int nslots, float sign, int mean_valid, long P, float* __restrict__ loss) {
  __shared__ double redd[16];
  __shared__ int redi[16];
  __shared__ float part[16][64];
  if (blockIdx.x == gridDim.x - 1 && loss != nullptr) {
    const int s = mean_valid ? cn_count(slots, nslots, redi) : 0;
    double a = 0.0;
    for (int i = threadIdx.x; i < nl; i += 1024) a += lsum[i];
    a = block_sum_d(a, redd);
    if (threadIdx.x == 0) loss[0] = (float)((double)sign * a / (double)(mean_valid ? max(s, 1) : P));
    return;
  }
  const bool isw = blockIdx.x < (unsigned)dw_blocks;
  const int el = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int i = (isw ? blockIdx.x : blockIdx.x - dw_blocks) * 64 + el, total = isw ? V * kC : V;
  const float* src = isw ? dwp : dbp;
  const size_t stride = isw ? dw_split : (size_t)db_split;
  float a = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int k = grp; k < splits; k += 16) a += src[k * stride + i];
  }
  part[grp][el] = a;
  __syncthreads();
  if (grp != 0 || i >= total) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) a += part[k][el];
  if (isw) {
    const int v = i / kC, c = i - v * kC;
    if (c < C) ActIO<WT>::st1(dw, (size_t)v * C + c, a);
  } else {
    db[i] = a;
  }
}

// ------------------------------------------------------------------------------------------------------------------------------ host
struct CnPlan {
  int KS, nch, Vp, nslots; long P, Pp, wgs; int njw, units, wpx, vblocks, tp, tiles, splits;
  size_t o_img, o_slots, o_lsum, o_fx, o_lse, o_gp, o_hot, o_lab, o_dw, o_db, total;
};
static CnPlan cn_plan(int N, int C, int V, int HW, int types, bool grad) {
  CnPlan k{};
  k.KS = C <= 16 ? 0 : cdiv(C, 32);
  const int kW = k.KS == 0 ? 16 : k.KS * 32; k.nch = cdiv(V, 64); k.Vp = k.nch * 64; k.P = (long)N * HW;
  k.wgs = (k.P + kCnNJ * 64 - 1) / (kCnNJ * 64);
  k.Pp = (k.P + 255) / 256 * 256;
  k.nslots = (int)std::min<long>(kCnPrep, k.P / 1024 + 1);
  k.njw = k.KS <= 2 && V > 32 ? 4 : 2;
  k.units = cdiv(V, 16 * k.njw);
  k.tp = k.KS <= 2 ? 128 : 64;
  k.wpx = k.units >= 3 ? 1 : (k.units == 2 ? 2 : 4);
  k.wpx = std::min(k.wpx, k.tp / 32);
  k.vblocks = cdiv(k.units, 4 / k.wpx);
  k.tiles = (int)((k.P + k.tp - 1) / k.tp);
  k.splits = (int)std::max<long>(1, std::min<long>(k.tiles, 512 / std::min(k.vblocks, 512)));
  size_t o = 0;
  auto take = [&](size_t n) { const size_t at = o; o += (n + 255) & ~(size_t)255; return at; };
  k.o_img = take((size_t)k.nch * ((size_t)((types & 2) ? 1 : 2) * 64 * kW * 2 + 1024));
  k.o_slots = take(kCnPrep * 4); k.o_lsum = take((size_t)k.wgs * 8);
  if (grad) {
    k.o_fx = take(k.Pp * 4); k.o_lse = take(k.Pp * 4); k.o_gp = take(k.Pp * 4); k.o_hot = take(k.Pp * 4); k.o_lab = take(k.Pp * 4);
    k.o_dw = take((size_t)k.splits * k.wpx * k.Vp * kW * 4);
    k.o_db = take((size_t)k.splits * k.wpx * k.Vp * 4);
  }
  k.total = o;
  return k;
}

bool ce_narrow_ok(int N, int C, int V, int HW) {
  // A wave's loop over classes is serial, 0.015 + 0.00027 C us a class until the rows fill the chip; the wide form spreads classes over workgroups, starts 15 us later and
  // takes 4e-6 us a row and class.  Training calls, fp32, narrow / wide in us: 64 channels, 600 classes: 48 / 39 at 64 rows, 54 / 61 at 4096, 117 / 245 at 65536;
  // 16 channels, 1536 classes: 49 / 40, 53 / 70, 119 / 470; 128 channels, 1536 classes: 111 / 44, 139 / 75, 367 / 606.
  const long P = (long)N * HW;
  return C <= 128 && P < (1L << 30) && (double)V * (0.015 + 0.00027 * C - 4e-6 * (double)P) <= 15.0;
}
size_t ce_narrow_ws_bytes(int N, int C, int V, int HW, int types, bool grad) { return cn_plan(N, C, V, HW, types, grad).total; }

template <typename HT, typename WT, int KS>
static int cn_run(const CeArgs& a, const CnPlan& k) {
  constexpr int WP = sizeof(WT) == 4 ? 2 : 1, kW = CnW<KS>::kW;
  const bool need_dw = a.dw != nullptr || a.db != nullptr, need_grad = need_dw || a.dh != nullptr;
  char* ws = (char*)a.ws;
  hipStream_t st = a.st;
  int* slots = (int*)(ws + k.o_slots);
  MS_LAUNCH((cn_prep_kernel<WT, WP, KS>), dim3(std::max(k.nch, a.mean_valid ? k.nslots : 1)), dim3(256), 0, st, a.w, a.b, a.labels, k.P, a.mean_valid, ws + k.o_img, slots, k.nslots, a.V, k.nch, a.C);
  if (int e = check_launch("class_ce_prep")) return e;
  CnArgs p{};
  p.h = a.h; p.w = a.w; p.labels = a.labels; p.img = ws + k.o_img; p.slots = slots; p.nslots = k.nslots;
  p.nll = a.nll; p.lse_out = a.lse; p.lse_in = a.lse_in; p.grad = a.grad; p.scale_dev = a.scale_dev; p.sign = a.sign; p.mean_valid = a.mean_valid; p.drop = need_grad ? 1 : 0;
  p.dh = a.dh; p.lsum = a.loss != nullptr ? (double*)(ws + k.o_lsum) : nullptr;
  if (need_dw) { p.fx = (float*)(ws + k.o_fx); p.lse2 = (float*)(ws + k.o_lse); p.gp = (float*)(ws + k.o_gp); p.hot = (float*)(ws + k.o_hot); p.lab = (int*)(ws + k.o_lab); }
  p.full = a.C == CnW<KS>::kW && (size_t)a.N * a.HW * a.C * sizeof(HT) <= 0xFFFFFFFFu;
  p.w_vec = a.C % 4 == 0 && (reinterpret_cast<uintptr_t>(a.w) & (4 * sizeof(WT) - 1)) == 0;
  p.P = k.P; p.C = a.C; p.HW = a.HW; p.V = a.V; p.nch = k.nch;
  const dim3 grid((unsigned)k.wgs), block(256);
  if (a.dh != nullptr) MS_LAUNCH((cn_pixels_kernel<HT, WT, KS, kCnNJ, true>), grid, block, 0, st, p);
  else MS_LAUNCH((cn_pixels_kernel<HT, WT, KS, kCnNJ, false>), grid, block, 0, st, p);
  if (int e = check_launch("class_ce_pixels")) return e;
  if (need_dw) {
    CnwArgs c{};
    c.h = a.h; c.img = p.img; c.fx = p.fx; c.lse2 = p.lse2; c.gp = p.gp; c.hot = p.hot; c.lab = p.lab;
    c.dwp = (float*)(ws + k.o_dw); c.dbp = (float*)(ws + k.o_db); c.dw_split = (size_t)k.Vp * kW; c.db_split = k.Vp;
    c.P = k.P; c.C = a.C; c.HW = a.HW; c.V = a.V; c.units = k.units; c.wpx = k.wpx; c.splits = k.splits; c.tiles = k.tiles;
    const dim3 gw((unsigned)k.splits, (unsigned)k.vblocks);
    const bool vec = a.HW % 8 == 0 && aligned16(a.h);          // 8-pixel groups that never cross an image, in whole vectors
    constexpr int TP = KS <= 2 ? 128 : 64;
    if constexpr (KS <= 2) {
      if (k.njw == 4 && vec) MS_LAUNCH((cn_classes_kernel<HT, WT, KS, 4, TP, true>), gw, block, 0, st, c);
      else if (k.njw == 4) MS_LAUNCH((cn_classes_kernel<HT, WT, KS, 4, TP, false>), gw, block, 0, st, c);
    }
    if (k.njw == 2 && vec) MS_LAUNCH((cn_classes_kernel<HT, WT, KS, 2, TP, true>), gw, block, 0, st, c);
    else if (k.njw == 2) MS_LAUNCH((cn_classes_kernel<HT, WT, KS, 2, TP, false>), gw, block, 0, st, c);
    if (int e = check_launch("class_ce_classes")) return e;
  }
  if (need_dw || a.loss != nullptr) {
    const int wb = a.dw != nullptr ? cdiv(a.V * kW, 64) : 0;
    const unsigned blocks = (unsigned)(wb + (a.db != nullptr ? cdiv(a.V, 64) : 0) + (a.loss != nullptr ? 1 : 0));
    MS_LAUNCH((cn_join_kernel<WT>), dim3(blocks), dim3(1024), 0, st, (const float*)(ws + k.o_dw), (const float*)(ws + k.o_db), (size_t)k.Vp * kW, k.Vp, k.splits * k.wpx, a.dw, a.db,
              a.V, a.C, kW, wb, p.lsum, (int)k.wgs, slots, k.nslots, a.sign, a.mean_valid, k.P, a.loss);
    if (int e = check_launch("class_ce_join")) return e;
  }
  return MS_OK;
}
template <typename HT, typename WT>
static int cn_dispatch(const CeArgs& a, const CnPlan& k) {
  switch (k.KS) {
    case 0: return cn_run<HT, WT, 0>(a, k);
    case 1: return cn_run<HT, WT, 1>(a, k);
    case 2: return cn_run<HT, WT, 2>(a, k);
    case 3: return cn_run<HT, WT, 3>(a, k);
    default: return cn_run<HT, WT, 4>(a, k);
  }
}
int ce_narrow_run(const CeArgs& a, bool grad, const char* who) {
  const CnPlan k = cn_plan(a.N, a.C, a.V, a.HW, a.types, grad);
  if (a.ws == nullptr || a.ws_bytes < k.total) { set_error("%s: workspace too small", who); return MS_ERR_WORKSPACE; }
  if (!aligned16(a.ws)) { set_error("%s: workspace not 16-byte aligned", who); return MS_ERR_ALIGN; }
  switch (a.types) {
    case 0: return cn_dispatch<float, float>(a, k);
    case 1: return cn_dispatch<ms_bf16, float>(a, k);
    case 2: return cn_dispatch<float, ms_bf16>(a, k);
    default: return cn_dispatch<ms_bf16, ms_bf16>(a, k);
  }
}
}  // namespace ms
