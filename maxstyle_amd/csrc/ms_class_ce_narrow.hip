// Head + softmax cross entropy over many classes, narrow form (C <= 128): no operand and no product ever leaves the chip; see ms_class_ce.h.
//
//   prep    w -> fp16 planes in the order the LDS wants them, 64 classes a chunk (an "image": the next kernel's DMA copies it as it lies); rows that take part counted
//   pixels  a wave keeps NJ x 16 pixels' features in registers (one read of h), runs over the classes twice: (max, sum exp) first, then G = exp(z - lse) - hot,
//           which is already in the register layout the second product wants, and dh += w^T G.  One read of h, one write of dh, w from L2.
//   classes roles exchanged: a wave keeps NJ x 16 classes' weights in registers and runs over pixels: z again, G, dw += h G^T, db += G.  Pixels are split over
//           workgroups; the partial dw are summed by
//   join    in a fixed order, with the loss.
// 10 P V C products instead of 8 (z is formed three times), but nothing of size P V is stored.  The vector unit, not the matrix cores, sets the time: about 6 operations
// a logit for the statistics, 11 for each G (exp2 counts 4).
#include <algorithm>
#include "ms_class_ce.h"
#include "ms_class_ce_narrow.h"
#include "maxstyle_hip.h"

namespace ms {

constexpr int kCnClasses = 64;        // classes of one image chunk
constexpr int kCnPrep = 256;          // most workgroups of the prep pass

// 16-byte chunk j of row r of a tile of KS * 32 columns lies at chunk j ^ cn_swz(r): both the row reads and the transposing reads below are then free of bank conflicts
template <int KS> __device__ __forceinline__ int cn_swz(int r) { return KS == 1 ? (r >> 1) & 3 : (KS == 3 ? (r >> 2) & 3 : r & 7); }
template <int KS, int WP> struct CnImage {
  static constexpr int kPlane = kCnClasses * KS * 32;                    // halves of one plane
  static constexpr int kBytes = WP * kPlane * 2 + 1024;                  // + 64 x {2^ew log2(e)}, 64 x {b log2(e)}, 64 x {ew}
};

// transposing read: lane (q, i) gets column mn + i of rows k .. k + 3, k = k0 + 4 q (swizzled tile of KS * 32 columns)
template <int KS>
__device__ __forceinline__ ms_h8 cn_tr2(const _Float16* tile, int k0, int k1, int mn, int lane) {
  const int q = lane >> 4, i = lane & 15;
  typedef __attribute__((address_space(3))) ms_s4* lp;
  union { ms_s4 s[2]; ms_h8 h; } u;
  const int ra = k0 + q * 4 + (i >> 2), rb = k1 + q * 4 + (i >> 2), ch = (mn >> 3) + ((i & 3) >> 1), off = (i & 1) * 4;
  u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(tile + ra * (KS * 32) + ((ch ^ cn_swz<KS>(ra)) * 8) + off));
  u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(tile + rb * (KS * 32) + ((ch ^ cn_swz<KS>(rb)) * 8) + off));
  return u.h;
}

// slots[block] = {rows that take part, max ew}; scal[1] is made ready for the pixel pass
template <typename WT, int WP, int KS>
__global__ __launch_bounds__(256) void cn_prep_kernel(const void* __restrict__ w, const float* __restrict__ b, const int64_t* __restrict__ labels, long P, int count,
                                                      char* __restrict__ img, int2* __restrict__ slots, int* __restrict__ scal, int V, int Vp, int C) {
  using IO = ActIO<WT>;
  using IM = CnImage<KS, WP>;
  __shared__ int red[2][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (blockIdx.x == 0 && threadIdx.x == 0) scal[1] = -100000;
  int emax = -100000;
  for (int v = blockIdx.x * 4 + wave; v < Vp; v += gridDim.x * 4) {
    float x[2];
    unsigned am = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = lane + 64 * k;
      x[k] = (v < V && c < C) ? IO::ld1(w, (size_t)v * C + c) : 0.f;
      am = max(am, __float_as_uint(x[k]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) am = max(am, (unsigned)__shfl_xor((int)am, off, 64));
    const int e = ce_exponent(__uint_as_float(am));
    const float inv = ce_pow2(-e);
    char* im = img + (size_t)(v >> 6) * IM::kBytes;
    _Float16* pl = (_Float16*)im;
    const int r = v & 63;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = lane + 64 * k;
      if (c < KS * 32) {
        _Float16 hi, lo;
        ce_split(x[k] * inv, hi, lo);
        const int at = r * (KS * 32) + (((c >> 3) ^ cn_swz<KS>(r)) * 8) + (c & 7);
        pl[at] = hi;
        if (WP == 2) pl[IM::kPlane + at] = lo;
      }
    }
    if (lane == 0) {
      float* t = (float*)(im + WP * IM::kPlane * 2);
      t[r] = ce_pow2(e) * kLog2e;
      t[64 + r] = v < V ? (b != nullptr ? b[v] * kLog2e : 0.f) : -__builtin_inff();
      t[128 + r] = (float)e;
      if (v < V) emax = max(emax, e);
    }
  }
  int k = 0;
  if (count) for (long p = (long)blockIdx.x * 256 + threadIdx.x; p < P; p += (long)gridDim.x * 256) { const int64_t l = labels[p]; k += (l >= 0 && l < V) ? 1 : 0; }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { k += __shfl_xor(k, off, 64); emax = max(emax, __shfl_xor(emax, off, 64)); }
  if (lane == 0) { red[0][wave] = k; red[1][wave] = emax; }
  __syncthreads();
  if (threadIdx.x == 0) slots[blockIdx.x] = make_int2(red[0][0] + red[0][1] + red[0][2] + red[0][3], max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3])));
}

// {rows that take part, max ew} from the prep pass's slots (at most 256: one a thread)
__device__ __forceinline__ int2 cn_slots(const int2* __restrict__ slots, int n, int* red /* 2 x waves */) {
  int2 s = threadIdx.x < (unsigned)n ? slots[threadIdx.x] : make_int2(0, -100000);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { s.x += __shfl_xor(s.x, off, 64); s.y = max(s.y, __shfl_xor(s.y, off, 64)); }
  if ((threadIdx.x & 63) == 0) { red[2 * (threadIdx.x >> 6)] = s.x; red[2 * (threadIdx.x >> 6) + 1] = s.y; }
  __syncthreads();
  return make_int2(red[0] + red[2] + red[4] + red[6], max(max(red[1], red[3]), max(red[5], red[7])));      // (the slots lie in the first four waves)
}

template <int WP, int KS>
__device__ __forceinline__ void cn_stage(const char* img, int chunk, unsigned lds, int wave, int lane) {
  constexpr int kN = CnImage<KS, WP>::kBytes / 1024;
  const ms_i32x4 rs = ms_dma_rsrc(img + (size_t)chunk * CnImage<KS, WP>::kBytes);
  for (int i = wave; i < kN; i += 4) ms_lds_dma16(rs, __builtin_amdgcn_readfirstlane(lds + i * 1024), i * 1024 + lane * 16, 0);
}

struct CnArgs {
  const void *h; const int64_t* labels; const char* img; const int2* slots; int nslots; int* scal;
  float *nll, *lse_out; const float *lse_in, *grad, *scale_dev; float sign; int mean_valid, drop;
  void* dh; double* lsum;
  float *fx, *lse2, *gp; int* lab;          // what the class pass needs of every row (NULL: it does not run)
  long P; int C, HW, V, nch;
};

template <typename HT, int HP, int WP, int KS, int NJ>
__global__ __launch_bounds__(256) void cn_pixels_kernel(CnArgs a) {
  using IO = ActIO<HT>;
  using IM = CnImage<KS, WP>;
  constexpr int CT = KS * 2;
  __shared__ __attribute__((aligned(1024))) char sm[2][IM::kBytes];
  __shared__ int redi[8];
  __shared__ double redd[16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const unsigned lds0 = ms_lds_addr(&sm[0][0]);
  const bool stats = a.lse_in == nullptr, grads = a.dh != nullptr;
  const int nch = a.nch, T = (stats ? nch : 0) + (grads ? nch : 0);
  const bool resident = nch <= 2;           // both chunks stay: the second run over the classes loads nothing
  auto chunk_of = [&](int t) { return t >= nch ? t - nch : t; };
  auto buf_of = [&](int t) { return resident ? chunk_of(t) : (t & 1); };
  if (T > 0) cn_stage<WP, KS>(a.img, 0, lds0, wave, lane);

  // ---- this wave's pixels: scaled fp16 planes in the layout of a matrix operand (column = pixel li, 8 channels 32 ks + 8 q + j)
  ms_h8 x[HP][KS][NJ];
  float fx[NJ];
  int lab[NJ];
  long pix[NJ];
  size_t base[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const long p = (long)blockIdx.x * (4 * NJ * 16) + wave * (NJ * 16) + j * 16 + li;
    pix[j] = p;
    int y = -1;
    if (p < a.P) { const int64_t l = a.labels[p]; y = (l >= 0 && l < a.V) ? (int)l : -1; }
    lab[j] = y;
    const bool live = p < a.P && (!a.drop || y >= 0);
    const int n = (int)p / a.HW;                     // (at most 2^30 rows)
    base[j] = (size_t)n * a.C * a.HW + (size_t)((int)p - n * a.HW);
    float v[KS][8];
    unsigned am = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = ks * 32 + q * 8 + k;
        v[ks][k] = (live && c < a.C) ? IO::ld1(a.h, base[j] + (size_t)c * a.HW) : 0.f;
      }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int k = 0; k < 8; ++k) am = max(am, __float_as_uint(v[ks][k]) & 0x7FFFFFFFu);
    am = max(am, (unsigned)__shfl_xor((int)am, 16, 64));
    am = max(am, (unsigned)__shfl_xor((int)am, 32, 64));
    const int e = ce_exponent(__uint_as_float(am));
    const float inv = ce_pow2(-e);
    fx[j] = ce_pow2(e);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        _Float16 hi, lo;
        ce_split(v[ks][k] * inv, hi, lo);
        x[0][ks][j][k] = hi;
        if (HP == 2) x[HP - 1][ks][j][k] = lo;
      }
  }
  const int2 prep = cn_slots(a.slots, a.nslots, redi);

  // one pair of 16-class tiles: z (without the row's scale) of classes t0 + 4 q + r
  auto logits = [&](const _Float16* wp, int t0, ms_f4 (&s)[2][NJ]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) s[t][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
      const int r = t0 + t * 16 + li;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int at = r * (KS * 32) + (((ks * 4 + q) ^ cn_swz<KS>(r)) * 8);
        const ms_h8 hi = *reinterpret_cast<const ms_h8*>(wp + at);
#pragma unroll
        for (int j = 0; j < NJ; ++j) s[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, x[0][ks][j], s[t][j], 0, 0, 0);
        if (HP == 2) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, x[HP - 1][ks][j], s[t][j], 0, 0, 0);
        }
        if (WP == 2) {
          const ms_h8 lo = *reinterpret_cast<const ms_h8*>(wp + IM::kPlane + at);
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, x[0][ks][j], s[t][j], 0, 0, 0);
        }
      }
    }
  };

  float m[NJ], l[NJ], zl[NJ];          // in units of log2
#pragma unroll
  for (int j = 0; j < NJ; ++j) { m[j] = -__builtin_inff(); l[j] = 0.f; zl[j] = 0.f; }
  int t = 0;
  auto next_chunk = [&]() {            // chunk t is in LDS for every wave; chunk t + 1 starts
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < T && !(resident && t + 1 >= nch)) cn_stage<WP, KS>(a.img, chunk_of(t + 1), lds0 + (unsigned)buf_of(t + 1) * (unsigned)IM::kBytes, wave, lane);
  };
  if (stats) {
    for (; t < nch; ++t) {
      next_chunk();
      const _Float16* wp = (const _Float16*)sm[buf_of(t)];
      const float* tb = (const float*)(sm[buf_of(t)] + WP * IM::kPlane * 2);
#pragma unroll 1
      for (int h2 = 0; h2 < 2; ++h2) {
        if (t * kCnClasses + h2 * 32 >= a.V) break;
        ms_f4 s[2][NJ];
        logits(wp, h2 * 32, s);
        bool any = false;
#pragma unroll
        for (int j = 0; j < NJ; ++j) any |= (lab[j] >> 5) == t * 2 + h2;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const float4 f = *reinterpret_cast<const float4*>(tb + h2 * 32 + tt * 16 + q * 4), b = *reinterpret_cast<const float4*>(tb + 64 + h2 * 32 + tt * 16 + q * 4);
          const float ff[4] = {f.x, f.y, f.z, f.w}, bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[tt][j][r] = __builtin_fmaf(s[tt][j][r] * ff[r], fx[j], bb[r]);
        }
        if (__any(any)) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const int y = lab[j] - (t * kCnClasses + h2 * 32 + q * 4);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
              for (int r = 0; r < 4; ++r) zl[j] = y == tt * 16 + r ? s[tt][j][r] : zl[j];
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          float mx = fmaxf(fmaxf(fmaxf(s[0][j][0], s[0][j][1]), fmaxf(s[0][j][2], s[0][j][3])), fmaxf(fmaxf(s[1][j][0], s[1][j][1]), fmaxf(s[1][j][2], s[1][j][3])));
          mx = fmaxf(m[j], mx);
          const float mm = mx == -__builtin_inff() ? 0.f : mx;
          float sum = l[j] * __builtin_amdgcn_exp2f(m[j] - mm);
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(s[tt][j][r] - mm);
          l[j] = sum; m[j] = mx;
        }
      }
    }
  }
  // ---- rows: join the four class quarters, loss, what the class pass needs
  const float cnt = (float)(a.mean_valid ? max(prep.x, 1) : a.P);
  float gp[NJ], lse2[NJ];
  double acc_l = 0.0;
  int emax = -100000;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const long p = pix[j];
    if (stats) {
#pragma unroll
      for (int off = 16; off <= 32; off <<= 1) {
        const float mo = __shfl_xor(m[j], off, 64), lo = __shfl_xor(l[j], off, 64), mn = fmaxf(m[j], mo), mm = mn == -__builtin_inff() ? 0.f : mn;
        l[j] = l[j] * __builtin_amdgcn_exp2f(m[j] - mm) + lo * __builtin_amdgcn_exp2f(mo - mm);
        m[j] = mn;
        zl[j] += __shfl_xor(zl[j], off, 64);          // (one lane of the four holds it, the others 0)
      }
      const float lg = __builtin_amdgcn_logf(l[j]);   // log2
      lse2[j] = m[j] + lg;
      const float ln2 = 0.693147180559945309f, nll = lab[j] >= 0 ? ((m[j] - zl[j]) + lg) * ln2 : 0.f;
      if (q == 0 && p < a.P) {
        if (a.nll != nullptr) { a.nll[p] = nll; a.lse_out[p] = lse2[j] * ln2; }
        acc_l += (double)nll;
      }
    } else {
      lse2[j] = p < a.P ? a.lse_in[p] * kLog2e : 0.f;
    }
    gp[j] = 0.f;
    if (lab[j] >= 0) gp[j] = a.grad != nullptr ? a.grad[p] : a.sign / cnt * (a.scale_dev != nullptr ? *a.scale_dev : 1.f);
    if (a.fx != nullptr) {
      const unsigned gb = __float_as_uint(gp[j]) & 0x7FFFFFFFu;
      if (gb != 0u && gb < 0x7F800000u) emax = max(emax, (int)(gb >> 23) - 126 + (int)(__float_as_uint(fx[j]) >> 23) - 127);
      if (q == 0) {                                   // (arrays padded to whole workgroups)
        a.fx[p] = fx[j]; a.gp[p] = gp[j]; a.lab[p] = lab[j];
        a.lse2[p] = gp[j] == 0.f ? __builtin_inff() : lse2[j];      // a row that takes no part: exp2(z - inf) = 0 whatever z is
      }
    }
  }
  if (a.lsum != nullptr) {
    acc_l = block_sum_d(acc_l, redd);
    if (threadIdx.x == 0) a.lsum[blockIdx.x] = acc_l;
  }
  if (a.fx != nullptr) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) emax = max(emax, __shfl_xor(emax, off, 64));
    if (lane == 0 && emax > -100000) atomicMax(&a.scal[1], emax);
  }
  if (!grads) return;

  // ---- dh = w^T G.  G is scaled by 2^(ew - max ew + 13) class by class: the power of two rides on the exponent's argument.
  ms_f4 o[CT][NJ];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[c][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
  const float top = (float)(kCeTopExp - prep.y);
  constexpr bool kG2 = HP == 2;          // planes of G (and of w, below): two for an fp32 dh
#pragma unroll 1
  for (; t < T; ++t) {
    next_chunk();
    const int ch = chunk_of(t);
    const _Float16* wp = (const _Float16*)sm[buf_of(t)];
    const float* tb = (const float*)(sm[buf_of(t)] + WP * IM::kPlane * 2);
#pragma unroll 1
    for (int h2 = 0; h2 < 2; ++h2) {
      if (ch * kCnClasses + h2 * 32 >= a.V) break;
      ms_f4 s[2][NJ];
      logits(wp, h2 * 32, s);
      ms_h8 gh[NJ], gl[NJ];
      bool any = false;
#pragma unroll
      for (int j = 0; j < NJ; ++j) any |= (lab[j] >> 5) == ch * 2 + h2;
      any = __any(any);
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const float4 f = *reinterpret_cast<const float4*>(tb + h2 * 32 + tt * 16 + q * 4), b = *reinterpret_cast<const float4*>(tb + 64 + h2 * 32 + tt * 16 + q * 4),
                     ew = *reinterpret_cast<const float4*>(tb + 128 + h2 * 32 + tt * 16 + q * 4);
        const float ff[4] = {f.x, f.y, f.z, f.w}, bb[4] = {b.x, b.y, b.z, b.w}, ee[4] = {ew.x + top, ew.y + top, ew.z + top, ew.w + top};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          float g[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) g[r] = __builtin_amdgcn_exp2f((__builtin_fmaf(s[tt][j][r] * ff[r], fx[j], bb[r]) - lse2[j]) + ee[r]);
          if (any) {
            const int y = lab[j] - (ch * kCnClasses + h2 * 32 + tt * 16 + q * 4);
#pragma unroll
            for (int r = 0; r < 4; ++r) g[r] -= y == r ? __builtin_amdgcn_exp2f(ee[r]) : 0.f;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            _Float16 hi, lo;
            ce_split(g[r], hi, lo);
            gh[j][tt * 4 + r] = hi; gl[j][tt * 4 + r] = lo;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const ms_h8 wh = cn_tr2<KS>(wp, h2 * 32, h2 * 32 + 16, c * 16, lane);
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, gh[j], o[c][j], 0, 0, 0);
        if (kG2) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, gl[j], o[c][j], 0, 0, 0);
          if (WP == 2) {
            const ms_h8 wl = cn_tr2<KS>(wp + IM::kPlane, h2 * 32, h2 * 32 + 16, c * 16, lane);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl, gh[j], o[c][j], 0, 0, 0);
          }
        }
      }
    }
  }
  const float back = ce_pow2(prep.y - kCeTopExp);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (pix[j] >= a.P) continue;
    const float f = gp[j] * back;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int cc = c * 16 + q * 4 + r;
        if (cc < a.C) IO::st1(a.dh, base[j] + (size_t)cc * a.HW, gp[j] == 0.f ? 0.f : o[c][j][r] * f);
      }
  }
}

// ------------------------------------------------------------------------------------------------------------------------------ dw, db
struct CnwArgs {
  const void* h; const char* img; const float *fx, *lse2, *gp; const int* lab; const int* scal;
  float *dwp, *dbp; size_t dw_split; int db_split;
  long P; int C, HW, V, units, wpx, splits, tiles;
};

// Pixel tile in LDS: [plane][channel][TP pixels], 16-byte chunk j of row c at j ^ (c & 7).
template <typename HT, int HP, int WP, int KS, int NJ, int TP, bool VEC>
__global__ __launch_bounds__(256) void cn_classes_kernel(CnwArgs a) {
  using IO = ActIO<HT>;
  using IM = CnImage<KS, WP>;
  constexpr int CT = KS * 2, kC = KS * 32, kTasks = kC * (TP / 8) / 256;
  __shared__ __attribute__((aligned(1024))) _Float16 xs[HP * kC * TP];
  __shared__ __attribute__((aligned(16))) float rows[4][TP];       // 2^ex, lse, g_p 2^ex 2^k, g_p
  __shared__ __attribute__((aligned(16))) int labs[TP];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, li = lane & 15;
  const int wv = 4 / a.wpx, unit = blockIdx.y * wv + wave % wv, wp_ = wave / wv;
  const bool busy = unit < a.units;
  const int v0 = unit * (NJ * 16);
  const int ge = a.scal[1];
  const int gexp = ge < -50000 ? 0 : min(max(kCeTopExp - ge, -120), 120);
  const float gn = ce_pow2(gexp);

  // this wave's classes
  ms_h8 w[WP][KS][NJ];
  float fw[NJ], bw[NJ], db[NJ];
  ms_f4 o[CT][NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int v = min(v0 + j * 16 + li, ((a.V + 63) & ~63) - 1), r = v & 63;      // (a class behind the last chunk repeats its last row and is not stored)
    const char* im = a.img + (size_t)(v >> 6) * IM::kBytes;
    const float* tb = (const float*)(im + WP * IM::kPlane * 2);
    fw[j] = tb[r]; bw[j] = tb[64 + r]; db[j] = 0.f;
#pragma unroll
    for (int pl = 0; pl < WP; ++pl)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) w[pl][ks][j] = *reinterpret_cast<const ms_h8*>((const _Float16*)im + pl * IM::kPlane + r * kC + (((ks * 4 + q) ^ cn_swz<KS>(r)) * 8));
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][j] = ms_f4{0.f, 0.f, 0.f, 0.f};
  }
  const int t0 = (int)((long)a.tiles * blockIdx.x / a.splits), t1 = (int)((long)a.tiles * (blockIdx.x + 1) / a.splits);

  float pre[kTasks][8];
  float prow[3];
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
      prow[0] = a.fx[p]; prow[1] = a.lse2[p]; prow[2] = a.gp[p]; plab = a.lab[p];
    }
  };
  if (t0 < t1) load(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();                           // nobody reads the tile before this one
    if (threadIdx.x < TP) {
      rows[0][threadIdx.x] = prow[0]; rows[1][threadIdx.x] = prow[1]; rows[2][threadIdx.x] = prow[2] * prow[0] * gn; rows[3][threadIdx.x] = prow[2];
      labs[threadIdx.x] = plab;
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
    __syncthreads();
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
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < HP; ++pl) {
              // rows of the operand = pixels, 8 channels 32 ks + 8 q + k: transposing reads of rows 4 at a time
              typedef __attribute__((address_space(3))) ms_s4* lp;
              union { ms_s4 s[2]; ms_h8 h; } u;
              const int c = ks * 32 + q * 8 + (li >> 2), chn = ((p0 + tt * 16) >> 3) + ((li & 3) >> 1), off = (li & 1) * 4;
              const _Float16* b = xs + pl * kC * TP;
              u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(b + c * TP + ((chn ^ (c & 7)) * 8) + off));
              u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(ms_s4*)(b + (c + 4) * TP + ((chn ^ ((c + 4) & 7)) * 8) + off));
#pragma unroll
              for (int j = 0; j < NJ; ++j) s[tt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u.h, w[0][ks][j], s[tt][j], 0, 0, 0);
              if (WP == 2 && pl == 0) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) s[tt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u.h, w[WP - 1][ks][j], s[tt][j], 0, 0, 0);
              }
            }
        }
        ms_h8 gh[NJ], gl[NJ];
        constexpr bool kG2 = WP == 2;          // planes of G: two for an fp32 dw
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int pr = p0 + tt * 16 + q * 4;
          const float4 f = *reinterpret_cast<const float4*>(&rows[0][pr]), ls = *reinterpret_cast<const float4*>(&rows[1][pr]), rr = *reinterpret_cast<const float4*>(&rows[2][pr]),
                       gg = *reinterpret_cast<const float4*>(&rows[3][pr]);
          const int4 yy = *reinterpret_cast<const int4*>(&labs[pr]);
          const float ff[4] = {f.x, f.y, f.z, f.w}, l4[4] = {ls.x, ls.y, ls.z, ls.w}, r4[4] = {rr.x, rr.y, rr.z, rr.w}, g4[4] = {gg.x, gg.y, gg.z, gg.w};
          const int y4[4] = {yy.x, yy.y, yy.z, yy.w};
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][j][r] * ff[r], fw[j], bw[j]) - l4[r]);
              e -= y4[r] == v0 + j * 16 + li ? 1.f : 0.f;
              db[j] = __builtin_fmaf(e, g4[r], db[j]);
              _Float16 x, y;
              ce_split(e * r4[r], x, y);
              gh[j][tt * 4 + r] = x; gl[j][tt * 4 + r] = y;
            }
        }
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
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh.h, gl[j], o[c][j], 0, 0, 0);
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
  const float back = ce_pow2(-gexp);
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
                                                       float* __restrict__ db, int V, int C, int kC, int dw_blocks, const double* __restrict__ lsum, int nl, const int2* __restrict__ slots,
                                                       int nslots, float sign, int mean_valid, long P, float* __restrict__ loss) {
  __shared__ double redd[16];
  __shared__ int redi[32];
  __shared__ float part[16][64];
  if (blockIdx.x == gridDim.x - 1 && loss != nullptr) {
    const int2 s = cn_slots(slots, nslots, redi);
    double a = 0.0;
    for (int i = threadIdx.x; i < nl; i += 1024) a += lsum[i];
    a = block_sum_d(a, redd);
    if (threadIdx.x == 0) loss[0] = (float)((double)sign * a / (double)(mean_valid ? max(s.x, 1) : P));
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
  int KS, nch, Vp, nslots; long P, Pp, wgs; int nj; int njw, units, wpx, vblocks, tp, tiles, splits;
  size_t o_img, o_slots, o_scal, o_lsum, o_fx, o_lse, o_gp, o_lab, o_dw, o_db, total;
};
static CnPlan cn_plan(int N, int C, int V, int HW, int types, bool grad) {
  CnPlan k{};
  k.KS = cdiv(C, 32); k.nch = cdiv(V, 64); k.Vp = k.nch * 64; k.P = (long)N * HW;
  // Pixels of a wave: as many as its registers hold, fewer where the launch would leave compute units idle.
  k.nj = k.KS <= 2 ? 4 : 2;
  if (k.nj == 4 && k.P < 256L * 256) k.nj = 2;
  k.wgs = (k.P + k.nj * 64 - 1) / (k.nj * 64);
  k.Pp = (k.P + 255) / 256 * 256;
  k.nslots = (int)std::min<long>(kCnPrep, std::max<long>(cdiv(k.Vp, 4), std::min<long>(k.P / 1024 + 1, kCnPrep)));
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
  k.o_img = take((size_t)k.nch * ((size_t)((types & 2) ? 1 : 2) * 64 * k.KS * 64 + 1024));
  k.o_slots = take(kCnPrep * 8); k.o_scal = take(64); k.o_lsum = take((size_t)k.wgs * 8);
  if (grad) {
    k.o_fx = take(k.Pp * 4); k.o_lse = take(k.Pp * 4); k.o_gp = take(k.Pp * 4); k.o_lab = take(k.Pp * 4);
    k.o_dw = take((size_t)k.splits * k.wpx * k.Vp * k.KS * 32 * 4);
    k.o_db = take((size_t)k.splits * k.wpx * k.Vp * 4);
  }
  k.total = o;
  return k;
}

bool ce_narrow_ok(int N, int C, int V, int HW) {
  // The class loop of a wave is serial: with many classes and few rows the wide form's tiles over classes fill the chip better.
  const long P = (long)N * HW;
  return C <= 128 && (V <= 1536 || P >= 32768) && P < (1L << 30);
}
size_t ce_narrow_ws_bytes(int N, int C, int V, int HW, int types, bool grad) { return cn_plan(N, C, V, HW, types, grad).total; }

template <typename HT, typename WT, int KS>
static int cn_run(const CeArgs& a, const CnPlan& k) {
  constexpr int HP = sizeof(HT) == 4 ? 2 : 1, WP = sizeof(WT) == 4 ? 2 : 1;
  const bool need_dw = a.dw != nullptr || a.db != nullptr, need_grad = need_dw || a.dh != nullptr;
  char* ws = (char*)a.ws;
  hipStream_t st = a.st;
  int2* slots = (int2*)(ws + k.o_slots);
  int* scal = (int*)(ws + k.o_scal);
  MS_LAUNCH((cn_prep_kernel<WT, WP, KS>), dim3(k.nslots), dim3(256), 0, st, a.w, a.b, a.labels, k.P, a.mean_valid, ws + k.o_img, slots, scal, a.V, k.Vp, a.C);
  if (int e = check_launch("class_ce_prep")) return e;
  CnArgs p{};
  p.h = a.h; p.labels = a.labels; p.img = ws + k.o_img; p.slots = slots; p.nslots = k.nslots; p.scal = scal;
  p.nll = a.nll; p.lse_out = a.lse; p.lse_in = a.lse_in; p.grad = a.grad; p.scale_dev = a.scale_dev; p.sign = a.sign; p.mean_valid = a.mean_valid; p.drop = need_grad ? 1 : 0;
  p.dh = a.dh; p.lsum = a.loss != nullptr ? (double*)(ws + k.o_lsum) : nullptr;
  if (need_dw) { p.fx = (float*)(ws + k.o_fx); p.lse2 = (float*)(ws + k.o_lse); p.gp = (float*)(ws + k.o_gp); p.lab = (int*)(ws + k.o_lab); }
  p.P = k.P; p.C = a.C; p.HW = a.HW; p.V = a.V; p.nch = k.nch;
  const dim3 grid((unsigned)k.wgs), block(256);
  if constexpr (KS <= 2) {
    if (k.nj == 4) MS_LAUNCH((cn_pixels_kernel<HT, HP, WP, KS, 4>), grid, block, 0, st, p);
    else MS_LAUNCH((cn_pixels_kernel<HT, HP, WP, KS, 2>), grid, block, 0, st, p);
  } else {
    MS_LAUNCH((cn_pixels_kernel<HT, HP, WP, KS, 2>), grid, block, 0, st, p);
  }
  if (int e = check_launch("class_ce_pixels")) return e;
  if (need_dw) {
    CnwArgs c{};
    c.h = a.h; c.img = p.img; c.fx = p.fx; c.lse2 = p.lse2; c.gp = p.gp; c.lab = p.lab; c.scal = scal;
    c.dwp = (float*)(ws + k.o_dw); c.dbp = (float*)(ws + k.o_db); c.dw_split = (size_t)k.Vp * KS * 32; c.db_split = k.Vp;
    c.P = k.P; c.C = a.C; c.HW = a.HW; c.V = a.V; c.units = k.units; c.wpx = k.wpx; c.splits = k.splits; c.tiles = k.tiles;
    const dim3 gw((unsigned)k.splits, (unsigned)k.vblocks);
    const bool vec = a.HW % 8 == 0 && aligned16(a.h);          // 8-pixel groups that never cross an image, in whole vectors
    constexpr int TP = KS <= 2 ? 128 : 64;
    if constexpr (KS <= 2) {
      if (k.njw == 4) {
        if (vec) MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 4, TP, true>), gw, block, 0, st, c);
        else MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 4, TP, false>), gw, block, 0, st, c);
      } else {
        if (vec) MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 2, TP, true>), gw, block, 0, st, c);
        else MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 2, TP, false>), gw, block, 0, st, c);
      }
    } else {
      if (vec) MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 2, TP, true>), gw, block, 0, st, c);
      else MS_LAUNCH((cn_classes_kernel<HT, HP, WP, KS, 2, TP, false>), gw, block, 0, st, c);
    }
    if (int e = check_launch("class_ce_classes")) return e;
  }
  if (need_dw || a.loss != nullptr) {
    const int wb = a.dw != nullptr ? cdiv(a.V * KS * 32, 64) : 0;
    const unsigned blocks = (unsigned)(wb + (a.db != nullptr ? cdiv(a.V, 64) : 0) + (a.loss != nullptr ? 1 : 0));
    MS_LAUNCH((cn_join_kernel<WT>), dim3(blocks), dim3(1024), 0, st, (const float*)(ws + k.o_dw), (const float*)(ws + k.o_db), (size_t)k.Vp * KS * 32, k.Vp, k.splits * k.wpx, a.dw, a.db,
              a.V, a.C, KS * 32, wb, p.lsum, (int)k.wgs, slots, k.nslots, a.sign, a.mean_valid, k.P, a.loss);
    if (int e = check_launch("class_ce_join")) return e;
  }
  return MS_OK;
}
template <typename HT, typename WT>
static int cn_dispatch(const CeArgs& a, const CnPlan& k) {
  switch (k.KS) {
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
