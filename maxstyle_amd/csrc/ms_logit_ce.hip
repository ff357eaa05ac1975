// Mean softmax cross entropy of a map of logits, the logits as they are: nll[p] = max_k z - z[y_p] + log sum_k exp(z[p,k] - max), 0 where y_p is outside [0,K);
// loss = sign sum nll / P.
//
// One read of the logits, nothing else of their size: a lane keeps 4 pixels (1 where rows are not made of whole vectors), their label's logit and a running maximum and sum.  No weights and
// no products take part, so a class may be masked with anything down to -infinity.  Bound by HBM: 16 x 21 x 512 x 512 in 75 us (5.1 TB/s; a copy moves 5.3), 16 x 150 x 256 x 256 in 118 (5.4).
// Small calls are the host's time: 13 us for two launches and two tensors.
#include <algorithm>
#include "ms_class_ce.h"
#include "maxstyle_hip.h"

namespace ms {

constexpr int kLcBlocks = 2048;        // workgroups at most: each leaves up to four partial sums

struct LcRun { float m, l, z; };       // sum of exp(z) = l exp(m); the label's z (where another wave has it: 0)
__device__ __forceinline__ void lc_join(LcRun& a, float m, float l) {
  const float mn = fmaxf(a.m, m), mm = mn == -__builtin_inff() ? 0.f : mn;
  a.l = a.l * __builtin_amdgcn_exp2f((a.m - mm) * kLog2e) + l * __builtin_amdgcn_exp2f((m - mm) * kLog2e);
  a.m = mn;
}

// GROUPS = 1: every wave has pixels of its own; 16: the 16 waves of a workgroup split the classes of the same pixels
template <int VEC, int GROUPS>
__global__ __launch_bounds__(GROUPS == 1 ? 256 : GROUPS * 64) void logit_ce_kernel(const float* __restrict__ z, const int64_t* __restrict__ labels, double* __restrict__ lsum, int K, int HW, long P) {
  constexpr int kAhead = 8;            // classes whose loads are in flight together
  constexpr int kOwn = GROUPS == 1 ? 4 : 1;          // tiles a workgroup has under way
  __shared__ LcRun run[GROUPS][64][VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = GROUPS == 1 ? 0 : wave, own = GROUPS == 1 ? wave : 0;
  double acc = 0.0;
  const long tiles = (P + 64 * VEC - 1) / (64 * VEC);
  for (long t = (long)blockIdx.x * kOwn + own; t < tiles; t += (long)gridDim.x * kOwn) {
    const long p = (t * 64 + lane) * VEC, pc = min(p, P - VEC);          // (clamped: the loads need no branch)
    const int n = (int)(pc / HW);
    const float* base = z + ((size_t)n * K) * HW + (size_t)(pc - (long)n * HW);
    LcRun r[VEC];
    int y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int64_t lb = labels[pc + e];
      y[e] = (lb >= 0 && lb < K) ? (int)lb : -1;
      r[e] = LcRun{-__builtin_inff(), 0.f, 0.f};
    }
    for (int k0 = grp * kAhead; k0 < K; k0 += GROUPS * kAhead) {
      float v[kAhead][VEC];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const float* src = base + (size_t)min(k0 + a, K - 1) * HW;
        if (VEC == 4) {
          const float4 f = *reinterpret_cast<const float4*>(src);
          const float ff[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[a][e] = ff[e];
        } else {
          v[a][0] = src[0];
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float m = r[e].m;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) m = fmaxf(m, v[a][e]);          // (a repeated last class changes no maximum)
        const float mm = m == -__builtin_inff() ? 0.f : m;
        float l = r[e].l * __builtin_amdgcn_exp2f((r[e].m - mm) * kLog2e);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) l += k0 + a < K ? __builtin_amdgcn_exp2f((v[a][e] - mm) * kLog2e) : 0.f;
        float zl = r[e].z;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) zl = k0 + a == y[e] ? v[a][e] : zl;          // (read here again it would come from memory: 4 M pixels x 21 classes 130 us)
        r[e] = LcRun{m, l, zl};
      }
    }
    if (GROUPS > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) run[grp][lane][e] = r[e];
      __syncthreads();
    }
    if (grp == 0 && p < P) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        for (int g = 1; g < GROUPS; ++g) {
          lc_join(r[e], run[g][lane][e].m, run[g][lane][e].l);
          r[e].z += run[g][lane][e].z;
        }
        if (y[e] >= 0) acc += (double)((r[e].m - r[e].z) + ce_log2(r[e].l) * 0.693147180559945309f);
      }
    }
    if (GROUPS > 1) __syncthreads();   // nobody overwrites `run` before it has been read
  }
  if (grp != 0) return;
  acc = wave_sum_d(acc);
  if (lane == 0) lsum[blockIdx.x * kOwn + own] = acc;
}
__global__ __launch_bounds__(1024) void logit_ce_sum_kernel(const double* __restrict__ lsum, int n, float sign, long P, float* __restrict__ loss) {
  __shared__ double redd[16];
  double a = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) a += lsum[i];
  a = block_sum_d(a, redd);
  if (threadIdx.x == 0) loss[0] = (float)((double)sign * a / (double)P);
}
}  // namespace ms

extern "C" size_t ms_logit_ce_ws_bytes(void) { return ms::kLcBlocks * 4 * sizeof(double); }
extern "C" int ms_logit_ce(const float* logits, const int64_t* labels, float* loss_out, int N, int K, int HW, float loss_sign, void* ws, size_t ws_bytes, void* stream) {
  using namespace ms;
  if (N < 1 || K < 1 || K > (1 << 30) || HW < 1 || (long long)N * HW > (1LL << 30)) { set_error("ms_logit_ce: invalid shape (up to 2^30 classes and 2^30 pixels)"); return MS_ERR_INVALID; }
  if (logits == nullptr || labels == nullptr || loss_out == nullptr) { set_error("ms_logit_ce: null pointer"); return MS_ERR_INVALID; }
  if (ws == nullptr || ws_bytes < ms_logit_ce_ws_bytes()) { set_error("ms_logit_ce: workspace too small"); return MS_ERR_WORKSPACE; }
  if (reinterpret_cast<uintptr_t>(ws) & 7u) { set_error("ms_logit_ce: workspace not 8-byte aligned"); return MS_ERR_ALIGN; }
  const long P = (long)N * HW;
  // Few pixels: one a lane, and 16 waves to a workgroup of 64 of them, each a sixteenth of the classes (1 x 1000 x 64 x 64: 21 us with
  // four pixels a lane in 16 workgroups, 13 so, the host's time)
  const bool few = P < 64 * 4 * 4 * (long)kNumCU && K >= 32, vec = !few && HW % 4 == 0 && aligned16(logits);
  const long tiles = (P + (vec ? 255 : 63)) / (vec ? 256 : 64);
  const int blocks = (int)std::min<long>(few ? tiles : (tiles + 3) / 4, kLcBlocks);
  double* lsum = (double*)ws;
  hipStream_t st = (hipStream_t)stream;
  if (few) MS_LAUNCH((logit_ce_kernel<1, 16>), dim3(blocks), dim3(1024), 0, st, logits, labels, lsum, K, HW, P);
  else if (vec) MS_LAUNCH((logit_ce_kernel<4, 1>), dim3(blocks), dim3(256), 0, st, logits, labels, lsum, K, HW, P);
  else MS_LAUNCH((logit_ce_kernel<1, 1>), dim3(blocks), dim3(256), 0, st, logits, labels, lsum, K, HW, P);
  if (int e = check_launch("logit_ce")) return e;
  MS_LAUNCH(logit_ce_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)lsum, few ? blocks : blocks * 4, loss_sign, P, loss_out);
  return check_launch("logit_ce_sum");
}
