/* maxstyle_hip.h - C ABI of libmaxstyle_hip.so (gfx950 / MI355X kernels for the MaxStyle inner loop).
 *
 * The reference (cherise215/MaxStyle) has no FFI layer: its hot path is eager PyTorch.  The drop-in
 * boundary is therefore the reference's three Python call signatures and THIS header is
 * the C ABI underneath them: every entry point names the reference lines whose arithmetic it replaces.
 *
 * Conventions
 *   - all tensors are fp32, NCHW, contiguous, device memory owned by the caller (PyTorch caching allocator);
 *     the library allocates nothing; scratch is a caller-provided workspace (size queries below)
 *   - kernels are enqueued asynchronously on `stream` (a hipStream_t passed as void*); no host sync, so every
 *     entry point may be captured into a hipGraph
 *   - return value: 0 = ok, <0 = MS_ERR_* (invalid argument / alignment / workspace), >0 = hipError_t;
 *     ms_last_error() returns a thread-local description; nothing throws across the ABI
 *   - re-entrant and thread-safe; the only mutable process-wide state is the option table (ms_set_option: which kernel FORM a dispatch picks, never what it
 *     computes) - nothing is read from the environment
 */
#ifndef MAXSTYLE_HIP_H
#define MAXSTYLE_HIP_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Two surfaces.  Both macros expand to nothing: they are labels a binding author can grep for.
 *   MS_STABLE    one entry point per operator of the reference path (convolution, BatchNorm finalize / apply / backward, pooling, heads, the MaxStyle layer and its
 *                backward, Adam / AdamW, weight gradients, running statistics, Dice confusion matrix) plus their size queries and `_bf16` twins: plain tensors in,
 *                plain tensors out, no precondition beyond shapes and alignment.  This is what INTEGRATION.md binds and what is kept source-compatible.
 *   MS_INTERNAL  engine-private fusions and their helpers (`_xfin`, `_ride`, residual tails, activation-backward epilogues, sub-pixel / small-channel forms, the
 *                fused step tail, planning and measurement queries).  They carry PRECONDITIONS the engine guarantees and a foreign caller would have to reproduce:
 *                launch epochs left in statistics tables by the producing conv, zero-initialised granule tables and error words, a GPU the launch does not share
 *                (`_xfin`, single-read MaxStyle kernel: every workgroup of the grid must be resident at once - grids are sized from the occupancy API for that, and
 *                NO dispatch order is assumed), a rider's channel count within ms_conv_ride_capacity.  Their results are bit-identical to the MS_STABLE sequence
 *                they replace (tests/test_round3_gpu.py); they may change between rounds. */
#define MS_STABLE
#define MS_INTERNAL
MS_STABLE int ms_version(void);
MS_STABLE const char* ms_last_error(void);

/* ---- library options ------------------------------------------------------------------------------------------------------------------------------------
 * The library reads NOTHING from the environment (round 5: 33 getenv switches inside the dispatch before).  Where more than one kernel form is
 * built for a shape, the dispatch consults these process-wide options; the DEFAULTS are the product, the other values exist for A/B timing and for the "same bits as the
 * form it replaces" tests.  Every form computes the same operator; an option never changes what an entry point means.
 *   name               default  values
 *   "conv.wide"        1        0: 3x3 stride-1 convs never take conv_wide_kernel (first-generation kernel everywhere)
 *   "conv.wino"        1        0: MS_FETCH_WINOGRAD is ignored (direct form) | 1: honoured per call | 2: Winograd form wherever legal, asked for or not
 *   "conv.wino32"      1        0: no 8 x 32-pixel Winograd tile for rows of 20..63 pixels
 *   "conv.wino_nt"     0        0: automatic | 1 / 2: channel blocks per staged Winograd tile
 *   "conv.wino_block"  1        0: never the 8x8 block form | 1: by fill | 2: wherever legal
 *   "conv.wide_rows"   0        0: 4-row tiles | 8: 8-row tiles of the direct-form wide kernel where they have work for the chip
 *   "conv.k1s" "conv.k1g" "conv.s2g2"   1   0: the streaming / GEMM 1x1 forms, the second-generation stride-2 form are not chosen
 *   "conv.k3n"         1        0: 3x3 stride-1 convs on rows of 12 / 14 / 16 pixels stay on the first-generation kernel (csrc/ms_conv_k3n.h is the second generation:
 *                               flattened-pixel M-tiles, LDS-DMA / hoisted-offset staging; the same bits in `out` where the first generation runs 16-channel chunks)
 *   "conv.k9"          1        ms_conv3x3_small_cin at Cin = 1, rows of whole 16-pixel M-tiles: the nine taps are the K dimension of the matrix instruction (3 MFMAs per
 *                               16 pixels; the same bits in `out` as ms_conv2d on that layer) | 0: the vector-ALU form (another rounding)
 *   "conv.force_nt"    0        1 / 2 / 4: output-channel blocks of 16 per workgroup of the first-generation kernel (tuning)
 *   "style.fused"      1        0: ms_style_fwd never takes the single-read kernel (three-launch path)
 *   "conv.wino_flat"   1        0: no flattened-tile Winograd form on images of 20 / 24 / 28-pixel rows (the 8 x 32-pixel tiles instead: the same bits in `out`) | 1: where it
 *                               saves a round of the persistent grid | 2: wherever legal
 *   "diag.conv_dbg"    0        timing-only ablation bits of the conv kernels - results are WRONG with any bit set
 * ms_set_option returns the previous value (>= 0) or MS_ERR_INVALID for an unknown name / a value out of range; ms_get_option the current value.  Setting an option
 * while launches of other threads are in flight is safe (relaxed atomics): such a launch takes one form or the other.  ms_option_count / ms_option_name enumerate. */
MS_STABLE int ms_set_option(const char* name, int value);
MS_STABLE int ms_get_option(const char* name);
MS_STABLE int ms_option_default(const char* name);
MS_STABLE int ms_option_count(void);
MS_STABLE const char* ms_option_name(int index);
/* diagnostic builds only (-DMS_CONV_TRACE_BUILD / -DMS_WGRAD_TRACE_BUILD): device buffers (conv: >= 128 KiB, wgrad: >= 8 KiB, or NULL) for the in-kernel cycle stamps */
MS_INTERNAL int ms_diag_set_trace(void* conv_trace, void* wgrad_trace);
/* Layer-chain probe (tools/chain_probe.py): L plain 3x3 layers C -> C on N images of H x 16 pixels as ONE persistent launch with a grid barrier
 * between layers (layer l reads a_buf / b_buf alternately and writes the other).  layers_dev: ms_diag_k3n_chain_bytes(L) bytes of device scratch; arrive: two device
 * words, zero before the first call, owned by the probe afterwards; err: set to 1 if a barrier times out.  Not used by any product path. */
MS_INTERNAL size_t ms_diag_k3n_chain_bytes(int L);
MS_INTERNAL int ms_diag_k3n_chain(const float* a_buf, float* b_buf, const float* w_packed, int N, int C, int H, int L, void* layers_dev, unsigned* arrive, int* err, void* stream);
/* bit of the `fetch` argument of the convolution entry points: the caller accepts the Winograd form for this call (see ms_conv2d) */
#define MS_FETCH_WINOGRAD 0x100
/* (bit 9, 0x200, was MS_FETCH_X3 - the three-way bf16 split form, built and measured 2x slower than the Winograd form in round 3, removed in round 5; the bit is rejected) */
/* with MS_FETCH_WINOGRAD: keep the Winograd form's ONE-channel-block variant (the input tile staged and transformed per 16 output channels) where the library would
 * stage it once per 32 (round 4).  Per output element both variants accumulate in the same order - the same bits; only the grouping of the BatchNorm partial sums
 * follows the work-item numbering.  An A/B and test switch, not a numerical choice. */
#define MS_FETCH_WINO_NT1 0x400
/* with MS_FETCH_WINOGRAD: w_packed carries the Winograd APPENDIX - the transformed weights U = G g G^T of every (input channel, output channel) pair behind the
 * packed taps, at float offset 9 * cin_pad * cout_pad, ms_wino_pack_floats(Cin, Cout) floats, filled by ms_wino_pack (below) - and the kernel may stage U from
 * there with LDS-DMA instead of transforming the nine taps of every chunk again in its staging waves (weights are constant over the K steps of a loop call and over
 * every call until the next optimiser step).  ms_wino_pack computes each value with the in-kernel expression, so results are bit-identical with and without the bit.
 * Ignored where the Winograd form is not taken. */
#define MS_FETCH_WINO_U 0x800
/* with MS_FETCH_WINOGRAD: take the BLOCK form of the Winograd kernel (four independent 8x8-pixel blocks per work item, see ms_conv2d_form) wherever it is legal,
 * not only where the dispatch finds it faster.  Same bits per output element as the tiled form.  A test and A/B switch. */
#define MS_FETCH_WINO_BLOCKS 0x1000
/* ms_conv2d epi_mode 6: the 2x2-POOLED store.  out is [N, Cout, H/2, W/2] and receives the sum of every 2x2 block of the convolution's result, in ms_pool2_sum's
 * order over the values as they would have been stored: the same bits as ms_conv2d + ms_pool2_sum, a quarter of the bytes written and none read back.  The
 * data-gradient of `conv3x3(nearest-up-sampled x)` (encoder_decoder.py:298-300, 323-337 backward) ends in exactly that sum.  Built for the Winograd form of the
 * wide kernel only (ks 3, stride 1, MS_FETCH_WINOGRAD; no bias / statistics): ask ms_conv2d_pool2_ok first. */
#define MS_EPI_POOL2 6
MS_INTERNAL int ms_conv2d_pool2_ok(int N, int Cin, int H, int W, int Cout, int pro_mode, int bf16);      /* bf16: 0 = the fp32 entry point, 1 = `_bf16`, 2 = `_bf16m` */
/* Which kernel form ms_conv2d(ks 3, stride 1, fetch) takes for this shape (16-byte aligned tensors assumed) - what the measurement tools print and price, asked of the
 * dispatch itself instead of re-deriving its rules: 0 first-generation kernel (conv_mfma_kernel) | 1 wide direct form (conv_wide_kernel) | 2 Winograd F(2x2,3x3), one
 * 16-channel block per staged tile (conv_wide_kernel<1, ..., ms_f32w*>) | 3 Winograd, two blocks (conv_wide_kernel<2, ...>: round 4) | 4 / 5 the same on independent
 * 8x8-pixel blocks instead of 4x64 / 8x32 tiles (ms_f32wb: rows that are not multiples of 32 / 64 pixels) | 6 the narrow-rows second generation (conv_k3n_kernel:
 * rows of 12 / 14 / 16 pixels, round 5) | 7 Winograd on the flattened tile list of 20-pixel images, two blocks (conv_wide_kernel<2, ..., ms_f32wf>: round 6; needs the
 * MS_FETCH_WINO_U appendix).  fetch = the call's fetch argument
 * (MS_FETCH_WINOGRAD / MS_FETCH_WINO_NT1 bits); a fused-fetch call (fetch & 0xFF != 0) is always 0. */
MS_INTERNAL int ms_conv2d_form(int N, int Cin, int H, int W, int Cout, int pro_mode, int bf16, int fetch);
/* The Winograd appendix of a packed 3x3 weight tensor (MS_FETCH_WINO_U): layout [ceil(Cout/16)][Cin/8][16 positions][8 input channels][16 output channels] fp32
 * (one 8 KB block per (16-channel output block, 8-channel chunk): what one LDS-DMA burst of a staging wave copies).  Needs Cin % 8 == 0 (ms_wino_pack_floats
 * returns 0 otherwise).  ms_wino_pack reads the taps at w_packed and writes the appendix behind them - call it after every (re-)pack of the weights. */
MS_INTERNAL size_t ms_wino_pack_floats(int Cin, int Cout);
MS_INTERNAL int ms_wino_pack(float* w_packed, int Cin, int Cout, void* stream);
/* Compute units of the current device (hipDeviceProp.multiProcessorCount, read once per device): every persistent grid and every
 * co-residency bound of the library is sized from it (a partitioned or CU-masked device reports fewer than MI355X's 256). */
MS_STABLE int ms_num_cus(void);
/* Measurement aid: register-only fp32-MFMA chains (iters x 64 per wave) on `workgroups` x `threads`; writes, for workgroup 0, {clock64() cycles,
 * 100 MHz ticks (s_memrealtime)} around the loop (tools/clock_probe.py). */
MS_INTERNAL int ms_clock_probe(int iters, int workgroups, int threads, long long* cycles_and_ticks, float* sink, void* stream);

/* ---- MaxStyle layer: src/advanced/maxstyle.py:140-189 ------------------------------------------------ */

/* bytes of workspace needed by ms_style_moments / ms_style_fwd / ms_style_bwd for a [B,C,H*W] tensor.
 * Contract: give every layer (shape) its OWN workspace, zero-fill it once after allocation and keep it for the layer's lifetime - its
 * tail holds the persistent launch-epoch state of the single-read forward kernel (the head is per-launch scratch). */
MS_STABLE size_t ms_style_ws_bytes(int B, int C, int HW);

/* mu = mean_HW(x), sig = sqrt(var_HW(x, unbiased) + eps) per plane.          maxstyle.py:157-159 */
MS_INTERNAL int ms_style_moments(const float* x, float* mu, float* sig, int planes, int HW, float eps, void* ws, size_t ws_bytes, void* stream);

/* Per-plane affine coefficients  A = sig(1-l)+sig[perm]l + gamma_noise*gamma_std,  S = mu(1-l)+mu[perm]l + beta_noise*beta_std
 * with l = clamp(lmda,0,1).  compute_std is a flag word.  bit 2 (ms_style_fwd only): the device is shared with kernels of other streams /
 * processes - the single-read kernel (whose progress argument needs its whole grid resident) is not used.  bit 0: gamma_std[c]=std_b(sig[:,c]), beta_std[c]=std_b(mu[:,c]) (unbiased) are
 * computed from mu/sig and stored (the reference caches them on the first forward), else they are read.  compute_std bit 1:
 * l = lmda without the clamp (MixStyle: src/advanced/mixstyle.py:91-92).
 * lmda == NULL: no style mixing (mix_style=False); gamma_noise == beta_noise == NULL: no_noise=True.  maxstyle.py:165-185 */
MS_INTERNAL int ms_style_coeffs(float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std, const float* lmda,
                    const float* gamma_noise, const float* beta_noise, const int64_t* perm, float* coefA, float* coefS,
                    int B, int C, void* stream);

/* y = A * ((x - mu) / sig) + S                                                 maxstyle.py:161,184-185 */
MS_INTERNAL int ms_style_apply(const float* x, float* y, const float* mu, const float* sig, const float* coefA, const float* coefS,
                   int planes, int HW, void* stream);

/* The fused forward: moments + coeffs + apply (K1 of SURVEY.md 2.2).  Outputs y, and mu/sig/coefA/coefS [B*C]
 * (kept for the backward pass), gamma_std/beta_std [C] (written when compute_std != 0). */
MS_STABLE int ms_style_fwd(const float* x, float* y, float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std,
                 const float* lmda, const float* gamma_noise, const float* beta_noise, const int64_t* perm,
                 float* coefA, float* coefS, int B, int C, int HW, float eps, void* ws, size_t ws_bytes, void* stream);

/* The two implementations behind ms_style_fwd (same arguments, same results to rounding):
 *   ms_style_fwd_fused  single-read persistent kernel: x crosses HBM once (8 B/element); eligible when H*W % 4 == 0, 2 <= B <= 256 and
 *                       one channel group (B x chunks) fits the grid - ms_style_fused_ws_bytes() returns 0 otherwise
 *                       here `ws` is ONLY the kernel's persistent state (>= ms_style_fused_ws_bytes, zero-filled once, one layer, one
 *                       stream at a time); ws[1] (int) is an error word set if a bounded spin ever times out
 *   ms_style_fwd_3k     moments / finalize / restyle as three launches (any shape; x is read twice) */
MS_INTERNAL size_t ms_style_fused_ws_bytes(int B, int C, int HW);
/* geometry the single-read kernel would use: threads per workgroup, float4 register slots per thread, chunks per plane, grid (diagnostics) */
MS_INTERNAL int ms_style_fused_plan(int B, int C, int HW, int* threads, int* nv, int* S, int* grid);
/* byte offset of the single-read kernel's state block inside a workspace of ms_style_ws_bytes() bytes ((size_t)-1: the shape has none);
 * the int at offset + 4 is its ERROR WORD.  A caller that syncs anyway can read it with its own copy; ms_style_fused_status does a
 * stream-ordered synchronous read of the word of `state` (= workspace + offset), clears it when set and leaves the reason in ms_last_error(). */
MS_INTERNAL size_t ms_style_ws_state_offset(int B, int C, int HW);
MS_INTERNAL int ms_style_fused_status(void* state, int* out_host, void* stream);
MS_INTERNAL int ms_style_fwd_fused(const float* x, float* y, float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std,
                       const float* lmda, const float* gamma_noise, const float* beta_noise, const int64_t* perm,
                       float* coefA, float* coefS, int B, int C, int HW, float eps, void* ws, size_t ws_bytes, void* stream);
MS_INTERNAL int ms_style_fwd_3k(const float* x, float* y, float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std,
                    const float* lmda, const float* gamma_noise, const float* beta_noise, const int64_t* perm,
                    float* coefA, float* coefS, int B, int C, int HW, float eps, void* ws, size_t ws_bytes, void* stream);

/* Backward of nn.UpsamplingNearest2d (ms_pool2_sum) + the accumulate of the 1x1 skip data-gradient + the output-activation backward of the block BELOW
 * (ms_act_bwd_reduce) in one pass: out = (pool2(in) [+ add]) * lrelu'(act); part2 as ms_act_bwd_reduce ([C][ms_act_bwd_parts(N,C,Ho*Wo)][2]). */
MS_INTERNAL int ms_pool2_actbwd(const float* in, const float* add, float* out, const float* act, const float* u, const float* coef4, float* part2,
                    int N, int C, int Ho, int Wo, float slope, void* stream);
/* ... that also writes pooled [N,C,Ho/2,Wo/2] = ms_pool2_sum(out) - the input of the NEXT block's 1x1 skip data-gradient (no pooling launch there): a thread owns a
 * 2x2 quad of output pixels instead of four pixels of a row, sums the STORED values in ms_pool2_sum's order (same bits); part2 agrees with ms_pool2_actbwd's to
 * rounding (the per-thread grouping of the sums follows the mapping).  Ho even, Wo % 4 == 0. */
MS_INTERNAL int ms_pool2_actbwd_pool(const float* in, const float* add, float* out, const float* act, const float* u, const float* coef4, float* part2,
                         int N, int C, int Ho, int Wo, float slope, float* pooled, void* stream);
/* ... whose first operand in_lo [N,C,Ho,Wo] is ALREADY pooled (the data-gradient conv in front stored the 2x2 sums itself: ms_conv2d epi_mode MS_EPI_POOL2);
 * pooled may be NULL (then: ms_pool2_actbwd's pixel mapping, else ms_pool2_actbwd_pool's). */
MS_INTERNAL int ms_add_actbwd(const float* in_lo, const float* add, float* out, const float* act, const float* u, const float* coef4, float* part2,
                  int N, int C, int Ho, int Wo, float slope, float* pooled, void* stream);

/* ms_head_ce (segmentation head + cross entropy + backward to the head input h, custom_loss.py:1043-1078) whose dh is already multiplied by lrelu'(h) - h is the
 * output of the last residual block - and which writes the BatchNorm-backward sums of that block's last BatchNorm (raw input bn_u, record bn_coef4) to
 * bn_part [C][ms_head_ce_actbwd_parts(N,C,HW)][2]: replaces ms_head_ce + ms_act_bwd_reduce.  C <= 16 (parts() returns 0 otherwise: use the two calls). */
MS_INTERNAL int ms_head_ce_actbwd_parts(int N, int C, int HW);
MS_INTERNAL int ms_head_ce_actbwd(const float* h, const float* w, const float* b, const int64_t* labels, float* dh, float* loss_out, const int* loss_slot_dev,
                      int N, int C, int K, int HW, float loss_sign, void* ws, size_t ws_bytes,
                      const float* bn_u, const float* bn_coef4, float* bn_part, float act_slope, void* stream);
/* ms_conv1x1_bnres (half-resolution skip) + ms_head_ce_actbwd in ONE pass over u: the output h = lrelu(bn(u) + skip[y/2][x/2]) of the segmentation decoder's last
 * residual block (encoder_decoder.py:344-346; final_conv + cross_entropy_2D, custom_loss.py:1043-1078) is formed inside the head kernel and never written.
 * u [N,C,H,W] the block's second conv output, coef4 its BatchNorm record {sc, sh, mean, invstd}, skip [N,C,H/2,W/2] the 1x1 skip conv (+ bias) at half
 * resolution (plain ms_conv2d).  dh, bn_part, loss_out (may be NULL: ms_step_tail), ws as ms_head_ce_actbwd.  Same arithmetic, same order: bit-identical.
 * pooled != NULL: a thread owns a 2x2 pixel quad instead of four pixels of a row and also writes pooled [N,C,H/2,W/2] = ms_pool2_sum(dh) (the sum of the STORED
 * values, in ms_pool2_sum's order: same bits) - the input of the block's 1x1 skip data-gradient; the per-thread grouping of the BatchNorm-backward sums changes
 * with the mapping, so bn_part agrees with the pooled == NULL form to rounding, not to the bit. */
MS_INTERNAL int ms_head_ce_tail(const float* u, const float* skip, const float* coef4, const float* w, const float* b, const int64_t* labels, float* dh, float* loss_out,
                    const int* loss_slot_dev, int N, int C, int K, int H, int W, float loss_sign, void* ws, size_t ws_bytes, float* bn_part, float act_slope, float* pooled,
                    void* stream);


/* ms_style_bwd for a layer that sits right behind a residual block (x = that block's output): dx is additionally multiplied by lrelu'(x) and the sums the
 * BatchNorm backward of the block's last BatchNorm needs are written to bn_part [C][ms_style_bwd_actbwd_parts(B,C,HW)][2] (the partial layout of
 * ms_act_bwd_reduce, consumed by ms_bn_bwd_coefs / ms_bn_bwd_full): bn_u = that BatchNorm's raw input [B,C,H,W], bn_coef4 = its {scale, shift, mean, invstd}.
 * Replaces ms_style_bwd + ms_act_bwd_reduce (encoder_decoder.py:344-346 backward); needs dx and H*W % 4 == 0.  The style gradients are unaffected. */
/* ms_head_bwd + ms_style_bwd[_actbwd] in ONE pass, for a MaxStyle layer that sits directly in front of a 1x1 head (apply_max_style: layer 4 -> final_conv ->
 * Sigmoid, encoder_decoder.py:619-627): the layer's incoming gradient dy[c] = sum_k head_w[k][c] * head_g[k] * out_k(1-out_k) is formed while streaming instead of
 * being written by ms_head_bwd and read back (a [B,C,H,W] tensor each way).  head_g, head_out [B,K,HW] (head_out NULL: no sigmoid), head_w [K][C], K <= 4.
 * Everything else as ms_style_bwd_actbwd; bn_u / bn_coef4 / bn_part may be NULL (plain ms_style_bwd), dx may be NULL.  Same arithmetic, same order: bit-identical. */
MS_INTERNAL int ms_style_bwd_head(const float* head_g, const float* head_out, const float* head_w, int K, const float* x, float* dx, const float* mu, const float* sig,
                      const float* coefA, const float* gamma_std, const float* beta_std, const float* lmda, const int64_t* perm,
                      float* d_gamma, float* d_beta, float* d_lmda, int B, int C, int HW, void* ws, size_t ws_bytes,
                      const float* bn_u, const float* bn_coef4, float* bn_part, float act_slope, void* stream);
MS_INTERNAL int ms_style_bwd_actbwd_parts(int B, int C, int HW);
MS_INTERNAL int ms_style_bwd_actbwd(const float* dy, const float* x, float* dx, const float* mu, const float* sig, const float* coefA,
                        const float* gamma_std, const float* beta_std, const float* lmda, const int64_t* perm,
                        float* d_gamma, float* d_beta, float* d_lmda, int B, int C, int HW, void* ws, size_t ws_bytes,
                        const float* bn_u, const float* bn_coef4, float* bn_part, float act_slope, void* stream);

/* bf16 ACTIVATION STORAGE variants ("`_bf16` I/O variants with fp32 statistics"): x / y / dy / dx are bf16 bit
 * patterns (uint16_t, NCHW, 16-byte aligned, H*W % 8 == 0) - half the HBM bytes of these bandwidth-bound kernels; mu / sig / coefficients / std / partial
 * sums / parameter gradients stay fp32 (fp64 merges) and all arithmetic is fp32.  Results equal the fp32 entry points evaluated on the bf16-rounded
 * input, with y / dx rounded to nearest-even bf16 on store (relative error <= 2^-9 per element).  Same workspace contract (ms_style_ws_bytes_bf16). */
MS_STABLE size_t ms_style_ws_bytes_bf16(int B, int C, int HW);
MS_INTERNAL size_t ms_style_fused_ws_bytes_bf16(int B, int C, int HW);
MS_STABLE int ms_style_fwd_bf16(const uint16_t* x, uint16_t* y, float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std,
                      const float* lmda, const float* gamma_noise, const float* beta_noise, const int64_t* perm,
                      float* coefA, float* coefS, int B, int C, int HW, float eps, void* ws, size_t ws_bytes, void* stream);
MS_INTERNAL int ms_style_fwd_fused_bf16(const uint16_t* x, uint16_t* y, float* mu, float* sig, float* gamma_std, float* beta_std, int compute_std,
                            const float* lmda, const float* gamma_noise, const float* beta_noise, const int64_t* perm,
                            float* coefA, float* coefS, int B, int C, int HW, float eps, void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_style_bwd_bf16(const uint16_t* dy, const uint16_t* x, uint16_t* dx, const float* mu, const float* sig, const float* coefA,
                      const float* gamma_std, const float* beta_std, const float* lmda, const int64_t* perm,
                      float* d_gamma, float* d_beta, float* d_lmda, int B, int C, int HW, void* ws, size_t ws_bytes, void* stream);

/* Backward of the layer (autograd of maxstyle.py:161-185 with mu/sig detached):
 *   dx = dy*A/sig (skipped when dx == NULL);  d_gamma = gamma_std*sum(dy*xhat);  d_beta = beta_std*sum(dy);
 *   d_lmda[b] = 1[0<=lmda<=1] * sum_c (sig[perm b]-sig[b])*S2 + (mu[perm b]-mu[b])*S1.   Any of d_* may be NULL. */
MS_STABLE int ms_style_bwd(const float* dy, const float* x, float* dx, const float* mu, const float* sig, const float* coefA,
                 const float* gamma_std, const float* beta_std, const float* lmda, const int64_t* perm,
                 float* d_gamma, float* d_beta, float* d_lmda, int B, int C, int HW, void* ws, size_t ws_bytes, void* stream);

/* torch.optim.Adam(lr, betas=(b1,b2), eps, weight_decay=0, amsgrad=False) single update on a flat buffer
 * (advanced_triplet_recon_segmentation_model.py:537,562).  step is 1-based; if step_dev != NULL the kernel uses
 * *step_dev + 1 instead (graph replay) - advance it with ms_counter_incr. */
MS_STABLE int ms_adam_step(float* p, const float* g, float* m, float* v, int n, float lr, float b1, float b2, float eps, int step,
                 const int* step_dev, void* stream);
MS_INTERNAL int ms_counter_incr(int* counter, void* stream);

/* The tail of one inner step of generate_max_style_image (advanced_triplet...py:559-562: loss.backward() has produced the layers' partial sums,
 * optimizer.step()) as ONE launch: for every inserted MaxStyle layer the reduction ms_style_bwd does behind its streaming pass (call ms_style_bwd /
 * ms_style_bwd_actbwd with d_gamma = d_beta = d_lmda = NULL: the per-plane partial sums stay in the layer's workspace, ms_style_bwd_slots() per plane),
 * torch.optim.Adam on those parameters (ms_adam_step's arithmetic), the cross-entropy sum of ms_head_ce_actbwd called with loss_out = NULL (ce_part = that
 * call's workspace, ce_nparts = ms_head_ce_actbwd_parts(); loss_out[*step_dev] = ce_scale * sum), and *step_dev += 1.  Bit-identical to the separate calls.
 * Parameters / gradients / moments are ONE flat buffer each (p, g, m, v); a layer names its rows by element offsets (-1: the layer has no such tensor),
 * learn_* = 0 leaves a tensor's parameters untouched (its gradient is still written).  `arrive`: one int, zero-initialised once, dedicated to this call site. */
#define MS_MAX_TAIL_LAYERS 8
typedef struct ms_tail_layer {
  const void* part;                 /* float2 [B*C][S] */
  const float* mu; const float* sig; const float* gamma_std; const float* beta_std;
  const int64_t* perm;              /* NULL: no style mixing (off_lmda = -1) */
  int off_gamma, off_beta, off_lmda;
  int learn_noise, learn_mix;
  int B, C, S;
} ms_tail_layer;
MS_INTERNAL int ms_style_bwd_slots(int B, int C, int HW, int bf16);
MS_INTERNAL int ms_step_tail(const ms_tail_layer* layers, int n_layers, const double* ce_part, int ce_nparts, double ce_scale, float* loss_out,
                 float* p, float* g, float* m, float* v, float lr, float b1, float b2, float eps, int* step_dev, int* arrive, void* stream);

/* ---- convolution stack: src/models/ebm/encoder_decoder.py:22-74, 289-357, 423-482, 561-596, 634-680 -------- */

/* Implicit-GEMM convolution on the exact-fp32 matrix cores.  Replaces nn.Conv2d(k=3,p=1,s=1|2), nn.Conv2d(k=1),
 * nn.ConvTranspose2d(k=2,s=2) and (with transformed weights) their data-gradients.
 *   in        [N,Cin,Hs,Ws]; in2 same shape (only for pro_mode 2)
 *   w_packed  [ks*ks][cin_pad][cout_pad] fp32, cin_pad = roundup(Cin,4), cout_pad = roundup(gemm_cols,64), zero padded,
 *             w_packed[ky*ks+kx][ci][co] = weight[co][ci][ky][kx]           (gemm_cols = Cout, or 4*Cout for epi_mode 2)
 *   ks/stride (3,1) (3,2) (1,1) (2,2); padding = 1 for ks 3 else 0
 *   fetch     0 normal | 1 nearest x2 up-sampling fused into the load | 2 zero-insertion x2 (stride-2 data-gradient)
 *             | MS_FETCH_WINOGRAD (bit 8, with fetch 0): the caller ACCEPTS the Winograd F(2x2,3x3) form of a 3x3 stride-1 convolution where it is built
 *             (fp32 or bf16 storage, Cin % 8 == 0, rows of >= 20 pixels with W % 4 == 0): 16 instead of 36 multiplications per 2x2 outputs, the same fp32
 *             matrix instruction.  On random data it is as close to fp64 as the direct form (2-4e-7 of the output range); on the networks'
 *             activations (non-zero channel means: the transforms add and subtract values of the size of the mean) its rounding error is about twice
 *             the direct form's, which doubles the activation-mask flips behind a backward pass - measured on the full-size training pass, weight
 *             gradients against the fp64 oracle: direct form 4.7e-4 mean / 3.3e-3 worst, Winograd 1.0e-3 / 1.0e-2, the fp32 CPU reference itself
 *             5.2e-4 / 4.2e-3.  The inner style-optimisation loop sets the bit (its parity tests hold unchanged); the training passes do not.
 *             Without the bit the result is the direct form's, bit for bit.
 *   pro_mode  0 none | 1 v = LeakyReLU_slope(pro_a[i]*v + pro_b[i]), i = (n*pro_nstride + ci)*pro_cstride  (BatchNorm apply +
 *             activation of the producer; pro_nstride = 0 per channel, = Cin per (n,c) plane; pro_cstride = 4 reads the
 *             interleaved coef4 records of ms_bn_finalize / ms_bn_bwd_coefs in place)
 *             | 2 v = pro_a[i]*v + pro_b[i]*in2 + pro_c[i], i = ci*pro_cstride   (BatchNorm backward apply)
 *             every activation slope of this library (slope, act_slope) must lie in [0, 1] - LeakyReLU (0.2) or ReLU (0), the only ones the
 *             reference uses (encoder_decoder.py:646,655); anything else is MS_ERR_INVALID (the kernels compute max(v, v*slope))
 *   epi_mode  0 out = acc + bias | 1 out += acc + bias | 2 ConvTranspose2d(k=2,s=2) pixel-shuffle store:
 *             GEMM column (dy*2+dx)*Cout+co -> out[n,co,2y+dy,2x+dx] (needs ks=1)
 *   stats     NULL or a table of ms_conv_stats_bytes() bytes receiving per-workgroup running (count, mean, M2, 0) of the outputs
 *             (float4 header {slots used} + float4[Cout][ms_conv_stats_parts()]) for ms_bn_finalize (BatchNorm batch statistics;
 *             model_util.py:468-510). */
MS_STABLE size_t ms_conv_stats_bytes(int N, int Cout, int Hout, int Wout);
MS_STABLE int ms_conv_stats_parts(int N, int Hout, int Wout);
MS_STABLE int ms_conv2d(const float* in, const float* in2, float* out, const float* w_packed, const float* bias,
              int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
              int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
              int epi_mode, float* stats, void* stream);

/* 3x3 stride-1 convolution with <= 4 INPUT channels and 16 output channels on the vector ALUs - the encoder's first conv on the image (`inc.0`, encoder_decoder.py:
 * 441-445 forward; on the matrix cores its single input channel is padded to an 8-channel chunk: 3 of 18 MFMAs per 16 pixels carry data).  out [N,16,H,W] =
 * conv3x3(in [N,Cin,H,W], w) + bias; w_packed = ms_conv2d's forward layout; stats (may be NULL) = ms_conv2d's statistics table of the outputs (one slot per
 * workgroup, header {slots, launch epoch}): ms_bn_finalize and the `_xfin` consumers read it like any other.  W % 4 == 0, 16-byte aligned tensors.
 * ms_conv3x3_small_cin_ok answers 1 where the entry point is also the FASTER choice (Cin == 1: 30 vs 34 us at 16x1x256x256), not merely accepted. */
MS_INTERNAL int ms_conv3x3_small_cin_ok(int Cin, int Cout, int W);
MS_INTERNAL int ms_conv3x3_small_cin(const float* in, float* out, const float* w_packed, const float* bias, int N, int Cin, int H, int W, int Cout, float* stats, void* stream);

/* 3x3 stride-1 convolution with <= 4 OUTPUT channels on the vector ALUs (csrc/ms_conv_small.hip): the data-gradient that reaches the image (`inc.0`,
 * encoder_decoder.py:441-445: 16 -> 1 channels at config 2, 64 -> 3 at config 4).  Same arithmetic contract as ms_conv2d(ks=3, stride=1) with pro_mode 0 or 2
 * (BatchNorm-backward prologue pro_a*in + pro_b*in2 + pro_c); w_packed = the packed weights [9][cin_pad][cout_pad].  W % 4 == 0; one image of the input
 * (Cin * H * W * 4 bytes) below 2 GiB (buffer-resource addressing: MS_ERR_INVALID otherwise).  The products of an output are summed channel by channel, tap by tap,
 * as fused multiply-adds (to rounding against ms_conv2d, which sums them in the matrix cores' order). */
MS_INTERNAL int ms_conv3x3_small_cout_ok(int Cout, int W);
MS_INTERNAL int ms_conv3x3_small_cout(const float* in, const float* in2, float* out, const float* w_packed, int N, int Cin, int H, int W, int Cout,
                          int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_cstride, void* stream);

/* Sub-pixel form of the two x2 resampling convolutions (csrc/ms_conv_subpix.h): same results as ms_conv2d with fetch = 1 / 2 to fp32 rounding, without
 * multiplying the duplicates / zeros the resampling inserts (2.25x / 4x fewer matrix instructions).  in [N,Cin,Hs,Ws], out [N,Cout,2Hs,2Ws]; ms_conv_subpix_eligible:
 * 1 = Ws % 4 == 0 (every form), 2 = Ws even (14-pixel rows of the shipped 224-pixel workload: the second generation's block geometry only - fp32 storage, mode 0 with w_sums).
 *   mode 0: nn.UpsamplingNearest2d(2) -> nn.Conv2d(3x3,p=1) (encoder_decoder.py:298-300, 323-337); w_packed = the FORWARD packed weights, bias optional,
 *           stats = optional BatchNorm statistics table of the outputs (ms_conv_stats_bytes);
 *   mode 1: data-gradient of nn.Conv2d(3x3,s=2,p=1) (res_convdown.down, encoder_decoder.py:40); `in` = dY [N,Cout_fwd,Hs,Ws], w_packed = the
 *           DATA-GRADIENT packed weights, Cout = Cin_fwd.  With ref != NULL the epilogue also does what ms_act_bwd_reduce would do on the result:
 *           out = dX * lrelu'(ref) (ref = the materialised activation output [N,Cout,2Hs,2Ws]) and tab gets the sums of out and out*(u - mean) per channel
 *           (u = that activation's raw BatchNorm input, coef4 = its {scale, shift, mean, invstd}; table as ms_conv2d_actbwd: ms_conv_actbwd_tab_bytes).
 *           ref == NULL with u != NULL: the activation lrelu(scale*u + shift) was never materialised - the mask is recomputed from u. */
MS_INTERNAL int ms_conv_subpix_eligible(int Hs, int Ws);
MS_INTERNAL int ms_conv_subpix(const float* in, float* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout, int mode,
                   float* stats, const float* ref, const float* u, const float* coef4, float act_slope, float* tab, void* stream);
/* Second generation (csrc/ms_conv_subpix2.h; fp32 storage): the same products in the same order per output element (`out` has ms_conv_subpix's bits; the statistics /
 * activation-backward tables agree to summation order), staged entirely by LDS-DMA.  Mode 0 reads its 16 sub-pixel weight matrices from w_sums, an appendix of
 * ms_subpix_pack_floats(Cin, Cout) floats that ms_subpix_pack() fills from the packed forward weights ONCE PER WEIGHT VERSION (repack after every change of the taps;
 * the sums are formed in the first generation's order: same bits).  w_sums == NULL in mode 0, bf16 storage or tensors beyond 2 GiB: the first generation runs.
 * flags: MS_SUBPIX_FIRST_GEN forces the first generation; MS_SUBPIX_TILES / MS_SUBPIX_BLOCKS force the work-item geometry (8 x 32-pixel tiles | sixteen 4 x 4-pixel
 * blocks from a flattened block list: every stored size that is a multiple of 4 fills its MFMA rows); neither: chosen by fill.  ms_conv_subpix = flags 0, w_sums NULL. */
#define MS_SUBPIX_FIRST_GEN 1
#define MS_SUBPIX_TILES 2
#define MS_SUBPIX_BLOCKS 4
MS_INTERNAL size_t ms_subpix_pack_floats(int Cin, int Cout);
MS_INTERNAL int ms_subpix_pack(const float* w_packed, float* w_sums, int Cin, int Cout, void* stream);
MS_INTERNAL int ms_conv_subpix2(const float* in, float* out, const float* w_packed, const float* w_sums, const float* bias, int N, int Cin, int Hs, int Ws, int Cout, int mode,
                    float* stats, const float* ref, const float* u, const float* coef4, float act_slope, float* tab, int flags, void* stream);
/* Every appendix of a weight version in ONE launch (ms_wino_pack / ms_subpix_pack jobs behind ms_repack_weights; same device functions: same bits).  desc_dev: a device
 * array of ndesc records {int64 begin; float* w_packed; float* w_sums; int kind (0 = ms_wino_pack, 1 = ms_subpix_pack); int Cin, Cout, cin_pad, cout_pad; int pad},
 * ms_appendix_desc_bytes() each, sorted by `begin` = the job's first thread (jobs are spaced by ms_appendix_job_threads(kind, Cin, Cout)); total = threads of all jobs. */
MS_INTERNAL size_t ms_appendix_desc_bytes(void);
MS_INTERNAL long long ms_appendix_job_threads(int kind, int Cin, int Cout);
MS_INTERNAL int ms_appendix_batch(const void* desc_dev, int ndesc, long long total, void* stream);

/* Tail of a residual block in one launch (res_convdown / res_up_family: `last_act(conv_input(x) + conv(x))`, encoder_decoder.py:62-64, 344-346):
 * the 1x1 skip convolution `conv_input` (packed weights, bias) whose epilogue reads the raw output `u` [N,Cout,H',W'] of the block's second 3x3
 * convolution, applies that layer's BatchNorm record coef4 = {scale, shift, ..} per channel and the LeakyReLU:
 *     out = lrelu((scale*u + shift) + (conv1x1(in) + bias)).
 * Replaces ms_conv2d(ks=1) + ms_bn_act(res_mode 1 / 2) - the skip tensor is never written (2 HBM passes and one launch less per block); same
 * arithmetic, bit for bit.  up2 = 1: `in` has HALF the resolution of u / out (up_type 'NN': nn.UpsamplingNearest2d commutes with a 1x1 conv). */
MS_INTERNAL int ms_conv1x1_bnres(const float* in, float* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout,
                     const float* u, const float* coef4, float slope, int up2, void* stream);

/* Cross-workgroup finalize (`_xfin`): ms_bn_finalize + its consumer in ONE launch.  The consumer launch derives the BatchNorm coefficients itself from the
 * statistics table `stats` of the conv that produced u (one wave per channel runs ms_bn_finalize's arithmetic - same bits -, writes the record to coef4 for
 * later kernels and publishes (scale, shift) as two tagged 8-byte granules in `gran`; the waves that need a channel poll its granules - bounded spin, *err = 1
 * on time-out).  Tag = the launch epoch the producing conv left in the table header, so nothing is cleared between launches: `gran` (ms_xfin_gran_bytes(C))
 * and `err` are zero-filled ONCE by the caller and dedicated to this BatchNorm layer.  Needs every workgroup of the launch co-resident (an exclusive device).
 * Replaces, per residual block, the ms_bn_finalize launch behind its second conv (~4.8 us of launch boundary in a replayed graph). */
MS_INTERNAL size_t ms_xfin_gran_bytes(int C);
/* The same for a consumer that needs the coefficients in its PROLOGUE: ms_conv2d with pro_mode 1 (kind 0: ms_bn_finalize folded in; tab = statistics table of the
 * producing conv, p0 = gamma, p1 = beta, eps) or pro_mode 2 (kind 1: ms_bn_bwd_coefs folded in; tab = the float2 table of ms_conv2d_actbwd / ms_conv_subpix, p0 =
 * the forward records {sc, sh, mean, invstd} [Cin][4], count = N*H*W).  The MFMA waves reduce and publish, then fill the launch's LDS coefficient table from
 * the granules while the staging waves' first global loads are in flight.  coef4 [Cin][4] receives the records ms_bn_finalize / ms_bn_bwd_coefs would write. */
MS_INTERNAL int ms_conv2d_xfin(const float* in, const float* in2, float* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride,
                   int fetch, int pro_mode, float slope, int epi_mode, float* stats, int kind, const float* tab, const float* p0, const float* p1, float eps, double count,
                   float* coef4, void* gran, int* err, void* stream);
MS_INTERNAL int ms_conv1x1_bnres_xfin(const float* in, float* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout,
                          const float* u, const float* stats, const float* gamma, const float* beta, float eps, float* coef4, void* gran, int* err,
                          float slope, int up2, void* stream);
/* ms_conv2d_actbwd (pro_mode 2) whose prologue coefficients are derived in the launch like ms_conv2d_xfin kind 1 does: xf_tab = the float2 table of the activation-backward
 * epilogue that produced `in`, xf_p0 = the forward records [Cin][4] of the BatchNorm being back-propagated, count = N*H*W; xf_coef4 [Cin][4] receives the records.  The same
 * bits in `out` and `tab` as ms_bn_bwd_coefs + ms_conv2d_actbwd (round 5: two launches of the encoder's backward per step). */
MS_INTERNAL int ms_conv2d_actbwd_xfin(const float* in, const float* in2, float* out, const float* w_packed, int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                          const float* u, const float* coef4, float act_slope, float* tab, const float* xf_tab, const float* xf_p0, double count, float* xf_coef4,
                          void* gran, int* err, void* stream);

/* ms_conv2d whose output is the gradient w.r.t. an activation LeakyReLU_act_slope(coef4[c].scale*u + coef4[c].shift) that the forward pass
 * never materialised (it was folded into the next convolution's prologue: encoder_decoder.py:44-46, 62-64): the epilogue multiplies by the
 * activation's derivative and accumulates, per output channel, {sum g, sum g*(u - coef4[c].mean)} - the result of
 * ms_act_bwd_reduce(ref = NULL) without its extra pass over the gradient (autograd: leaky_relu_backward + the reductions of
 * native_batch_norm_backward).  No bias, plain store.
 *   u [N,Cout,Hout,Wout], coef4 float4[Cout] from ms_bn_finalize, tab: ms_conv_actbwd_tab_bytes(Cout) bytes, float2 header {slots used}
 *   + float2[Cout][slots]; hand it to ms_bn_bwd_coefs / ms_bn_bwd_full with nparts = 0. */
MS_STABLE size_t ms_conv_actbwd_tab_bytes(int Cout);
MS_INTERNAL int ms_conv2d_actbwd(const float* in, const float* in2, float* out, const float* w_packed,
                     int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                     int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                     const float* u, const float* coef4, float act_slope, float* tab, void* stream);

/* ms_conv2d (a 1x1 conv: ks == 1) that also CARRIES a coefficient job for the launch behind it.  ride_kind 0 = ms_bn_bwd_coefs: one MFMA wave per channel
 * c < ride_C reduces that channel's BatchNorm-backward partial sums (ride_tab [ride_C][ride_nparts][2], or - ride_nparts == 0 - the table of ms_conv2d_actbwd /
 * ms_conv_subpix; ride_p0 = the forward records [C][4], ride_count = N*H*W) with ms_bn_bwd_coefs' arithmetic in its order (same bits) and writes
 * ride_out4[c] = {al, be, de, 0}, while the workgroup's staging waves fetch their first chunk.  ride_kind 1 = ms_bn_finalize: ride_tab = the statistics table of
 * the conv in front (ms_conv2d `stats`), ride_p0 / ride_p1 = gamma / beta, ride_eps -> ride_out4[c] = {scale, shift, mean, invstd}.
 * The conv neither reads nor waits for ride_out4: it is for the NEXT launch on the stream (the residual block's data-gradient conv, whose prologue needs it
 * - model_util.py:468-510 backward; the 1x1 skip data-gradient runs between producer and consumer anyway, so the ~5 us coefficient launch disappears).
 * MFMA wave w of workgroup b takes channels 4b + w, 4b + w + 4*grid, ...: any grid carries the whole job; within ride_C <= ms_conv_ride_capacity(N, Hout, Wout) a wave has
 * at most one channel (the speed the rider is meant to have). */
/* Streaming form of the 1x1 convolutions (csrc/ms_conv_k1s.h: every wave streams 64-pixel units with 16 loads in flight, no LDS / barrier on the activation path; the
 * channels are accumulated in the tiled kernel's order: same bits).  Chosen by ms_conv2d / ms_conv2d_ride / ms_conv1x1_bnres(_xfin) themselves for fp32 storage, no
 * prologue, Cin a power of two in 16..128, H W % 4 == 0, no statistics, and at least one 64-pixel unit per CU.  Option "conv.k1s" (ms_set_option)
 * switches the choice off / on for the process (A/B runs, the same-bits tests). */
/* Second generation of the 3x3 stride-2 forward conv (csrc/ms_conv_s2.h: LDS-DMA staging, 64-bit A-fragment reads of the interleaved patch, 1 / 2 / 4 channel blocks per
 * staged patch, 4 x 4-block work items on small outputs), taken by ms_conv2d(ks 3, stride 2) itself for fp32 storage without prologue / statistics.  Same products per output
 * element; the 4-channel groups are accumulated in ascending order (the first generation's order where it uses 4-channel chunks).  Option "conv.s2g2": off / on for
 * the process. */
/* LDS-tiled GEMM form of the 1x1 convolutions with >= 256 input channels (csrc/ms_conv_k1g.h: 64-pixel units of a flattened (image, unit) list, LDS-DMA staging, 1 / 2 / 4
 * sixteen-channel blocks per staged tile; plain and residual-tail epilogues, rider, cross-workgroup finalize; same bits as the tiled kernel), chosen by the 1x1 entry points
 * themselves.  Option "conv.k1g": off / on for the process. */
MS_INTERNAL int ms_conv_k1s_would_run(int N, int Cin, int H, int W, int Cout, int epi_mode);      /* the choice for this shape (epi_mode 0 plain, 2 ConvTranspose GEMM, 4 residual tail) */
MS_INTERNAL int ms_conv_ride_capacity(int N, int Hout, int Wout);
MS_INTERNAL int ms_conv2d_ride(const float* in, const float* in2, float* out, const float* w_packed, const float* bias,
                   int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                   int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                   int epi_mode, float* stats, int ride_kind, const float* ride_tab, int ride_nparts, const float* ride_p0, const float* ride_p1, float ride_eps, double ride_count,
                   float* ride_out4, int ride_C, void* stream);

/* Chan-merge of the per-workgroup statistics in fp64 -> coef4[c] = {scale=gamma*invstd, shift=beta-mean*scale, mean, invstd}
 * (biased variance + eps: nn.BatchNorm2d training-mode normalisation with frozen affine). */
MS_STABLE int ms_bn_finalize(const float* stats, int nparts, const float* gamma, const float* beta, float eps, float* coef4, int C, void* stream);

/* ---- streaming kernels around the convolutions ------------------------------------------------------------- */

/* out = LeakyReLU_slope(coef4[c].scale*u + coef4[c].shift + res): BatchNorm apply + residual add + activation
 * (encoder_decoder.py:62-64, 344-346; slope 0.2, or 0 for nn.ReLU; 0 <= slope <= 1).  res_mode 0 none | 1 same shape | 2 res is
 * [N,C,H/2,W/2] and is nearest-up-sampled on the fly (conv1x1 commutes with nn.UpsamplingNearest2d). */
MS_STABLE int ms_bn_act(const float* u, const float* coef4, const float* res, int res_mode, float* out, int N, int C, int H, int W, float slope, void* stream);

/* ms_bn_finalize + ms_bn_act(res_mode 0) in one launch, for a BatchNorm whose only consumer is its own activation (the encoder's code z_i, the code decoupler's z_s:
 * encoder_decoder.py:646, 655): coef4 receives ms_bn_finalize's record, out = LeakyReLU_slope(scale*u + shift).  Same arithmetic in the same order as the two calls:
 * the same bits.  stats / nparts / gamma / beta / eps as ms_bn_finalize; u, out [N,C,H,W]. */
MS_INTERNAL int ms_bn_finalize_act(const float* stats, int nparts, const float* gamma, const float* beta, float eps, float* coef4, const float* u, float* out,
                       int N, int C, int H, int W, float slope, void* stream);

/* Backward through the activation + the two BatchNorm-backward reductions in one pass:
 *   gout = gin * (r > 0 ? 1 : slope), r = ref (the saved activation output) or coef4.scale*u+coef4.shift when ref == NULL;
 *   part2[c][ms_act_bwd_parts()] = per-workgroup {sum gout, sum gout*(u - mean_c)} with mean_c = coef4[c].mean (centred, as
 *   native_batch_norm_backward does: the uncentred form cancels catastrophically for channels with a large mean).  gout may alias gin. */
MS_STABLE int ms_act_bwd_parts(int N, int C, int HW);
MS_STABLE int ms_act_bwd_reduce(const float* gin, const float* ref, const float* u, const float* coef4, float* gout, float* part2,
                      int N, int C, int HW, float slope, void* stream);

/* native_batch_norm_backward (input gradient only, batch statistics): du = al*g + be*u + de, coef_out4[c] = {al,be,de,0}
 * (SURVEY.md A.7).  count = N*H*W.  Feed coef_out4 to ms_conv2d(pro_mode=2) of the data-gradient convolution.
 * nparts = 0: part2 is the table written by ms_conv2d_actbwd (its header holds the slot count). */
MS_STABLE int ms_bn_bwd_coefs(const float* part2, int nparts, const float* coef4, double count, float* coef_out4, int C, void* stream);

/* out[p,y,x] (+)= in[p,2y,2x]+in[p,2y,2x+1]+in[p,2y+1,2x]+in[p,2y+1,2x+1]: gradient of nn.UpsamplingNearest2d(2) */
MS_STABLE int ms_pool2_sum(const float* in, float* out, int planes, int Ho, int Wo, int accumulate, void* stream);

/* ---- weight gradients for the outer update: autograd's convolution_backward w.r.t. `weight` when loss.backward()
 * runs after standard_training / hard_example_traininng (train_adv_supervised_segmentation_triplet.py:532-535).
 *   dw[m][n][ty][tx] (+)= sum_{img,y,x} P[img,m,y,x] * Q[img,n, stride*y+ty-pad, stride*x+tx-pad]        pad = 1 for ks 3, else 0
 * Conv2d (ks 3 stride 1|2, ks 1): P = gradient w.r.t. the conv output [N][M=Cout][Hp][Wp], Q = conv input [N][Nq=Cin][Hq][Wq],
 *   dw = weight.grad [Cout][Cin][ks][ks].  ConvTranspose2d (ks 2, stride 2): P = its input, Q = gradient w.r.t. its output,
 *   dw = weight.grad [Cin][Cout][2][2].
 * q_fetch 1: Q is stored at half resolution and read through nearest 2x up-sampling (nn.UpsamplingNearest2d before the conv, ks 3 stride 1 only).
 * p_mode 2: P = pa[m]*p + pb[m]*p2 + pc[m] (BatchNorm backward of the masked gradient p with the raw conv output p2 - what ms_conv2d's
 *   pro_mode 2 applies on the data-gradient side); q_mode 1: Q = LeakyReLU_slope(qa[n]*q + qb[n]) (BatchNorm apply + activation of the
 *   producer layer); coefficient arrays are read with stride coef_stride (4 for the float4 tables of ms_bn_finalize / ms_bn_bwd_coefs).
 * Built combinations: 3x3 stride 1: (p_mode,q_mode) in {(0,0),(2,0),(2,1)}; 1x1: (0,0),(2,0); stride 2 (3x3, ConvTranspose 2x2): (0,0) - the ones
 * the networks need; anything else returns an error.
 * Deterministic: per-workgroup partials in `ws` (ms_conv_wgrad_ws_bytes), summed in a fixed order; accumulate != 0 adds to dw. */
MS_STABLE size_t ms_conv_wgrad_ws_bytes(int N, int M, int Nq, int Hp, int Wp, int ks, int stride);
MS_STABLE int ms_conv_wgrad(const float* p, const float* p2, const float* q, float* dw, int N, int M, int Nq, int Hp, int Wp, int Hq, int Wq,
                  int ks, int stride, int q_fetch, int p_mode, const float* pa, const float* pb, const float* pc,
                  int q_mode, const float* qa, const float* qb, int coef_stride, float slope, int accumulate,
                  void* ws, size_t ws_bytes, void* stream);

/* BatchNorm backward from the partial sums of ms_act_bwd_reduce: coefficients as ms_bn_bwd_coefs (coef_out4 may be NULL) plus
 * BatchNorm weight.grad (dgamma) / bias.grad (dbeta) and dsum = sum of the masked gradient (bias.grad of the residual 1x1 conv that
 * shares it); each may be NULL.  accumulate != 0 adds.  In the hard-example pass the BatchNorm affine is frozen
 * (model_util.py:468-510): pass NULL for dgamma/dbeta there.  nparts = 0: part2 is the table of ms_conv2d_actbwd. */
MS_STABLE int ms_bn_bwd_full(const float* part2, int nparts, const float* coef4, double count, float* coef_out4, float* dgamma, float* dbeta, float* dsum,
                   int accumulate, int C, void* stream);

/* out[c] (+)= sum_{n,hw} x[n,c,hw]: bias.grad of a convolution from the gradient of its output. */
MS_STABLE size_t ms_channel_sum_ws_bytes(int N, int C);
MS_STABLE int ms_channel_sum(const float* x, int N, int C, int HW, float* out, int accumulate, void* ws, size_t ws_bytes, void* stream);

/* weight.grad [K][C] / bias.grad [K] (db may be NULL) of a 1x1 head, d computed on the fly:
 *   mode 0: d = scale*(softmax(aux) - onehot(target int64 [N,HW]))   aux = logits [N,K,HW]      (cross_entropy_2D, custom_loss.py:1043-1078)
 *   mode 1: d = scale*(aux - target)*aux*(1-aux)                      aux = sigmoid output, target float [N,K,HW]   (0.5*MSE, :718-729)
 *   mode 2: d = scale*aux. */
MS_STABLE size_t ms_head_wgrad_ws_bytes(int N, int C, int K, int HW);
MS_STABLE int ms_head_wgrad(const float* h, const float* aux, const void* target, int mode, float scale, float* dw, float* db,
                  int N, int C, int K, int HW, int accumulate, void* ws, size_t ws_bytes, void* stream);

/* loss_out[0] = loss_scale * sum (x-target)^2 (loss_out may be NULL); dx = grad_scale*(x-target) (dx may be NULL).
 * compute_image_recon_loss 'l2' (advanced_triplet...py:718-722): loss_scale = 0.5/n, grad_scale = upstream/n. */
MS_STABLE size_t ms_mse_ws_bytes(void);
MS_STABLE int ms_mse_loss(const float* x, const float* target, size_t n, float loss_scale, float grad_scale, float* loss_out, float* dx,
                void* ws, size_t ws_bytes, void* stream);
/* `_ds`: the three launches that seed a backward pass (ms_head_ce's dh, ms_head_wgrad's d, ms_mse_loss's dx) with the UPSTREAM gradient as a device scalar
 * (*..._dev multiplies the host-side scale inside the kernel; NULL = 1): `loss.backward()` hands the training pass its incoming gradient as a GPU tensor, and reading it
 * on the host would make the host wait for everything queued before it - the inner loop included (advanced_triplet...py:731-786, train_adv...py:532-535). */
MS_STABLE int ms_head_wgrad_ds(const float* h, const float* aux, const void* target, int mode, float scale, const float* scale_dev, float* dw, float* db,
                     int N, int C, int K, int HW, int accumulate, void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_mse_loss_ds(const float* x, const float* target, size_t n, float loss_scale, float grad_scale, const float* grad_scale_dev, float* loss_out, float* dx,
                   void* ws, size_t ws_bytes, void* stream);

/* torch.optim.AdamW (weight_decay > 0: p *= 1 - lr*wd first) / torch.optim.Adam (weight_decay = 0) on a flat buffer
 * (advanced_triplet...py:1055-1086); step semantics as ms_adam_step. */
MS_STABLE int ms_adamw_step(float* p, const float* g, float* m, float* v, size_t n, float lr, float b1, float b2, float eps, float weight_decay,
                  int step, const int* step_dev, void* stream);

/* After an optimiser step: re-pack every convolution weight from the flat parameter buffer into ms_conv2d's forward and data-gradient
 * layouts with one launch.  desc_dev: device array of ndesc records of ms_repack_desc_bytes() bytes each
 *   { int64 begin (prefix sum of element counts), int64 src_off (floats into flat), float* dst_fwd, float* dst_dgrad,
 *     int32 kind (0 Conv2d [Cout][Cin][k][k], 1 ConvTranspose2d k2s2 [Cin][Cout][2][2]), d0, d1, k, cin_pad_fwd, cout_pad_fwd, cin_pad_dgrad, cout_pad_dgrad };
 * total = sum of element counts.  Padding of the packed buffers is left untouched (zero from allocation). */
MS_INTERNAL size_t ms_repack_desc_bytes(void);
MS_STABLE int ms_repack_weights(const float* flat, const void* desc_dev, int ndesc, long long total, void* stream);

/* Running statistics of a tracking BatchNorm forward from the coefficient table of ms_bn_finalize (mean, invstd):
 * running = (1-momentum)*running + momentum*batch, variance unbiased (count/(count-1)). */
MS_STABLE int ms_bn_running_update(const float* coef4, float* running_mean, float* running_var, int C, double count, float momentum, float eps, void* stream);
/* ... for all BatchNorm layers of a pass in one launch; desc_dev: nlayers records of ms_bn_running_desc_bytes() bytes
 *   { const float* coef4, float* running_mean, float* running_var, int32 C, float count } (same momentum for all). */
MS_INTERNAL size_t ms_bn_running_desc_bytes(void);
MS_INTERNAL int ms_bn_running_update_batch(const void* desc_dev, int nlayers, float momentum, float eps, void* stream);

/* The two halves of ms_conv_wgrad for a whole backward pass: ms_conv_wgrad_partials runs only the MFMA kernel (partials stay in `ws`, the
 * number of partial slots is returned in *nslots_out), ms_wgrad_reduce_batch then sums the partials of MANY tensors with one launch.
 * desc_dev: device array of ndesc records of ms_wgrad_batch_desc_bytes() bytes:
 *   { int64 block_begin (prefix sum of ceil(numel/64)), const float* partial, float* dst, int32 numel, nslots, accumulate, pad };
 * total_blocks = sum of ceil(numel/64). */
MS_INTERNAL int ms_conv_wgrad_partials(const float* p, const float* p2, const float* q, int N, int M, int Nq, int Hp, int Wp, int Hq, int Wq,
                           int ks, int stride, int q_fetch, int p_mode, const float* pa, const float* pb, const float* pc,
                           int q_mode, const float* qa, const float* qb, int coef_stride, float slope,
                           void* ws, size_t ws_bytes, int* nslots_out, void* stream);
MS_INTERNAL size_t ms_wgrad_batch_desc_bytes(void);
MS_INTERNAL int ms_wgrad_reduce_batch(const void* desc_dev, int ndesc, long long total_blocks, void* stream);

/* Per-plane min-max rescale y = (x - min)/(max - min + eps)*(new_max - new_min) + new_min: rescale_intensity
 * (common_utils/basic_operations.py:257-281), applied to the stylised image right after the path (advanced_triplet...py:868-869). */
MS_STABLE int ms_rescale_intensity(const float* x, float* y, int planes, int HW, float new_min, float new_max, float eps, void* stream);

/* cm[label*K + argmax(logits)] += 1 over all pixels (accumulates; zero cm first). Evaluation: common_utils/metrics.py:12-52 (confusion
 * matrix), :216-218 (Dice = 2|A n B| / (|A|+|B|) per class, medpy.metric.binary.dc). K <= 4. */
MS_STABLE int ms_confusion(const float* logits, const int64_t* labels, unsigned long long* cm, int N, int K, int HW, void* stream);

/* Heads (1x1 conv with K <= 4 outputs from C <= 64 channels; w is [K][C]):
 *   ms_head_fwd  out = sigmoid?(w h + b)         MyDecoder.final_conv + nn.Sigmoid (encoder_decoder.py:582,594)
 *   ms_head_bwd  dh = w^T (dout * out*(1-out))   (apply_sigmoid=0: dh = w^T dout)
 *   ms_head_ce   logits = w h + b; loss = loss_sign * cross_entropy_2D(logits, labels) (custom_loss.py:1043-1078: sum of
 *                pixel NLL / (N*H*W)); writes loss_out[*loss_slot_dev or 0], dh = d loss / d h (NULL to skip) and the
 *                logits (NULL to skip).  The inner loop uses loss_sign = -1 (advanced_triplet...py:555). */
MS_STABLE int ms_head_fwd(const float* h, const float* w, const float* b, float* out, int N, int C, int K, int HW, int apply_sigmoid, void* stream);
/* ms_style_fwd's restyle + ms_head_fwd in one pass, for a MaxStyle layer that sits directly in front of the 1x1 head (apply_max_style: layer 4 -> final_conv ->
 * Sigmoid, encoder_decoder.py:598-631): x [N,C,HW] is the layer's INPUT, (mu, sig, coefA, coefS) [N*C] what ms_style_fwd - called with y = NULL: statistics and
 * coefficients only - left; y = coefA/sig * (x - mu) + coefS (maxstyle.py:157-188) is formed per element with the layer's own expression and rounding and never
 * written: same bits in `out` as ms_style_fwd + ms_head_fwd. */
MS_INTERNAL int ms_head_fwd_styled(const float* x, const float* mu, const float* sig, const float* coefA, const float* coefS, const float* w, const float* b, float* out,
                       int N, int C, int K, int HW, int apply_sigmoid, void* stream);
MS_STABLE int ms_head_bwd(const float* dout, const float* out, const float* w, float* dh, int N, int C, int K, int HW, int apply_sigmoid, void* stream);
MS_STABLE size_t ms_head_ce_ws_bytes(int N, int HW);
MS_STABLE int ms_head_ce(const float* h, const float* w, const float* b, const int64_t* labels, float* dh, float* logits, float* loss_out,
               const int* loss_slot_dev, int N, int C, int K, int HW, float loss_sign, void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_head_ce_ds(const float* h, const float* w, const float* b, const int64_t* labels, float* dh, float* logits, float* loss_out,
                  const int* loss_slot_dev, int N, int C, int K, int HW, float loss_sign, const float* grad_scale_dev, void* ws, size_t ws_bytes, void* stream);

/* Mean softmax cross entropy of logits as they are, any number of classes (custom_loss.py:1043-1078): loss_out[0] = loss_sign * sum_p (log sum_k exp z[n,k,hw] - z[n,labels,hw]) / (N*HW);
 * a label outside [0,K) adds nothing.  logits [N][K][HW] fp32, read once; masked classes may be anything down to -infinity.  Deterministic.  ws: ms_logit_ce_ws_bytes(), 8-byte aligned. */
MS_STABLE size_t ms_logit_ce_ws_bytes(void);
MS_STABLE int ms_logit_ce(const float* logits, const int64_t* labels, float* loss_out, int N, int K, int HW, float loss_sign, void* ws, size_t ws_bytes, void* stream);

/* ---- head + softmax cross entropy over MANY classes, the logits never kept ------------------------------------------------------------------------
 * ms_head_ce's operator without its limits (K <= 4, C <= 64), with all gradients in the one call:
 *   z[p,v] = sum_c w[v,c] h[p,c] + b[v];  lse[p] = log sum_v exp z[p,v];  nll[p] = lse[p] - z[p,labels[p]], 0 where the label is outside [0,V)
 *   loss = loss_sign * sum_p nll / (N*HW, or with mean_valid the rows whose label is a class; no such row: loss and gradients are 0)   (custom_loss.py:1043-1078)
 *   dh = d loss/d h, dw = d loss/d w, db = d loss/d b, times *grad_scale_dev (NULL: 1); each may be NULL.
 * h [N][C][HW] (rows of features [T][C]: N = T, HW = 1), w [V][C], b [V] or NULL, labels [N][HW]; dh like h, dw like w.  types: bit 0 h / dh are bf16, bit 1 w / dw
 * are bf16, otherwise fp32; b, db, loss, nll, lse are fp32.  Up to 8192 channels, 2^20 classes, 2^30 rows.  A row whose label is not a class gives nothing to the
 * loss and exactly 0 to every gradient, whatever its features hold; b may be -infinity for classes that are switched off.
 * Numbers: an fp32 element of h or w enters the products to 2^-22 of itself or 2^-39 of the largest of its row (up to 128 channels: of 64 neighbouring classes), a bf16
 * one as it is; G = g (softmax - hot) to 2^-22 of itself or 2^-41 g, or 2^-11 and 2^-29 g where h AND w are bf16 - for rows, classes and upstream gradients g within
 * 2^30 of the largest; sums are fp32 or wider.  ms_class_ce_bwd's softmax = exp(z - lse) carries the 2^-24 |lse| of the fp32 lse; ms_class_ce's does not.
 * ms_class_ce_fwd: nll and lse of every row, ms_class_ce_bwd: the gradients for an upstream gradient of every row (grad [N][HW]) and the lse of that forward.
 * Deterministic.  ws: ms_class_ce_ws_bytes(.., need_grad = 1 when any gradient is asked for), 16-byte aligned, free again when the stream has passed the call. */
MS_STABLE size_t ms_class_ce_ws_bytes(int N, int C, int V, int HW, int types, int need_grad);
MS_STABLE int ms_class_ce(const void* h, const void* w, const float* b, const int64_t* labels, float* loss_out, void* dh, void* dw, float* db, int N, int C, int V, int HW,
                int types, float loss_sign, int mean_valid, const float* grad_scale_dev, void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_class_ce_fwd(const void* h, const void* w, const float* b, const int64_t* labels, float* nll, float* lse, int N, int C, int V, int HW, int types,
                    void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_class_ce_bwd(const void* h, const void* w, const float* b, const int64_t* labels, const float* lse, const float* grad, void* dh, void* dw, float* db,
                    int N, int C, int V, int HW, int types, void* ws, size_t ws_bytes, void* stream);

/* ---- activation checkpoints in 8 bits ---------------------------------------------------------------------------------------------------------------
 * A plane (n,c) of x [N][C][HW] in blocks of ms_act8_block() = 256 elements (the last may be shorter): with d = x - centre_c,
 *   s = max|d| / 127 (fp32), q = rint(d / s), and the sign of d where that is 0 although d is not;  x' = centre_c + q s.       q [N][C][HW], s [N][C][ceil(HW/256)]
 * coef4 (NULL: centre 0) is a BatchNorm record of ms_bn_finalize {scale, shift, mean, invstd} per channel: centre_c = -shift/scale where that lies within 4 standard
 * deviations of the mean, else the mean - the sign of scale x + shift is then kept exactly.  A block below 2^-120 is kept as zeros, one with an infinity or NaN
 * reads back as NaN.
 *   ms_act8_bwd_reduce   ms_act_bwd_reduce out of a checkpoint: g' = g * (r > 0 ? 1 : slope), r = ref_q (the checkpoint, without a record, of the saved activation
 *                        output: only its signs are read) or scale x' + shift when ref_q == NULL; part2 [C][ms_act8_bwd_parts()][2] = {sum g', sum g'(x' - mean)} for
 *                        ms_bn_bwd_full; gout (g', may alias gin) and uout (x') may be NULL.  coef4 must be the record the checkpoint was made with.
 *   ms_act8_bn_act_bwd   the whole backward of BatchNorm (batch statistics) + LeakyReLU: du, dgamma, dbeta (may not be NULL; du may alias g).
 * Deterministic; any alignment and any HW; up to 2^26 runs of 1024 elements inside the planes, the backward entries up to 2^24 of up to 16384. */
MS_STABLE int ms_act8_block(void);
MS_STABLE int ms_act8_pack(const float* x, const float* coef4, int8_t* q, float* s, int N, int C, int HW, void* stream);
MS_STABLE int ms_act8_unpack(const int8_t* q, const float* s, const float* coef4, float* x, int N, int C, int HW, void* stream);
MS_STABLE int ms_act8_bwd_parts(int N, int C, int HW);
MS_STABLE int ms_act8_bwd_reduce(const float* gin, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, float* gout, float* uout, float* part2,
                       int N, int C, int HW, float slope, void* stream);
MS_STABLE size_t ms_act8_bwd_ws_bytes(int N, int C, int HW);
MS_STABLE int ms_act8_bn_act_bwd(const float* g, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, float* du, float* dgamma, float* dbeta,
                       int N, int C, int HW, float slope, void* ws, size_t ws_bytes, void* stream);
MS_STABLE int ms_act8_pack_bf16(const uint16_t* x, const float* coef4, int8_t* q, float* s, int N, int C, int HW, void* stream);
MS_STABLE int ms_act8_unpack_bf16(const int8_t* q, const float* s, const float* coef4, uint16_t* x, int N, int C, int HW, void* stream);
MS_STABLE int ms_act8_bwd_reduce_bf16(const uint16_t* gin, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, uint16_t* gout, uint16_t* uout, float* part2,
                            int N, int C, int HW, float slope, void* stream);
MS_STABLE int ms_act8_bn_act_bwd_bf16(const uint16_t* g, const int8_t* ref_q, const int8_t* q, const float* s, const float* coef4, uint16_t* du, float* dgamma, float* dbeta,
                            int N, int C, int HW, float slope, void* ws, size_t ws_bytes, void* stream);

/* ---- bf16 ACTIVATION STORAGE for the conv stack (SURVEY.md 8(b) "`_bf16` I/O variants with fp32 statistics") -----------------
 * Twins of the fp32 entry points above with the same argument lists and semantics; every ACTIVATION tensor (conv inputs / outputs, raw conv
 * outputs u, gradients, residuals, head inputs / outputs) is a tensor of bf16 bit patterns (uint16_t), everything else - packed weights, biases,
 * BatchNorm coefficient records, statistics / partial tables, losses, logits - stays fp32 (fp64 where the fp32 entry point uses it).  Arithmetic is
 * unchanged: loads widen bf16 to fp32 exactly, the convolutions run on the fp32 matrix cores, BatchNorm statistics are taken from the fp32
 * accumulators BEFORE the output is rounded, stores round to nearest-even bf16 (relative error <= 2^-9 per stored element).  Requirements: the
 * vector paths of the fp32 entry points (rows of W % 4 == 0 elements - W % 2 for fetch 1 -, 16-byte aligned tensors); MS_ERR_INVALID otherwise.
 */
MS_STABLE int ms_conv2d_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, const float* bias,
                   int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                   int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                   int epi_mode, float* stats, void* stream);
/* `_bf16m`: bf16 storage AND bf16 matrix arithmetic.  3x3 stride-1 convolutions with rows of >= 16 pixels (W % 4 == 0) run v_mfma_f32_16x16x16_bf16 with
 * fp32 accumulation: the contraction operands - the prologue's output and the weights - are rounded to bf16 on their way into LDS (relative error <= 2^-9
 * per operand; the accumulation, the BatchNorm statistics and the epilogue are those of ms_conv2d_bf16).  Every other shape runs ms_conv2d_bf16 unchanged.
 * Measured against fp64 on the rounded operands: 3.5e-3 of the output range = the bf16 rounding of the stored output. */
MS_STABLE int ms_conv2d_bf16m(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, const float* bias,
                    int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                    int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                    int epi_mode, float* stats, void* stream);
MS_INTERNAL int ms_conv2d_actbwd_bf16m(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed,
                           int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                           int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                           const uint16_t* u, const float* coef4, float act_slope, float* tab, void* stream);
MS_INTERNAL int ms_conv1x1_bnres_bf16(const uint16_t* in, uint16_t* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout,
                          const uint16_t* u, const float* coef4, float slope, int up2, void* stream);
MS_INTERNAL int ms_conv2d_actbwd_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed,
                          int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                          int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                          const uint16_t* u, const float* coef4, float act_slope, float* tab, void* stream);
MS_INTERNAL int ms_style_bwd_actbwd_parts_bf16(int B, int C, int HW);
MS_INTERNAL int ms_style_bwd_actbwd_bf16(const uint16_t* dy, const uint16_t* x, uint16_t* dx, const float* mu, const float* sig, const float* coefA,
                             const float* gamma_std, const float* beta_std, const float* lmda, const int64_t* perm,
                             float* d_gamma, float* d_beta, float* d_lmda, int B, int C, int HW, void* ws, size_t ws_bytes,
                             const uint16_t* bn_u, const float* bn_coef4, float* bn_part, float act_slope, void* stream);
MS_INTERNAL int ms_conv_subpix_bf16(const uint16_t* in, uint16_t* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout, int mode,
                        float* stats, const uint16_t* ref, const uint16_t* u, const float* coef4, float act_slope, float* tab, void* stream);
MS_INTERNAL int ms_conv3x3_small_cin_bf16(const uint16_t* in, uint16_t* out, const float* w_packed, const float* bias, int N, int Cin, int H, int W, int Cout, float* stats, void* stream);
MS_INTERNAL int ms_conv3x3_small_cout_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, int N, int Cin, int H, int W, int Cout,
                               int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_cstride, void* stream);
MS_STABLE int ms_bn_act_bf16(const uint16_t* u, const float* coef4, const uint16_t* res, int res_mode, uint16_t* out, int N, int C, int H, int W, float slope, void* stream);
MS_INTERNAL int ms_bn_finalize_act_bf16(const float* stats, int nparts, const float* gamma, const float* beta, float eps, float* coef4, const uint16_t* u, uint16_t* out,
                            int N, int C, int H, int W, float slope, void* stream);
MS_STABLE int ms_act_bwd_reduce_bf16(const uint16_t* gin, const uint16_t* ref, const uint16_t* u, const float* coef4, uint16_t* gout, float* part2,
                           int N, int C, int HW, float slope, void* stream);
MS_STABLE int ms_pool2_sum_bf16(const uint16_t* in, uint16_t* out, int planes, int Ho, int Wo, int accumulate, void* stream);
MS_INTERNAL int ms_pool2_actbwd_bf16(const uint16_t* in, const uint16_t* add, uint16_t* out, const uint16_t* act, const uint16_t* u, const float* coef4, float* part2,
                         int N, int C, int Ho, int Wo, float slope, void* stream);
MS_INTERNAL int ms_conv2d_ride_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, const float* bias,
                        int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride, int fetch,
                        int pro_mode, const float* pro_a, const float* pro_b, const float* pro_c, int pro_nstride, int pro_cstride, float slope,
                        int epi_mode, float* stats, int ride_kind, const float* ride_tab, int ride_nparts, const float* ride_p0, const float* ride_p1, float ride_eps, double ride_count,
                        float* ride_out4, int ride_C, void* stream);
MS_INTERNAL int ms_conv2d_xfin_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride,
                        int fetch, int pro_mode, float slope, int epi_mode, float* stats, int kind, const float* tab, const float* p0, const float* p1, float eps, double count,
                        float* coef4, void* gran, int* err, void* stream);
MS_INTERNAL int ms_conv2d_actbwd_xfin_bf16(const uint16_t* in, const uint16_t* in2, uint16_t* out, const float* w_packed, int N, int Cin, int Hs, int Ws, int Cout, int ks, int stride,
                               int fetch, const uint16_t* u, const float* coef4, float act_slope, float* tab, const float* xf_tab, const float* xf_p0, double count,
                               float* xf_coef4, void* gran, int* err, void* stream);
MS_INTERNAL int ms_conv1x1_bnres_xfin_bf16(const uint16_t* in, uint16_t* out, const float* w_packed, const float* bias, int N, int Cin, int Hs, int Ws, int Cout,
                               const uint16_t* u, const float* stats, const float* gamma, const float* beta, float eps, float* coef4, void* gran, int* err,
                               float slope, int up2, void* stream);
MS_INTERNAL int ms_pool2_actbwd_pool_bf16(const uint16_t* in, const uint16_t* add, uint16_t* out, const uint16_t* act, const uint16_t* u, const float* coef4, float* part2,
                              int N, int C, int Ho, int Wo, float slope, uint16_t* pooled, void* stream);
MS_INTERNAL int ms_add_actbwd_bf16(const uint16_t* in_lo, const uint16_t* add, uint16_t* out, const uint16_t* act, const uint16_t* u, const float* coef4, float* part2,
                       int N, int C, int Ho, int Wo, float slope, uint16_t* pooled, void* stream);
MS_STABLE int ms_head_fwd_bf16(const uint16_t* h, const float* w, const float* b, uint16_t* out, int N, int C, int K, int HW, int apply_sigmoid, void* stream);
MS_INTERNAL int ms_head_fwd_styled_bf16(const uint16_t* x, const float* mu, const float* sig, const float* coefA, const float* coefS, const float* w, const float* b, uint16_t* out,
                            int N, int C, int K, int HW, int apply_sigmoid, void* stream);
MS_STABLE int ms_head_bwd_bf16(const uint16_t* dout, const uint16_t* out, const float* w, uint16_t* dh, int N, int C, int K, int HW, int apply_sigmoid, void* stream);
MS_STABLE int ms_head_ce_bf16(const uint16_t* h, const float* w, const float* b, const int64_t* labels, uint16_t* dh, float* logits, float* loss_out,
                    const int* loss_slot_dev, int N, int C, int K, int HW, float loss_sign, void* ws, size_t ws_bytes, void* stream);
MS_INTERNAL int ms_head_ce_tail_bf16(const uint16_t* u, const uint16_t* skip, const float* coef4, const float* w, const float* b, const int64_t* labels, uint16_t* dh, float* loss_out,
                         const int* loss_slot_dev, int N, int C, int K, int H, int W, float loss_sign, void* ws, size_t ws_bytes, float* bn_part, float act_slope, uint16_t* pooled,
                         void* stream);
MS_INTERNAL int ms_head_ce_actbwd_bf16(const uint16_t* h, const float* w, const float* b, const int64_t* labels, uint16_t* dh, float* loss_out, const int* loss_slot_dev,
                           int N, int C, int K, int HW, float loss_sign, void* ws, size_t ws_bytes,
                           const uint16_t* bn_u, const float* bn_coef4, float* bn_part, float act_slope, void* stream);

#ifdef __cplusplus
}
#endif
#endif
