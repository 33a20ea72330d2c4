/*
 * omniwave_b200 -- C ABI of the B200-native BiGEMM operator.
 *
 * BiGEMM (OmniWeave's structured two-sided tiled GEMM) maps an NHWC activation
 * x[B,H,W,C] to a residual delta of the same shape.  For every spatial tile q_s
 * (16 tokens chosen by a route plan) and channel group q_c (d channels):
 *
 *     T = x[b, tok_idx[q_s,:], ch_idx[q_c,:]]                 (16 x d)
 *     U = A_u T B_u[q_c],  V = A_v T B_v[q_c]                (16 x rd)
 *     Z = silu(U) * V
 *     delta = (A_o Z B_o[q_c]) * mask * gamma[ch]            (16 x d)
 *
 * and delta is scattered back to the positions it was gathered from.  This is
 * the computation of the reference's ``bigemm_delta_reference``
 * (omniweave/ops/reference.py:120-173) with ``pack_tiles`` (:16-64) and
 * ``unpack_tiles`` (:67-117) folded into the kernels' loads and stores.
 *
 * Conventions
 *  - All tensor pointers are device pointers owned by the caller; the library
 *    only borrows them for the duration of the call.  It keeps no state
 *    between calls except immutable per-device kernel attributes, the
 *    per-device fault word (ow_device_fault) and, for
 *    ow_bigemm_fwd_noalloc only, that entry point's fixed scratch array and
 *    its cached device address (see its comment).
 *  - ``stream`` is a ``cudaStream_t`` passed as ``void*``.  Calls are
 *    asynchronous on that stream and never synchronise the device.
 *  - Every entry point returns OW_OK (0) or an error code; no C++ exception
 *    crosses the ABI.  ``ow_last_error()`` returns a thread-local message for
 *    the last failing call made by the calling thread.
 *  - Functions are reentrant: concurrent calls on different streams are safe
 *    as long as their workspaces do not overlap.  The exception is
 *    ow_bigemm_fwd_noalloc, whose calls share one scratch array and must not
 *    overlap on the GPU (see its comment).
 */
#ifndef OMNIWAVE_B200_H
#define OMNIWAVE_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OW_ABI_VERSION 8

#if defined(__GNUC__)
#define OW_API __attribute__((visibility("default")))
#else
#define OW_API
#endif

/* Element types. */
enum {
  OW_DTYPE_F32 = 0,
  OW_DTYPE_F64 = 1,
  OW_DTYPE_BF16 = 2,
  OW_DTYPE_F16 = 3
};

/* Status codes. */
enum {
  OW_OK = 0,
  OW_ERR_INVALID = 1,      /* bad argument: null pointer, shape mismatch, ... */
  OW_ERR_UNSUPPORTED = 2,  /* valid but not supported (dtype, tile size, device) */
  OW_ERR_CUDA = 3,         /* a CUDA runtime call or kernel launch failed */
  OW_ERR_WORKSPACE = 4     /* workspace missing or smaller than required */
};

/*
 * Route description of one BiGEMM call.  Mirrors the reference ``RoutePlan``
 * (omniweave/models/routing.py:17-33): ``tok_idx`` is
 * ``plan.token_indices`` and ``ch_idx`` is ``plan.channel_indices``, both as
 * int32 device arrays, with pad index H*W for tokens and C for channels.
 * Pad entries are exactly the masked-off entries of the reference's masks.
 * Valid (non-pad) token indices must be distinct, and so must valid channel
 * indices (every plan the reference builds satisfies this).
 */
typedef struct ow_route_t {
  int32_t batch, height, width, channels; /* B, H, W, C of the NHWC activation */
  int32_t q_s, q_c;                       /* number of spatial tiles / channel groups */
  int32_t g, d, rd;                       /* tile tokens (16), channel tile, expanded tile */
  const int32_t* tok_idx;                 /* [q_s * g] */
  const int32_t* ch_idx;                  /* [q_c * d] */
  /* Channel-layout hint: 0 = unknown (any table); S >= 1 = the caller
   * states that channel group q is ch_idx[q*d + k] = c0(q) + S*k for every
   * k (S == 1: one run of d consecutive channels starting on a multiple of 8;
   * the radix routes at levels 1 and 2 give S = q_c).  The hint only selects
   * a kernel: with S == 1 the forward gathers the group's rows with TMA
   * straight from x.  The kernels verify it against the table; a group that
   * does not match is not computed and the device fault word reports code 2
   * (ow_device_fault). */
  int32_t ch_stride;
} ow_route_t;

/*
 * Inputs of a forward (and of the matching backward).
 *
 * Operator mode (``rstd == NULL``, ``residual == 0``) computes exactly the
 * reference ``bigemm(x=..., plan=..., ...)`` delta.  Block mode
 * (``rstd != NULL``, ``residual == 1``) fuses ``OmniWeaveBlock.forward``
 * (omniweave/models/block.py:80-108): the tile loads apply RMSNorm
 * ``x * rstd[token] * norm_w[c]`` and the stores write ``x + scale[b]*delta``.
 */
typedef struct ow_bigemm_args_t {
  ow_route_t route;
  const void* x;            /* [B,H,W,C] contiguous, dtype x_dtype */
  int32_t x_dtype;
  int32_t compute_dtype;    /* F64/F32: exact CUDA-core path; BF16/F16: tensor-core path */
  const void* rstd;         /* [B*H*W], F64 when compute is F64 else F32; NULL in operator mode */
  const void* norm_w;       /* [C] RMSNorm weight (block mode only) */
  const void* a_u;          /* [g,g] */
  const void* a_v;          /* [g,g] */
  const void* a_o;          /* [g,g] */
  const void* b_u;          /* [q_c,d,rd] */
  const void* b_v;          /* [q_c,d,rd] */
  const void* b_o;          /* [q_c,rd,d] */
  const void* gamma;        /* [C] LayerScale */
  int32_t w_dtype;          /* dtype of norm_w, a_*, b_*, gamma as stored */
  const float* sample_scale;/* [B] per-sample drop-path scale, or NULL */
  int32_t residual;         /* 1: out = x + delta (block mode) */
  void* out;                /* [B,H,W,C], dtype out_dtype (forward only) */
  int32_t out_dtype;
  void* workspace;          /* device scratch, >= ow_bigemm_workspace_size() bytes */
  size_t workspace_bytes;
} ow_bigemm_args_t;

/* Gradients written by ow_bigemm_bwd (all outputs overwrite, never accumulate). */
typedef struct ow_bigemm_grads_t {
  const void* dout;   /* [B,H,W,C] gradient of the forward's out, dtype out_dtype */
  void* dx;           /* [B,H,W,C] dtype x_dtype (block mode: includes the residual path) */
  void* da_u;         /* [g,g]     dtype w_dtype */
  void* da_v;
  void* da_o;
  void* db_u;         /* [q_c,d,rd] */
  void* db_v;
  void* db_o;         /* [q_c,rd,d] */
  void* dgamma;       /* [C] */
  void* dnorm_w;      /* [C] block mode only, else ignored */
} ow_bigemm_grads_t;

/*
 * Number of kernels this library has launched in this process (all devices,
 * all threads).  Lets a caller check that work really ran on the GPU.
 */
OW_API uint64_t ow_launch_count(void);

/*
 * Kernel timing for measurement tools.  While set, every call in this
 * process (any host thread) records the caller's CUDA events (cudaEvent_t
 * cast to void*) on the call's stream immediately before and after one of
 * its kernels:
 *   OW_PROF_FWD   the tensor-core forward kernel,
 *   OW_PROF_PACK  the backward pack kernel (operand images),
 *   OW_PROF_BWD   the backward role kernel,
 *   OW_PROF_FPACK the forward pack kernel (P_u | P_v images).
 * Passing NULL for both events stops recording for that kernel.  Returns
 * OW_ERR_INVALID for an unknown ``kernel``.  No counterpart in the reference
 * (it is a measurement aid, not part of the operator).
 */
#define OW_PROF_FWD 0
#define OW_PROF_PACK 1
#define OW_PROF_BWD 2
#define OW_PROF_FPACK 3
OW_API int ow_profile_events(int kernel, void* start, void* stop);

/* ABI version compiled into the library (OW_ABI_VERSION). */
OW_API int ow_abi_version(void);

/* Message of the last failing call on this thread ("" if none). */
OW_API const char* ow_last_error(void);

/*
 * Returns 1 if ``device`` can run this library's kernels (sm_100a), else 0.
 * Does not change the current device.
 */
OW_API int ow_device_supported(int device);

/*
 * Fault word of this library's kernels on ``device``: 0 when no kernel ever
 * gave up on a bounded wait (every wait on the GPU is bounded at 2 s), else a
 * nonzero code (1: a wait ran out; 2: a channel group did not match the
 * route's ch_stride hint; the outputs of that call are undefined).
 * One word per device is shared by every kernel of the library.  Calls are
 * asynchronous, so a fault surfaces here, not in the failing call's status:
 * this function synchronises the device first.  ``reset`` != 0 clears the
 * word after reading it.  Returns -1 if the device cannot be queried.
 */
OW_API int ow_device_fault(int device, int reset);

/*
 * Wait-timeout self-check, a test aid with no counterpart in the reference.
 * While ``probe_ns`` is nonzero (at most 1e9), every mbarrier-pipelined
 * kernel launched afterwards first waits ``probe_ns`` nanoseconds on a
 * barrier that nothing arrives on, before it issues any copy or MMA; the
 * wait runs out, the kernel skips its work and records code 1 in the fault
 * word.  Outputs of calls made while it is set are undefined.  Pass 0 to
 * turn it off.  Returns OW_ERR_INVALID above the limit.
 */
OW_API int ow_debug_wait_probe(uint32_t probe_ns);

/*
 * Bytes of workspace a forward (``for_backward == 0``) or backward
 * (``for_backward == 1``) call with these arguments needs.  Only the shape
 * and dtype fields of ``args`` are read.
 */
OW_API size_t ow_bigemm_workspace_size(const ow_bigemm_args_t* args, int for_backward);

/*
 * Per-token reciprocal RMS for the fused block: ``rstd[r] = 1/sqrt(mean_c
 * x[r,c]^2 + eps)``, the mean taken in float32 as the reference does
 * (omniweave/models/block.py:83-84).  ``rstd`` is F64 when compute_dtype is
 * F64, else F32.
 */
OW_API int ow_rmsnorm_rstd(const void* x, int32_t x_dtype, int32_t compute_dtype,
                    int64_t rows, int32_t channels, double eps, void* rstd, void* stream);

/*
 * Forward.  Replaces the reference's ``bigemm(...)`` dispatch target
 * (omniweave/ops/bigemm.py:24-73) for backend "cuda", and in block mode the
 * body of ``OmniWeaveBlock.forward`` (omniweave/models/block.py:80-108).
 */
OW_API int ow_bigemm_fwd(const ow_bigemm_args_t* args, void* stream);

/*
 * Allocation-free variant of ow_bigemm_fwd, for callers that cannot allocate
 * device memory when they run the operator (plugin hosts that pass only input
 * and output buffers, code that must not enter the process's allocator).  It
 * has no counterpart in the reference.  Same arguments as ow_bigemm_fwd except
 * that ``workspace``/``workspace_bytes`` are ignored: scratch comes from a
 * fixed array of ow_noalloc_scratch_limit() bytes (4 MiB) in the library's
 * device memory, which every GPU that loads the library holds until exit.
 * Shapes needing more scratch are rejected with OW_ERR_WORKSPACE.  The first
 * call on a device (with that device current) looks up the array's device
 * address; make it before any stream capture.  All calls share the array, so
 * calls that overlap on the GPU race; no scratch contents need to start at
 * zero.  Allocates nothing (no cudaMalloc/cudaFree).
 */
OW_API int ow_bigemm_fwd_noalloc(const ow_bigemm_args_t* args, void* stream);

/* Scratch bytes available to ow_bigemm_fwd_noalloc (no reference counterpart). */
OW_API size_t ow_noalloc_scratch_limit(void);

/*
 * Backward of ow_bigemm_fwd with the same ``args`` (``out`` is ignored).
 * Replaces the autograd backward the reference takes through
 * ``bigemm_delta_reference`` (and, in block mode, through RMSNorm and the
 * residual add).  Weight gradients are reduced in a fixed order, so results
 * are bitwise reproducible run to run.
 */
OW_API int ow_bigemm_bwd(const ow_bigemm_args_t* args, const ow_bigemm_grads_t* grads, void* stream);

/*
 * Space-to-depth + Linear, the OmniWeave-T stem and downsamples
 * (omniweave/models/backbone.py:14-27 ``space_to_depth_nhwc`` followed by the
 * bias-free ``nn.Linear`` of :121 and :128-132, as called at :176-187), as one
 * tensor-core GEMM that reads the rearranged rows straight from x:
 *
 *   out[b, i, j, n] = sum_{dy, dx, c} s(b, i, j, dy, dx, c) * weight[n, (dy f + dx) C + c]
 *   s = x[b, f i + dy, f j + dx, c]    layout OW_LAYOUT_NHWC (downsample)
 *   s = x[b, c, f i + dy, f j + dx]    layout OW_LAYOUT_NCHW (stem: the image
 *                                      batch before its NHWC permute, :173)
 *
 * ``out`` is NHWC [batch, height/factor, width/factor, out_features] in
 * ``out_dtype`` (bf16 or f16), which is also the dtype the products are
 * taken in (f32 accumulation), as under the reference's autocast.  weight is
 * [out_features, factor^2 channels] row-major (f32 or out_dtype; f32 is
 * rounded).  Supported: NHWC with x_dtype == out_dtype, channels % 64 == 0,
 * width/factor <= 128 and out_features % 256 == 0; NCHW with channels == 3,
 * factor == 4, x f32 or out_dtype and out_features a multiple of 128 up to
 * 512.  x and out 16-byte aligned.  Anything else returns OW_ERR_UNSUPPORTED.
 */
#define OW_LAYOUT_NHWC 0
#define OW_LAYOUT_NCHW 1
typedef struct ow_s2d_linear_t {
  const void* x;
  int32_t x_dtype;
  int32_t layout;          /* OW_LAYOUT_NHWC or OW_LAYOUT_NCHW */
  int32_t batch, height, width, channels, factor;
  const void* weight;
  int32_t w_dtype;
  int32_t out_features;
  void* out;
  int32_t out_dtype;
  void* workspace;         /* ow_s2d_linear_workspace_size() bytes */
  size_t workspace_bytes;
} ow_s2d_linear_t;

/* Workspace bytes ow_s2d_linear_fwd needs (0 if the arguments are unsupported). */
OW_API size_t ow_s2d_linear_workspace_size(const ow_s2d_linear_t* args);
OW_API int ow_s2d_linear_fwd(const ow_s2d_linear_t* args, void* stream);

/*
 * Linear followed by depth-to-space, the input gradient of the downsample
 * above: the autograd of ``Linear(space_to_depth_nhwc(x, f))``
 * (omniweave/models/backbone.py:14-27, :128-132) with respect to x, without
 * the rearranged intermediate:
 *
 *   out[b, f i + dy, f j + dx, c] = sum_n y[b, i, j, n] * weight[n, (dy f + dx) C + c]
 *
 * y is NHWC [batch, height/factor, width/factor, in_features] (bf16 or f16,
 * the compute type: products in it, f32 accumulation); weight
 * [in_features, factor^2 channels] row-major (f32 or y's dtype; the folded
 * anchor weight W_a W_d where there is one); out NHWC
 * [batch, height, width, channels] in out_dtype: y's dtype, or f32 holding
 * the values rounded to y's dtype (as autocast's backward casts the 16-bit
 * input gradient to an f32 input's dtype).
 * Supported: channels and in_features multiples of 64, factor^2 channels a
 * multiple of 256, width/factor <= 128; y and out 16-byte aligned.  Anything
 * else returns OW_ERR_UNSUPPORTED.
 */
typedef struct ow_d2s_linear_t {
  const void* y;
  int32_t y_dtype;
  int32_t batch, height, width, channels, factor;   /* of the output image */
  int32_t in_features;
  const void* weight;
  int32_t w_dtype;
  void* out;
  int32_t out_dtype;
  void* workspace;         /* ow_d2s_linear_workspace_size() bytes */
  size_t workspace_bytes;
} ow_d2s_linear_t;

/* Workspace bytes ow_d2s_linear_fwd needs (0 if the arguments are unsupported). */
OW_API size_t ow_d2s_linear_workspace_size(const ow_d2s_linear_t* args);
OW_API int ow_d2s_linear_fwd(const ow_d2s_linear_t* args, void* stream);

/*
 * Global average pool + classifier head, the backbone's tail
 * (omniweave/models/backbone.py:193-197: ``pooled = stage4.mean(dim=(1, 2))``
 * then ``self.head(pooled)``, an ``nn.Linear`` with bias), as one kernel in
 * which the pooled matrix feeds the tensor-core GEMM from shared memory:
 *
 *   pooled[b, c] = round(sum_t x[b, t, c] / tokens)                 (f32 sum)
 *   out[b, n]    = round(bias[n] + sum_c weight[n, c] pooled[b, c])  (f32 acc)
 *
 * round() is to ``compute_dtype`` (bf16 or f16), which is also the dtype of
 * ``out`` [batch, classes] and of ``pooled`` [batch, channels] (written only
 * when non-NULL; the head's backward needs it), as under the reference's
 * autocast, where the f32 mean, weight and bias are cast before the GEMM.
 * x is [batch, tokens, channels] (the NHWC stage-4 map, f32 or compute_dtype);
 * weight [classes, channels] f32 or compute_dtype; bias [classes] (f32, bf16
 * or f16; rounded to compute_dtype) or NULL.  Supported: channels a multiple
 * of 512 up to 2048 and classes up to 1024; x, weight and pooled 16-byte
 * aligned.  Anything else returns OW_ERR_UNSUPPORTED.  Results are bitwise
 * reproducible (fixed summation order).
 */
typedef struct ow_pool_head_t {
  const void* x;
  int32_t x_dtype;
  int32_t batch, tokens, channels;
  const void* weight;
  int32_t w_dtype;
  const void* bias;
  int32_t bias_dtype;
  int32_t classes;
  int32_t compute_dtype;
  void* out;
  void* pooled;
  void* workspace;         /* ow_pool_head_workspace_size() bytes */
  size_t workspace_bytes;
} ow_pool_head_t;

/* Workspace bytes ow_pool_head_fwd needs (0 if the arguments are
 * unsupported): 256, plus room for the converted weight when weight is f32. */
OW_API size_t ow_pool_head_workspace_size(const ow_pool_head_t* args);
OW_API int ow_pool_head_fwd(const ow_pool_head_t* args, void* stream);

/*
 * AdamW over many tensors at once, the optimizer of the reference's training
 * engine (``torch.optim.AdamW`` at omniweave/training/engine.py:411, with the
 * clipping and the finite checks of :229-251), moments in 32 or in 8 bits:
 *
 *   g  = clip * grad
 *   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2
 *   p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
 *
 * in f32, rounded once to the parameter's dtype.  All tensors of a call share
 * a dtype (f32, bf16 or f16; the gradient has the parameter's) and the
 * hyperparameters; every tensor counts its own steps t.
 *
 * State is flat: tensor i owns the slots [slots[i], slots[i + 1]), multiples of
 * OW_ADAMW_BLOCK, of which its first elements are used.  With
 * state_bits == 32 the moments are f32.  With 8 they are e4m3 codes, with one
 * f32 scale (largest magnitude / 448) for each block of OW_ADAMW_BLOCK slots;
 * they are rounded stochastically by a hash of (slot, step), so a run is
 * reproducible bit for bit.  A positive second moment is held as the smallest
 * code at least; a block of which none is above 2^-100 is held as zeros, its
 * first moments too.  eps must be positive with 8 bits.
 *
 * ``params``, ``grads`` and ``slots`` are host arrays, read during the call
 * (a captured graph keeps the pointers it was captured with).  A NULL
 * gradient leaves its tensor, its state and its step count as they are.  A
 * gradient that is inf or NaN and does not call the step off makes its own
 * parameter and moments NaN, and no others.  A finite one whose square is past
 * f32 (above 6e20 with b2 = 0.999) is no reason to call a step off: its v is inf
 * and its update 0, for good with 32 bits; with 8 its m is then held as 0 and
 * its v as its block's largest finite one, and it goes on from there.  Neither
 * function allocates or synchronises.
 */
#define OW_ADAMW_BLOCK 256
#define OW_ADAMW_CONTROL_BYTES 64
typedef struct ow_adamw_t {
  int32_t tensors;
  int32_t dtype;
  void* const* params;              /* host [tensors] */
  const void* const* grads;         /* host [tensors] */
  const int64_t* slots;             /* host [tensors + 1] */
  const int32_t* dev_blocks;        /* device, 16-byte aligned: four ints for each block of OW_ADAMW_BLOCK
                                     * slots: its tensor, the how manieth block of that tensor it is, the
                                     * number of its slots in use (1 to OW_ADAMW_BLOCK), 0 */
  void* control;                    /* device, OW_ADAMW_CONTROL_BYTES, zero before its first use, this
                                     * optimizer's own: calls that overlap must not share it */
  int32_t state_bits;               /* 32 or 8 */
  void* exp_avg;                    /* flat m */
  void* exp_avg_sq;                 /* flat v */
  float* exp_avg_scale;             /* 8 bits: one a block */
  float* exp_avg_sq_scale;
  float* dev_steps;                 /* device [tensors]: steps done, counted up by the call */
  double lr, beta1, beta2, eps, weight_decay;
  const float* lr_ptr;              /* device learning rate in the place of ``lr``, or NULL */
  const float* found;               /* device flag, or NULL: nonzero calls the step off */
  int32_t use_norm;                 /* 1: apply what ow_grad_norm left in ``control`` */
} ow_adamw_t;

/*
 * Norm of all gradients (the tensors of several calls when only the last has
 * ``finish`` set: each adds ow_grad_norm_partials() sums from ``first`` on).
 * The last call leaves in ``control`` the clip coefficient
 * min(1, max_norm / (norm + 1e-6)) (1 when max_norm <= 0) and, with
 * skip_nonfinite, whether a gradient is inf or NaN, which ``found`` gets as
 * well.  The squares are added in f64 in a fixed order.
 */
typedef struct ow_grad_norm_t {
  double* partials;       /* device */
  int32_t first, capacity;
  int32_t finish;
  float max_norm;
  int32_t skip_nonfinite;
  float* norm;            /* device, or NULL */
  float* found;           /* device, or NULL: set to 1 when a gradient is not finite */
} ow_grad_norm_t;

OW_API int32_t ow_grad_norm_partials(const ow_adamw_t* args);
OW_API int ow_grad_norm(const ow_adamw_t* args, const ow_grad_norm_t* options, void* stream);
OW_API int ow_adamw_step(const ow_adamw_t* args, void* stream);

/*
 * RMSNorm before and after a block, fused with the block's gate, the
 * per-sample residual scale and the residual add (the norm, LayerScale and
 * drop-path of omniweave/models/block.py:80-108 around an operator that is
 * normalised on both sides).  x, delta, h and n are [samples, tokens,
 * channels]; rms(v) = v rsqrt(mean(v^2) + eps) over the channels:
 *
 *   h = x + sample_scale[b] * gate[c] * rms(delta) * post_w[c]
 *   n = rms(h) * next_w[c]
 *
 * in f32, each output rounded once; n is taken from the f32 h.  delta NULL:
 * h is x, only n is written (the plain RMSNorm).  next_w NULL: only h is.
 * gate_rows: 0 no gate, 1 a gate [channels], samples a gate [samples,
 * channels].  dtypes are f32, bf16 or f16, each array its own; h has x's.
 * rstd_delta and rstd_h [samples * tokens] are written by the forward when
 * not NULL and read by the backward.
 *
 * The backward takes dh (x's dtype, NULL for zero) and dn (n's dtype, needed
 * with next_w) and writes dx, ddelta and, where not NULL, the weights'
 * gradients in their dtypes; these are added in f32 in a fixed order.
 */
typedef struct ow_norm_t {
  int64_t samples, tokens;
  int32_t channels;
  const void* x;
  int32_t x_dtype;
  const void* delta;
  int32_t delta_dtype;
  const void* post_w;
  int32_t post_dtype;
  const void* gate;
  int32_t gate_dtype;
  int64_t gate_rows;
  const float* sample_scale;   /* [samples] or NULL */
  const void* next_w;
  int32_t next_dtype;
  double eps;
  void* h;                     /* forward only */
  void* n;                     /* forward only */
  int32_t n_dtype;
  float* rstd_delta;
  float* rstd_h;
  void* workspace;             /* backward only: ow_norm_bwd_workspace_size() bytes */
  size_t workspace_bytes;
} ow_norm_t;

typedef struct ow_norm_grads_t {
  const void* dh;
  const void* dn;
  void* dx;
  void* ddelta;
  void* dpost;
  void* dgate;
  void* dnext;
} ow_norm_grads_t;

/* Workspace bytes of ow_norm_bwd (0 if the arguments are invalid). */
OW_API size_t ow_norm_bwd_workspace_size(const ow_norm_t* args);
OW_API int ow_norm_fwd(const ow_norm_t* args, void* stream);
OW_API int ow_norm_bwd(const ow_norm_t* args, const ow_norm_grads_t* grads, void* stream);

/*
 * Layer norm over the channels of x [rows, channels]:
 *
 *   n = (x - mean(x)) rsqrt(mean((x - mean(x))^2) + eps) * weight + bias
 *
 * in f32, n rounded once.  bias may be NULL.  dtypes are f32, bf16 or f16,
 * each array its own.  mean and rstd [rows] are written by the forward when
 * not NULL (both or neither) and read by the backward, which takes dn (n's
 * dtype) and writes, where not NULL, dx (x's dtype) and the gradients of
 * weight and bias in their dtypes; these are added in f32 in a fixed order.
 */
typedef struct ow_layernorm_t {
  int64_t rows;
  int32_t channels;
  const void* x;
  int32_t x_dtype;
  const void* weight;
  int32_t weight_dtype;
  const void* bias;            /* or NULL */
  int32_t bias_dtype;
  double eps;
  void* n;                     /* forward only */
  int32_t n_dtype;
  float* mean;
  float* rstd;
  void* workspace;             /* backward only: ow_layernorm_bwd_workspace_size() bytes */
  size_t workspace_bytes;
} ow_layernorm_t;

typedef struct ow_layernorm_grads_t {
  const void* dn;
  void* dx;
  void* dweight;
  void* dbias;                 /* of bias_dtype */
} ow_layernorm_grads_t;

/* Workspace bytes of ow_layernorm_bwd (0 if the arguments are invalid). */
OW_API size_t ow_layernorm_bwd_workspace_size(const ow_layernorm_t* args);
OW_API int ow_layernorm_fwd(const ow_layernorm_t* args, void* stream);
OW_API int ow_layernorm_bwd(const ow_layernorm_t* args, const ow_layernorm_grads_t* grads, void* stream);

/*
 * Linear layer with its epilogue, for the 16-bit compute types:
 *
 *   z = x W^T + bias;   out = act(z) + residual
 *
 * x [rows, in_features] with row stride ldx, weight [out_features,
 * in_features] with row stride ldw, residual [rows, out_features] with row
 * stride ldr, all of ``dtype`` (bf16 or f16) with unit column stride; bias
 * [out_features] f32, bf16 or f16, or NULL; out [rows, out_features]
 * contiguous.  The sums and the activation are f32, out is rounded once.
 * ``z`` (NULL, or [rows, ldz] with ldz = out_features rounded up to 8) gets z
 * rounded to ``dtype`` for the backward of an activation.
 *
 * Backward: dz = dout act'(z); dx = dz W; dweight = dz^T x; dbias = column
 * sums of dz (in bias_dtype).  The residual's gradient is dout itself.  dz is
 * rounded to ``dtype`` when there is an activation.  NULL outputs are not
 * computed.  All sums are taken in a fixed order.
 */
#define OW_ACT_NONE 0
#define OW_ACT_RELU 1
#define OW_ACT_SILU 2
#define OW_ACT_GELU 3 /* z Phi(z), by erf */
typedef struct ow_linear_t {
  int64_t rows;
  int32_t in_features, out_features;
  int32_t dtype, activation;
  const void* x;
  int64_t ldx;
  const void* weight;
  int64_t ldw;
  const void* bias;
  int32_t bias_dtype;
  const void* residual;
  int64_t ldr;
  void* out;
  void* z;
  void* workspace;             /* ow_linear_workspace_size() bytes */
  size_t workspace_bytes;
} ow_linear_t;

typedef struct ow_linear_grads_t {
  const void* dout;            /* [rows, out_features] contiguous */
  void* dx;                    /* [rows, in_features] contiguous, or NULL */
  void* dweight;               /* [out_features, in_features] contiguous, or NULL */
  int32_t dweight_dtype;       /* dtype, or f32 */
  void* dbias;                 /* or NULL */
} ow_linear_grads_t;

/* Workspace bytes of the forward (grads NULL) or of the backward; reads the
 * shapes, dtypes, strides and pointers (their alignment).  0: invalid. */
OW_API size_t ow_linear_workspace_size(const ow_linear_t* args, const ow_linear_grads_t* grads);
OW_API int ow_linear_fwd(const ow_linear_t* args, void* stream);
OW_API int ow_linear_bwd(const ow_linear_t* args, const ow_linear_grads_t* grads, void* stream);

/*
 * Gated feed-forward block, for the 16-bit compute types:
 *
 *   g = x Wg^T + gate_bias;  u = x Wu^T + up_bias;  h = act(g) u
 *   out = h Wd^T + down_bias + residual
 *
 * x [rows, in_features] with row stride ldx, gate_weight and up_weight [hidden,
 * in_features] with row strides ldg and ldu, down_weight [out_features, hidden]
 * with row stride ldd, residual [rows, out_features] with row stride ldr, all of
 * ``dtype`` (bf16 or f16) with unit column stride; biases f32, bf16 or f16, or
 * NULL; out [rows, out_features] contiguous.  Sums and activation are f32.  h
 * [rows, ldh], ldh = hidden rounded up to 8, gets h rounded to ``dtype``; act and
 * slope (both NULL, or [rows, ldh]) act(g) and u act'(g), for the backward.
 *
 * Backward, from dout: NULL outputs are not computed; dgate_weight and dup_weight
 * come together, with one dtype.  h is needed for ddown_weight only, act, slope and
 * down_weight for all gradients but the projection back's.  dg and du are rounded
 * to ``dtype``, dh is not; dgate_bias and dup_bias are f32 sums of dg and du, rounded
 * unless dh's product is split.  In f16, act and slope end at its largest value.  All
 * sums are taken in a fixed order.
 */
typedef struct ow_ffn_t {
  int64_t rows;
  int32_t in_features, hidden, out_features;
  int32_t dtype, activation;
  const void* x;
  int64_t ldx;
  const void* gate_weight;
  int64_t ldg;
  const void* up_weight;
  int64_t ldu;
  const void* down_weight;
  int64_t ldd;
  const void* gate_bias;
  int32_t gate_bias_dtype;
  const void* up_bias;
  int32_t up_bias_dtype;
  const void* down_bias;
  int32_t down_bias_dtype;
  const void* residual;
  int64_t ldr;
  void* out;
  void* h;
  void* act;
  void* slope;
  void* workspace;             /* ow_ffn_workspace_size() bytes */
  size_t workspace_bytes;
} ow_ffn_t;

typedef struct ow_ffn_grads_t {
  const void* dout;            /* [rows, out_features] contiguous */
  void* dx;                    /* [rows, in_features] contiguous, or NULL, as the weights' and biases' */
  void* dgate_weight;
  int32_t dgate_dtype;         /* dtype, or f32 */
  void* dup_weight;
  int32_t dup_dtype;
  void* ddown_weight;
  int32_t ddown_dtype;
  void* dgate_bias;            /* of their biases' dtypes */
  void* dup_bias;
  void* ddown_bias;
} ow_ffn_grads_t;

/* Workspace bytes of the forward (grads NULL) or of the backward; reads the
 * shapes, dtypes, strides and pointers (their alignment).  0: invalid. */
OW_API size_t ow_ffn_workspace_size(const ow_ffn_t* args, const ow_ffn_grads_t* grads);
OW_API int ow_ffn_fwd(const ow_ffn_t* args, void* stream);
OW_API int ow_ffn_bwd(const ow_ffn_t* args, const ow_ffn_grads_t* grads, void* stream);

/*
 * Loss of a classifier that learns from a teacher's top logits and from labels.
 * logits [rows, classes] with row stride ld; a row has ``top`` entries of the
 * teacher, top_logits t_j for top_classes c_j (both [rows, top]), and a label.
 * With q_T = softmax(logits / T) and p = softmax(t / T) over the row's entries:
 *
 *   soft = T^2 sum_j p_j (log p_j - log q_T[c_j]);   hard = -log q_1[label]
 *
 * An entry whose class is negative is padding; a row without entries, or with
 * none above -inf, has no soft, one with a negative label no hard.  A class or
 * label that is not below ``classes`` makes its row NaN.  Entries may name a
 * class more than once.  reduction NONE: loss [rows] = weight soft + (1 - weight)
 * hard, a term that a row lacks being 0.  SUM: loss [1], the sum of these.  MEAN:
 * weight times the mean of soft over the rows that have one, plus (1 - weight)
 * times that of hard.  weight 0 leaves soft out, 1 hard.
 *
 * All in f32, sums over rows in f64, in a fixed order.  The forward leaves in
 * stats [5 rows] and factors [2] (not with NONE) what the backward takes, which
 * writes dlogits [rows, classes] of logits' dtype from dloss ([rows] with NONE,
 * else [1]).
 */
#define OW_REDUCE_NONE 0
#define OW_REDUCE_MEAN 1
#define OW_REDUCE_SUM 2
typedef struct ow_distill_t {
  int64_t rows;
  int32_t classes, top;        /* top at most 1024 */
  const void* logits;
  int32_t dtype;               /* f32, bf16 or f16 */
  int64_t ld;
  const void* top_logits;
  int32_t top_dtype;           /* f32, bf16 or f16 */
  const void* top_classes;
  int32_t class_bytes;         /* 4 or 8: of a signed integer */
  const void* labels;          /* [rows], or NULL */
  int32_t label_bytes;
  double temperature, weight;
  int32_t reduction;
  float* loss;                 /* forward only */
  float* stats;
  float* factors;
  void* workspace;             /* forward only: ow_distill_workspace_size() bytes */
  size_t workspace_bytes;
} ow_distill_t;

typedef struct ow_distill_grads_t {
  const float* dloss;
  void* dlogits;
} ow_distill_grads_t;

/* Workspace bytes of ow_distill_fwd (0 if the arguments are invalid). */
OW_API size_t ow_distill_workspace_size(const ow_distill_t* args);
OW_API int ow_distill_fwd(const ow_distill_t* args, void* stream);
OW_API int ow_distill_bwd(const ow_distill_t* args, const ow_distill_grads_t* grads, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* OMNIWAVE_B200_H */
