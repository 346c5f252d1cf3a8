/*
 * libmixmoe -- MI355X (gfx950) executor for mixlab's MoE feed-forward op
 * (IR op 74, OP_MOE_FEED_FORWARD).
 *
 * This is the C ABI that replaces, for op 74 only, the path
 *   gpu/lower.go:117-170 (LowerIRProgram)  ->  mlx_ir_program_create/add_op
 *   gpu/mlx_bridge.h:83-90                  ->  mlx_ir_eval_program_named_outputs
 *   gpu/mlx_bridge.h:172-181                ->  ir_interpret_outputs
 *   gpu/ir.cpp:4816-4824 (case OP_MOE_FEED_FORWARD) -> moe_feed_forward
 *   gpu/ir.cpp:1073-1164.
 * The op keeps the reference encoding (arch/ir.go:692-698):
 *   IntParams   = [B, T, D, E, topK, expertType, ffn, activation]
 *   FloatParams = [leakySlope]
 *   Inputs      = [x, router_w, then per expert (gate, up, down) or (up, down)]
 *   Outputs     = [delta [B*T, D] fp32, aux [1] fp32, entropy [1] fp32]
 *
 * Conventions follow gpu/mlx_bridge.h: opaque int64 handles with 0 meaning
 * failure (gpu/mlx_bridge.h:70-83), int status codes (gpu/mlx_bridge.cpp:
 * 814-823): 0 = OK, -10 = an argument the call cannot accept (shape, dtype,
 * index, size limit, NULL pointer), -11 = the HIP runtime or device could not
 * be initialised, -12 = not a live op handle, -1 = any other failure (a HIP
 * error, a call out of sequence); no C++ exception ever crosses the
 * boundary (gpu/mlx_bridge.cpp:64-82): the message of the last failure on the
 * calling thread is available from mxm_last_error.  Tensor dtype codes extend
 * mlx_tensor_input's (0 = int32, 1 = float32; gpu/mlx_bridge.h:92-99).
 *
 * Every call on one op handle is serialised by the caller (one HIP stream per
 * handle); distinct handles are independent.
 */
#ifndef MIXMOE_H
#define MIXMOE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MXM_OK 0
#define MXM_ERR -1       /* HIP error, call out of sequence */
#define MXM_ERR_ARGS -10 /* gpu/mlx_bridge.cpp:814-815: argument error */
#define MXM_ERR_INIT -11 /* gpu/mlx_bridge.cpp:818-819: runtime / device not initialised */
#define MXM_ERR_OP -12   /* gpu/mlx_bridge.cpp:821-822: bad op handle */

#define MXM_DTYPE_INT32 0 /* gpu/mlx_bridge.h:94 */
#define MXM_DTYPE_F32 1   /* gpu/mlx_bridge.h:94 */
#define MXM_DTYPE_BF16 2  /* compute_dtype "bf16" (gpu/ir_trainer.cpp:1395-1412) */
#define MXM_DTYPE_I8 3    /* symmetric int8 weights with fp32 per-output-channel scales */

#define MXM_OP_MOE_FEED_FORWARD 74 /* arch/ir.go:67, gpu/ir.h:81 */

/* mxm_moe_create flags */
#define MXM_FLAG_FORCE_SIMT 1 /* use the exact-order SIMT expert kernels even where MFMA tiles fit */
#define MXM_FLAG_DEBUG_PROBS 2 /* keep the router probabilities of the last forward */
/* MFMA tile family (bits 2-3); 0 picks 256x256 where the dimensions allow,
 * else 128x128 */
#define MXM_FLAG_MFMA_TILE128 4       /* 128 x 128 x 64 tiles, 4 waves, 2 LDS stages */
#define MXM_FLAG_MFMA_TILE256x128 8   /* 256 x 128 x 32 tiles, 4 waves, 3 LDS stages */
#define MXM_FLAG_MFMA_TILE256x256 12  /* 256 x 256 x 64 tiles, 8 waves, 2 LDS stages */
#define MXM_FLAG_MFMA_TILE_MASK 12
#define MXM_FLAG_INT8_WEIGHTS 16 /* expert weights are int8 + per-output-channel scales
                                    (mxm_moe_set_input_q8); bf16 compute */
/* Each mxm_moe_forward keeps the op's own copy of x, its routing and router
 * probabilities and, where the backward runs in bf16 (bf16 compute on the
 * MFMA family, D a multiple of 128), its raw up projections, for
 * mxm_moe_backward_kept: the backward of that forward,
 * which then does not run the forward again, as the reference's autodiff
 * keeps the forward's values for its backward.  No counterpart flag in the
 * reference (its graph keeps them implicitly). */
#define MXM_FLAG_KEEP_FOR_BACKWARD 32

/* Stages timed by mxm_moe_stage_times, in launch order.  ROUTER includes the
 * zero-padded copy of x where D is not a multiple of 64 (the router reads it);
 * SCAN is the dispatch (counts, offsets, permutation, aux and entropy) of the
 * tiled router's batches, all of it: SCATTER has no launch of its own and times
 * an empty gap. */
#define MXM_STAGE_ROUTER 0
#define MXM_STAGE_SCAN 1
#define MXM_STAGE_SCATTER 2
#define MXM_STAGE_GEMM_UP 3
#define MXM_STAGE_GEMM_DOWN 4
#define MXM_STAGE_COMBINE 5
#define MXM_NUM_STAGES 6

/* Initialise the HIP runtime on the current device.  Replaces mlx_init
 * (gpu/mlx_bridge.h:15).  0 on success, MXM_ERR_INIT on failure. */
int mxm_init(void);

/* Device name ("AMD Instinct MI355X ..."); replaces mlx_device_name
 * (gpu/mlx_bridge.h:53).  Never NULL. */
const char* mxm_device_name(void);

/* Copy the last failure message of the calling thread into buf (NUL
 * terminated, truncated to n bytes).  Returns the full message length.
 * Replaces the stderr logging of log_bridge_exception
 * (gpu/mlx_bridge.cpp:80-82). */
int mxm_last_error(char* buf, int n);

/* Device memory for callers that hold inputs and outputs in HBM (the cgo
 * side keeps these instead of MLX array handles, gpu/mlx_bridge.h:70-80). */
int mxm_malloc(void** ptr, int64_t bytes);
int mxm_free(void* ptr);
int mxm_memcpy_h2d(void* dst, const void* src, int64_t bytes);
int mxm_memcpy_d2h(void* dst, const void* src, int64_t bytes);
int mxm_memcpy_d2d(void* dst, const void* src, int64_t bytes);
int mxm_device_synchronize(void);

/* Create an op-74 executor.  Replaces mlx_ir_program_create(n_weights) +
 * mlx_ir_program_add_op(prog, 74, ...) (gpu/mlx_bridge.h:83-90) for one MoE
 * op.  int_params/float_params are the op's IntParams/FloatParams
 * (arch/ir.go:697); n_inputs is len(Op.Inputs).  Parameter checks and their
 * messages are those of gpu/ir.cpp:1076-1104.  compute_dtype is
 * MXM_DTYPE_F32 or MXM_DTYPE_BF16 (weights are cast to it, as
 * gpu/ir_trainer.cpp:1395-1412 does).  Returns a handle, 0 on failure. */
int64_t mxm_moe_create(const float* float_params, int n_float_params, const int32_t* int_params,
                       int n_int_params, int n_inputs, int compute_dtype, int flags);

/* Release an executor and its device memory; replaces
 * mlx_ir_program_destroy + mlx_free_handles (gpu/mlx_bridge.h:79-90). */
int mxm_moe_destroy(int64_t op);

/* Bind weight input `input_index` (position in Op.Inputs: 1 = router_w
 * [D, E], then expert e's matrices at 2 + e*wpe + j, in x.W layout
 * [in, out] as arch/moe.go:126-142 declares them).  dtype is MXM_DTYPE_F32
 * or MXM_DTYPE_BF16; data is host memory (on_device = 0) or device memory
 * (on_device = 1), copied and converted, so the caller keeps ownership.
 * Replaces mlx_from_data_shape (gpu/mlx_bridge.h:71) plus the w<i> name
 * lookup of gpu/ir.cpp:3730-3734; shape checks and messages are those of
 * gpu/ir.cpp:1098-1140. */
int mxm_moe_set_input(int64_t op, int input_index, int dtype, const int64_t* shape, int ndim,
                      const void* data, int on_device);

/* Bind expert weight input `input_index` (2 + e*wpe + j, as for
 * mxm_moe_set_input) as symmetric int8: q [in, out] in x.W layout and fp32
 * scales [out], i.e. W = q * scales[None, :] (per output channel).  Only for
 * ops created with MXM_FLAG_INT8_WEIGHTS.  This has no counterpart in the
 * reference, whose bridge takes fp32 weights only (gpu/mlx_bridge.cpp:210-217);
 * it serves decode-shaped serving, where the expert weights are the traffic.
 * Any D and ffn (widths that are not multiples of 64 are padded with zero
 * weights inside the library; one expert's matrix below 2^31 entries).  An
 * op whose batch routes 96 or more rows per expert (B*T*topK >= 96*E), which
 * is compute-bound, keeps the integers as bf16 (exact; twice the int8
 * bytes) for the bf16 MFMA tiles, which apply the scales to the fp32
 * accumulators: the same products and activation as the int8 kernels. */
int mxm_moe_set_input_q8(int64_t op, int input_index, const int8_t* q, const float* scales,
                         const int64_t* shape, int ndim, int on_device);

/* Run the op on x [rows = B*T, D] (dtype MXM_DTYPE_BF16 or MXM_DTYPE_F32;
 * fp32 x is rounded to bf16 first under bf16 compute), writing delta
 * [rows, D] fp32, aux [1] fp32 and entropy [1] fp32.  All pointers are
 * device memory; the call is asynchronous on the op's stream.  aux and
 * entropy may be NULL.  Replaces the case OP_MOE_FEED_FORWARD dispatch
 * (gpu/ir.cpp:4816-4824) of moe_feed_forward (gpu/ir.cpp:1073-1164).
 * A row whose logits are not finite (a NaN or infinity in x or router_w)
 * gets NaN probabilities and gates and still picks K distinct experts
 * (the lowest ids), so the dispatch of every other row is unaffected. */
int mxm_moe_forward(int64_t op, const void* x, int x_dtype, int64_t rows, float* delta,
                    float* aux, float* entropy);

/* Same with host buffers; synchronous (copies in, runs, copies out).  This
 * is the shape of mlx_ir_eval_program_named_outputs (gpu/mlx_bridge.h:172-181)
 * for the three outputs of op 74. */
int mxm_moe_forward_host(int64_t op, const void* x, int x_dtype, int64_t rows, float* delta,
                         float* aux, float* entropy);

/* Device scratch of mxm_moe_forward_noalloc, per GPU (64 MiB). */
#define MXM_NOALLOC_MAX_BYTES (64ll << 20)

/* mxm_moe_forward that allocates nothing.  It has no counterpart in the
 * reference: it is for callers that cannot call hipMalloc -- code under HIP
 * graph capture, tight serving loops, harnesses that forbid allocation.
 * Every buffer the forward writes besides its outputs (routing, dispatch,
 * H, Y) lives in one file-scope device array per GPU of
 * MXM_NOALLOC_MAX_BYTES, held until the process ends; an op whose workspace
 * is larger is rejected with an error.  Same arguments, kernels and results
 * as mxm_moe_forward (device pointers, asynchronous on the op's stream).
 * All calls on one GPU share that array: calls that overlap on one GPU (two
 * streams, two threads) race; each call leaves it ready for the next.  Call
 * mxm_init on each device before capturing (it looks up and clears the
 * array).  After this call mxm_moe_routing reads the array, which the next
 * no-allocation call on that GPU overwrites. */
int mxm_moe_forward_noalloc(int64_t op, const void* x, int x_dtype, int64_t rows, float* delta,
                            float* aux, float* entropy);

/* The whole MoE block of arch/moe.go:152-213 (emitMoEIR + emitMoEDeltaIR):
 *   xn     = RMSNorm(x, norm_scale, eps)        gpu/ir.cpp:4949-4960 (OP_RMSNORM)
 *   (delta, aux_raw, entropy) = op 74 on xn     gpu/ir.cpp:1073-1164
 *   delta *= moe_scale   (when moe_scale != NULL; block scales, arch/moe.go:199-204)
 *   x_out  = x + delta                          (the residual Add, arch/moe.go:164)
 *   aux    = aux_weight * aux_raw               (ScalarMul, arch/moe.go:197)
 * x [rows, D] is bf16 bits or fp32 (x_dtype); norm_scale and moe_scale [D]
 * have scale_dtype (fp32 or bf16 bits); x_out [rows, D], aux and entropy are
 * fp32.  xn is computed in the op's compute dtype.  The emitter uses
 * eps = 1e-5 and aux_weight = the block's effective load_balance_loss_weight.
 * Dropout (training only) is not applied.  Replaces the four IR ops the
 * emitter produces for one block (RMSNorm, op 74, ScalarMul, Add); device
 * pointers, asynchronous on the op's stream. */
int mxm_moe_block_forward(int64_t op, const void* x, int x_dtype, int64_t rows,
                          const void* norm_scale, const void* moe_scale, int scale_dtype, float eps,
                          float aux_weight, float* x_out, float* aux, float* entropy);

/* Same with host buffers; synchronous. */
int mxm_moe_block_forward_host(int64_t op, const void* x, int x_dtype, int64_t rows,
                               const void* norm_scale, const void* moe_scale, int scale_dtype,
                               float eps, float aux_weight, float* x_out, float* aux,
                               float* entropy);

/* Backward of op 74 (the gradients MLX's autodiff takes through
 * gpu/ir.cpp:1073-1164; the reference exercises them in
 * gpu/moe_feed_forward_test.go:84-151), computed in fp32.  Under bf16 compute
 * it uses the bf16 flow's values (x and weights rounded to bf16, the
 * forward's bf16 expert outputs); int8-weight ops have no backward.  Given
 * x [rows, D] (fp32, or bf16 bits under bf16 compute) and the upstream
 * gradients d_delta [rows, D] fp32, d_aux and
 * d_entropy (scalars), runs the forward on x (routing held fixed, as top-k
 * indices carry no gradient) and writes dx [rows, D], d_router_w [D, E] and
 * d_experts: the expert weight gradients in Op.Inputs order (per expert
 * w_gate, w_up, w_down -- or w_up, w_down -- each in x.W layout, as
 * mxm_moe_set_input takes them).  Device pointers; the call is asynchronous
 * on the op's stream (every expert product is a ragged grouped product whose
 * row ranges come from the device-side routing).  Under fp32 compute each
 * expert product runs as a bf16 MFMA product over the operands' hi / lo
 * planes (hi = bf16(v), lo = bf16(v - hi); about 2^-16 relative).  The first
 * call allocates the backward's workspace (on MI355X, 128 MiB of it holds the
 * weight gradients' split-reduction partials). */
int mxm_moe_backward(int64_t op, const void* x, int x_dtype, int64_t rows, const float* d_delta,
                     float d_aux, float d_entropy, float* dx, float* d_router_w, float* d_experts);

/* The backward of the op's last call, which must be an mxm_moe_forward on
 * an op created with MXM_FLAG_KEEP_FOR_BACKWARD: the gradients at the x that
 * forward read (the op kept its own copy, so the caller's buffer may have
 * changed since), from the routing and projections it kept.  Outputs as
 * mxm_moe_backward's.  Any other call that runs the op -- another forward
 * (plain, host, no-allocation or block), a backward -- or a weight update
 * with mxm_moe_set_input[_q8] drops the kept forward; without one this
 * returns MXM_ERR.  Replaces the backward half of the trainer's
 * value_and_grad over the graph (gpu/ir_trainer.cpp:2790-2816), which
 * differentiates the forward it just ran. */
int mxm_moe_backward_kept(int64_t op, const float* d_delta, float d_aux, float d_entropy, float* dx,
                          float* d_router_w, float* d_experts);

/* Same with host buffers; synchronous. */
int mxm_moe_backward_host(int64_t op, const void* x, int x_dtype, int64_t rows,
                          const float* d_delta, float d_aux, float d_entropy, float* dx,
                          float* d_router_w, float* d_experts);

/* Wait for all work queued on the op's stream. */
int mxm_moe_synchronize(int64_t op);

/* Routing of the last forward (synchronous copy): top_idx [rows, K] int32
 * (argsort(-probs)[:, :K], gpu/ir.cpp:1108-1109), gates [rows, K] fp32
 * (top_norm, gpu/ir.cpp:1110-1111), counts [E], offsets [E+1] and perm
 * [rows*K] (expert-grouped token ids).  Any pointer may be NULL.  to_host
 * selects host (1) or device (0) destinations.  A forward of the decode
 * flow (mxm_moe_info entry 7) computes only the per-token picks and
 * gates; this call then computes counts, offsets and perm from them on the
 * device first (the same tables, bit for bit). */
int mxm_moe_routing(int64_t op, int32_t* top_idx, float* gates, int32_t* counts,
                    int32_t* offsets, int32_t* perm, int to_host);

/* Router probabilities [rows, E] of the last forward; requires
 * MXM_FLAG_DEBUG_PROBS.  Host destination. */
int mxm_moe_probs(int64_t op, float* probs);

/* Per-stage HIP-event timing on the op's stream.  mxm_moe_set_profiling
 * (re)starts a recording: every later forward records events between its
 * kernels (enable = 0 stops it).  With enable = R > 1 each stage is launched
 * R times between its events (the stages are idempotent, so outputs are
 * unchanged), which times short kernels without the events' own gaps.
 * mxm_moe_stage_times waits for the recorded forwards and writes the mean
 * duration of one launch of each of the MXM_NUM_STAGES stages in
 * milliseconds; it returns the number of forwards averaged (> 0) or an error
 * code. */
int mxm_moe_set_profiling(int64_t op, int enable);
int mxm_moe_stage_times(int64_t op, float* ms, int n);

/* Executor facts: info[0] = expert kernel family (0 SIMT, 1 bf16 MFMA, 2 int8
 * weights on the int8 kernels, 3 int8 weights on the bf16 MFMA tiles: the
 * integers as bf16, the scales applied to the fp32 accumulators, for batches
 * past the decode sizes, 4 bf16 MFMA family whose forwards stream the
 * weights through the decode kernels: bf16 ops at decode sizes with fewer
 * than 96 routed rows per expert, not created with
 * MXM_FLAG_KEEP_FOR_BACKWARD; they hold the weights in both layouts, and
 * their backward runs on the tiles), info[1] = workspace bytes, info[2] = row-tile
 * height that the up projection's kernel runs most rows at, info[3] = number of router tiles, info[4] = the
 * expert width the kernels run at (ffn, or ffn rounded up to the tiles: 128
 * for MFMA, 64 for the int8 kernels, with zero weights in the padding),
 * info[5] = the down
 * projection's output width (D, or D rounded up to 128 / 16), info[6] = the
 * up projection's reduction length (D, or D rounded up to 64), info[7] = how
 * the last forward routed: 0 the tiled router and the dispatch (two launches,
 * three for many tiles), 1 the one-launch router (a workgroup per token, or per
 * four past 256, the dispatch in its last workgroup), 2 the decode flow of the decode kernels (int8, or
 * bf16 streamed: the one-launch router's per-token results only; the expert
 * kernels find their rows from the top-k picks), -1 no forward yet.  Returns the number of entries written (at most
 * n, at most 8). */
int mxm_moe_info(int64_t op, int64_t* info, int n);

/* ---- around the op's training step ----
 *
 * The handles below run on a stream of their own, or on that of another live
 * handle (`stream_of`: an op or any of these; 0: a new
 * stream on the current device).  Handles that share a stream run in call
 * order without any wait on the host, so a block's norms, its op and its
 * optimizer go on one stream; work on another stream is ordered by the caller
 * (mxm_stream, mxm_synchronize).  The stream lives as long as its last handle.
 * Calls on one handle are serialised by the caller, as an op's are; calls on
 * handles that share nothing but the stream may come from several threads.
 * Every call is asynchronous and runs on the handle's device, whichever device
 * is current.  Tensors are contiguous device memory aligned to their elements.
 * After creation (and mxm_grads_bind) no call allocates or waits, so all of
 * them can be captured into a HIP graph on the handle's stream; the scalars
 * given by value (rows, lr, max_norm, ...) are then the captured ones.  A
 * handle's workspace is its own: two graphs captured from one handle must not
 * run at once, and none runs after the handle's destruction.  None of this has a counterpart in the reference's bridge,
 * whose graph compiler fuses such work itself. */

/* Residual norm: what stands between a block's branch and the next block.
 * Row n, channel d; x the residual stream, delta the branch's output:
 *   z = delta / sqrt(mean_d(delta^2) + eps) with MXM_RESNORM_POST_NORM, else delta
 *   h = x + gate[n / gateRows] * branch_scale * post_scale * z
 *   y = norm_scale * h / sqrt(mean_d(h^2) + eps)    with MXM_RESNORM_NORM
 * (moe_scale and the residual Add of arch/moe.go:199-204, :164, and the RMSNorm
 * of gpu/ir.cpp:4949-4960, in one pass).  y is computed from h as it is kept,
 * i.e. after h's rounding to the stream's type; sums are in fp32, so a row's
 * squares have to add up to less than 3.4e38. */
#define MXM_RESNORM_BRANCH 1       /* h = x + ...; without it h is x itself */
#define MXM_RESNORM_POST_NORM 2    /* the branch is normalised first */
#define MXM_RESNORM_NORM 4         /* the sum is normalised: y */
#define MXM_RESNORM_GATE_SIGMOID 8 /* the gate is the sigmoid of what is given */
#define MXM_RESNORM_BACKWARD 16    /* the handle also runs backward (holds its workspace) */
#define MXM_RESNORM_MAX_D 16384
#define MXM_GATE_NONE 0
#define MXM_GATE_ROW 1     /* gate [ceil(rows / gateRows)] */
#define MXM_GATE_CHANNEL 2 /* gate [ceil(rows / gateRows)][D] */

/* params = [D, maxRows, streamDtype, branchDtype, outDtype, scaleDtype,
 * gradDtype, flags, gate, gateRows]; dtypes are MXM_DTYPE_F32 or
 * MXM_DTYPE_BF16: x and h, delta, y, the scales and the gate, and the gradients
 * dh, dy, dx and d_delta.  Returns a handle, 0 on failure. */
int64_t mxm_resnorm_create(const int64_t* params, int n_params, float eps, int64_t stream_of);
int mxm_resnorm_destroy(int64_t h);

/* h and y for rows <= maxRows rows (rows behind them are left as they were).
 * Scales may be NULL (ones).  h or y may be x or delta where the types agree, or
 * one buffer, which then holds y; any other overlap of an output with a tensor of
 * the call is refused.
 * delta, h and gate are ignored without a branch or gate, y without a norm. */
int mxm_resnorm_forward(int64_t handle, int64_t rows, const void* x, const void* delta,
                        const void* post_scale, const void* branch_scale, const void* gate,
                        const void* norm_scale, void* h, void* y);

/* Gradients at the forward's h (x for a handle without a branch) and delta,
 * for upstream gradients dh and dy.  With a norm dh may be NULL (zeros), without
 * one dy is ignored and dx, which then equals dh, may be NULL.  dx or d_delta may
 * be any of h, delta, dh and dy where the types agree, or one buffer, which then
 * holds d_delta, and the gradient of an fp32 scale or gate may take its place; any
 * other overlap of an output is refused.  The scales' and the gate's gradients are fp32 (overwritten, not added to; NULL:
 * not computed), summed in a fixed order: equal inputs give equal bits. */
int mxm_resnorm_backward(int64_t handle, int64_t rows, const void* h, const void* delta,
                         const void* post_scale, const void* branch_scale, const void* gate,
                         const void* norm_scale, const void* dh, const void* dy, void* dx,
                         void* d_delta, float* d_post_scale, float* d_branch_scale, float* d_gate,
                         float* d_norm_scale);

/* Gradient set: n tensors of sizes[i] elements whose gradients are dtypes[i]
 * (MXM_DTYPE_F32 or MXM_DTYPE_BF16); decay[i] multiplies the weight decay of
 * tensor i (NULL: 1 each).  Returns a handle, 0 on failure. */
int64_t mxm_grads_create(const int64_t* sizes, const int32_t* dtypes, const float* decay, int n,
                         int64_t stream_of);
int mxm_grads_destroy(int64_t h);

/* Where the tensors are: host arrays of n device pointers (any value for a tensor
 * of no elements).  clipped (the type of the gradients) is where mxm_grads_clip
 * writes, NULL or the gradient's own pointer: in place.  params, m and v (fp32)
 * are AdamW's, all or none; params_bf16, or NULL, gets the updated params
 * rounded to bf16.  No two of the tensors may overlap.  Waits for the handle's stream; calls use the
 * pointers bound last, those captured into a graph too (a captured mxm_grads_adamw
 * that runs while no params are bound updates nothing and sets *skipped to 1). */
int mxm_grads_bind(int64_t h, const void* const* grads, void* const* clipped, void* const* params,
                   void* const* m, void* const* v, void* const* params_bf16);

/* norm [1] fp32 = sqrt(sum of squares over all tensors), summed in 64 bits in a
 * fixed order; infinite where it is past fp32's largest value.  The two calls
 * below go by this fp32 value. */
int mxm_grads_norm(int64_t h, float* norm);

/* clipped = g * min(1, max_norm / (norm + 1e-6)), a factor in fp32; where the norm
 * is not finite the gradients are copied as they are.  norm may be NULL. */
int mxm_grads_clip(int64_t h, double max_norm, float* norm);

/* One AdamW step on the clipped gradients (max_norm 0: not clipped), which are
 * not written back: with t = ++*step (device memory; below 0 taken as 0)
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
 *   p -= lr weight_decay decay[i] p + lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)
 * A gradient norm that is not finite leaves params, m, v, the bf16 copies and
 * *step as they were (gpu/optimizer_step_guard.h:12-71 rejects such a step) and
 * sets *skipped to 1, else to 0.  norm and skipped may be NULL. */
int mxm_grads_adamw(int64_t h, double lr, double beta1, double beta2, double eps,
                    double weight_decay, double max_norm, int64_t* step, float* norm,
                    int32_t* skipped);

/* ---- the vocabulary's two ends of a training step ----
 *
 * Handles as the residual norm's and the gradient set's above: shared streams,
 * asynchronous calls without allocation or waiting (all can be captured), contiguous
 * device tensors aligned to their elements, a workspace that is the handle's own.
 * None is created on a stream that is being captured.
 * An output may not overlap any other tensor of its call.  Every sum is taken in
 * an order that the call's sizes and whole-number inputs decide: equal inputs give
 * equal bits. */
#define MXM_VOCAB_MAX 4194304

/* Token embedding: out[n] = scale * table[tokens[n]], n < rows, for a table [V, D];
 * a token outside [0, V) gives a row of zeros.
 * params = [V, D, maxRows, tableDtype, outDtype, gradDtype, tableGradDtype, flags];
 * dtypes (MXM_DTYPE_F32 or MXM_DTYPE_BF16) are those of table, out, d_out and
 * d_table.  D is at most MXM_RESNORM_MAX_D, V at most MXM_VOCAB_MAX.  Returns a
 * handle, 0 on failure. */
#define MXM_EMBED_BACKWARD 1 /* the handle also runs backward (holds its workspace) */
int64_t mxm_embed_create(const int64_t* params, int n_params, float scale, int64_t stream_of);
int mxm_embed_destroy(int64_t h);

/* tokens [rows] int32, rows <= maxRows; rows of out behind them are left as they were. */
int mxm_embed_forward(int64_t h, int64_t rows, const int32_t* tokens, const void* table, void* out);

/* d_table[v] = scale * sum of d_out[n] over the n with tokens[n] = v, for every v
 * (zeros where there is none); with accumulate the sums are added to d_table, and
 * the rows of tokens that do not occur are left as they were (a table tied to a
 * token loss: its dw first).  Sums in fp32, one rounding.  d_out's rows of tokens
 * outside [0, V) are not read. */
int mxm_embed_backward(int64_t h, int64_t rows, const int32_t* tokens, const void* d_out,
                       void* d_table, int accumulate);

/* Token loss: softmax cross entropy of hidden rows x [rows, D] against a table
 * weight [V, D] (the embedding's, where they are tied), without keeping the logits
 * of more than a piece of the rows.  A row takes part where its target is in [0, V)
 * and its weight is not 0; of any other row nothing else is read, and its loss, lse
 * and dx are 0.
 *   l = x . weight[v]                      with a softcap: softcap * tanh(l / softcap)
 *   lse[n] = log sum_v exp(l[v]),  loss[n] = lse[n] - l[targets[n]]
 *   total = sum of row_weights[n] * loss[n]    MXM_XENT_MEAN: / sum of row_weights[n]
 * over the rows that take part (0 where none does).
 * params = [V, D, maxRows, dtype, dxDtype, dwDtype, flags]; dtype is that of x and
 * weight.  Under bf16 the products are exact and summed in fp32, and the backward
 * rounds the logits' gradient to bf16 before the products with it (from fp16: what is
 * below 2^-29 of a row's largest keeps fewer bits, below 2^-39 of it none).  Under fp32 a
 * row's elements keep 22 bits down to 2^-17 of its largest and 2^-40 of it below,
 * and so does a row's gradient of the logits (under a softcap, of what it is before
 * the cap's slope); the dw of an entry whose gradient is 2^-k of every row's largest
 * keeps 36 - k bits at least, of 22.  An entry (row of weight) that minus infinity or the type's
 * lowest value keeps from coming has no share in any result (but that dx of a bf16
 * table with infinities is not a number, 0 times those; under fp32 the logit of an
 * entry with infinities has the sign of their sum times x, and is 0 where that is 0);
 * as a target it makes the loss infinite (or as large), and then dx and dw are of no
 * use.  A row of x that is not finite spoils its own results and dw.  softcap is
 * 0 (none) or in [1/64, 1024]; capped logits are off by a few 2^-24 of it, and minus
 * infinity is -softcap under it.  Returns a handle, 0 on failure. */
#define MXM_XENT_MEAN 1
#define MXM_XENT_BACKWARD 2 /* the handle also runs backward (holds its workspace) */
int64_t mxm_xent_create(const int64_t* params, int n_params, float softcap, int64_t stream_of);
int mxm_xent_destroy(int64_t h);

/* targets [rows] int32, row_weights [rows] fp32 or NULL (ones); loss and lse [rows]
 * and total [1] fp32, each NULL where it is not wanted, not all of them. */
int mxm_xent_forward(int64_t h, int64_t rows, const void* x, const void* weight,
                     const int32_t* targets, const float* row_weights, float* loss, float* lse,
                     float* total);

/* The forward and the gradients of d_total * total: dx [rows, D] and dw [V, D]
 * (overwritten), either NULL where it is not wanted.  loss, lse and total may all be
 * NULL.  It runs the forward on what it is given: no mxm_xent_forward before it. */
int mxm_xent_backward(int64_t h, int64_t rows, const void* x, const void* weight,
                      const int32_t* targets, const float* row_weights, float d_total, float* loss,
                      float* lse, float* total, void* dx, void* dw);

/* The hipStream_t that a handle (an op's too) runs on, to order other work with
 * it or to capture its calls. */
int mxm_stream(int64_t handle, void** stream);
/* Wait for all work queued on a handle's stream. */
int mxm_synchronize(int64_t handle);

#ifdef __cplusplus
}
#endif

#endif /* MIXMOE_H */
