// Kernels around the MoE op's training step and its residual stream: the
// residual norm (mxm_resnorm.hip) and the gradient set's norm, clipping and
// AdamW step (mxm_optim.hip).  mxm_train.hip owns every buffer; these structs
// carry raw device pointers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxm_numerics.h"

// ---- residual norm ----
//
// Row n, channel d; stream x, branch delta, all sums in fp32:
//   rp = 1 / sqrt(mean_d(delta^2) + eps)           (post norm; else 1)
//   z = delta * rp,  f = scale * post,  a = gate or sigmoid(gate) of row n / gate_rows
//   h = x + a * f * z                              rounded to the stream's type
//   rn = 1 / sqrt(mean_d(h^2) + eps),  y = h * rn * w     of the rounded h
// and backwards, given dh and dy:
//   u = w * dy,  hn = rn * h,  t = dh + rn * (u - hn * mean_d(u * hn))
//   dx = t,  dw = sum_n dy * hn
//   e = t * a * f,  d_delta = rp * (e - z * mean_d(e * z))               (post norm; else e)
//   q = t * z,  d_scale = post * sum_n a q,  d_post = scale * sum_n a q,
//   d_gate = a' * sum over the gate's rows (and over d, for a gate per row) of f q
struct ResNormArgs {
  int N, D;
  float eps, inv_d;                     // inv_d = (float)(1.0 / D)
  bool branch, post_norm, norm, sigmoid;
  bool x_bf16, delta_bf16, y_bf16, p_bf16, g_bf16;  // stream, branch, y, scales and gate, gradients
  int gate;                             // 0 none, 1 one value per row, 2 one per channel
  int gate_rows;                        // rows of x per row of the gate
  const void *x, *delta;                // [N, D]; x unused backwards
  const void *post, *scale, *w, *gatep; // [D] each (null: ones), gate [ceil(N / gate_rows)][1 or D]
  void* h;                              // [N, D]: out forwards, in backwards
  void* y;                              // [N, D]
  // backward
  const void *dh, *dy;                  // [N, D]; dh null: zeros
  void *dx, *d_delta;                   // [N, D]
  float *d_post, *d_scale, *d_w, *d_gate;  // null: not wanted
  // Column sums go over chunks of rows, one a row's threads; a workgroup's chunks
  // make a part: part [2][parts][D] (w, then a q) and, for gates whose rows span
  // several parts, gate_part [parts][1 or D].  Set by the launcher.
  float *part, *gate_part;
  int chunks, parts, chunk_rows;   // (forwards chunk_rows: rows a thread walks)
  int group_chunks, group_parts;   // per group of gate rows, each within one; 0: whole groups
  int max_parts;                   // that part and gate_part have room for
  int n_cu;
};
void mxm_launch_resnorm(const ResNormArgs& a, hipStream_t s);
// false, and no launch, where max_parts is too few.
bool mxm_launch_resnorm_bw(const ResNormArgs& a, hipStream_t s);
// Most parts of any backward of up to max_rows rows; bf16: stream and gradients;
// groups: of several rows per row of the gate.
int64_t mxm_resnorm_max_parts(int64_t max_rows, int D, bool bf16, bool groups, int n_cu);

// ---- gradient sets ----
// A piece of one tensor, with where it is (a launch reads one descriptor and
// then the data).
struct GradChunk {
  const void* g;      // gradients, fp32 or bf16
  void* clipped;      // where clip writes (g itself: in place)
  float *p, *m, *v;
  uint16_t* p16;      // bf16 copy of p, or null
  int32_t count;      // elements
  float decay;        // multiplies the call's weight decay
  int64_t bf16;       // the gradients' type
};
// What the norm leaves for the launches after it.
struct GradScalars {
  float coef;         // multiplies every gradient
  float step_size;    // lr / (1 - beta1^t)
  float root2;        // 1 / sqrt(1 - beta2^t)
  int32_t skip;       // the norm is not finite, or no params are bound
};
struct GradArgs {
  const GradChunk* chunks;
  int n_chunks;
  int chunk_elems;       // elements of a chunk (a tensor's last one may be shorter)
  bool all_bf16;         // every tensor's gradients are bf16
  int keep_from;         // (set by the norm's launcher) chunks from here on stay in the caches
  int slices;            // workgroups per chunk, and the one that a launch's first
  int first_slice;       // workgroup takes (set by the launchers of clip and AdamW)
  double* partial;       // [n_chunks or fewer]
  int32_t* ticket;       // zero between calls
  GradScalars* scalars;
  double max_norm;       // 0: no clipping
  float* norm;           // or null
  // AdamW
  bool adamw;
  int64_t* step;
  int32_t* skipped;      // or null
  // (in 64 bits: 1 - beta in 32 loses digits for beta next to 1)
  double lr, beta1, beta2, eps, weight_decay;
  float b1, c1, b2, c2, eps32, lr_decay;  // set by the launcher: c = 1 - b
};
int mxm_grad_chunk_elems(int64_t total, int n_cu);
int mxm_grad_norm_blocks(int n_chunks);
// again: a launch that reads the gradients again follows.
void mxm_launch_grad_norm(const GradArgs& a, bool again, hipStream_t s);
void mxm_launch_grad_clip(const GradArgs& a, hipStream_t s);
void mxm_launch_grad_adamw(const GradArgs& a, hipStream_t s);
