// Kernels at the vocabulary's two ends of a training step: the token embedding
// (mxm_embed.hip) and the token loss (mxm_xent.hip).  mxm_vocab.hip owns every
// buffer; these structs carry raw device pointers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxm_numerics.h"

// ---- token embedding ----
//
//   out[n] = scale * table[t_n]                            zeros for t_n outside [0, V)
//   d_table[v] = scale * sum over n with t_n = v of d_out[n]   (+ d_table[v]: accumulate)
// The backward sorts the tokens' places by token (equal ones by place), sums runs
// of equal tokens over chunks of sorted places and joins the runs that cross
// chunks, all in an order that the tokens alone decide.
struct EmbedArgs {
  int64_t rows;
  int V, D;
  float scale;
  bool table_bf16, out_bf16, grad_bf16, dtable_bf16, accumulate;
  const int32_t* tokens;  // [rows]
  const void* table;      // [V, D]
  void* out;              // [rows, D]
  const void* d_out;      // [rows, D]
  void* d_table;          // [V, D]
  // backward's workspace
  int2* sorted;           // [rows]: place, token
  int32_t* starts;        // [V + 1]: first sorted place of token v
  float* part;            // [chunks][2][D]: sums of runs that a chunk shares
  int64_t max_rows;
  int n_cu;
};
void mxm_launch_embed(const EmbedArgs& a, hipStream_t s);
void mxm_launch_embed_bw(const EmbedArgs& a, hipStream_t s);
// Most chunks of a backward of up to max_rows rows (part's first extent).
int64_t mxm_embed_max_chunks(int64_t max_rows);

// ---- token loss ----
//
// Rows n with a target t in [0, V) and a weight w_n that is not 0 take part:
//   z = x W^T,  l = cap tanh(z / cap)   (softcap; else z)
//   loss = log(1 + sum_{v != t} exp(l_v - l_t)),  lse = loss + l_t
//   total = sum_n w_n loss_n             (mean: / sum_n w_n)
//   g_n = d_total w_n                    (mean: / sum_n w_n)
//   dz = g (softmax(l) - [v = t]) (1 - (l / cap)^2),  dx = dz W,  dW = dz^T x
// Rows that take part are gathered (in order); the logits of a piece of them
// exist at a time.
struct XentArgs {
  int64_t rows;
  int V, D;
  float softcap;            // 0: none
  bool bf16;                // x and weight
  bool dx_bf16, dw_bf16, mean;
  float d_total;
  const void* x;            // [rows, D]
  const void* weight;       // [V, D]
  const int32_t* targets;   // [rows]
  const float* row_weights; // [rows] or null: ones
  float *loss, *lse;        // [rows] or null
  float* total;             // [1] or null
  void *dx, *dw;            // [rows, D], [V, D], or null
  bool backward;
  // workspace
  int32_t* map;             // [rows] the rows that take part
  struct XentScalars* scalars;
  float* nll;               // [rows] loss of the rows that take part
  float* logits;            // [piece_rows][V]
  float* dw32;              // [V][D] or null: dw is fp32 itself
  int64_t piece_rows;
  int n_cu;
};
struct XentScalars {
  double weight_sum;        // of the rows that take part
  int32_t rows;             // that take part
};
void mxm_launch_xent(const XentArgs& a, hipStream_t s);
