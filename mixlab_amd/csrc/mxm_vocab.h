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
  float* part;            // [chunks][2][D up to 8]: sums of runs that a chunk shares
  int64_t max_rows;
  int n_cu;
};
void mxm_launch_embed(const EmbedArgs& a, hipStream_t s);
void mxm_launch_embed_bw(const EmbedArgs& a, hipStream_t s);
// Floats of part, for a backward of up to max_rows rows.
int64_t mxm_embed_part_floats(int64_t max_rows, int D);

// ---- token loss ----
//
// Rows n with a target t in [0, V) and a weight w_n that is not 0 take part:
//   z = x W^T,  l = cap tanh(z / cap)   (softcap; else z)
//   loss = log(1 + sum_{v != t} exp(l_v - l_t)),  lse = loss + l_t
//   total = sum_n w_n loss_n             (mean: / sum_n w_n)
//   g_n = d_total w_n                    (mean: / sum_n w_n)
//   dz = g (softmax(l) - [v = t]) (1 - (l / cap)^2),  dx = dz W,  dW = dz^T x
// The rows that take part are packed (in order) into x_pack, zero-padded to whole
// 64-wide stages.
//
// fp32 operands become two fp16 planes: a row of x or weight is 2^exp (hi + lo) with
// its largest element's hi in [2^14, 2^15), 22 bits of every element down to 2^-17 of
// the largest and 2^-40 of the largest below.  Products of two such operands are
// hi lo + lo hi + hi hi (lo lo, up to 2^-22 of the product, is left out), each exact in fp32.
// Exponents of rows along m or n of a product are applied to its sums; along k they
// have to agree.  With W_v = 2^c_v W'_v and x_n = 2^X_n x'_n:
//   dz'[n, v] = dz 2^(c_v - E_n),  dx = 2^E_n dz' W'
//   x''_n = x'_n 2^(E_n + X_n - C),  dW_v = 2^(C - c_v) dz'^T x'',  C = max_n (E_n + X_n)
// E_n is the largest of |dz| 2^c_v, taken where the summands are, so that an entry of
// any size without a share in the gradient has none in it.  c_v is the exponent w_v of
// the row of weight, but where that is so small that dz' would lose digits, which dW_v
// needs whatever the row holds (zeros, say): no smaller than L = max_n of the others'
// largest |dz| 2^w_v over the others' largest |dz| (under a softcap, before its slope),
// less XENT_SLACK: next to the exponents of the rows that the gradients go to.  Rows of
// W' below L are taken down to it before product 2 (with the slack, few if any of a table
// of alike rows; a step of 733 rows of D 1528 and 256 entries took 206 us without, 76 with
// it).  So dz' keeps 2^-36 of a row's largest |dz|, whatever the entry's row of weight.
// (Over the largest |dz| of all, the target's, L was lower by the others' shares: with
// 50257 entries dW of rows of zeros was off by 1.6e-4 of it, 4e-7 so.)
// A row of weight with infinite elements is its infinities' signs and the exponent
// XENT_INF, one of zeros has XENT_ZERO.
//
// Then, for a piece of the rows that take part at a time:
//   product 1 (mxm_xent_gemm.hip): logits of a tile of vocabulary x rows in the
//     accumulators; of each row and block of the vocabulary the sum over v != t of
//     2^(l log2 e - ref) with a ref of the block (a whole number, or next to one);
//     backwards also each summand (under a softcap times a quarter of 1 - (l / cap)^2),
//     relative to that ref;
//   join (mxm_xent.hip): each row's loss and the factors of its gradient;
//   finish: the summands to dz, in place (fp32: to planes; x' to x'');
//   product 2: dx = dz W;  product 3: dW (+)= dz^T x.
struct XentScalars {
  double weight_sum;        // of the rows that take part
  int32_t rows;             // that take part
  int32_t dw_exp;           // C
  int32_t low[2];           // L of the pieces so far, by the last one's parity
};
constexpr int XENT_INF = 1 << 20;
constexpr int XENT_ZERO = -(1 << 18);
constexpr int XENT_SLACK = 4;
constexpr int XENT_NO_EXP = -(1 << 20);  // of nothing
constexpr float XENT_NO_REF = -3.4028235e38f;  // ref of a block without an entry: the least
struct XentRow {            // of a row that takes part
  float ref;                // M: the summands' common exponent
  float scale;              // g / sum of all 2^(l log2 e - M), times 4 under a softcap
  float at_target;          // dz of the target
  int32_t target;
  // fp32: |dz| 2^w < 2^(e + 15) and |dz| < 2^(g + 15), XENT_NO_EXP for a row without a
  // gradient
  int32_t e, g;
};
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
  int Dp, Vp;               // D rounded up to whole stages; V to an odd number of them
  int planes;               // 1 (bf16) or 2 (fp32)
  int32_t* map;             // [rows] a row that takes part, by its place among those
  int32_t* target;          // [rows] of those that take part
  int32_t* counts;          // [XENT_CHUNKS] of rows that take part, and their weights' sums
  double* weights;
  XentScalars* scalars;
  float* nll;               // [rows] loss of the rows that take part
  float* at_target;         // [rows] their target's logit, before the cap
  XentRow* row;             // [rows]
  uint16_t* x_pack;         // [planes][x_rows][Dp]
  int64_t x_rows;
  uint16_t* w_pack;         // [planes][V][Dp], unused where weight is read in place
  bool w_direct;            // weight itself: bf16 rows of whole 16 bytes
  int32_t *x_exp, *w_exp;   // [rows], [V up to whole tiles]: X, w (fp32)
  int32_t* e_row;           // [rows]: E
  int4* c_part;             // of each workgroup that joins rows the largest others' e - g,
  int c_parts;              // e + X and g + X
  float2* stat;             // [blocks][stat_ld]: sum, ref
  int32_t* stat_exp;        // [blocks][stat_ld] (fp32 backward): the exponent of summand 2^w
  void* summands;           // [piece_rows][Vp]: fp16 (bf16) or fp32
  uint16_t* dz;             // [planes][piece_rows][Vp]: the summands' place under bf16
  float* partial;           // tiles of products that are split along their sums
  float* dw32;              // [V][D] sums of the pieces before the last, or null: dw itself
  const uint16_t* zeros;    // 4 KB of zeros
  int64_t piece_rows, stat_ld;
  int n_cu;
};
constexpr int XENT_CHUNKS = 4096;  // most chunks of a call's rows
// Bytes of partial, for handles that run backward.
int64_t mxm_xent_partial_bytes(int n_cu);
// Most blocks of stat times rows, for pieces of `rows`.
int64_t mxm_xent_stats(int64_t rows, int V, int n_cu);
// Columns of the vocabulary per block of stat, for a piece of `rows` rows.
int mxm_xent_block(int64_t rows, int V, int n_cu);
// low: where the pieces before left L, or null.
// gather: the kernel itself finds the rows that take part and reads them in place.
void mxm_launch_xent_logits(const XentArgs& a, int64_t r0, int64_t rows, const int32_t* low, bool gather,
                            hipStream_t s);
// Most rows of a forward that are read in place.
constexpr int XENT_GATHER = 32;
// dx and dw, as far as they are wanted; last: no piece comes after this one.
void mxm_launch_xent_grads(const XentArgs& a, int64_t r0, int64_t rows, bool last, const int32_t* low,
                           hipStream_t s);
void mxm_launch_xent(const XentArgs& a, hipStream_t s);

// Whether a row of weight w and target t takes part.
__device__ __forceinline__ bool mxm_xent_takes_part(const int32_t* targets, const float* row_weights, int V,
                                                    int64_t n, int& t, float& w) {
  t = targets[n];
  w = row_weights ? row_weights[n] : 1.0f;
  return t >= 0 && t < V && w != 0.0f;
}

// Rows of the piece that starts at row r0 of those that take part.
__device__ __forceinline__ int mxm_xent_rows(const XentArgs& a, int64_t r0) {
  const int64_t left = a.scalars->rows - r0;
  return left <= 0 ? 0 : (int)(left < a.piece_rows ? left : a.piece_rows);
}

// tanh(z / cap) = 1 - 2 / (1 + exp(2 z / cap)), k2 = 2 log2 e / cap: off by a few 2^-24
// of 1.
__device__ __forceinline__ float mxm_xent_capped(float z, float k2) {
  return fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * k2)), 1.0f);
}

// The slope 1 - tanh^2, as 4 times this, from e = exp(2 z / cap) and r = 1 / (1 + e), tanh =
// 1 - 2 r: it keeps its digits where tanh is next to 1 or -1 (taken from tanh it is off by
// 6e-5 at z = 4 cap, by 8e-3 at 7, and zero from 9 on).  e r is 1 where e is infinite.
__device__ __forceinline__ float mxm_xent_cap_slope(float e, float r) { return r * fminf(e * r, 1.0f); }
