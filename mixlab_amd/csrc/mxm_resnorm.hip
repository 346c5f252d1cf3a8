// The residual norm forwards (formulas in mxm_train.h): the branch's output
// normalised, scaled and gated, added to the stream, and the next sublayer's
// norm of the sum, in one pass over the rows.
#include <algorithm>

#include "mxm_resnorm.h"

namespace {

using namespace resnorm;

constexpr int ROWS_PER_WG_LOOP = 4;  // row rounds of a workgroup that loops

template <int V, int NV, int LPR, int XT, int DT, int YT>
__global__ __launch_bounds__(LPR ? THREADS : 1024) void resnorm_kernel(ResNormArgs a) {
  constexpr int E = V * NV;
  __shared__ float red[2][2][LPR ? 1 : 16];
  const int lane = LPR ? threadIdx.x % (LPR ? LPR : 1) : threadIdx.x;
  const int stride = LPR ? LPR : blockDim.x;
  const int rows = LPR ? THREADS / (LPR ? LPR : 1) : 1;
  const int D = a.D;
  int at[NV];
  float f[E], w[E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at[i] = (i * stride + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) f[i * V + j] = w[i * V + j] = 0.0f;
    if (at[i] < D) {
      float p[V];
      load_scale<V>(a.scale, a.p_bf16, at[i], f + i * V);
      load_scale<V>(a.post, a.p_bf16, at[i], p);
#pragma unroll
      for (int j = 0; j < V; ++j) f[i * V + j] *= p[j];
      if (a.norm) load_scale<V>(a.w, a.p_bf16, at[i], w + i * V);
    }
  }
  // (at most 2^30 rows and a workgroup's more)
  const int first =
      (int)blockIdx.x * rows * a.chunk_rows + (LPR ? (int)threadIdx.x / (LPR ? LPR : 1) : 0);
  for (int it = 0; it < a.chunk_rows; ++it) {
    const int n = first + it * rows;
    const bool valid = n < a.N;  // (a workgroup of one row: for all of it)
    const size_t row = (size_t)n * D;
    float h[E], dl[E], ga[E], sum[1];
    // (values past the row's end and rows past the last stay zero)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) h[i * V + j] = dl[i * V + j] = ga[i * V + j] = 0.0f;
      if (valid && at[i] < D) {
        load<XT, V>(a.x, a.x_bf16, row + at[i], h + i * V);
        if (a.branch) load<DT, V>(a.delta, a.delta_bf16, row + at[i], dl + i * V);
      }
    }
    if (a.branch) {
      if (a.gate == 2) {
        const size_t grow = (size_t)(n / a.gate_rows) * D;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (valid && at[i] < D) load_scale<V>(a.gatep, a.p_bf16, grow + at[i], ga + i * V);
#pragma unroll
        for (int e = 0; e < E; ++e) ga[e] = gate_of(a, ga[e]) * f[e];
      } else {
        float g = 1.0f;
        if (a.gate == 1 && valid) {
          load_scale<1>(a.gatep, a.p_bf16, (size_t)(n / a.gate_rows), &g);
          g = gate_of(a, g);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) ga[e] = g * f[e];
      }
      float rp = 1.0f;
      if (a.post_norm) {
        sum[0] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[0] = __builtin_fmaf(dl[e], dl[e], sum[0]);
        row_sum<LPR>(sum, red[0][it & 1]);
        rp = 1.0f / __builtin_sqrtf(sum[0] * a.inv_d + a.eps);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = h[e] + ga[e] * (dl[e] * rp);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (valid && at[i] < D) store<XT, V>(a.h, a.x_bf16, row + at[i], h + i * V);
    }
    if (!a.norm) continue;
    sum[0] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[0] = __builtin_fmaf(h[e], h[e], sum[0]);
    row_sum<LPR>(sum, red[1][it & 1]);
    const float rn = 1.0f / __builtin_sqrtf(sum[0] * a.inv_d + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!valid || at[i] >= D) continue;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = (h[i * V + j] * rn) * w[i * V + j];
      store<YT, V>(a.y, a.y_bf16, row + at[i], y);
    }
  }
}

template <int V, int NV, int LPR, int XT, int DT, int YT>
void launch(const ResNormArgs& args, const Shape& sh, hipStream_t s) {
  ResNormArgs a = args;
  const int64_t rounds = ((int64_t)a.N + sh.rows() - 1) / sh.rows();
  a.chunk_rows = rounds >= 4096 * ROWS_PER_WG_LOOP ? ROWS_PER_WG_LOOP : 1;
  const int64_t blocks = (rounds + a.chunk_rows - 1) / a.chunk_rows;
  hipLaunchKernelGGL((resnorm_kernel<V, NV, LPR, XT, DT, YT>), dim3((unsigned)blocks),
                     dim3(sh.threads), 0, s, a);
}

}  // namespace

void mxm_launch_resnorm(const ResNormArgs& a, hipStream_t s) {
  if (a.N <= 0) return;
  const bool vectors = a.D % 4 == 0 && aligned(a.x, a.x_bf16) &&
                       (!a.branch || (aligned(a.delta, a.delta_bf16) && aligned(a.h, a.x_bf16))) &&
                       (!a.norm || aligned(a.y, a.y_bf16));
  const Shape sh = shape_of(a.D, vectors);
  if (vectors)
    with_shape4(sh, [&](auto nv, auto lpr) {
      with_types(a.x_bf16, a.delta_bf16, a.y_bf16, [&](auto xt, auto dt, auto yt) {
        launch<4, nv(), lpr(), xt(), dt(), yt()>(a, sh, s);
      });
    });
  else
    with_shape1(sh, [&](auto nv, auto lpr) { launch<1, nv(), lpr(), ANY, ANY, ANY>(a, sh, s); });
}
