// The residual norm forwards (formulas in mxm_train.h): the branch's output
// normalised, scaled and gated, added to the stream, and the next sublayer's
// norm of the sum, in one pass over the rows.  Bound by memory: 65,536 rows of
// 2048 channels, fp32 with a bf16 y and a gate per token, 306 us (1.88 GB at 6.1
// TB/s; 383 us at a large copy's rate), few rows by one row's chain of load, sum,
// root, sum, root, store (3.9 us for 8 rows of 1024).
#include <algorithm>

#include "mxm_resnorm.h"

namespace {

using namespace resnorm;

template <int NV, int LPR, int XT, int DT, int YT, int ODD>
__global__ __launch_bounds__(most_threads(LPR)) void resnorm_kernel(ResNormArgs a) {
  constexpr int E = V * NV;
  __shared__ float red[2][2][LPR > 0 ? 1 : 16];
  const int lane = LPR > 0 ? threadIdx.x % (LPR > 0 ? LPR : 1) : threadIdx.x;
  const int stride = LPR > 0 ? LPR : blockDim.x;
  const int rows = LPR > 0 ? THREADS / (LPR > 0 ? LPR : 1) : 1;
  const int D = a.D;
  int at[NV];
  float f[E], w[E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at[i] = (i * stride + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) f[i * V + j] = w[i * V + j] = 0.0f;
    if (at[i] < D) {
      if (a.branch) {
        float p[V];
        load_scale<ODD>(a.scale, a.p_bf16, 0, at[i], D, f + i * V);
        load_scale<ODD>(a.post, a.p_bf16, 0, at[i], D, p);
#pragma unroll
        for (int j = 0; j < V; ++j) f[i * V + j] *= p[j];
      }
      if (a.norm) load_scale<ODD>(a.w, a.p_bf16, 0, at[i], D, w + i * V);
    }
  }
  // (at most 2^30 rows and a workgroup's more)
  const int first = (int)blockIdx.x * rows * a.chunk_rows + row_slot<LPR>();
  Raw<XT> rx[NV];
  Raw<DT> rd[NV];
  float rg = 0.0f;  // a gate per row
  // (values past the row's end and rows past the last are zero)
  auto fetch = [&](int n) {
    const size_t row = (size_t)n * D;
    if (a.gate == 1 && n < a.N) rg = load_one(a.gatep, a.p_bf16, (size_t)(n / a.gate_rows));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      rx[i] = Raw<XT>{};
      rd[i] = Raw<DT>{};
      if (n < a.N && at[i] < D) {
        rx[i] = load<XT, ODD>(a.x, row, at[i], D);
        if (a.branch) rd[i] = load<DT, ODD>(a.delta, row, at[i], D);
      }
    }
  };
  fetch(first);
  for (int it = 0; it < a.chunk_rows; ++it) {
    const int n = first + it * rows;
    const bool valid = n < a.N;  // (a workgroup of one row: for all of it)
    const size_t row = (size_t)n * D;
    float h[E], dl[E], ga[E], sum[1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<XT, ODD>(rx[i], at[i], D, h + i * V);
      unpack<DT, ODD>(rd[i], at[i], D, dl + i * V);
    }
    float g = a.gate == 1 ? rg : 1.0f;
    if (it + 1 < a.chunk_rows) fetch(n + rows);
    if (a.branch) {
      // (the gate's values go through the sigmoid after the sum, which hides its load)
      if (a.gate == 2) {
        const size_t grow = (size_t)(n / a.gate_rows) * D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int j = 0; j < V; ++j) ga[i * V + j] = 0.0f;
          if (valid && at[i] < D) load_scale<ODD>(a.gatep, a.p_bf16, grow, at[i], D, ga + i * V);
        }
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
      for (int e = 0; e < E; ++e) ga[e] = a.gate == 2 ? gate_of(a, ga[e]) * f[e] : f[e];
      g = (a.gate == 1 ? gate_of(a, g) : 1.0f) * rp;
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = __builtin_fmaf(g * dl[e], ga[e], h[e]);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (valid && at[i] < D) store<XT, ODD>(a.h, row, at[i], D, h + i * V);
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
      store<YT, ODD>(a.y, row, at[i], D, y);
    }
  }
}

// Rows that a thread walks, which share its loads of the scales: few enough that
// all CUs have several workgroups.  134 M elements at 1024 and 2048 channels with
// 1 / 2 / 4 / 8 rows, fp32 302-328 / 302-305 / 320-332 / 341-349 us, bf16 206-210 /
// 178-182 / 174-178 / 174-194: rows of half the bytes pay for twice as many.
int rows_per_thread(const ResNormArgs& a, const Shape& sh) {
  const int64_t rounds = ((int64_t)a.N + sh.rows() - 1) / sh.rows();
  const int most = a.x_bf16 && (a.delta_bf16 || !a.branch) ? 4 : 2;
  // (a launch's threads are counted in 32 bits)
  const int64_t least = (rounds * sh.threads + ((int64_t)1 << 31) - 1) >> 31;
  return (int)std::max(std::min<int64_t>(std::max<int64_t>(rounds / (8 * a.n_cu), 1), most), least);
}

template <int NV, int LPR, int XT, int DT, int YT, int ODD>
void launch(const ResNormArgs& args, const Shape& sh, hipStream_t s) {
  ResNormArgs a = args;
  a.chunk_rows = rows_per_thread(a, sh);
  const int64_t per = (int64_t)a.chunk_rows * sh.rows();
  hipLaunchKernelGGL((resnorm_kernel<NV, LPR, XT, DT, YT, ODD>), dim3((unsigned)((a.N + per - 1) / per)),
                     dim3(sh.threads), 0, s, a);
}

}  // namespace

void mxm_launch_resnorm(const ResNormArgs& a, hipStream_t s) {
  if (a.N <= 0) return;
  const bool vectors = a.D % 4 == 0 && aligned(a.x, a.x_bf16) &&
                       (!a.branch || (aligned(a.delta, a.delta_bf16) && aligned(a.h, a.x_bf16))) &&
                       (!a.norm || aligned(a.y, a.y_bf16));
  const Shape sh = shape_of(a.D, false, a.N);
  with_shape<false>(sh, [&](auto nv, auto lpr) {
    with_types(a.x_bf16, a.delta_bf16, a.y_bf16, !vectors, [&](auto xt, auto dt, auto yt, auto odd) {
      launch<nv(), lpr(), xt(), dt(), yt(), odd() ? lpr() == 16 ? 2 : 1 : 0>(a, sh, s);
    });
  });
}
