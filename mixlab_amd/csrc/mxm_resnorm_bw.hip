// The residual norm's backward (formulas in mxm_train.h): one pass over the rows
// with the gradients of the stream and the branch, column sums of the scales'
// and the gate's gradients kept in registers over a chunk of rows, and a second
// launch that joins the chunks in their order.
#include <algorithm>

#include "mxm_resnorm.h"

namespace {

using namespace resnorm;

// Rows [*lo, *hi) of chunk c.
__device__ __forceinline__ void chunk_range(const ResNormArgs& a, int c, int* lo, int* hi) {
  int64_t r0, r1;
  if (c >= a.chunks) {
    r0 = r1 = a.N;
  } else if (a.group_chunks > 0) {
    const int64_t g = c / a.group_chunks, sub = c % a.group_chunks;
    r0 = g * a.gate_rows + sub * a.chunk_rows;
    r1 = min(r0 + a.chunk_rows, (g + 1) * (int64_t)a.gate_rows);
  } else {
    r0 = (int64_t)c * a.chunk_rows;
    r1 = r0 + a.chunk_rows;
  }
  *lo = (int)min(r0, (int64_t)a.N);
  *hi = (int)min(r1, (int64_t)a.N);
}

// CH: a gate per channel.  A row's threads walk one chunk; the chunks of a
// workgroup add their column sums in LDS and store one partial.
template <int V, int NV, int LPR, int XT, int DT, int GT, bool CH>
__global__ __launch_bounds__(LPR ? THREADS : 1024) void resnorm_bw_kernel(ResNormArgs a) {
  constexpr int E = V * NV;
  // of a row's sums (LPR = 0), or of the workgroup's column sums at the end
  __shared__ float red[LPR ? THREADS * E : 2 * 2 * 16 * 3];
  const int lane = LPR ? threadIdx.x % (LPR ? LPR : 1) : threadIdx.x;
  const int stride = LPR ? LPR : blockDim.x;
  const int rows = LPR ? THREADS / (LPR ? LPR : 1) : 1;
  const int proc = LPR ? threadIdx.x / (LPR ? LPR : 1) : 0;
  const int c = blockIdx.x * rows + proc, D = a.D;
  const bool post = a.branch && a.post_norm;
  int at[NV];
  float f[E], w[E], aw[E], aq[E], ag[CH ? E : 1], ga[CH ? E : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at[i] = (i * stride + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = i * V + j;
      f[e] = w[e] = aw[e] = aq[e] = 0.0f;
      if (CH) ag[CH ? e : 0] = ga[CH ? e : 0] = 0.0f;
    }
    if (at[i] < D) {
      if (a.branch) {
        float p[V];
        load_scale<V>(a.scale, a.p_bf16, at[i], f + i * V);
        load_scale<V>(a.post, a.p_bf16, at[i], p);
#pragma unroll
        for (int j = 0; j < V; ++j) f[i * V + j] *= p[j];
      }
      if (a.norm) load_scale<V>(a.w, a.p_bf16, at[i], w + i * V);
    }
  }
  if (!CH) {
    ag[0] = 0.0f;
    ga[0] = 1.0f;
  }
  int lo, hi;
  chunk_range(a, c, &lo, &hi);
  int group = a.gate ? lo / a.gate_rows : 0;
  int left = a.gate ? a.gate_rows - (lo - group * a.gate_rows) : 0;  // rows to the group's end
  bool fresh = true;                                                  // the gate is not loaded yet
  // (the same number of rounds in every lane: the sums use whole waves)
  const int rounds = LPR ? a.chunk_rows : hi - lo;
  for (int it = 0; it < rounds; ++it) {
    const int n = lo + it;
    const bool valid = n < hi;
    const size_t row = (size_t)n * D;
    float h[E], dl[E], t[E], dy[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = i * V + j;
        h[e] = dl[e] = t[e] = dy[e] = 0.0f;
      }
      if (!valid || at[i] >= D) continue;
      if (a.norm) {
        load<XT, V>(a.h, a.x_bf16, row + at[i], h + i * V);
        load<GT, V>(a.dy, a.g_bf16, row + at[i], dy + i * V);
      }
      if (a.branch) load<DT, V>(a.delta, a.delta_bf16, row + at[i], dl + i * V);
      if (a.dh) load<GT, V>(a.dh, a.g_bf16, row + at[i], t + i * V);
    }
    if (a.gate && fresh && valid) {
      if (CH) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (at[i] < D)
            load_scale<V>(a.gatep, a.p_bf16, (size_t)group * D + at[i], ga + (CH ? i * V : 0));
#pragma unroll
        for (int e = 0; e < (CH ? E : 1); ++e) ga[e] = gate_of(a, ga[e]);
      } else {
        load_scale<1>(a.gatep, a.p_bf16, (size_t)group, ga);
        ga[0] = gate_of(a, ga[0]);
      }
      fresh = false;
    }
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s[0] = __builtin_fmaf(h[e], h[e], s[0]);
      s[1] = __builtin_fmaf(w[e] * dy[e], h[e], s[1]);
      s[2] = __builtin_fmaf(dl[e], dl[e], s[2]);
    }
    if (a.norm || post) row_sum<LPR>(s, red + (it & 1) * 48);
    if (a.norm) {
      const float rn = 1.0f / __builtin_sqrtf(s[0] * a.inv_d + a.eps);
      const float kn = rn * rn * rn * (s[1] * a.inv_d);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        t[e] = t[e] + (rn * (w[e] * dy[e]) - h[e] * kn);
        if (valid) aw[e] = aw[e] + dy[e] * h[e] * rn;
      }
    }
    if (a.branch) {
      const float rp = post ? 1.0f / __builtin_sqrtf(s[2] * a.inv_d + a.eps) : 1.0f;
      float q[2] = {0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float td = f[e] * t[e] * dl[e];
        q[0] = __builtin_fmaf(ga[CH ? e : 0], td, q[0]);  // e * delta
        q[1] = q[1] + td * rp;                            // f * q
      }
      if (post || a.gate == 1) row_sum<LPR>(q, red + 96 + (it & 1) * 32);
      const float kp = post ? rp * rp * rp * (q[0] * a.inv_d) : 0.0f;
      float d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float g = ga[CH ? e : 0];
        const float tz = t[e] * (dl[e] * rp);
        if (valid) {
          aq[e] = aq[e] + g * tz;
          if (CH) ag[CH ? e : 0] = ag[CH ? e : 0] + f[e] * tz;
        }
        d[e] = rp * (t[e] * (g * f[e])) - dl[e] * kp;
      }
      if (!CH && valid) ag[0] = ag[0] + q[1];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (valid && at[i] < D) store<GT, V>(a.d_delta, a.g_bf16, row + at[i], d + i * V);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (valid && at[i] < D && a.dx) store<GT, V>(a.dx, a.g_bf16, row + at[i], t + i * V);
    // the group's last row here: its gate's gradient goes out
    if (a.gate && valid && (--left == 0 || n + 1 == hi)) {
      if (a.d_gate) {
        float* out = a.group_chunks > 0 ? a.gate_part + (size_t)c * (CH ? D : 1)
                                        : a.d_gate + (size_t)group * (CH ? D : 1);
        if (CH) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int e = CH ? i * V + j : 0;
              if (at[i] < D) out[at[i] + j] = a.sigmoid ? ag[e] * (ga[e] * (1.0f - ga[e])) : ag[e];
              ag[e] = 0.0f;
            }
        } else {
          if (lane == 0) out[0] = a.sigmoid ? ag[0] * (ga[0] * (1.0f - ga[0])) : ag[0];
          ag[0] = 0.0f;
        }
      }
      ++group;
      left = a.gate_rows;
      fresh = true;
    }
  }
  if (a.gate && a.group_chunks > 0 && a.d_gate && lo >= hi && c < a.chunks) {
    // (a chunk past the last row of a short group)
    if (CH) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at[i] < D) a.gate_part[(size_t)c * D + at[i] + j] = 0.0f;
    } else if (lane == 0) {
      a.gate_part[c] = 0.0f;
    }
  }
  auto join = [&](float(&acc)[E], int kind) {
    float* part = a.part + ((size_t)kind * a.parts + blockIdx.x) * D;
    if (LPR) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) red[LPR ? e * THREADS + threadIdx.x : 0] = acc[e];
      __syncthreads();
      if (proc > 0) return;
#pragma unroll
      for (int e = 0; e < E; ++e)
        for (int p = 1; p < rows; ++p) acc[e] += red[LPR ? e * THREADS + p * LPR + lane : 0];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at[i] < D) part[at[i] + j] = acc[i * V + j];
  };
  if (a.norm && a.d_w) join(aw, 0);
  if (a.branch && (a.d_scale || a.d_post)) join(aq, 1);
}

// Joins the workgroups' column sums: 32 columns a workgroup, 32 slices of the
// partials, each summed in order, then the slices in order.  blockIdx.y 0 writes
// the next norm's scale gradient, 1 the branch's, 2 ... the gate's groups.
constexpr int JOIN_COLS = 32, JOIN_SLICES = 32;
__global__ __launch_bounds__(JOIN_COLS* JOIN_SLICES) void resnorm_join_kernel(ResNormArgs a) {
  __shared__ float red[JOIN_SLICES][JOIN_COLS + 1];
  const int col = threadIdx.x % JOIN_COLS, slice = threadIdx.x / JOIN_COLS;
  const int kind = blockIdx.y < 2 ? (int)blockIdx.y : 2;
  const int width = kind == 2 && a.gate == 1 ? 1 : a.D;
  if (kind == 0 && !(a.norm && a.d_w)) return;
  if (kind == 1 && !(a.branch && (a.d_scale || a.d_post))) return;
  const int d = blockIdx.x * JOIN_COLS + col;
  const int group = (int)blockIdx.y - 2;
  const int count = kind == 2 ? a.group_chunks : a.parts;
  const float* src = kind == 2 ? a.gate_part + (size_t)group * a.group_chunks * width
                               : a.part + (size_t)kind * a.parts * a.D;
  float s = 0.0f;
  if (d < width)
    for (int p = slice; p < count; p += JOIN_SLICES) s += src[(size_t)p * width + d];
  red[slice][col] = s;
  __syncthreads();
  if (slice != 0 || d >= width) return;
  s = 0.0f;
  for (int i = 0; i < JOIN_SLICES; ++i) s += red[i][col];
  float other[1];
  if (kind == 0) {
    a.d_w[d] = s;
  } else if (kind == 1) {
    load_scale<1>(a.post, a.p_bf16, d, other);
    if (a.d_scale) a.d_scale[d] = s * other[0];
    load_scale<1>(a.scale, a.p_bf16, d, other);
    if (a.d_post) a.d_post[d] = s * other[0];
  } else {
    a.d_gate[(size_t)group * width + d] = s;
  }
}

// Chunks that a backward aims at, and the fewest rows of one.
constexpr int WGS_PER_CU = 4, MIN_CHUNK_ROWS = 4;
int64_t target_chunks(const Shape& sh, int n_cu) { return (int64_t)WGS_PER_CU * n_cu * sh.rows(); }

// Splits a.N rows into chunks.
void plan(ResNormArgs& a, const Shape& sh) {
  const int64_t target = target_chunks(sh, a.n_cu);
  const int rows = (int)std::max<int64_t>((a.N + target - 1) / target, MIN_CHUNK_ROWS);
  a.group_chunks = 0;
  a.chunk_rows = rows;
  const int T = std::min(a.gate_rows, a.N);  // rows of the longest group
  if (a.gate && a.gate_rows > 1 && T > rows) {
    a.group_chunks = (T + rows - 1) / rows;
    a.chunk_rows = (T + a.group_chunks - 1) / a.group_chunks;
    a.group_chunks = (T + a.chunk_rows - 1) / a.chunk_rows;
    const int groups = (int)(((int64_t)a.N + a.gate_rows - 1) / a.gate_rows);
    a.chunks = groups * a.group_chunks;
  } else {
    // whole groups (or part of the only one)
    if (a.gate && a.gate_rows <= rows) a.chunk_rows = rows / a.gate_rows * a.gate_rows;
    a.chunks = (a.N + a.chunk_rows - 1) / a.chunk_rows;
  }
  a.parts = (a.chunks + sh.rows() - 1) / sh.rows();
}

template <int V, int NV, int LPR, int XT, int DT, int GT>
void launch(const ResNormArgs& a, const Shape& sh, hipStream_t s) {
  if (a.gate == 2)
    hipLaunchKernelGGL((resnorm_bw_kernel<V, NV, LPR, XT, DT, GT, true>), dim3(a.parts),
                       dim3(sh.threads), 0, s, a);
  else
    hipLaunchKernelGGL((resnorm_bw_kernel<V, NV, LPR, XT, DT, GT, false>), dim3(a.parts),
                       dim3(sh.threads), 0, s, a);
}

template <int NV, int LPR>
void launch_typed(const ResNormArgs& a, const Shape& sh, hipStream_t s) {
  const int types = (a.x_bf16 ? 4 : 0) | (a.delta_bf16 ? 2 : 0) | (a.g_bf16 ? 1 : 0);
  switch (types) {
    case 0: return launch<4, NV, LPR, F32, F32, F32>(a, sh, s);
    case 1: return launch<4, NV, LPR, F32, F32, BF16>(a, sh, s);
    case 2: return launch<4, NV, LPR, F32, BF16, F32>(a, sh, s);
    case 3: return launch<4, NV, LPR, F32, BF16, BF16>(a, sh, s);
    case 4: return launch<4, NV, LPR, BF16, F32, F32>(a, sh, s);
    case 5: return launch<4, NV, LPR, BF16, F32, BF16>(a, sh, s);
    case 6: return launch<4, NV, LPR, BF16, BF16, F32>(a, sh, s);
    default: return launch<4, NV, LPR, BF16, BF16, BF16>(a, sh, s);
  }
}

void launch_rows(const ResNormArgs& a, const Shape& sh, hipStream_t s) {
  if (sh.V == 4) {
    if (sh.lpr == 16) return launch_typed<1, 16>(a, sh, s);
    if (sh.lpr == 32) return launch_typed<1, 32>(a, sh, s);
    if (sh.lpr == 64) return sh.NV == 1 ? launch_typed<1, 64>(a, sh, s) : launch_typed<2, 64>(a, sh, s);
    return sh.NV == 2 ? launch_typed<2, 0>(a, sh, s) : launch_typed<4, 0>(a, sh, s);
  }
  if (sh.lpr == 64) return launch<1, 4, 64, ANY, ANY, ANY>(a, sh, s);
  return sh.NV == 4 ? launch<1, 4, 0, ANY, ANY, ANY>(a, sh, s) : launch<1, 16, 0, ANY, ANY, ANY>(a, sh, s);
}

}  // namespace

int64_t mxm_resnorm_max_chunks(int64_t max_rows, int D, bool groups, int n_cu) {
  // Without groups at most the target's; whole groups make chunks of at least
  // half the rows aimed at; chunks within groups are at most one more per group
  // than rows / chunk rows, and the groups fewer than that.
  int64_t most = 0;
  for (const bool vectors : {false, true})
    most = std::max(most, target_chunks(shape_of(D, vectors), n_cu));
  most = std::min(most, (max_rows + MIN_CHUNK_ROWS - 1) / MIN_CHUNK_ROWS);
  return groups ? 3 * most + 1 : most;
}

void mxm_launch_resnorm_bw(const ResNormArgs& args, hipStream_t s) {
  ResNormArgs a = args;
  const bool vectors =
      a.D % 4 == 0 && (!a.norm || (aligned(a.h, a.x_bf16) && aligned(a.dy, a.g_bf16))) &&
      (!a.branch || (aligned(a.delta, a.delta_bf16) && aligned(a.d_delta, a.g_bf16))) &&
      aligned(a.dh, a.g_bf16) && aligned(a.dx, a.g_bf16);
  const Shape sh = shape_of(a.D, vectors);
  a.chunks = a.parts = a.group_chunks = 0;
  if (a.N > 0) {
    plan(a, sh);
    launch_rows(a, sh, s);
  }
  // (without rows the scales' gradients are zero)
  const bool columns = (a.norm && a.d_w) || (a.branch && (a.d_scale || a.d_post));
  const bool gates = a.gate && a.group_chunks > 0 && a.d_gate;
  if (!columns && !gates) return;
  const dim3 grid((a.D + JOIN_COLS - 1) / JOIN_COLS, 2 + (gates ? a.chunks / a.group_chunks : 0));
  hipLaunchKernelGGL(resnorm_join_kernel, grid, dim3(JOIN_COLS * JOIN_SLICES), 0, s, a);
}
