// The residual norm, forwards and backwards (formulas in mxm_train.h): the
// branch's output normalised, scaled and gated, added to the stream, and the
// next sublayer's norm of the sum.
#include "mxm_kernels.h"
#include "mxm_train.h"

namespace {

constexpr int GEN_THREADS = 256;

__device__ __forceinline__ float ld1(const void* p, bool bf, size_t i) {
  return bf ? mxm_bf2f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}
// Rounds to the type it is kept in and returns the kept value.
__device__ __forceinline__ float st1(void* p, bool bf, size_t i, float v) {
  if (bf) {
    const uint16_t b = mxm_f2bf(v);
    static_cast<uint16_t*>(p)[i] = b;
    return mxm_bf2f(b);
  }
  static_cast<float*>(p)[i] = v;
  return v;
}
__device__ __forceinline__ float scale_at(const void* p, bool bf, int d) {
  return p ? ld1(p, bf, d) : 1.0f;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v = v + mxm_xor_lane_f(v, s);
  return v;
}

// Sums of K values over the workgroup, in every thread; `red` holds K floats a
// wave.  Ends with a barrier, so that the next call may write `red`.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* red) {
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += red[w * K + k];
    v[k] = s;
  }
  __syncthreads();
}

// The gate's value and its derivative by what was given.
__device__ __forceinline__ float gate_value(const ResNormArgs& a, size_t i, float* slope) {
  const float g = ld1(a.gatep, a.p_bf16, i);
  if (!a.sigmoid) {
    *slope = 1.0f;
    return g;
  }
  const float s = mxm_sigmoid(g);
  *slope = s * (1.0f - s);
  return s;
}

// One workgroup per row, any D: every pass reads the row again.
__global__ __launch_bounds__(GEN_THREADS) void resnorm_any_kernel(ResNormArgs a) {
  __shared__ float red[GEN_THREADS / 64];
  const int tid = threadIdx.x, D = a.D;
  for (int n = blockIdx.x; n < a.N; n += gridDim.x) {
    const size_t row = (size_t)n * D;
    const size_t grow = a.gate ? (size_t)(n / a.gate_rows) * (a.gate == 2 ? D : 1) : 0;
    float rp = 1.0f, sum[1], slope, ga = 1.0f;
    if (a.branch && a.post_norm) {
      sum[0] = 0.0f;
      for (int d = tid; d < D; d += GEN_THREADS) {
        const float v = ld1(a.delta, a.delta_bf16, row + d);
        sum[0] = __builtin_fmaf(v, v, sum[0]);
      }
      block_sum(sum, red);
      rp = 1.0f / __builtin_sqrtf(sum[0] * a.inv_d + a.eps);
    }
    if (a.gate == 1) ga = gate_value(a, grow, &slope);
    sum[0] = 0.0f;
    for (int d = tid; d < D; d += GEN_THREADS) {
      float h = ld1(a.x, a.x_bf16, row + d);
      if (a.branch) {
        if (a.gate == 2) ga = gate_value(a, grow + d, &slope);
        const float f = scale_at(a.scale, a.p_bf16, d) * scale_at(a.post, a.p_bf16, d);
        h = st1(a.h, a.x_bf16, row + d, h + (ga * f) * (ld1(a.delta, a.delta_bf16, row + d) * rp));
      }
      sum[0] = __builtin_fmaf(h, h, sum[0]);
    }
    if (!a.norm) continue;
    block_sum(sum, red);
    const float rn = 1.0f / __builtin_sqrtf(sum[0] * a.inv_d + a.eps);
    // (h may be x's own buffer: the sum is read back from where it was kept)
    const void* src = a.branch ? a.h : a.x;
    for (int d = tid; d < D; d += GEN_THREADS)
      st1(a.y, a.y_bf16, row + d,
          (ld1(src, a.x_bf16, row + d) * rn) * scale_at(a.w, a.p_bf16, d));
  }
}

// Rows [*lo, *hi) of chunk c.
__device__ __forceinline__ void chunk_range(const ResNormArgs& a, int c, int* lo, int* hi) {
  int64_t r0, r1;
  if (a.group_chunks > 0) {
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

// One workgroup per chunk of rows, any D: three passes over each row, the
// column sums kept in the chunk's own rows of `part`.
__global__ __launch_bounds__(GEN_THREADS) void resnorm_bw_any_kernel(ResNormArgs a) {
  __shared__ float red[3 * (GEN_THREADS / 64)];
  const int tid = threadIdx.x, D = a.D, c = blockIdx.x;
  const bool post = a.branch && a.post_norm;
  float* part_w = a.part + (size_t)c * D;
  float* part_q = a.part + (size_t)(a.chunks + c) * D;
  for (int d = tid; d < D; d += GEN_THREADS) {
    if (a.norm) part_w[d] = 0.0f;
    if (a.branch) part_q[d] = 0.0f;
    if (a.gate == 2 && a.group_chunks > 0) a.gate_part[(size_t)c * D + d] = 0.0f;
  }
  float gsum = 0.0f;  // a gate per row: the sum over its group's rows so far
  int lo, hi;
  chunk_range(a, c, &lo, &hi);
  for (int n = lo; n < hi; ++n) {
    const size_t row = (size_t)n * D;
    const int group = a.gate ? n / a.gate_rows : 0;
    const size_t grow = (size_t)group * (a.gate == 2 ? D : 1);
    const bool first = a.gate && n % a.gate_rows == 0;
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int d = tid; d < D; d += GEN_THREADS) {
      if (a.norm) {
        const float h = ld1(a.h, a.x_bf16, row + d);
        const float u = ld1(a.dy, a.g_bf16, row + d) * scale_at(a.w, a.p_bf16, d);
        s[0] = __builtin_fmaf(h, h, s[0]);
        s[1] = __builtin_fmaf(u, h, s[1]);
      }
      if (post) {
        const float v = ld1(a.delta, a.delta_bf16, row + d);
        s[2] = __builtin_fmaf(v, v, s[2]);
      }
    }
    block_sum(s, red);
    const float rn = 1.0f / __builtin_sqrtf(s[0] * a.inv_d + a.eps);
    const float kn = rn * rn * rn * (s[1] * a.inv_d);
    const float rp = post ? 1.0f / __builtin_sqrtf(s[2] * a.inv_d + a.eps) : 1.0f;
    auto upstream = [&](int d) {
      float t = a.dh ? ld1(a.dh, a.g_bf16, row + d) : 0.0f;
      if (a.norm) {
        const float u = ld1(a.dy, a.g_bf16, row + d) * scale_at(a.w, a.p_bf16, d);
        t = t + (rn * u - ld1(a.h, a.x_bf16, row + d) * kn);
      }
      return t;
    };
    float ga = 1.0f, slope = 1.0f;
    if (a.gate == 1) ga = gate_value(a, grow, &slope);
    float q[2] = {0.0f, 0.0f};
    if (a.branch && (post || a.gate == 1)) {
      for (int d = tid; d < D; d += GEN_THREADS) {
        if (a.gate == 2) ga = gate_value(a, grow + d, &slope);
        const float f = scale_at(a.scale, a.p_bf16, d) * scale_at(a.post, a.p_bf16, d);
        const float td = upstream(d) * f * ld1(a.delta, a.delta_bf16, row + d);
        q[0] = __builtin_fmaf(ga, td, q[0]);  // e * delta
        q[1] = q[1] + td * rp;                // f * q
      }
      block_sum(q, red);
    }
    const float kp = post ? rp * rp * rp * (q[0] * a.inv_d) : 0.0f;
    if (a.gate == 1) {
      gsum = (first ? 0.0f : gsum) + q[1] * slope;
      if (tid == 0 && a.d_gate) {
        if (a.group_chunks > 0)
          a.gate_part[c] = gsum;
        else
          a.d_gate[group] = gsum;
      }
    }
    for (int d = tid; d < D; d += GEN_THREADS) {
      const float t = upstream(d);
      const float dy = a.norm ? ld1(a.dy, a.g_bf16, row + d) : 0.0f;
      const float h = a.norm ? ld1(a.h, a.x_bf16, row + d) : 0.0f;
      const float dl = a.branch ? ld1(a.delta, a.delta_bf16, row + d) : 0.0f;
      if (a.dx) st1(a.dx, a.g_bf16, row + d, t);
      if (a.norm) part_w[d] = part_w[d] + dy * h * rn;
      if (!a.branch) continue;
      if (a.gate == 2) ga = gate_value(a, grow + d, &slope);
      const float f = scale_at(a.scale, a.p_bf16, d) * scale_at(a.post, a.p_bf16, d);
      const float tz = t * (dl * rp);
      part_q[d] = part_q[d] + ga * tz;
      if (a.gate == 2 && a.d_gate) {
        float* g = a.group_chunks > 0 ? a.gate_part + (size_t)c * D + d : a.d_gate + grow + d;
        // (a group's first row starts its sum where the chunk holds whole groups)
        const float before = a.group_chunks == 0 && first ? 0.0f : *g;
        *g = before + f * tz * slope;
      }
      const float e = t * (ga * f);
      st1(a.d_delta, a.g_bf16, row + d, post ? rp * e - dl * kp : e);
    }
  }
  if (a.gate == 1 && a.group_chunks > 0 && lo >= hi && tid == 0) a.gate_part[c] = 0.0f;
}

// Joins the chunks' column sums: 32 columns a workgroup, 32 slices of the
// chunks, each summed in order, then the slices in order.  blockIdx.y 0 writes
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
  const int c0 = kind == 2 ? group * a.group_chunks : 0;
  const int count = kind == 2 ? a.group_chunks : a.chunks;
  const float* src = kind == 2 ? a.gate_part : a.part + (size_t)kind * a.chunks * a.D;
  float s = 0.0f;
  if (d < width)
    for (int c = slice; c < count; c += JOIN_SLICES) s += src[(size_t)(c0 + c) * width + d];
  red[slice][col] = s;
  __syncthreads();
  if (slice != 0 || d >= width) return;
  s = 0.0f;
  for (int i = 0; i < JOIN_SLICES; ++i) s += red[i][col];
  if (kind == 0) {
    a.d_w[d] = s;
  } else if (kind == 1) {
    if (a.d_scale) a.d_scale[d] = s * scale_at(a.post, a.p_bf16, d);
    if (a.d_post) a.d_post[d] = s * scale_at(a.scale, a.p_bf16, d);
  } else {
    a.d_gate[(size_t)group * width + d] = s;
  }
}

// Chunks that a backward aims at, and the fewest rows of one.
int target_chunks(int n_cu) { return 4 * n_cu; }
constexpr int MIN_CHUNK_ROWS = 4;

}  // namespace

int64_t mxm_resnorm_max_chunks(int64_t max_rows, int D, int gate, int gate_rows, int n_cu) {
  // ungrouped: at most the target; whole groups: rows per chunk are at least
  // half of what was aimed at; chunks within groups: at most one more per group
  // and one more group than rows / chunk rows
  const int64_t aim = (max_rows + MIN_CHUNK_ROWS - 1) / MIN_CHUNK_ROWS;
  return 3 * (aim < target_chunks(n_cu) ? aim : target_chunks(n_cu)) + 1;
}

void mxm_resnorm_plan(ResNormArgs& a, int n_cu) {
  const int target = target_chunks(n_cu);
  int rows = (a.N + target - 1) / target;
  if (rows < MIN_CHUNK_ROWS) rows = MIN_CHUNK_ROWS;
  a.group_chunks = 0;
  a.chunk_rows = rows;
  if (a.gate && a.gate_rows > 1) {
    const int T = a.gate_rows < a.N ? a.gate_rows : a.N;  // rows of the longest group
    if (T <= rows) {
      a.chunk_rows = a.gate_rows <= rows ? rows / a.gate_rows * a.gate_rows : rows;
    } else {
      a.group_chunks = (T + rows - 1) / rows;
      a.chunk_rows = (T + a.group_chunks - 1) / a.group_chunks;
      a.group_chunks = (T + a.chunk_rows - 1) / a.chunk_rows;
      const int groups = (int)(((int64_t)a.N + a.gate_rows - 1) / a.gate_rows);
      a.chunks = groups * a.group_chunks;
      return;
    }
  }
  a.chunks = (a.N + a.chunk_rows - 1) / a.chunk_rows;
}

void mxm_launch_resnorm(const ResNormArgs& a, hipStream_t s) {
  if (a.N <= 0) return;
  const int blocks = a.N < 65536 ? a.N : 65536;
  hipLaunchKernelGGL(resnorm_any_kernel, dim3(blocks), dim3(GEN_THREADS), 0, s, a);
}

void mxm_launch_resnorm_bw(const ResNormArgs& a, hipStream_t s) {
  if (a.chunks > 0)
    hipLaunchKernelGGL(resnorm_bw_any_kernel, dim3(a.chunks), dim3(GEN_THREADS), 0, s, a);
  // (without rows the scales' gradients are zero)
  const bool columns = (a.norm && a.d_w) || (a.branch && (a.d_scale || a.d_post));
  const bool gates = a.gate && a.group_chunks > 0 && a.d_gate;
  if (!columns && !gates) return;
  const dim3 grid((a.D + JOIN_COLS - 1) / JOIN_COLS, 2 + (gates ? a.chunks / a.group_chunks : 0));
  hipLaunchKernelGGL(resnorm_join_kernel, grid, dim3(JOIN_COLS * JOIN_SLICES), 0, s, a);
}
