// The residual norm's backward (formulas in mxm_train.h): one pass over the rows
// with the gradients of the stream and the branch, column sums of the scales'
// and the gate's gradients kept in registers over a chunk of rows, and a second
// launch that joins the chunks in their order.  Bound by memory: 65,536 rows of
// 2048 channels in fp32 559 us (3.22 GB over six streams at 5.8 TB/s; 656 us at a
// large copy's rate), the join 4.8 of them.
#include <algorithm>

#include "mxm_resnorm.h"

namespace {

using namespace resnorm;

// The rows of a chunk: first, first + step, ... (count of them).  Neighbouring
// chunks hold neighbouring rows, so that the workgroups sweep over memory side
// by side; chunks of whole groups of gate rows hold theirs in a row.
struct Rows {
  int first, step, count;
};
__device__ __forceinline__ Rows rows_of(const ResNormArgs& a, int c) {
  if (c >= a.chunks) return {0, 1, 0};
  int first = c, step = a.chunks, end = a.N;
  if (a.group_chunks > 0) {
    const int g = c / a.group_chunks;
    first = (int)min((int64_t)g * a.gate_rows + c % a.group_chunks, (int64_t)a.N);
    step = a.group_chunks;
    end = (int)min((int64_t)(g + 1) * a.gate_rows, (int64_t)a.N);
  } else if (a.gate && a.gate_rows > 1) {
    first = (int)min((int64_t)c * a.chunk_rows, (int64_t)a.N);
    step = 1;
    end = (int)min((int64_t)first + a.chunk_rows, (int64_t)a.N);
  }
  return {first, step, first < end ? (int)(((int64_t)end - first + step - 1) / step) : 0};
}

// A gate between its load and its gradient.  Of a sigmoid a that is a where a < 1/2,
// else -(1 - a), for its slope a (1 - a): 1 - a has few digits where a is next to 1
// (the slope 10 % off at 15 and 0 past 17), and two values an element do not fit
// the registers.  k - floor(k) is a again, at most 1 - 2^-24.
constexpr float LEAST_TAIL = 1.17549435e-38f;  // (so that 1 has a sign)
__device__ __forceinline__ float gate_kept(const ResNormArgs& a, float g) {
  if (!a.sigmoid) return g;
  const float tail = mxm_sigmoid(-__builtin_fabsf(g));
  return g < 0.0f ? tail : tail < LEAST_TAIL ? -LEAST_TAIL : -tail;
}
__device__ __forceinline__ float gate_value(const ResNormArgs& a, float k) {
  return a.sigmoid ? __builtin_amdgcn_fractf(k) : k;
}
__device__ __forceinline__ float gate_slope(float k) {
  const float tail = __builtin_fabsf(k);
  return tail <= LEAST_TAIL ? 0.0f : tail * (1.0f - tail);
}

// CH: a gate per channel.  A row's threads walk one chunk; the chunks of a
// workgroup add their column sums in LDS and store one partial.
template <int NV, int LPR, int XT, int DT, int GT, int ODD, bool CH>
__global__ __launch_bounds__(most_threads(LPR)) void resnorm_bw_kernel(ResNormArgs a) {
  constexpr int E = V * NV;
  // of a row's sums (a workgroup a row), or of the workgroup's column sums at the end
  __shared__ float red[LPR > 0 ? THREADS * E : 2 * 16 * 3 + 2 * 16];
  const int lane = LPR > 0 ? threadIdx.x % (LPR > 0 ? LPR : 1) : threadIdx.x;
  const int stride = LPR > 0 ? LPR : blockDim.x;
  const int rows = LPR > 0 ? THREADS / (LPR > 0 ? LPR : 1) : 1;
  const int proc = row_slot<LPR>();
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
        load_scale<ODD>(a.scale, a.p_bf16, 0, at[i], D, f + i * V);
        load_scale<ODD>(a.post, a.p_bf16, 0, at[i], D, p);
#pragma unroll
        for (int j = 0; j < V; ++j) f[i * V + j] *= p[j];
      }
      if (a.norm) load_scale<ODD>(a.w, a.p_bf16, 0, at[i], D, w + i * V);
    }
  }
  if (!CH) {
    ag[0] = 0.0f;
    ga[0] = 1.0f;
  }
  const Rows mine = rows_of(a, c);
  int group = a.gate ? mine.first / a.gate_rows : 0;
  // the chunk's rows before its group ends: whole groups (in a row), or one group
  int left = a.group_chunks > 0 ? mine.count : a.gate_rows;
  bool fresh = true;  // the group's gate is not loaded yet
  Raw<XT> rh[NV];
  Raw<DT> rd[NV];
  Raw<GT> rt[NV], ry[NV];
  float rg = 0.0f;  // a gate of the row alone
  const bool row_gate = !CH && a.gate && a.gate_rows == 1;
  // (values past the row's end and rows past the chunk's are zero)
  auto fetch = [&](int it) {
    const size_t row = ((size_t)mine.first + (size_t)it * mine.step) * D;
    if (row_gate && it < mine.count)
      rg = load_one(a.gatep, a.p_bf16, (size_t)mine.first + (size_t)it * mine.step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      rh[i] = Raw<XT>{};
      rd[i] = Raw<DT>{};
      rt[i] = Raw<GT>{};
      ry[i] = Raw<GT>{};
      if (it < mine.count && at[i] < D) {
        if (a.norm) {
          rh[i] = load<XT, ODD>(a.h, row, at[i], D);
          ry[i] = load<GT, ODD>(a.dy, row, at[i], D);
        }
        if (a.branch) rd[i] = load<DT, ODD>(a.delta, row, at[i], D);
        if (a.dh) rt[i] = load<GT, ODD>(a.dh, row, at[i], D);
      }
    }
  };
  if (LPR >= 0) fetch(0);
  // (the same number of rounds in every lane: the sums use whole waves)
  const int rounds = LPR > 0 ? a.chunk_rows : mine.count;
  for (int it = 0; it < rounds; ++it) {
    const bool valid = LPR <= 0 || it < mine.count;
    const size_t row = ((size_t)mine.first + (size_t)it * mine.step) * D;
    float h[E], dl[E], t[E], dy[E];
    if (LPR < 0) fetch(it);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<XT, ODD>(rh[i], at[i], D, h + i * V);
      unpack<DT, ODD>(rd[i], at[i], D, dl + i * V);
      unpack<GT, ODD>(rt[i], at[i], D, t + i * V);
      unpack<GT, ODD>(ry[i], at[i], D, dy + i * V);
    }
    // (the gate's values go through the sigmoid after the sums, which hide its load)
    const bool new_gate = a.gate && fresh && valid;
    if (row_gate) ga[0] = rg;
    if (LPR >= 0 && it + 1 < rounds) fetch(it + 1);
    if (new_gate && !row_gate) {
      if (CH) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (at[i] < D)
            load_scale<ODD>(a.gatep, a.p_bf16, (size_t)group * D, at[i], D, ga + (CH ? i * V : 0));
      } else {
        ga[0] = load_one(a.gatep, a.p_bf16, (size_t)group);
      }
    }
    float s[3] = {0.0f, 0.0f, 0.0f};
    if (a.norm) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[0] = __builtin_fmaf(h[e], h[e], s[0]);
        s[1] = __builtin_fmaf(w[e] * dy[e], h[e], s[1]);
      }
    }
    if (post) {
#pragma unroll
      for (int e = 0; e < E; ++e) s[2] = __builtin_fmaf(dl[e], dl[e], s[2]);
    }
    if (a.norm || post) row_sum<LPR>(s, red + (it & 1) * 48);
    if (a.norm) {
      const float rn = 1.0f / __builtin_sqrtf(s[0] * a.inv_d + a.eps);
      const float k = rn * (s[1] * a.inv_d);  // (rn^3 leaves fp32's range where rn does not)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float hn = rn * h[e];
        t[e] = __builtin_fmaf(rn, __builtin_fmaf(-k, hn, w[e] * dy[e]), t[e]);
        if (valid) aw[e] = __builtin_fmaf(dy[e], hn, aw[e]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!(valid && at[i] < D && a.dx)) continue;
      float out[V];
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = t[i * V + j];
      store<GT, ODD>(a.dx, row, at[i], D, out);
    }
    if (new_gate) {
#pragma unroll
      for (int e = 0; e < (CH ? E : 1); ++e) ga[e] = gate_kept(a, ga[e]);
      fresh = false;
    }
    if (a.branch) {
      const float rp = post ? 1.0f / __builtin_sqrtf(s[2] * a.inv_d + a.eps) : 1.0f;
      // q = sum f t z, times the gate where that differs by channel
      float q[1] = {0.0f};
      const float g = CH || !a.gate ? 1.0f : gate_value(a, ga[0]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dl[e] = rp * dl[e];  // z
        const float tz = t[e] * dl[e];
        const float gv = CH ? gate_value(a, ga[CH ? e : 0]) : 1.0f;
        const float gt = CH ? gv * tz : tz;
        if (valid) {  // (past the chunk's rows 1 / sqrt(eps) or a gate times 0 need not be 0)
          aq[e] = __builtin_fmaf(g, gt, aq[e]);
          if (CH) ag[CH ? e : 0] = __builtin_fmaf(f[e], tz, ag[CH ? e : 0]);
        }
        q[0] = __builtin_fmaf(f[e], gt, q[0]);
        t[e] = (CH ? gv * f[e] : f[e]) * t[e];
      }
      if (post || a.gate == 1) row_sum<LPR>(q, red + 96 + (it & 1) * 16);
      if (!CH && valid) ag[0] = ag[0] + q[0];
      if (post) {  // (else nothing of delta, which may be infinite)
        const float k = q[0] * a.inv_d;
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = __builtin_fmaf(-k, dl[e], t[e]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!(valid && at[i] < D)) continue;
        float out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = (g * rp) * t[i * V + j];
        store<GT, ODD>(a.d_delta, row, at[i], D, out);
      }
    }
    // the group's last row here
    if (a.gate && valid && (--left == 0 || it + 1 == mine.count)) {
      if (a.sigmoid) {
#pragma unroll
        for (int e = 0; e < (CH ? E : 1); ++e) ag[e] = ag[e] * gate_slope(ga[e]);
      }
      if (a.group_chunks == 0) {  // the group is whole: its gate's gradient goes out
        if (a.d_gate) {
          float* out = a.d_gate + (size_t)group * (CH ? D : 1);
          if (CH) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
              if (at[i] < D)
#pragma unroll
                for (int j = 0; j < V; ++j)
                  if (!ODD || at[i] + j < D) out[at[i] + j] = ag[CH ? i * V + j : 0];
          } else if (lane == 0) {
            out[0] = ag[0];
          }
        }
#pragma unroll
        for (int e = 0; e < (CH ? E : 1); ++e) ag[e] = 0.0f;
      }
      group += a.gate_rows == 1 ? mine.step : 1;
      left = a.gate_rows;
      fresh = true;
    }
  }
  // One partial a workgroup, of its rows' sums in their order: n values a thread
  // in columns, or one (a gate per row).
  auto join = [&](auto& acc, float* part) {
    constexpr int n = sizeof acc / sizeof acc[0];
    if (LPR > 0) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < n; ++e) red[LPR > 0 ? e * THREADS + threadIdx.x : 0] = acc[e];
      __syncthreads();
      if (proc > 0) return;
#pragma unroll
      for (int e = 0; e < n; ++e)
        for (int p = 1; p < rows; ++p) acc[e] += red[LPR > 0 ? e * THREADS + p * LPR + lane : 0];
    }
    if constexpr (n == 1) {
      if (lane == 0) part[0] = acc[0];
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at[i] < D)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!ODD || at[i] + j < D) part[at[i] + j] = acc[i * V + j];
    }
  };
  if (a.norm && a.d_w) join(aw, a.part + (size_t)blockIdx.x * D);
  if (a.branch && (a.d_scale || a.d_post)) join(aq, a.part + ((size_t)a.parts + blockIdx.x) * D);
  if (a.gate && a.group_chunks > 0 && a.d_gate)
    join(ag, a.gate_part + (size_t)blockIdx.x * (CH ? D : 1));
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
  const int count = kind == 2 ? a.group_parts : a.parts;
  const float* src = kind == 2 ? a.gate_part + (size_t)group * a.group_parts * width
                               : a.part + (size_t)kind * a.parts * a.D;
  float s = 0.0f;
  if (d < width) {
    int p = slice;
    for (; p + 7 * JOIN_SLICES < count; p += 8 * JOIN_SLICES) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = src[(size_t)(p + k * JOIN_SLICES) * width + d];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; p < count; p += JOIN_SLICES) s += src[(size_t)p * width + d];
  }
  red[slice][col] = s;
  __syncthreads();
  if (slice != 0 || d >= width) return;
  s = 0.0f;
  for (int i = 0; i < JOIN_SLICES; ++i) s += red[i][col];
  if (kind == 0) {
    a.d_w[d] = s;
  } else if (kind == 1) {
    // (both before the stores: a gradient may take its scale's place)
    const float post = a.post ? load_one(a.post, a.p_bf16, d) : 1.0f;
    const float scale = a.scale ? load_one(a.scale, a.p_bf16, d) : 1.0f;
    if (a.d_scale) a.d_scale[d] = s * post;
    if (a.d_post) a.d_post[d] = s * scale;
  } else {
    a.d_gate[(size_t)group * width + d] = s;
  }
}

// Chunks that a backward of N rows aims at: some workgroups a CU, of no fewer
// rows than pay for a partial.  134 M elements in fp32 at 512, 1024, 2048 and 4096
// channels with 2 / 4 / 8 workgroups a CU: 545 / 603 / 608, 576 / 589 / 593, 568 /
// 659 / 645 and 564 / 628 / 664 us (5.7 TB/s with 2): each has its next row's loads
// on their way, and fewer streams at once suit the memory better.  Rows of one
// vector a thread need 4 for as many bytes on their way (64 and 256 channels 655
// / 629 and 637 / 629), and three waves a row in bf16 3 (1032 and 1536 channels
// 537 / 421 and 377 / 311).
int wgs_per_cu(const Shape& sh, bool bf16) {
  return sh.NV == 1 ? 4 : bf16 && sh.lpr == 0 && sh.threads < 256 ? 3 : 2;
}
int fewest_rows(const Shape& sh) { return sh.lpr > 0 && sh.lpr < 64 ? 1 : 2; }
int rows_per_chunk(const Shape& sh, bool bf16, int64_t N, int n_cu) {
  const int64_t target = (int64_t)wgs_per_cu(sh, bf16) * n_cu * sh.rows();
  return (int)std::max<int64_t>((N + target - 1) / target, fewest_rows(sh));
}

// Splits a.N rows into chunks.
void plan(ResNormArgs& a, const Shape& sh) {
  const int rows = rows_per_chunk(sh, a.x_bf16 && a.g_bf16, a.N, a.n_cu);
  const int T = std::min(a.gate_rows, a.N);  // rows of the longest group
  a.group_chunks = a.group_parts = 0;
  a.chunk_rows = rows;
  if (a.gate && a.gate_rows > 1) {
    const int groups = (int)(((int64_t)a.N + a.gate_rows - 1) / a.gate_rows);
    if (T >= (int64_t)rows * sh.rows()) {
      // a group fills workgroups: whole workgroups of chunks for each
      a.group_parts = (int)(((int64_t)T + (int64_t)rows * sh.rows() - 1) / ((int64_t)rows * sh.rows()));
      a.group_chunks = a.group_parts * sh.rows();
      a.chunk_rows = (T + a.group_chunks - 1) / a.group_chunks;
      a.chunks = groups * a.group_chunks;
      a.parts = groups * a.group_parts;
      return;
    }
    // chunks of whole groups (or of the only one)
    a.chunk_rows = T <= rows ? rows / T * T : T;
  }
  a.chunks = (a.N + a.chunk_rows - 1) / a.chunk_rows;
  if (!(a.gate && a.gate_rows > 1)) a.chunk_rows = (a.N + a.chunks - 1) / a.chunks;
  a.parts = (a.chunks + sh.rows() - 1) / sh.rows();
}

template <int NV, int LPR, int XT, int DT, int GT, int ODD>
void launch(const ResNormArgs& a, const Shape& sh, hipStream_t s) {
  if (a.gate == 2)
    hipLaunchKernelGGL((resnorm_bw_kernel<NV, LPR, XT, DT, GT, ODD, true>), dim3(a.parts),
                       dim3(sh.threads), 0, s, a);
  else
    hipLaunchKernelGGL((resnorm_bw_kernel<NV, LPR, XT, DT, GT, ODD, false>), dim3(a.parts),
                       dim3(sh.threads), 0, s, a);
}

}  // namespace

int64_t mxm_resnorm_max_parts(int64_t max_rows, int D, bool bf16, bool groups, int n_cu) {
  // A workgroup's R = rows() * rows_per_chunk rows.  Without groups ceil(N / R)
  // parts, at most the target and at most ceil(N / (rows() * fewest)); chunks of
  // whole groups hold more than half of the rows aimed at; groups that fill
  // workgroups (T >= R) have at most T / R + 1 parts each, and there are at most
  // N / T + 1 of them: N / R + T / R + N / T + 1 <= 3 N / R + 1.
  int64_t most = 0;
  for (const int64_t rows : {max_rows, std::min<int64_t>(max_rows, FEW_ROWS)}) {
    const Shape sh = shape_of(D, true, rows);
    const int64_t R = (int64_t)sh.rows() * fewest_rows(sh);
    most = std::max(most, std::min<int64_t>((int64_t)wgs_per_cu(sh, bf16) * n_cu, (rows + R - 1) / R));
  }
  return groups ? 3 * most + 1 : most;
}

bool mxm_launch_resnorm_bw(const ResNormArgs& args, hipStream_t s) {
  ResNormArgs a = args;
  const bool vectors =
      a.D % 4 == 0 && (!a.norm || (aligned(a.h, a.x_bf16) && aligned(a.dy, a.g_bf16))) &&
      (!a.branch || (aligned(a.delta, a.delta_bf16) && aligned(a.d_delta, a.g_bf16))) &&
      aligned(a.dh, a.g_bf16) && aligned(a.dx, a.g_bf16);
  const Shape sh = shape_of(a.D, true, a.N);
  a.chunks = a.parts = a.group_chunks = a.group_parts = 0;
  if (a.N > 0) {
    plan(a, sh);
    if (a.parts > a.max_parts) return false;
    with_shape<true>(sh, [&](auto nv, auto lpr) {
      with_types(a.x_bf16, a.delta_bf16, a.g_bf16, !vectors, [&](auto xt, auto dt, auto gt, auto odd) {
        launch<nv(), lpr(), xt(), dt(), gt(), odd() ? lpr() == 16 ? 2 : 1 : 0>(a, sh, s);
      });
    });
  }
  // (without rows the scales' gradients are zero)
  const bool columns = (a.norm && a.d_w) || (a.branch && (a.d_scale || a.d_post));
  const bool gates = a.gate && a.group_chunks > 0 && a.d_gate;
  if (columns || gates) {
    const dim3 grid((a.D + JOIN_COLS - 1) / JOIN_COLS, 2 + (gates ? a.parts / a.group_parts : 0));
    hipLaunchKernelGGL(resnorm_join_kernel, grid, dim3(JOIN_COLS * JOIN_SLICES), 0, s, a);
  }
  return true;
}
