// The token loss (mxm_vocab.h) around its three products: which rows take part,
// the operands' planes, the rows' losses and the logits' gradient.
#include <algorithm>

#include "mxm_vocab.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float load1(const void* p, bool bf16, int64_t at) {
  return bf16 ? mxm_bf2f(static_cast<const uint16_t*>(p)[at]) : static_cast<const float*>(p)[at];
}

__device__ __forceinline__ bool takes_part(const XentArgs& a, int64_t n, float& w) {
  const int t = a.targets[n];
  w = a.row_weights ? a.row_weights[n] : 1.0f;
  return t >= 0 && t < a.V && w != 0.0f;
}

// The rows that take part, in order, and the sum of their weights; zeros for the
// others' loss and lse.
constexpr int PLAN_NT = 1024;
__global__ __launch_bounds__(PLAN_NT) void xent_plan_kernel(XentArgs a) {
  __shared__ int wave_count[16];
  __shared__ double wave_weight[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t base = 0;
  double sum = 0.0;
  for (int64_t n0 = 0; n0 < a.rows; n0 += PLAN_NT) {
    const int64_t n = n0 + threadIdx.x;
    float w = 0.0f;
    const bool in = n < a.rows && takes_part(a, n, w);
    const unsigned long long m = __ballot(in);
    if (lane == 0) wave_count[wave] = __popcll(m);
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 16; ++i) {
      before += i < wave ? wave_count[i] : 0;
      all += wave_count[i];
    }
    const int64_t at = base + before + __popcll(m & ((1ull << lane) - 1));
    if (in) {
      a.map[at] = (int32_t)n;
      sum += (double)w;
    } else if (n < a.rows) {
      if (a.loss) a.loss[n] = 0.0f;
      if (a.lse) a.lse[n] = 0.0f;
    }
    if (n < a.rows) a.slot[n] = in ? (int32_t)at : -1;
    base += all;
    __syncthreads();
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) wave_weight[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < 16; ++i) s += wave_weight[i];
    a.scalars->weight_sum = s;
    a.scalars->rows = (int32_t)base;
  }
}

// v as hi + mid + lo, each a bf16: 24 bits, all of v's.  The differences are exact.
// Infinities become the largest bf16 (an infinite plane times another operand's
// mid plane, of any sign or zero, would make a NaN of every product).
__device__ __forceinline__ void planes3(float v, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
  const float c = v != v ? v : fminf(fmaxf(v, -3.3895313892515355e38f), 3.3895313892515355e38f);
  hi = mxm_f2bf_fast(c);
  const float r = c - mxm_bf2f(hi);
  mid = mxm_f2bf_fast(r);
  lo = mxm_f2bf_fast(r - mxm_bf2f(mid));
}

constexpr int NT = 256;

// Row `src` of x or weight to row `to` of its pack of `rows` rows, zeros behind D.
__device__ __forceinline__ void pack_row(const XentArgs& a, const void* p, int64_t src, uint16_t* pack,
                                         int64_t rows, int64_t to, int t, int T) {
  for (int d = t; d < a.Dp; d += T) {
    const int64_t at = to * a.Dp + d;
    if (a.planes == 1) {
      pack[at] = d < a.D ? static_cast<const uint16_t*>(p)[src * a.D + d] : (uint16_t)0;
    } else {
      uint16_t hi = 0, mid = 0, lo = 0;
      if (d < a.D) planes3(static_cast<const float*>(p)[src * a.D + d], hi, mid, lo);
      const int64_t plane = rows * a.Dp;
      pack[at] = hi;
      pack[at + plane] = mid;
      pack[at + 2 * plane] = lo;
    }
  }
}

// x's rows that take part to their places, and dx's others to zeros.
__global__ __launch_bounds__(NT) void xent_pack_x_kernel(XentArgs a) {
  const int lane = threadIdx.x & 63;
  for (int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); n < a.rows; n += (int64_t)gridDim.x * 4) {
    const int to = a.slot[n];
    if (to >= 0) {
      pack_row(a, a.x, n, a.x_pack, a.x_rows, to, lane, 64);
    } else if (a.dx) {
      for (int d = lane; d < a.D; d += 64) {
        if (a.dx_bf16)
          static_cast<uint16_t*>(a.dx)[n * a.D + d] = 0;
        else
          static_cast<float*>(a.dx)[n * a.D + d] = 0.0f;
      }
    }
  }
}

__global__ __launch_bounds__(NT) void xent_pack_w_kernel(XentArgs a) {
  const int lane = threadIdx.x & 63;
  for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < a.V; v += (int64_t)gridDim.x * 4)
    pack_row(a, a.weight, v, a.w_pack, a.V, v, lane, 64);
}

// 16 rows by 16 threads: each row's blocks joined.
constexpr int JOIN_ROWS = 16;
__global__ __launch_bounds__(NT) void xent_join_kernel(XentArgs a, int64_t r0, int blocks) {
  __shared__ float red[2][16][JOIN_ROWS];
  const int rows = mxm_xent_rows(a, r0);
  const int m = blockIdx.x * JOIN_ROWS + (threadIdx.x & 15), part = threadIdx.x >> 4;
  if (blockIdx.x * JOIN_ROWS >= rows) return;
  const bool in = m < rows;
  float top = -__builtin_inff(), sum = 0.0f;
  for (int b = part; in && b < blocks; b += 16) {
    const float2 e = a.stat[(int64_t)b * a.stat_ld + m];
    const float up = fmaxf(top, e.y);
    // (ref and top agree where both are infinite: no difference to take)
    sum = sum * (top == up ? 1.0f : __builtin_amdgcn_exp2f(top - up)) +
          e.x * (e.y == up ? 1.0f : __builtin_amdgcn_exp2f(e.y - up));
    top = up;
  }
  red[0][part][threadIdx.x & 15] = top;
  red[1][part][threadIdx.x & 15] = sum;
  __syncthreads();
  if (part != 0 || !in) return;
  for (int p = 1; p < 16; ++p) {
    const float t = red[0][p][m & 15], s = red[1][p][m & 15], up = fmaxf(top, t);
    sum = sum * (top == up ? 1.0f : __builtin_amdgcn_exp2f(top - up)) +
          s * (t == up ? 1.0f : __builtin_amdgcn_exp2f(t - up));
    top = up;
  }
  // the others' sum is sum * 2^top, the target's exponential 2^(top - d)
  const float lt = a.at_target[r0 + m], d = fmaf(-lt, LOG2E, top);
  const float et = __builtin_amdgcn_exp2f(-d), whole = sum + et;
  // (next to the target's probability of one the loss keeps its digits)
  const bool near = d <= 60.0f;
  const float over = logf(whole);
  const float loss = near ? log1pf(sum * __builtin_amdgcn_exp2f(d)) : d * LN2 + over;
  const int64_t n = a.map[r0 + m];
  a.nll[r0 + m] = loss;
  if (a.loss) a.loss[n] = loss;
  if (a.lse) a.lse[n] = near ? lt + loss : top * LN2 + over;
  if (a.backward) {
    const double w = a.row_weights ? (double)a.row_weights[n] : 1.0;
    const float g = (float)((double)a.d_total * w / (a.mean ? a.scalars->weight_sum : 1.0));
    XentRow r;
    r.ref = top;
    r.scale = g / whole;
    float slope = 1.0f;
    if (a.softcap > 0.0f) {
      const float u = lt / a.softcap;
      slope = 1.0f - u * u;
    }
    r.at_target = -g * (sum / whole) * slope;
    r.target = a.targets[n];
    a.row[r0 + m] = r;
  }
}

// The summands of a piece to dz, 8 of a row per thread.
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <int PLANES>
__global__ __launch_bounds__(NT) void xent_finish_kernel(XentArgs a, int64_t r0, int block) {
  const int rows = mxm_xent_rows(a, r0), units = a.Vp / 8;
  for (int m = blockIdx.y; m < rows; m += gridDim.y) {
    const XentRow r = a.row[r0 + m];
    for (int u = blockIdx.x * NT + threadIdx.x; u < units; u += gridDim.x * NT) {
      const int v = u * 8;
      // (the last units may lie in padding behind the last block)
      const float ref = v < a.V ? a.stat[(int64_t)(v / block) * a.stat_ld + m].y : r.ref;
      const float f = r.scale * (ref == r.ref ? 1.0f : __builtin_amdgcn_exp2f(ref - r.ref));
      float e[8];
      const int64_t at = (int64_t)m * a.Vp + v;
      if constexpr (PLANES == 1) {
        const f16x8_t h = *reinterpret_cast<const f16x8_t*>(static_cast<const uint16_t*>(a.summands) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (float)h[i] * f;
      } else {
        const f32x4_t* q = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(a.summands) + at);
        const f32x4_t lo = q[0], hi = q[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = lo[i] * f, e[4 + i] = hi[i] * f;
      }
      const int t = r.target - v;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i == t ? r.at_target : (v + i < a.V ? e[i] : 0.0f);
      if constexpr (PLANES == 1) {
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mxm_pack_bf2_fast(e[2 * i], e[2 * i + 1]);
        *reinterpret_cast<u32x4_t*>(a.dz + at) = o;
      } else {
        uint16_t p[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) planes3(e[i], p[0][i], p[1][i], p[2][i]);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          u32x4_t o;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = p[k][2 * i] | (uint32_t)p[k][2 * i + 1] << 16;
          *reinterpret_cast<u32x4_t*>(a.dz + (int64_t)k * a.piece_rows * a.Vp + at) = o;
        }
      }
    }
  }
}

__global__ __launch_bounds__(PLAN_NT) void xent_total_kernel(XentArgs a) {
  __shared__ double part[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < a.scalars->rows; i += PLAN_NT)
    s += (double)a.nll[i] * (a.row_weights ? (double)a.row_weights[a.map[i]] : 1.0);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < 16; ++i) s += part[i];
    if (a.mean && a.scalars->rows > 0) s /= a.scalars->weight_sum;
    a.total[0] = (float)s;
  }
}

}  // namespace

void mxm_launch_xent(const XentArgs& a0, hipStream_t s) {
  XentArgs a = a0;
  a.w_direct = a.bf16 && a.D % 8 == 0 && (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0;
  const auto rows_grid = [&](int64_t n) { return (unsigned)std::min<int64_t>((n + 3) / 4, (int64_t)a.n_cu * 16); };
  xent_plan_kernel<<<1, PLAN_NT, 0, s>>>(a);
  if (a.rows > 0) {
    xent_pack_x_kernel<<<rows_grid(a.rows), NT, 0, s>>>(a);
    if (!a.w_direct) xent_pack_w_kernel<<<rows_grid(a.V), NT, 0, s>>>(a);
  }
  const int64_t pieces = std::max<int64_t>(1, (a.rows + a.piece_rows - 1) / a.piece_rows);
  for (int64_t p = 0; p < pieces; ++p) {
    const int64_t r0 = p * a.piece_rows, rows = std::min(a.rows - r0, a.piece_rows);
    if (rows > 0) {
      const int block = mxm_xent_block(rows);
      a.stat_ld = rows;
      mxm_launch_xent_logits(a, r0, rows, s);
      xent_join_kernel<<<(unsigned)((rows + JOIN_ROWS - 1) / JOIN_ROWS), NT, 0, s>>>(
          a, r0, (a.V + block - 1) / block);
      if (a.backward) {
        const unsigned gx = (unsigned)std::min((a.Vp / 8 + NT - 1) / NT, 64);
        const dim3 grid(gx, (unsigned)std::min<int64_t>(rows, std::max(1u, (unsigned)a.n_cu * 32 / gx)));
        if (a.planes == 1)
          xent_finish_kernel<1><<<grid, NT, 0, s>>>(a, r0, block);
        else
          xent_finish_kernel<3><<<grid, NT, 0, s>>>(a, r0, block);
      }
      if (a.dx) mxm_launch_xent_dx(a, r0, rows, s);
    }
    if (a.dw) mxm_launch_xent_dw(a, r0, rows, p == pieces - 1, s);
  }
  if (a.total) xent_total_kernel<<<1, PLAN_NT, 0, s>>>(a);
}
