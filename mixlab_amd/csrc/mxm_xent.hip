// The token loss (mxm_vocab.h): softmax cross entropy of hidden rows against the
// vocabulary's table.
#include <algorithm>

#include "mxm_vocab.h"

namespace {

__device__ __forceinline__ float load1(const void* p, bool bf16, int64_t at) {
  return bf16 ? mxm_bf2f(static_cast<const uint16_t*>(p)[at]) : static_cast<const float*>(p)[at];
}
__device__ __forceinline__ void store1(void* p, bool bf16, int64_t at, float v) {
  if (bf16)
    static_cast<uint16_t*>(p)[at] = mxm_f2bf(v);
  else
    static_cast<float*>(p)[at] = v;
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
    if (n < a.rows && !in) {
      if (a.loss) a.loss[n] = 0.0f;
      if (a.lse) a.lse[n] = 0.0f;
    }
    const unsigned long long m = __ballot(in);
    if (lane == 0) wave_count[wave] = __popcll(m);
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 16; ++i) {
      before += i < wave ? wave_count[i] : 0;
      all += wave_count[i];
    }
    if (in) {
      a.map[base + before + __popcll(m & ((1ull << lane) - 1))] = (int32_t)n;
      sum += (double)w;
    }
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

// A 64 x 64 tile of sum_k A(m, k) B(k, n), 16 x 16 threads of 4 x 4.
template <class FA, class FB>
__device__ __forceinline__ void tile64(int K, FA A, FB B, float (&c)[4][4]) {
  __shared__ float sa[16][65], sb[16][65];
  const int t = threadIdx.x, tm = t / 16, tn = t % 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.0f;
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int i = t; i < 1024; i += 256) {
      sa[i % 16][i / 16] = k0 + i % 16 < K ? A(i / 16, k0 + i % 16) : 0.0f;
      sb[i / 64][i % 64] = k0 + i / 64 < K ? B(k0 + i / 64, i % 64) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = sa[k][tm * 4 + i], bv[i] = sb[k][tn * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[i][j] = fmaf(av[i], bv[j], c[i][j]);
    }
    __syncthreads();
  }
}

// The rows of the piece that starts at row r0.
__device__ __forceinline__ int piece_rows(const XentArgs& a, int64_t r0) {
  const int64_t left = a.scalars->rows - r0;
  return left <= 0 ? 0 : (int)(left < a.piece_rows ? left : a.piece_rows);
}

__global__ __launch_bounds__(256) void xent_logits_kernel(XentArgs a, int64_t r0) {
  const int rows = piece_rows(a, r0), tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  const int n0 = blockIdx.x * 64;
  for (int m0 = blockIdx.y * 64; m0 < rows; m0 += gridDim.y * 64) {
    float c[4][4];
    tile64(
        a.D,
        [&](int m, int k) {
          return m0 + m < rows ? load1(a.x, a.bf16, (int64_t)a.map[r0 + m0 + m] * a.D + k) : 0.0f;
        },
        [&](int k, int n) {
          return n0 + n < a.V ? load1(a.weight, a.bf16, (int64_t)(n0 + n) * a.D + k) : 0.0f;
        },
        c);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + tm * 4 + i, n = n0 + tn * 4 + j;
        if (m < rows && n < a.V) {
          float z = c[i][j];
          if (a.softcap > 0.0f) z = a.softcap * tanhf(z / a.softcap);
          a.logits[(int64_t)m * a.V + n] = z;
        }
      }
  }
}

__device__ __forceinline__ float block_reduce(float v, bool max_of, float* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o);
    v = max_of ? fmaxf(v, u) : v + u;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int i = 1; i < 4; ++i) v = max_of ? fmaxf(v, lds[i]) : v + lds[i];
  __syncthreads();
  return v;
}

// A row's loss, and its logits' gradient in their place.
__global__ __launch_bounds__(256) void xent_row_kernel(XentArgs a, int64_t r0) {
  __shared__ float lds[4];
  const int rows = piece_rows(a, r0);
  for (int m = blockIdx.x; m < rows; m += gridDim.x) {
    float* l = a.logits + (int64_t)m * a.V;
    const int64_t n = a.map[r0 + m];
    const int t = a.targets[n];
    const float lt = l[t];
    float top = -__builtin_inff();
    for (int v = threadIdx.x; v < a.V; v += 256)
      if (v != t) top = fmaxf(top, l[v]);
    top = fmaxf(block_reduce(top, true, lds), lt);
    float s = 0.0f;
    for (int v = threadIdx.x; v < a.V; v += 256)
      if (v != t) s += expf(l[v] - top);
    s = block_reduce(s, false, lds);
    const float et = expf(lt - top), whole = s + et;
    const float loss = lt == top ? log1pf(s) : logf(whole) + (top - lt);
    if (threadIdx.x == 0) {
      a.nll[r0 + m] = loss;
      if (a.loss) a.loss[n] = loss;
      if (a.lse) a.lse[n] = lt == top ? log1pf(s) + lt : logf(whole) + top;
    }
    if (a.backward) {
      const float w = a.row_weights ? a.row_weights[n] : 1.0f;
      const float g = (float)((double)a.d_total * w / (a.mean ? a.scalars->weight_sum : 1.0));
      for (int v = threadIdx.x; v < a.V; v += 256) {
        const float z = l[v];
        float d = v == t ? -s / whole : expf(z - top) / whole;
        d *= g;
        if (a.softcap > 0.0f) {
          const float u = z / a.softcap;
          d *= 1.0f - u * u;
        }
        l[v] = d;
      }
    }
  }
}

__global__ __launch_bounds__(256) void xent_dx_kernel(XentArgs a, int64_t r0) {
  const int rows = piece_rows(a, r0), tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  const int d0 = blockIdx.x * 64;
  for (int m0 = blockIdx.y * 64; m0 < rows; m0 += gridDim.y * 64) {
    float c[4][4];
    tile64(
        a.V, [&](int m, int k) { return m0 + m < rows ? a.logits[(int64_t)(m0 + m) * a.V + k] : 0.0f; },
        [&](int k, int n) {
          return d0 + n < a.D ? load1(a.weight, a.bf16, (int64_t)k * a.D + d0 + n) : 0.0f;
        },
        c);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + tm * 4 + i, d = d0 + tn * 4 + j;
        if (m < rows && d < a.D)
          store1(a.dx, a.dx_bf16, (int64_t)a.map[r0 + m] * a.D + d, c[i][j]);
      }
  }
}

__global__ __launch_bounds__(256) void xent_dw_kernel(XentArgs a, int64_t r0, bool last) {
  const int rows = piece_rows(a, r0), tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  const int d0 = blockIdx.x * 64;
  for (int v0 = blockIdx.y * 64; v0 < a.V; v0 += gridDim.y * 64) {
    float c[4][4];
    tile64(
        rows, [&](int m, int k) { return v0 + m < a.V ? a.logits[(int64_t)k * a.V + v0 + m] : 0.0f; },
        [&](int k, int n) {
          return d0 + n < a.D ? load1(a.x, a.bf16, (int64_t)a.map[r0 + k] * a.D + d0 + n) : 0.0f;
        },
        c);
    float* acc = a.dw_bf16 ? a.dw32 : static_cast<float*>(a.dw);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int v = v0 + tm * 4 + i, d = d0 + tn * 4 + j;
        if (v < a.V && d < a.D) {
          const int64_t at = (int64_t)v * a.D + d;
          const float s = r0 > 0 ? acc[at] + c[i][j] : c[i][j];
          if (last)
            store1(a.dw, a.dw_bf16, at, s);
          else
            acc[at] = s;
        }
      }
  }
}

// Zeros in dx for the rows that take no part.
__global__ __launch_bounds__(256) void xent_zero_kernel(XentArgs a) {
  for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
    float w;
    if (takes_part(a, n, w)) continue;
    for (int d = threadIdx.x; d < a.D; d += 256) store1(a.dx, a.dx_bf16, n * a.D + d, 0.0f);
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

void mxm_launch_xent(const XentArgs& a, hipStream_t s) {
  xent_plan_kernel<<<1, PLAN_NT, 0, s>>>(a);
  const int64_t pieces = std::max<int64_t>(1, (a.rows + a.piece_rows - 1) / a.piece_rows);
  const auto tiles = [](int64_t n, int64_t most) { return (unsigned)std::min((n + 63) / 64, most); };
  for (int64_t p = 0; p < pieces; ++p) {
    const int64_t r0 = p * a.piece_rows, rows = std::min(a.rows - r0, a.piece_rows);
    if (rows > 0) {
      xent_logits_kernel<<<dim3(tiles(a.V, 1 << 20), tiles(rows, 64)), 256, 0, s>>>(a, r0);
      xent_row_kernel<<<(unsigned)std::min<int64_t>(rows, 8192), 256, 0, s>>>(a, r0);
    }
    if (rows > 0 && a.dx) xent_dx_kernel<<<dim3(tiles(a.D, 1024), tiles(rows, 4096)), 256, 0, s>>>(a, r0);
    if (a.dw) xent_dw_kernel<<<dim3(tiles(a.D, 1024), tiles(a.V, 4096)), 256, 0, s>>>(a, r0, p == pieces - 1);
  }
  if (a.dx && a.rows > 0) xent_zero_kernel<<<(unsigned)std::min<int64_t>(a.rows, 8192), 256, 0, s>>>(a);
  if (a.total) xent_total_kernel<<<1, PLAN_NT, 0, s>>>(a);
}
