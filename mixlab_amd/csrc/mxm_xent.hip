// The token loss (mxm_vocab.h) around its three products: which rows take part,
// the operands' planes, the rows' losses and the logits' gradient.
#include <algorithm>

#include "mxm_vocab.h"

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ bool takes_part(const XentArgs& a, int64_t n, int& t, float& w) {
  return mxm_xent_takes_part(a.targets, a.row_weights, a.V, n, t, w);
}
__device__ __forceinline__ void leave_out(const XentArgs& a, int64_t n) {
  if (a.loss) a.loss[n] = 0.0f;
  if (a.lse) a.lse[n] = 0.0f;
}

// How many rows of each chunk take part, and the sum of their weights; a wave per chunk.
constexpr int NT = 256;
__global__ __launch_bounds__(NT) void xent_count_kernel(XentArgs a, int64_t chunk, int chunks) {
  const int lane = threadIdx.x & 63, c = blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (c >= chunks) return;
  int count = 0;
  double sum = 0.0;
  const int64_t from = c * chunk, to = min(from + chunk, a.rows);
  for (int64_t n = from + lane; n < to; n += 64) {
    int t;
    float w;
    if (takes_part(a, n, t, w)) {
      ++count;
      sum += (double)w;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    count += __shfl_xor(count, o);
    sum += __shfl_xor(sum, o);
  }
  if (lane == 0) {
    a.counts[c] = count;
    a.weights[c] = sum;
  }
}

// v as hi + lo of fp16 (the difference is exact; an infinity has no lo).
__device__ __forceinline__ void planes2(float v, uint16_t& hi, uint16_t& lo) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(__builtin_isinf((float)h) ? 0.0f : v - (float)h);
  hi = __builtin_bit_cast(uint16_t, h);
  lo = __builtin_bit_cast(uint16_t, l);
}
__device__ __forceinline__ void planes2x8(const float (&v)[8], u32x4_t (&q)[2]) {
  uint16_t p[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) planes2(v[i], p[0][i], p[1][i]);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) q[k][i] = p[k][2 * i] | (uint32_t)p[k][2 * i + 1] << 16;
}

// The 8 elements at p, of which `left` are a row's, zeros behind them: vectors at the
// elements' alignment, so that rows of any width and place are read alike (the losses of
// 67 rows of D 1001 against 50257 entries 85 us with element loads, 65 so).
__device__ __forceinline__ u32x4_t load8(const uint16_t* p, int left) {
  typedef unsigned int at2_t __attribute__((ext_vector_type(4), aligned(2)));
  if (left >= 8) return *reinterpret_cast<const at2_t*>(p);
  u32x4_t q = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) q[i / 2] |= (uint32_t)p[i] << 16 * (i % 2);
  return q;
}
__device__ __forceinline__ void load8(const float* p, int left, float (&v)[8]) {
  typedef float at4_t __attribute__((ext_vector_type(4), aligned(4)));
  if (left >= 8) {
    const f32x4_t lo = *reinterpret_cast<const at4_t*>(p), hi = *reinterpret_cast<const at4_t*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.0f;
  }
}

// Row `src` of x or weight to row `to` of its pack of `rows` rows, zeros behind D, by a
// wave.
__device__ __forceinline__ void pack_row(const XentArgs& a, const void* p, int64_t src, uint16_t* pack, int64_t to,
                                         int lane) {
  const uint16_t* from = static_cast<const uint16_t*>(p) + src * a.D;
  pack += to * a.Dp;
  for (int d = lane * 8; d < a.Dp; d += 512) *reinterpret_cast<u32x4_t*>(pack + d) = load8(from + d, a.D - d);
}

// The same of an fp32 row, to planes; returns its exponent.
template <bool WEIGHT>
__device__ __forceinline__ int pack_row32(const XentArgs& a, const void* p, int64_t src, uint16_t* pack, int64_t rows,
                                          int64_t to, int lane) {
  const float* from = static_cast<const float*>(p) + src * a.D;
  const int64_t plane = rows * a.Dp;
  pack += to * a.Dp;
  // the largest finite element (of their bits, which are ordered alike), any infinity
  uint32_t top = 0;
  bool inf = false;
  for (int d = lane * 8; d < a.D; d += 512) {
    float v[8];
    load8(from + d, a.D - d, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = mxm_f2u(v[i]) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);
      inf |= u == 0x7f800000u;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  const bool signs = WEIGHT && __ballot(inf) != 0;
  int e = WEIGHT ? XENT_ZERO : 0;
  if (top != 0) {
    (void)frexpf(mxm_u2f(top), &e);
    e = max(e - 15, -126);
  }
  auto scaled = [&](float v) {
    if (!signs) return ldexpf(v, -e);
    return v != v ? v : __builtin_isinf(v) ? __builtin_copysignf(1.0f, v) : 0.0f;
  };
  for (int d = lane * 8; d < a.Dp; d += 512) {
    float v[8];
    load8(from + d, a.D - d, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = scaled(v[i]);
    u32x4_t q[2];
    planes2x8(v, q);
    *reinterpret_cast<u32x4_t*>(pack + d) = q[0];
    *reinterpret_cast<u32x4_t*>(pack + plane + d) = q[1];
  }
  return signs ? XENT_INF : e;
}

// x's rows that take part to their places, dx's others to zeros; a workgroup per chunk
// of rows, a wave per row.  The places are in the rows' order; every workgroup counts the
// rows before its own: PLAN, for up to PLAN_ROWS rows, by itself, else from the chunks'
// counts (the losses of 2000 rows of D 64 and 1000 entries take 18.1 us by chunks and 15.8
// so; of 4000 21.2, 19.8; counted by one workgroup, those of 48000 took 89 us and by chunks
// 71).
constexpr int PLAN_ROWS = 4096;
// The workgroups behind the first x_blocks pack the table.
template <bool PLAN>
__global__ __launch_bounds__(NT) void xent_pack_kernel(XentArgs a, int x_blocks, int64_t chunk) {
  __shared__ int count[2][4];
  __shared__ double weight[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= x_blocks) {
    for (int64_t v = (int64_t)(blockIdx.x - x_blocks) * 4 + wave; v < a.V; v += (int64_t)(gridDim.x - x_blocks) * 4) {
      if (a.planes == 1) {
        pack_row(a, a.weight, v, a.w_pack, v, lane);
      } else {
        const int e = pack_row32<true>(a, a.weight, v, a.w_pack, a.V, v, lane);
        if (lane == 0) a.w_exp[v] = e;
      }
    }
    return;
  }
  const int64_t from = blockIdx.x * chunk, end = min(from + chunk, a.rows);
  int before = 0, all = 0;
  double sum = 0.0;
  if constexpr (PLAN) {
#pragma unroll 4
    for (int k = threadIdx.x; k < (int)a.rows; k += NT) {
      int t;
      float w = 0.0f;
      if (takes_part(a, k, t, w)) {
        before += k < from;
        ++all;
        sum += (double)w;
      }
    }
  } else {
#pragma unroll 4
    for (int c = threadIdx.x; c < x_blocks; c += NT) {
      const int n = a.counts[c];
      before += c < (int)blockIdx.x ? n : 0;
      all += n;
      if (blockIdx.x == 0) sum += a.weights[c];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    before += __shfl_xor(before, o);
    all += __shfl_xor(all, o);
    sum += __shfl_xor(sum, o);
  }
  if (lane == 0) count[0][wave] = before, count[1][wave] = all, weight[wave] = sum;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.scalars->rows = count[1][0] + count[1][1] + count[1][2] + count[1][3];
    a.scalars->weight_sum = ((weight[0] + weight[1]) + weight[2]) + weight[3];
  }
  int at = count[0][0] + count[0][1] + count[0][2] + count[0][3];
  for (int64_t first = from; first < end; first += 4) {
    const int64_t n = first + wave;
    int to = -1, target = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // (uniform in the wave)
      int t;
      float w;
      const bool in = first + k < end && takes_part(a, first + k, t, w);
      if (k == wave && in) to = at, target = t;
      at += in;
    }
    if (n >= end) continue;
    if (lane == 0) {
      if (to >= 0) {
        a.map[to] = (int32_t)n;
        a.target[to] = target;
      } else {
        leave_out(a, n);
      }
    }
    if (to >= 0) {
      if (a.planes == 1) {
        pack_row(a, a.x, n, a.x_pack, to, lane);
      } else {
        const int e = pack_row32<false>(a, a.x, n, a.x_pack, a.x_rows, to, lane);
        if (lane == 0) a.x_exp[to] = e;
      }
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

// What a set of exponentials sums to: sum * 2^top; exp: that of the largest summand times
// 2^w, over 2^top too.
struct Sum {
  float top, sum;
  int exp;
};
__device__ __forceinline__ int moved(int exp, float top, float up) {
  return top == up ? exp : max(exp + (int)fmaxf(top - up, (float)XENT_NO_EXP), XENT_NO_EXP);
}
__device__ __forceinline__ Sum join(Sum p, Sum q) {
  // (no difference of equal ones: they may be infinite)
  const float up = fmaxf(p.top, q.top);
  return {up,
          p.sum * (p.top == up ? 1.0f : __builtin_amdgcn_exp2f(p.top - up)) +
              q.sum * (q.top == up ? 1.0f : __builtin_amdgcn_exp2f(q.top - up)),
          max(moved(p.exp, p.top, up), moved(q.exp, q.top, up))};
}
__device__ __forceinline__ Sum of_lane(Sum s, int mask) {
  return {__shfl_xor(s.top, mask), __shfl_xor(s.sum, mask), __shfl_xor(s.exp, mask)};
}
// Blocks part, part + parts, ... of row m.
__device__ __forceinline__ Sum blocks_of(const XentArgs& a, int m, int part, int parts, int blocks) {
  constexpr int AHEAD = 8;
  const bool exps = a.backward && a.planes != 1;
  Sum all = {-__builtin_inff(), 0.0f, XENT_NO_EXP};
  for (int b = part; b < blocks; b += AHEAD * parts) {
    float2 e[AHEAD];
    int x[AHEAD];
    if (exps) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        x[k] = b + k * parts < blocks ? a.stat_exp[(int64_t)(b + k * parts) * a.stat_ld + m] : XENT_NO_EXP;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      e[k] = b + k * parts < blocks ? a.stat[(int64_t)(b + k * parts) * a.stat_ld + m]
                                    : make_float2(0.0f, -__builtin_inff());
    float up = all.top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) up = fmaxf(up, e[k].y);
    float s = all.sum * (all.top == up ? 1.0f : __builtin_amdgcn_exp2f(all.top - up));
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) s += e[k].x * (e[k].y == up ? 1.0f : __builtin_amdgcn_exp2f(e[k].y - up));
    int most = XENT_NO_EXP;
    if (exps) {
      most = moved(all.exp, all.top, up);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) most = max(most, moved(x[k], e[k].y, up));
    }
    all = {up, s, most};
  }
  return all;
}

// Largest exponents of some rows: c_part's.
struct Exps {
  int low, e, g;
  __device__ __forceinline__ void take(const Exps& o) {
    low = max(low, o.low);
    e = max(e, o.e);
    g = max(g, o.g);
  }
  __device__ __forceinline__ void take_wave() {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      take({__shfl_xor(low, o), __shfl_xor(e, o), __shfl_xor(g, o)});
  }
};

constexpr Exps NO_EXPS{XENT_NO_EXP, XENT_NO_EXP, XENT_NO_EXP};

// Row m's loss and the factors of its gradient from the others' sum.
__device__ __forceinline__ float finish_row(const XentArgs& a, int64_t r0, int m, Sum others, Exps& exps) {
  // the others' sum is sum * 2^top, the target's exponential 2^(top - d)
  const float top = others.top, sum = others.sum;
  float lt = a.at_target[r0 + m], slope = 1.0f;
  if (a.softcap > 0.0f) {
    const float e = __builtin_amdgcn_exp2f(lt * (2.0f * LOG2E / a.softcap)), r = __builtin_amdgcn_rcpf(1.0f + e);
    lt = a.softcap * fmaf(-2.0f, r, 1.0f);
    slope = 4.0f * mxm_xent_cap_slope(e, r);
  }
  // (no other entry comes: d is whatever makes the target's share one)
  const bool alone = sum == 0.0f;
  const float d = alone ? -200.0f : fmaf(-lt, LOG2E, top);
  const float et = __builtin_amdgcn_exp2f(-d), whole = sum + et;
  // (next to the target's probability of one the loss keeps its digits; a share of the
  // others' below 2^-113 leaves no gradient)
  const bool near = d <= 60.0f;
  const float over = logf(whole);
  const float loss = alone ? lt - lt : near ? log1pf(sum * __builtin_amdgcn_exp2f(d)) : d * LN2 + over;
  const int64_t n = a.map[r0 + m];
  a.nll[r0 + m] = loss;
  if (a.loss) a.loss[n] = loss;
  if (a.lse) a.lse[n] = near ? lt + loss : top * LN2 + over;
  if (a.backward) {
    const double w = a.row_weights ? (double)a.row_weights[n] : 1.0;
    const float g = (float)((double)a.d_total * w / (a.mean ? a.scalars->weight_sum : 1.0));
    XentRow r;
    r.ref = top;
    r.scale = (a.softcap > 0.0f ? 4.0f * g : g) / whole;
    r.at_target = -g * (sum / whole) * slope;
    r.target = a.target[r0 + m];
    r.e = r.g = XENT_NO_EXP;
    if (a.planes != 1) {
      // no |dz| of the row is above |g| times the others' share, none of the others' above
      // 2^15 (a summand's most) times scale
      const float most = __builtin_fabsf(g) * (sum / whole);
      if (most > 0.0f && most < __builtin_inff()) {
        int e_most, e_scale, e_target;
        (void)frexpf(most, &e_most);
        (void)frexpf(r.scale, &e_scale);
        (void)frexpf(r.at_target, &e_target);
        const int w = a.w_exp[r.target];
        const bool any = others.exp > XENT_NO_EXP / 2, at = w < XENT_INF && r.at_target != 0.0f;
        r.e = max(any ? others.exp + e_scale - 15 : XENT_NO_EXP, at ? w + e_target - 15 : XENT_NO_EXP);
        r.g = max(min(e_most, e_scale + 15), at ? e_target : XENT_NO_EXP) - 15;
        exps.take({any  ? others.exp - 15 - XENT_SLACK
                   : at ? w - XENT_SLACK
                        : XENT_NO_EXP,
                   r.e + a.x_exp[r0 + m], r.g + a.x_exp[r0 + m]});
      }
    }
    a.row[r0 + m] = r;
  }
  return loss;
}

// Few rows: WAVES waves each (1, or 4 for sums of many blocks: 21 rows' of 1713 blocks took
// 16.7 us with one, 12 so).  With one workgroup for all of them it also sums the total.
constexpr int JOIN_WAVES = 16, JOIN_FEW = 512, LONG_JOIN = 512;
template <int WAVES>
__global__ __launch_bounds__(64 * JOIN_WAVES) void xent_join_few_kernel(XentArgs a, int64_t r0, int blocks,
                                                                        bool total) {
  __shared__ double part[JOIN_WAVES];
  __shared__ Exps each[JOIN_WAVES];
  __shared__ Sum sums[JOIN_WAVES];
  const int rows = mxm_xent_rows(a, r0), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = blockIdx.x * (JOIN_WAVES / WAVES) + wave / WAVES;
  Exps exps = NO_EXPS;
  double sum = 0.0;
  Sum s = {-__builtin_inff(), 0.0f, XENT_NO_EXP};
  if (m < rows) {
    s = blocks_of(a, m, wave % WAVES * 64 + lane, 64 * WAVES, blocks);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s = join(s, of_lane(s, o));
  }
  if constexpr (WAVES > 1) {
    if (lane == 0) sums[wave] = s;
    __syncthreads();
#pragma unroll
    for (int i = 1; i < WAVES; ++i)
      if (wave % WAVES == 0) s = join(s, sums[wave + i]);
  }
  if (m < rows && wave % WAVES == 0 && lane == 0) {
    const float loss = finish_row(a, r0, m, s, exps);
    sum = (double)loss * (a.row_weights ? (double)a.row_weights[a.map[r0 + m]] : 1.0);
  }
  if (a.backward && a.planes != 1) {
    if (lane == 0) each[wave] = exps;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < JOIN_WAVES; ++i) exps.take(each[i]);
      a.c_part[blockIdx.x] = make_int4(exps.low, exps.e, exps.g, 0);
    }
  }
  if (!total) return;
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int i = 0; i < JOIN_WAVES; ++i) sum += part[i];
    if (a.mean && rows > 0) sum /= a.scalars->weight_sum;
    a.total[0] = (float)sum;
  }
}

// 16 rows by 16 threads.
constexpr int JOIN_ROWS = 16;
__global__ __launch_bounds__(NT) void xent_join_kernel(XentArgs a, int64_t r0, int blocks) {
  __shared__ Sum red[4][JOIN_ROWS];
  const int rows = mxm_xent_rows(a, r0);
  const int k = threadIdx.x & 15, m = blockIdx.x * JOIN_ROWS + k;
  const bool exponents = a.backward && a.planes != 1;
  if (blockIdx.x * JOIN_ROWS >= rows) {
    if (exponents && threadIdx.x == 0) a.c_part[blockIdx.x] = make_int4(XENT_NO_EXP, XENT_NO_EXP, XENT_NO_EXP, 0);
    return;
  }
  Sum s = blocks_of(a, min(m, rows - 1), threadIdx.x >> 4, 16, blocks);
  s = join(s, of_lane(s, 16));
  s = join(s, of_lane(s, 32));
  if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][k] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  Exps exps = NO_EXPS;
  if (threadIdx.x < 16 && m < rows)
    finish_row(a, r0, m, join(join(red[0][k], red[1][k]), join(red[2][k], red[3][k])), exps);
  if (exponents) {
    exps.take_wave();
    if (threadIdx.x == 0) a.c_part[blockIdx.x] = make_int4(exps.low, exps.e, exps.g, 0);
  }
}

// The total, by a workgroup.
template <int T>
__device__ __forceinline__ void sum_total(const XentArgs& a, double* part) {
  const int rows = a.scalars->rows;
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += T)
    s += (double)a.nll[i] * (a.row_weights ? (double)a.row_weights[a.map[i]] : 1.0);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < T / 64; ++i) s += part[i];
    if (a.mean && rows > 0) s /= a.scalars->weight_sum;
    a.total[0] = (float)s;
  }
}

// The summands of a piece to dz, 8 of a row per thread; under fp32 the first workgroups
// of the rows also take x' to x'', and all of them the rows of W' below L to it (in
// place: the piece's logits are done).  The last workgroup sums the total, where it is
// wanted (of the last piece).  ONCE: past the last-level cache.
template <bool F16, bool ONCE>
__global__ __launch_bounds__(NT) void xent_finish_kernel(XentArgs a, int64_t r0, int block, int parity,
                                                           bool first, bool total) {
  if (total && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) {
    __shared__ double part[NT / 64];
    sum_total<NT>(a, part);
  }
  constexpr int AHEAD = ONCE ? 4 : 1;  // units of a thread in flight
  const auto put = [](u32x4_t v, u32x4_t* to) {
    if constexpr (ONCE)
      __builtin_nontemporal_store(v, to);
    else
      *to = v;
  };
  const int rows = mxm_xent_rows(a, r0), units = a.Vp / 8;
  int c_top = 0, low = XENT_NO_EXP;
  if constexpr (F16) {
    __shared__ Exps each[NT / 64];
    Exps all = NO_EXPS;
    for (int i = threadIdx.x; i < a.c_parts; i += NT) {
      const int4 c = a.c_part[i];
      all.take({c.x, c.y, c.z});
    }
    all.take_wave();
    if ((threadIdx.x & 63) == 0) each[threadIdx.x >> 6] = all;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) all.take(each[i]);
    const int before = first ? XENT_NO_EXP : a.scalars->low[parity ^ 1];
    low = max(all.low, before);
    c_top = all.g == XENT_NO_EXP ? 0 : max(all.e, all.g + max(low, XENT_ZERO));
    const int id = blockIdx.y * gridDim.x + blockIdx.x;
    if (id == 0 && threadIdx.x == 0) {
      a.scalars->dw_exp = c_top;
      a.scalars->low[parity] = low;
    }
    if (a.dx) {
      const int lane = threadIdx.x & 63;
      // (neighbours go to different waves: where many need it, in a small table, all work)
      const int waves = gridDim.x * gridDim.y * (NT / 64);
      for (int v0 = id * (NT / 64) + (threadIdx.x >> 6); v0 < a.V; v0 += 64 * waves) {
        const int v = v0 + lane * waves, w = v < a.V ? a.w_exp[v] : XENT_ZERO;
        const int now = max(w, before);
        unsigned long long todo = __ballot(w != XENT_ZERO && now < low);
        while (todo != 0) {
          const int at = __ffsll(todo) - 1;
          todo &= todo - 1;
          const int64_t row = v0 + at * waves;
          const int by = __shfl(now, at) - low;
          for (int u = lane; u < 2 * (a.Dp / 8); u += 64) {
            const int pl = u >= a.Dp / 8;
            f16x8_t* q = reinterpret_cast<f16x8_t*>(a.w_pack + (pl * (int64_t)a.V + row) * a.Dp) + (u - pl * (a.Dp / 8));
            f16x8_t h = *q;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = (_Float16)ldexpf((float)h[i], by);
            *q = h;
          }
        }
      }
    }
  }
  for (int m = blockIdx.y; m < rows; m += gridDim.y) {
    const XentRow r = a.row[r0 + m];
    int row_exp = 0;
    if constexpr (F16) {
      if (r.g != XENT_NO_EXP) row_exp = max(r.e, r.g + max(low, XENT_ZERO));
      if (blockIdx.x == 0) {
        if (threadIdx.x == 0) a.e_row[r0 + m] = row_exp;
        if (a.dw) {
          const float f = r.g == XENT_NO_EXP ? 0.0f : ldexpf(1.0f, row_exp + a.x_exp[r0 + m] - c_top);
          for (int u = threadIdx.x; u < 2 * (a.Dp / 8); u += NT) {
            const int pl = u >= a.Dp / 8;
            f16x8_t* q = reinterpret_cast<f16x8_t*>(a.x_pack + pl * (a.x_rows * a.Dp) + (r0 + m) * a.Dp) +
                         (u - pl * (a.Dp / 8));
            f16x8_t v = *q;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (_Float16)((float)v[i] * f);
            *q = v;
          }
        }
      }
    }
    for (int u0 = blockIdx.x * NT * AHEAD + threadIdx.x; u0 < units; u0 += gridDim.x * NT * AHEAD) {
      u32x4_t raw[AHEAD][F16 ? 2 : 1];
      float ref[AHEAD];
      i32x4_t we[F16 ? AHEAD : 1][2];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        // (units behind the last one: it again, not stored; a row's last ones may lie in
        // padding behind the last block)
        const int v = min(u0 + k * NT, units - 1) * 8;
        const int64_t at = (int64_t)m * a.Vp + v;
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.summands) + at * (F16 ? 4 : 2));
        raw[k][0] = ONCE ? __builtin_nontemporal_load(from) : from[0];
        if constexpr (F16) {
          raw[k][1] = ONCE ? __builtin_nontemporal_load(from + 1) : from[1];
          const i32x4_t* w = reinterpret_cast<const i32x4_t*>(a.w_exp + (v < a.V ? v : 0));
          we[k][0] = w[0];
          we[k][1] = w[1];
        }
        ref[k] = v < a.V ? a.stat[(int64_t)(v / block) * a.stat_ld + m].y : r.ref;
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (u0 + k * NT >= units) break;
        const int v = (u0 + k * NT) * 8;
        const int64_t at = (int64_t)m * a.Vp + v;
        const float f = r.scale * (ref[k] == r.ref ? 1.0f : __builtin_amdgcn_exp2f(ref[k] - r.ref));
        float e[8];
        if constexpr (!F16) {
          const f16x8_t h = __builtin_bit_cast(f16x8_t, raw[k][0]);
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = (float)h[i] * f;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            e[i] = ldexpf(mxm_u2f(raw[k][i / 4][i % 4]) * f, max(we[k][i / 4][i % 4], low) - row_exp);
        }
        const int t = r.target - v;
        float at_target = r.at_target;
        if constexpr (F16) {
          if (t >= 0 && t < 8) at_target = ldexpf(at_target, max(a.w_exp[r.target], low) - row_exp);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i == t ? at_target : (v + i < a.V ? e[i] : 0.0f);
        if constexpr (!F16) {
          // (to bf16 as the table and x are, whose products are at the matrix cores' full
          // rate and exact: this rounding and that of the results to bf16 leave 1.8e-3 to
          // 2.3e-3 of dx and dw in the 2-norm, the results' alone 1.66e-3)
          u32x4_t o;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = mxm_pack_bf2_fast(e[2 * i], e[2 * i + 1]);
          put(o, reinterpret_cast<u32x4_t*>(a.dz + at));
        } else {
          u32x4_t q[2];
          planes2x8(e, q);
          put(q[0], reinterpret_cast<u32x4_t*>(a.dz + at));
          put(q[1], reinterpret_cast<u32x4_t*>(a.dz + a.piece_rows * a.Vp + at));
        }
      }
    }
  }
}

constexpr int TOTAL_NT = 1024;
__global__ __launch_bounds__(TOTAL_NT) void xent_total_kernel(XentArgs a) {
  __shared__ double part[TOTAL_NT / 64];
  sum_total<TOTAL_NT>(a, part);
}

}  // namespace

void mxm_launch_xent(const XentArgs& a0, hipStream_t s) {
  XentArgs a = a0;
  a.w_direct = a.bf16 && a.D % 8 == 0 && (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0;
  // (one row's loss at D 2048 and 50257 entries, in the caches: 39.4 us with the
  // packing's launch, 36.4 without)
  const bool gather = a.rows > 0 && !a.backward && a.w_direct && a.rows <= XENT_GATHER &&
                      (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  if (!gather) {
    const auto waves = [&](int64_t n) { return std::min<int64_t>((n + 3) / 4, (int64_t)a.n_cu * 16); };
    const int64_t chunk = ((a.rows + XENT_CHUNKS - 1) / XENT_CHUNKS + 3) / 4 * 4;
    const int64_t gx = chunk ? (a.rows + chunk - 1) / chunk : 1, gw = a.w_direct || a.rows == 0 ? 0 : waves(a.V);
    const auto pack = [&](auto kernel) { kernel<<<(unsigned)(gx + gw), NT, 0, s>>>(a, (int)gx, chunk); };
    if (a.rows <= PLAN_ROWS) {
      pack(xent_pack_kernel<true>);
    } else {
      xent_count_kernel<<<(unsigned)((gx + 3) / 4), NT, 0, s>>>(a, chunk, (int)gx);
      pack(xent_pack_kernel<false>);
    }
  }
  const int64_t pieces = std::max<int64_t>(1, (a.rows + a.piece_rows - 1) / a.piece_rows);
  bool total_there = false;  // one workgroup joins all rows and sums their total
  for (int64_t p = 0; p < pieces; ++p) {
    const int64_t r0 = p * a.piece_rows, rows = std::min(a.rows - r0, a.piece_rows);
    const int parity = (int)(p & 1);
    if (rows > 0) {
      const int block = mxm_xent_block(rows, a.V, a.n_cu);
      a.stat_ld = rows;
      mxm_launch_xent_logits(a, r0, rows, a.planes != 1 && a.dx && p > 0 ? a.scalars->low + (parity ^ 1) : nullptr,
                             gather, s);
      const int blocks = (a.V + block - 1) / block;
      if (rows <= JOIN_FEW) {
        // Four waves a row for long sums; but up to 15 rows' losses with their total, of
        // some 24000 blocks in all, take one workgroup with a wave a row and no launch for
        // the total (us so / with four waves a row and that launch: 10 rows against 58527
        // entries, 18000 blocks, 12.6 / 14.3; 13 rows, 24000, 15.0 / 15.1; 11 against 131072,
        // 45000, 20.7 / 18.7; 16 rows against 33000, 16500, 16.1 / 14.1, and against a
        // million 275 / 115).
        const bool alone = !a.backward && a.total && a.rows > JOIN_WAVES / 4 && a.rows < JOIN_WAVES &&
                           a.rows * blocks <= 24000;
        const bool long_joins = blocks > LONG_JOIN && !alone;
        const int each = long_joins ? JOIN_WAVES / 4 : JOIN_WAVES;
        a.c_parts = (int)((rows + each - 1) / each);
        total_there = a.total && a.rows <= each;
        const auto launch = [&](auto kernel) {
          kernel<<<a.c_parts, 64 * JOIN_WAVES, 0, s>>>(a, r0, blocks, total_there);
        };
        long_joins ? launch(xent_join_few_kernel<4>) : launch(xent_join_few_kernel<1>);
      } else {
        a.c_parts = (int)((rows + JOIN_ROWS - 1) / JOIN_ROWS);
        xent_join_kernel<<<a.c_parts, NT, 0, s>>>(a, r0, blocks);
      }
      if (a.backward) {
        // What is far past the 256 MB of the last-level cache goes around it: a step of
        // 1.6 GB of summands 1856 us, so 1776; of 538 MB 784, so 792; of 188 MB 552, so 558.
        const bool once = rows * a.Vp * (a.planes == 1 ? 2 : 8) > (int64_t)1 << 30;
        const int per = NT * (once ? 4 : 1);
        const unsigned gx = (unsigned)std::min((a.Vp / 8 + per - 1) / per, 64);
        unsigned gy = (unsigned)std::min<int64_t>(rows, std::max(1u, (unsigned)a.n_cu * 32 / gx));
        // (few rows' workgroups would be few for the rows of W' below L: a step of one row
        // against 32768 entries at D 512, whose rows' sizes spread over 2^8, 250-296 us, 112 so)
        if (a.planes != 1 && a.dx) gy = std::max(gy, (unsigned)std::min(a.n_cu * 4, (a.V + 3) / 4) / gx);
        const dim3 grid(gx, gy);
        const bool total_late = a.total && !total_there && p == pieces - 1;
        const auto launch = [&](auto kernel) { kernel<<<grid, NT, 0, s>>>(a, r0, block, parity, p == 0, total_late); };
        if (a.planes == 1)
          once ? launch(xent_finish_kernel<false, true>) : launch(xent_finish_kernel<false, false>);
        else
          once ? launch(xent_finish_kernel<true, true>) : launch(xent_finish_kernel<true, false>);
      }
    }
    if (a.backward) mxm_launch_xent_grads(a, r0, rows, p == pieces - 1, a.scalars->low + parity, s);
  }
  if (a.total && !total_there && !(a.backward && a.rows > 0)) xent_total_kernel<<<1, TOTAL_NT, 0, s>>>(a);
}
