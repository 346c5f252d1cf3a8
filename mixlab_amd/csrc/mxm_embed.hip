// The token embedding (mxm_vocab.h): lookup with scaling, and its gradient by
// sorted tokens.
#include <algorithm>

#include "mxm_vocab.h"

namespace {

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// U elements at p as fp32, U = 8 from 16-byte aligned rows, else 1.
template <int U>
__device__ __forceinline__ void load_unit(const void* p, bool bf16, int64_t at, float (&v)[U]) {
  if constexpr (U == 8) {
    if (bf16) {
      const u32x4_t q = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = mxm_u2f(q[i] << 16);
        v[2 * i + 1] = mxm_u2f(q[i] & 0xffff0000u);
      }
    } else {
      const f32x4_t* q = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + at);
      const f32x4_t a = q[0], b = q[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    }
  } else {
    v[0] = bf16 ? mxm_bf2f(static_cast<const uint16_t*>(p)[at]) : static_cast<const float*>(p)[at];
  }
}
template <int U>
__device__ __forceinline__ void store_unit(void* p, bool bf16, int64_t at, const float (&v)[U]) {
  if constexpr (U == 8) {
    if (bf16) {
      u32x4_t q;
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = mxm_pack_bf2_fast(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p) + at) = q;
    } else {
      f32x4_t a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = v[i], b[i] = v[4 + i];
      f32x4_t* q = reinterpret_cast<f32x4_t*>(static_cast<float*>(p) + at);
      q[0] = a;
      q[1] = b;
    }
  } else if (bf16) {
    static_cast<uint16_t*>(p)[at] = mxm_f2bf_fast(v[0]);
  } else {
    static_cast<float*>(p)[at] = v[0];
  }
}

constexpr int NT = 256;

// A row per T threads, ROWS of them in flight: their tokens, then their elements.
constexpr int ROWS = 4;
template <int U>
__global__ __launch_bounds__(NT) void embed_kernel(EmbedArgs a, int T) {
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * per;
  for (int64_t n0 = (int64_t)blockIdx.x * per + sub; n0 < a.rows; n0 += ROWS * step) {
    int v[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) v[k] = n0 + k * step < a.rows ? a.tokens[n0 + k * step] : -1;
    for (int d = t * U; d < a.D; d += T * U) {
      float e[ROWS][U];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        if (v[k] >= 0 && v[k] < a.V) {
          load_unit<U>(a.table, a.table_bf16, (int64_t)v[k] * a.D + d, e[k]);
#pragma unroll
          for (int i = 0; i < U; ++i) e[k][i] *= a.scale;
        } else {
#pragma unroll
          for (int i = 0; i < U; ++i) e[k][i] = 0.0f;
        }
      }
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (n0 + k * step < a.rows) store_unit<U>(a.out, a.out_bf16, (n0 + k * step) * a.D + d, e[k]);
    }
  }
}

// ---- backward: the places sorted by token ----
//
// Workgroup o owns the tokens [o * span, (o + 1) * span).  Its waves each walk
// their own stretch of the tokens twice: counting, per wave, how often each owned
// token occurs (and how many tokens are smaller than the first owned one, which is
// where the owned ones start), then writing the owned places in order.
constexpr int SORT_WAVES = 16;
constexpr int SORT_SPAN = 512;  // most tokens a workgroup owns
constexpr int SORT_AHEAD = 4;   // tokens in flight per lane

// LDS written by lanes of this wave is read by other lanes of it afterwards.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__global__ __launch_bounds__(64 * SORT_WAVES) void embed_sort_kernel(EmbedArgs a, int span) {
  __shared__ int cnt[SORT_WAVES][SORT_SPAN];
  __shared__ int tot[SORT_SPAN];
  __shared__ int lower[SORT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lo = blockIdx.x * span, own = min(span, a.V - lo);
  for (int i = threadIdx.x; i < SORT_WAVES * SORT_SPAN; i += blockDim.x) (&cnt[0][0])[i] = 0;
  __syncthreads();
  // stretches of whole groups of 64
  const int64_t groups = (a.rows + 63) / 64, each = (groups + SORT_WAVES - 1) / SORT_WAVES;
  const int64_t from = min((int64_t)wave * each * 64, a.rows);
  const int64_t to = min(from + each * 64, a.rows);
  int below = 0;
  for (int64_t n = from; n < to; n += 64 * SORT_AHEAD) {
    int v[SORT_AHEAD];
#pragma unroll
    for (int q = 0; q < SORT_AHEAD; ++q) {
      const int64_t i = n + 64 * q + lane;
      v[q] = i < to ? a.tokens[i] : -1;
    }
#pragma unroll
    for (int q = 0; q < SORT_AHEAD; ++q) {
      below += v[q] >= 0 && v[q] < lo;
      const unsigned b = (unsigned)v[q] - (unsigned)lo;
      if (b < (unsigned)own) atomicAdd(&cnt[wave][b], 1);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
  if (lane == 0) lower[wave] = below;
  __syncthreads();
  // where each wave's first place of each token goes
  for (int b = threadIdx.x; b < own; b += blockDim.x) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = cnt[w][b];
      cnt[w][b] = s;
      s += c;
    }
    tot[b] = s;
  }
  __syncthreads();
  if (wave == 0) {
    int base = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) base += lower[w];
    for (int b0 = 0; b0 < own; b0 += 64) {
      const int b = b0 + lane, c = b < own ? tot[b] : 0;
      int x = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (b < own) {
        tot[b] = base + x - c;
        a.starts[lo + b] = base + x - c;
      }
      base += __shfl(x, 63);
    }
    if (lane == 0 && lo + own == a.V) a.starts[a.V] = base;
  }
  __syncthreads();
  for (int64_t n = from; n < to; n += 64 * SORT_AHEAD) {
    int v[SORT_AHEAD];
#pragma unroll
    for (int q = 0; q < SORT_AHEAD; ++q) {
      const int64_t i = n + 64 * q + lane;
      v[q] = i < to ? a.tokens[i] : -1;
    }
#pragma unroll
    for (int q = 0; q < SORT_AHEAD; ++q) {
      const unsigned b = (unsigned)v[q] - (unsigned)lo;
      const bool mine = b < (unsigned)own;
      // the lanes that hold the same token: a ballot per bit of its place in the span
      unsigned long long same = __ballot(mine);
      if (!same) continue;
      for (unsigned bit = 1; bit < (unsigned)span; bit <<= 1) {
        const bool set = b & bit;
        const unsigned long long m = __ballot(set);
        same &= set ? m : ~m;
      }
      int left = 0;  // of the first of them: how many there are
      if (mine) {
        const unsigned long long before = same & ((1ull << lane) - 1);
        const int at = tot[b] + cnt[wave][b];
        a.sorted[at + __popcll(before)] = make_int2((int)(n + 64 * q + lane), v[q]);
        if (!before) left = __popcll(same);
      }
      wave_lds_sync();  // every lane has read its count
      if (left) cnt[wave][b] += left;
      wave_lds_sync();
    }
  }
}

// Sorted places [c * C, (c + 1) * C) per T threads: each run of one token that lies
// within them to the table, the first and last run's sums to part where they go on
// outside.  Workgroups behind the chunks': zeros for the tokens that occur nowhere.
template <int U>
__device__ __forceinline__ void put_row(const EmbedArgs& a, int v, int d, float (&s)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i) s[i] *= a.scale;
  const int64_t at = (int64_t)v * a.D + d;
  if (a.accumulate) {
    float o[U];
    load_unit<U>(a.d_table, a.dtable_bf16, at, o);
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] += o[i];
  }
  store_unit<U>(a.d_table, a.dtable_bf16, at, s);
}

constexpr int AHEAD = 4;  // rows in flight
template <int U>
__device__ __forceinline__ void sum_chunk(const EmbedArgs& a, int T, int t, int C, int64_t c, int64_t all) {
  const int64_t from = c * C, to = min(from + C, all);
  if (from >= to) return;
  for (int d = t * U; d < a.D; d += T * U) {
    float s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] = 0.0f;
    int v = a.sorted[from].y;
    bool first = true;  // the chunk's first run
    for (int64_t p0 = from; p0 < to; p0 += AHEAD) {
      int2 e[AHEAD];
      float g[AHEAD][U];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) e[k] = a.sorted[min(p0 + k, to - 1)];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) load_unit<U>(a.d_out, a.grad_bf16, (int64_t)e[k].x * a.D + d, g[k]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (p0 + k >= to) break;
        if (e[k].y != v) {
          if (first && a.starts[v] < from) {
            float* q = a.part + c * 2 * a.D + d;
#pragma unroll
            for (int i = 0; i < U; ++i) q[i] = s[i];
          } else {
            put_row<U>(a, v, d, s);
          }
          first = false;
          v = e[k].y;
#pragma unroll
          for (int i = 0; i < U; ++i) s[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] += g[k][i];
      }
    }
    const bool before = first && a.starts[v] < from, after = a.starts[v + 1] > to;
    if (before || after) {
      float* q = a.part + (c * 2 + (before ? 0 : 1)) * a.D + d;
#pragma unroll
      for (int i = 0; i < U; ++i) q[i] = s[i];
    } else {
      put_row<U>(a, v, d, s);
    }
  }
}

template <int U>
__global__ __launch_bounds__(NT) void embed_sum_kernel(EmbedArgs a, int T, int C, int64_t chunks,
                                                       int64_t items) {
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t all = a.starts[a.V];
  for (int64_t i = (int64_t)blockIdx.x * per + sub; i < items; i += (int64_t)gridDim.x * per) {
    if (i < chunks) {
      sum_chunk<U>(a, T, t, C, i, all);
    } else {
      const int64_t v = i - chunks;
      if (a.starts[v] != a.starts[v + 1]) continue;
      float z[U];
#pragma unroll
      for (int k = 0; k < U; ++k) z[k] = 0.0f;
      for (int d = t * U; d < a.D; d += T * U) store_unit<U>(a.d_table, a.dtable_bf16, v * a.D + d, z);
    }
  }
}

// The run that starts in chunk c and goes on behind it: its sums in order.
template <int U>
__device__ __forceinline__ void join_chunk(const EmbedArgs& a, int T, int t, int C, int64_t c, int64_t all) {
  if ((c + 1) * C >= all) return;
  const int v = a.sorted[(c + 1) * C - 1].y;
  const int64_t from = a.starts[v], to = a.starts[v + 1];
  if (from < c * C || to <= (c + 1) * C) return;
  const int64_t last = (to - 1) / C;
  for (int d = t * U; d < a.D; d += T * U) {
    float s[U];
    const float* q = a.part + (c * 2 + 1) * a.D + d;
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] = q[i];
    int64_t k = c + 1;
    for (; k + 8 <= last + 1; k += 8) {
      float e[8][U];
#pragma unroll
      for (int h = 0; h < 8; ++h) load_unit<U>(a.part, false, (k + h) * 2 * a.D + d, e[h]);
#pragma unroll
      for (int h = 0; h < 8; ++h)
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] += e[h][i];
    }
    for (; k <= last; ++k) {
      float e[U];
      load_unit<U>(a.part, false, k * 2 * a.D + d, e);
#pragma unroll
      for (int i = 0; i < U; ++i) s[i] += e[i];
    }
    put_row<U>(a, v, d, s);
  }
}

template <int U>
__global__ __launch_bounds__(NT) void embed_join_kernel(EmbedArgs a, int T, int C, int64_t chunks) {
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t all = a.starts[a.V];
  for (int64_t c = (int64_t)blockIdx.x * per + sub; c < chunks; c += (int64_t)gridDim.x * per)
    join_chunk<U>(a, T, t, C, c, all);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Threads that walk one row of `units`: the least power of two that covers it, at
// most a workgroup.
int threads_per_row(int64_t units) {
  int t = 8;
  while (t < NT && t < units) t *= 2;
  return t;
}

// Sorted places per chunk.
constexpr int64_t LONG_BATCH = 32768;
int chunk_rows(int64_t rows) { return rows >= LONG_BATCH ? 32 : 8; }

unsigned grid_of(int64_t items, int per, int n_cu) {
  return (unsigned)std::min<int64_t>((items + per - 1) / per, (int64_t)n_cu * 64);
}

}  // namespace

int64_t mxm_embed_max_chunks(int64_t max_rows) {
  return std::max((std::min(max_rows, LONG_BATCH - 1) + 7) / 8, (max_rows + 31) / 32);
}

void mxm_launch_embed(const EmbedArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  const bool wide = a.D % 8 == 0 && aligned(a.table) && aligned(a.out);
  const int T = threads_per_row(wide ? a.D / 8 : a.D);
  const unsigned grid = grid_of(a.rows, NT / T, a.n_cu);
  if (wide)
    embed_kernel<8><<<grid, NT, 0, s>>>(a, T);
  else
    embed_kernel<1><<<grid, NT, 0, s>>>(a, T);
}

void mxm_launch_embed_bw(const EmbedArgs& a, hipStream_t s) {
  const bool wide = a.D % 8 == 0 && aligned(a.d_out) && aligned(a.d_table);
  const int T = threads_per_row(wide ? a.D / 8 : a.D), per = NT / T;
  const int span = std::min(SORT_SPAN, std::max(16, (a.V + a.n_cu - 1) / a.n_cu));
  embed_sort_kernel<<<(a.V + span - 1) / span, 64 * SORT_WAVES, 0, s>>>(a, span);
  const int C = chunk_rows(a.rows);
  const int64_t chunks = (a.rows + C - 1) / C, items = chunks + (a.accumulate ? 0 : a.V);
  if (items > 0) {
    const unsigned grid = grid_of(items, per, a.n_cu);
    if (wide)
      embed_sum_kernel<8><<<grid, NT, 0, s>>>(a, T, C, chunks, items);
    else
      embed_sum_kernel<1><<<grid, NT, 0, s>>>(a, T, C, chunks, items);
  }
  if (chunks > 1) {
    const unsigned grid = grid_of(chunks, per, a.n_cu);
    if (wide)
      embed_join_kernel<8><<<grid, NT, 0, s>>>(a, T, C, chunks);
    else
      embed_join_kernel<1><<<grid, NT, 0, s>>>(a, T, C, chunks);
  }
}
