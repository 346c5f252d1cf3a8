// The token embedding (mxm_vocab.h): lookup with scaling, and its gradient by
// sorted tokens.
#include <algorithm>

#include "mxm_vocab.h"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// U elements of a row of fp32 or bf16 (ODD: at the elements' alignment, the row's last
// unit of as many as are left).
template <int N, bool ODD>
struct Words {
  typedef unsigned int type __attribute__((ext_vector_type(N)));
};
template <int N>
struct Words<N, true> {
  typedef unsigned int type __attribute__((ext_vector_type(N), aligned(2)));
};
template <bool ODD>
struct Floats {
  typedef float type __attribute__((ext_vector_type(4)));
};
template <>
struct Floats<true> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
// ONCE: read past the caches.
template <int U, bool ODD, bool ONCE = false>
__device__ __forceinline__ void load_unit(const void* p, bool bf16, int64_t at, int left, float (&v)[U]) {
  if (ODD && left < U) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      v[i] = i >= left ? 0.0f
             : bf16    ? mxm_bf2f(static_cast<const uint16_t*>(p)[at + i])
                       : static_cast<const float*>(p)[at + i];
  } else if (bf16) {
    typedef typename Words<U / 2, ODD>::type words_t;
    const words_t* from = reinterpret_cast<const words_t*>(static_cast<const uint16_t*>(p) + at);
    const typename Words<U / 2, false>::type q = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
    for (int i = 0; i < U / 2; ++i) {
      v[2 * i] = mxm_u2f(q[i] << 16);
      v[2 * i + 1] = mxm_u2f(q[i] & 0xffff0000u);
    }
  } else {
    typedef typename Floats<ODD>::type floats_t;
    const floats_t* q = reinterpret_cast<const floats_t*>(static_cast<const float*>(p) + at);
#pragma unroll
    for (int h = 0; h < U / 4; ++h) {
      const f32x4_t a = ONCE ? __builtin_nontemporal_load(q + h) : q[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = a[i];
    }
  }
}
template <int U, bool ODD>
__device__ __forceinline__ void store_unit(void* p, bool bf16, int64_t at, int left, const float (&v)[U]) {
  if (ODD && left < U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= left) continue;
      if (bf16)
        static_cast<uint16_t*>(p)[at + i] = mxm_f2bf_fast(v[i]);
      else
        static_cast<float*>(p)[at + i] = v[i];
    }
  } else if (bf16) {
    typename Words<U / 2, false>::type q;
#pragma unroll
    for (int i = 0; i < U / 2; ++i) q[i] = mxm_pack_bf2_fast(v[2 * i], v[2 * i + 1]);
    typedef typename Words<U / 2, ODD>::type words_t;
    __builtin_nontemporal_store(q, reinterpret_cast<words_t*>(static_cast<uint16_t*>(p) + at));
  } else {
    typedef typename Floats<ODD>::type floats_t;
    floats_t* q = reinterpret_cast<floats_t*>(static_cast<float*>(p) + at);
#pragma unroll
    for (int h = 0; h < U / 4; ++h) {
      const f32x4_t a = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
      __builtin_nontemporal_store(a, q + h);
    }
  }
}

constexpr int NT = 256;

// A row per T threads, ROWS of them in flight: their tokens, then their elements.
constexpr int ROWS = 4;
template <int U, bool ODD>
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
          load_unit<U, ODD>(a.table, a.table_bf16, (int64_t)v[k] * a.D + d, a.D - d, e[k]);
#pragma unroll
          for (int i = 0; i < U; ++i) e[k][i] *= a.scale;
        } else {
#pragma unroll
          for (int i = 0; i < U; ++i) e[k][i] = 0.0f;
        }
      }
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (n0 + k * step < a.rows) store_unit<U, ODD>(a.out, a.out_bf16, (n0 + k * step) * a.D + d, a.D - d, e[k]);
    }
  }
}

// ---- backward: the places sorted by token ----
//
// Workgroup o owns the tokens [o * span, (o + 1) * span).  Its waves each take their
// own stretch of the places: they count, per wave, how often each owned token occurs
// (and how many tokens are smaller than the first owned one, which is where the owned
// ones start), then write the owned places in order.  What bounds it is the tokens'
// latency and, where one span holds many of them, their ranks, which are one CU's: 65536
// places take 18 us of tokens spread evenly over 50257, 30 where token v occurs like
// 1 / (v + 1) (49 with a ballot per bit of the token instead of the bits' word).  The
// next batch is loaded while one is worked on; the loops stay rolled (unrolled over 64
// places a lane, with the tokens kept in registers between the two walks, the code's
// own way into the instruction cache made it 57 us).
constexpr int SORT_SPAN = 512;    // most tokens a workgroup owns
constexpr int SORT_FEW = 2048;    // places up to which it has 4 waves, not 16

// LDS written by lanes of this wave is read by other lanes of it afterwards.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// f(first place, token) for the wave's groups of 64 places in from .. to - 1; behind
// them ~0.  (As unsigned numbers, tokens below 0 are past the vocabulary.)
template <int AHEAD, class F>
__device__ __forceinline__ void each_group(const int32_t* tokens, int64_t from, int64_t to, int lane, F f) {
  unsigned v[AHEAD];
  auto fetch = [&](int64_t n) {
    const int32_t* t = tokens + n + lane;
    if (n + 64 * AHEAD <= to) {
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) v[q] = (unsigned)t[64 * q];
    } else {
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) v[q] = n + 64 * q + lane < to ? (unsigned)t[64 * q] : ~0u;
    }
  };
  fetch(from);
  for (int64_t n = from; n < to; n += 64 * AHEAD) {
    unsigned now[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) now[q] = v[q];
    if (n + 64 * AHEAD < to) fetch(n + 64 * AHEAD);
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) f(n + 64 * q, now[q]);
  }
}

template <int SORT_WAVES>
struct SortLds {
  int cnt[SORT_WAVES][SORT_SPAN];
  unsigned long long same[SORT_WAVES][SORT_SPAN];
  int tot[SORT_SPAN + 1];  // where each owned token starts, and the end
  int lower[SORT_WAVES];
};
// put(sorted place, place, token) for every owned place; LOCAL: the sorted places start at
// the workgroup's own.
template <int SORT_WAVES, bool LOCAL, class Put>
__device__ __forceinline__ void sort_span(const EmbedArgs& a, int span, SortLds<SORT_WAVES>& lds, Put put) {
  auto& cnt = lds.cnt;
  auto& same = lds.same;
  auto& tot = lds.tot;
  auto& lower = lds.lower;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lo = blockIdx.x * span, own = min(span, a.V - lo);
  // stretches of whole groups of 64
  const int64_t groups = (a.rows + 63) / 64, each = (groups + SORT_WAVES - 1) / SORT_WAVES * 64;
  const int64_t from = min(wave * each, a.rows), to = min(from + each, a.rows);
  for (int i = threadIdx.x; i < SORT_WAVES * span; i += blockDim.x) {
    const int w = i / span, b = i - w * span;
    cnt[w][b] = 0;
    same[w][b] = 0;
  }
  __syncthreads();
  int below = 0;
  each_group<16>(a.tokens, from, to, lane, [&](int64_t, unsigned v) {
    below += v < (unsigned)lo;
    const unsigned b = v - (unsigned)lo;
    if (__ballot(b < (unsigned)own) && b < (unsigned)own) atomicAdd(&cnt[wave][b], 1);
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
  if (lane == 0) lower[wave] = below;
  __syncthreads();
  // where each wave's first place of each token goes, within the token's
  for (int b = threadIdx.x; b < own; b += blockDim.x) {
    int c[SORT_WAVES], s = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) c[w] = cnt[w][b];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      cnt[w][b] = s;
      s += c[w];
    }
    tot[b] = s;
  }
  __syncthreads();
  if (wave == 0) {
    int base = 0;
    if constexpr (!LOCAL) {
#pragma unroll
      for (int w = 0; w < SORT_WAVES; ++w) base += lower[w];
    }
    for (int b0 = 0; b0 < own; b0 += 64) {
      const int b = b0 + lane, c = b < own ? tot[b] : 0;
      int x = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (b < own) tot[b] = base + x - c;
      base += __shfl(x, 63);
    }
    if (lane == 0) tot[own] = base;
  }
  __syncthreads();
  each_group<8>(a.tokens, from, to, lane, [&](int64_t n, unsigned v) {
    const unsigned b = v - (unsigned)lo;
    const bool mine = b < (unsigned)own;
    const unsigned long long any = __ballot(mine);
    if (!any) return;
    // the lanes that hold the same token: a bit each, in the token's word (64 lanes of one
    // token would go there one after the other: those need no word)
    const unsigned lead = __builtin_amdgcn_readlane(b, __builtin_ctzll(any));
    const bool one = __ballot(mine && b == lead) == any;
    if (!one) {
      if (mine) atomicOr(&same[wave][b], 1ull << lane);
      wave_lds_sync();
    }
    int before = 0, all = 0;
    if (mine) {
      const unsigned long long m = one ? any : same[wave][b];
      before = __popcll(m & ((1ull << lane) - 1));
      all = __popcll(m);
      put(tot[b] + cnt[wave][b] + before, (int)(n + lane), (int)v);
    }
    wave_lds_sync();  // every lane has read its word and count
    if (mine && before == 0) {
      cnt[wave][b] += all;
      same[wave][b] = 0;
    }
    wave_lds_sync();
  });
}

template <int SORT_WAVES>
__global__ __launch_bounds__(64 * SORT_WAVES) void embed_sort_kernel(EmbedArgs a, int span) {
  __shared__ SortLds<SORT_WAVES> lds;
  sort_span<SORT_WAVES, false>(a, span, lds, [&](int at, int n, int v) { a.sorted[at] = make_int2(n, v); });
  const int lo = blockIdx.x * span, own = min(span, a.V - lo);
  for (int b = threadIdx.x; b < own + (lo + own == a.V); b += blockDim.x) a.starts[lo + b] = lds.tot[b];
}

// Floats from one chunk's sum to the next: whole aligned units.
__host__ __device__ inline int part_row(int D) { return (D + 7) / 8 * 8; }

// The sorted places as the sums see them: place and token of one, where a token starts
// and ends, and the chunks' sums.
struct Runs {
  const EmbedArgs& a;
  __device__ __forceinline__ int2 at(int64_t p) const { return a.sorted[p]; }
  __device__ __forceinline__ int64_t start(int v) const { return a.starts[v]; }
  __device__ __forceinline__ float* part(int64_t row) const { return a.part + row * part_row(a.D); }
};

// Sorted places [c * C, (c + 1) * C) per T threads: each run of one token that lies
// within them to the table, the first and last run's sums to part where they go on
// outside.
template <int U, bool ODD>
__device__ __forceinline__ void put_row(const EmbedArgs& a, int v, int d, float (&s)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i) s[i] *= a.scale;
  const int64_t at = (int64_t)v * a.D + d;
  if (a.accumulate) {
    float o[U];
    load_unit<U, ODD>(a.d_table, a.dtable_bf16, at, a.D - d, o);
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] += o[i];
  }
  store_unit<U, ODD>(a.d_table, a.dtable_bf16, at, a.D - d, s);
}

// (read again by the join: kept in the caches)
template <int U>
__device__ __forceinline__ void store_part(float* q, const float (&s)[U]) {
#pragma unroll
  for (int h = 0; h < U / 4; ++h) {
    const f32x4_t v = {s[4 * h], s[4 * h + 1], s[4 * h + 2], s[4 * h + 3]};
    reinterpret_cast<f32x4_t*>(q)[h] = v;
  }
}

constexpr int AHEAD = 8;  // rows in flight
template <int U, bool ODD, class R>
__device__ __forceinline__ void sum_chunk(const EmbedArgs& a, const R& runs, int T, int t, int C, int64_t c,
                                          int64_t all) {
  const int64_t from = c * C, to = min(from + C, all);
  if (from >= to) return;
  for (int d = t * U; d < a.D; d += T * U) {
    float s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] = 0.0f;
    int v = runs.at(from).y;
    bool first = true;  // the chunk's first run
    for (int64_t p0 = from; p0 < to; p0 += AHEAD) {
      int2 e[AHEAD];
      float g[AHEAD][U];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) e[k] = runs.at(min(p0 + k, to - 1));
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) load_unit<U, ODD, true>(a.d_out, a.grad_bf16, (int64_t)e[k].x * a.D + d, a.D - d, g[k]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (p0 + k >= to) break;
        if (e[k].y != v) {
          if (first && runs.start(v) < from) {
            store_part<U>(runs.part(c * 2) + d, s);
          } else {
            put_row<U, ODD>(a, v, d, s);
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
    const bool before = first && runs.start(v) < from, after = runs.start(v + 1) > to;
    if (before || after) {
      store_part<U>(runs.part(c * 2 + (before ? 0 : 1)) + d, s);
    } else {
      put_row<U, ODD>(a, v, d, s);
    }
  }
}

template <int U, bool ODD>
__global__ __launch_bounds__(NT) void embed_sum_kernel(EmbedArgs a, int T, int C, int64_t chunks) {
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t all = a.starts[a.V];
  for (int64_t c = (int64_t)blockIdx.x * per + sub; c < chunks; c += (int64_t)gridDim.x * per)
    sum_chunk<U, ODD>(a, Runs{a}, T, t, C, c, all);
}

// The run that starts in chunk c and goes on behind it: its sums in order.
constexpr int JOIN_AHEAD = 16;
template <int U, bool ODD, class R>
__device__ __forceinline__ void join_chunk(const EmbedArgs& a, const R& runs, int T, int t, int C, int64_t c,
                                           int64_t all) {
  if ((c + 1) * C >= all) return;
  const int v = runs.at((c + 1) * C - 1).y;
  const int64_t from = runs.start(v), to = runs.start(v + 1);
  if (from < c * C || to <= (c + 1) * C) return;
  const int64_t last = (to - 1) / C;
  for (int d = t * U; d < a.D; d += T * U) {
    float s[U];
    load_unit<U, false>(runs.part(c * 2 + 1), false, d, U, s);
    int64_t k = c + 1;
    for (; k + JOIN_AHEAD <= last + 1; k += JOIN_AHEAD) {
      float e[JOIN_AHEAD][U];
#pragma unroll
      for (int h = 0; h < JOIN_AHEAD; ++h) load_unit<U, false>(runs.part((k + h) * 2), false, d, U, e[h]);
#pragma unroll
      for (int h = 0; h < JOIN_AHEAD; ++h)
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] += e[h][i];
    }
    for (; k <= last; ++k) {
      float e[U];
      load_unit<U, false>(runs.part(k * 2), false, d, U, e);
#pragma unroll
      for (int i = 0; i < U; ++i) s[i] += e[i];
    }
    put_row<U, ODD>(a, v, d, s);
  }
}

// The runs over several chunks, then zeros for the tokens that occur nowhere (behind the
// runs, whose partials come one after the other: a launch of theirs took 15 us more).
template <int U, bool ODD>
__global__ __launch_bounds__(NT) void embed_join_kernel(EmbedArgs a, int T, int C, int64_t joins, int64_t items) {
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t all = a.starts[a.V];
  for (int64_t i = (int64_t)blockIdx.x * per + sub; i < items; i += (int64_t)gridDim.x * per) {
    if (i < joins) {
      join_chunk<U, ODD>(a, Runs{a}, T, t, C, i, all);
    } else {
      const int64_t v = i - joins;
      if (a.starts[v] != a.starts[v + 1]) continue;
      float z[U];
#pragma unroll
      for (int k = 0; k < U; ++k) z[k] = 0.0f;
      for (int d = t * U; d < a.D; d += T * U) store_unit<U, ODD>(a.d_table, a.dtable_bf16, v * a.D + d, a.D - d, z);
    }
  }
}

// A batch whose chunks' sums fit into LDS, in one launch: a workgroup per span of tokens
// sorts its places and sums them.  1024 rows of D 64 into 1024 tokens take 13.6 us in
// three launches, 9.3 so; 8 rows of D 2048 on top of a table 14.3 and 8.4.  Zeros for a
// large table keep to the join, whose many workgroups write them faster (8 rows into 50257
// tokens of D 2048 84 us there, 92 so).
constexpr int FEW_SUMS = 16384;                 // floats of LDS for them
constexpr int FEW_CHUNK = 8;
constexpr int64_t FEW_ZEROS = (int64_t)1 << 25; // elements of a table that it writes zeros to
struct LocalRuns {
  const EmbedArgs& a;
  const int* list;  // place | token of the span << 16
  const int* tot;
  float* sums;
  int lo;
  __device__ __forceinline__ int2 at(int64_t p) const {
    return make_int2(list[p] & 0xffff, lo + (list[p] >> 16));
  }
  __device__ __forceinline__ int64_t start(int v) const { return tot[v - lo]; }
  __device__ __forceinline__ float* part(int64_t row) const { return sums + row * part_row(a.D); }
};
template <int U, bool ODD>
__global__ __launch_bounds__(NT) void embed_few_kernel(EmbedArgs a, int span, int T) {
  __shared__ SortLds<NT / 64> lds;
  __shared__ int list[SORT_FEW];
  __shared__ __attribute__((aligned(16))) float sums[FEW_SUMS];
  const int lo = blockIdx.x * span, own = min(span, a.V - lo);
  sort_span<NT / 64, true>(a, span, lds, [&](int at, int n, int v) { list[at] = n | (v - lo) << 16; });
  __syncthreads();
  const LocalRuns runs{a, list, lds.tot, sums, lo};
  const int all = lds.tot[own], chunks = (all + FEW_CHUNK - 1) / FEW_CHUNK;
  const int per = NT / T, sub = threadIdx.x / T, t = threadIdx.x % T;
  for (int c = sub; c < chunks; c += per) sum_chunk<U, ODD>(a, runs, T, t, FEW_CHUNK, c, all);
  __syncthreads();
  for (int c = sub; c < chunks - 1; c += per) join_chunk<U, ODD>(a, runs, T, t, FEW_CHUNK, c, all);
  if (a.accumulate) return;
  float z[U];
#pragma unroll
  for (int k = 0; k < U; ++k) z[k] = 0.0f;
  for (int b = sub; b < own; b += per) {
    if (lds.tot[b] != lds.tot[b + 1]) continue;
    for (int d = t * U; d < a.D; d += T * U) store_unit<U, ODD>(a.d_table, a.dtable_bf16, (int64_t)(lo + b) * a.D + d, a.D - d, z);
  }
}

// Elements per thread and step: 8 where both tensors are bf16, 4 where fp32 is among
// them (16 bytes of it, so that a wave's accesses lie side by side: two halves of 32 bytes
// a lane took 221 us for a backward's sums of 65536 x 2048, against 197).
int unit_of(bool p_bf16, bool q_bf16) { return p_bf16 && q_bf16 ? 8 : 4; }
// Whether those do not divide the rows, or their places (an element a thread, such a
// lookup of 65536 rows of D 1001 took 129 us, 67 in units at the elements' alignment; a
// gradient of 20000 rows of D 1289 into 20000 tokens 103, 80).
bool odd(int u, int D, const void* p, bool p_bf16, const void* q, bool q_bf16) {
  const auto fits = [&](const void* at, bool bf16) {
    return reinterpret_cast<uintptr_t>(at) % (u * (bf16 ? 2 : 4)) == 0;
  };
  return D % u != 0 || !fits(p, p_bf16) || !fits(q, q_bf16);
}

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

template <int U, bool ODD>
void launch_bw(const EmbedArgs& a, int span, hipStream_t s) {
  const unsigned spans = (unsigned)((a.V + span - 1) / span);
  // (a chunk has two sums)
  if (a.rows <= SORT_FEW && (a.rows + FEW_CHUNK - 1) / FEW_CHUNK * 2 * part_row(a.D) <= FEW_SUMS &&
      (a.accumulate || (int64_t)a.V * a.D <= FEW_ZEROS)) {
    embed_few_kernel<U, ODD><<<spans, NT, 0, s>>>(a, span, threads_per_row((a.D + U - 1) / U));
    return;
  }
  if (a.rows <= SORT_FEW)
    embed_sort_kernel<4><<<spans, 256, 0, s>>>(a, span);
  else
    embed_sort_kernel<16><<<spans, 1024, 0, s>>>(a, span);
  const int T = threads_per_row((a.D + U - 1) / U), per = NT / T, C = chunk_rows(a.rows);
  const int64_t chunks = (a.rows + C - 1) / C, joins = chunks > 1 ? chunks - 1 : 0;
  const int64_t items = joins + (a.accumulate ? 0 : a.V);
  if (chunks > 0) embed_sum_kernel<U, ODD><<<grid_of(chunks, per, a.n_cu), NT, 0, s>>>(a, T, C, chunks);
  if (items > 0) embed_join_kernel<U, ODD><<<grid_of(items, per, a.n_cu), NT, 0, s>>>(a, T, C, joins, items);
}

}  // namespace

int64_t mxm_embed_part_floats(int64_t max_rows, int D) {
  return std::max((std::min(max_rows, LONG_BATCH - 1) + 7) / 8, (max_rows + 31) / 32) * 2 * part_row(D);
}

void mxm_launch_embed(const EmbedArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  const int U = unit_of(a.table_bf16, a.out_bf16);
  const int T = threads_per_row((a.D + U - 1) / U);
  const unsigned grid = grid_of(a.rows, NT / T, a.n_cu);
  const auto launch = [&](auto kernel) { kernel<<<grid, NT, 0, s>>>(a, T); };
  if (odd(U, a.D, a.table, a.table_bf16, a.out, a.out_bf16))
    U == 8 ? launch(embed_kernel<8, true>) : launch(embed_kernel<4, true>);
  else
    U == 8 ? launch(embed_kernel<8, false>) : launch(embed_kernel<4, false>);
}

void mxm_launch_embed_bw(const EmbedArgs& a, hipStream_t s) {
  const int span = std::min(SORT_SPAN, (a.V + a.n_cu - 1) / a.n_cu);
  // (bf16 rows of D 100, 5000 into 2000 tokens: 19.7 us in whole units of 4, 26.0 in 8 and
  // a part)
  const auto uneven = [&](int u) { return odd(u, a.D, a.d_out, a.grad_bf16, a.d_table, a.dtable_bf16); };
  if (unit_of(a.grad_bf16, a.dtable_bf16) == 8 && !uneven(8))
    launch_bw<8, false>(a, span, s);
  else if (!uneven(4))
    launch_bw<4, false>(a, span, s);
  else
    launch_bw<4, true>(a, span, s);
}
