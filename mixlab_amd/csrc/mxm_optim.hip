// A set of gradients: their global norm, clipping by it, and the AdamW step
// with that clipping in it.
//
//   norm = sqrt(sum g^2)                                   in 64 bits
//   coef = min(1, max_norm / (norm + 1e-6))                (1 where the norm is not finite in fp32)
//   g' = coef g
//   m = beta1 m + (1 - beta1) g',  v = beta2 v + (1 - beta2) g'^2
//   p = p - lr decay p - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)
// Such a norm leaves p, m, v and the step count as they were.
// Bound by memory: the norm of 201 M fp32 gradients 120 us (6.7 TB/s; 115 at the
// rate of a plain read stream), AdamW over 403 M parameters with bf16 copies 2.00
// ms of 12.1 GB (6.0 TB/s) after the norm's 0.23.
#include <algorithm>

#include "mxm_kernels.h"
#include "mxm_train.h"

namespace {

constexpr int THREADS = 256;

constexpr int UNROLL = 4;  // vectors in flight per thread and tensor

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// The same at any element's address.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));

// A vector that is read or written once; EVEN: at its own boundary.
template <bool EVEN, class T, class U>
__device__ __forceinline__ T get(const void* p, int i) {
  if constexpr (EVEN)
    return __builtin_nontemporal_load(static_cast<const T*>(p) + i);
  else
    return static_cast<const U*>(p)[i];
}
template <bool EVEN, class T, class U>
__device__ __forceinline__ void put(void* p, int i, T v) {
  if constexpr (EVEN)
    __builtin_nontemporal_store(v, static_cast<T*>(p) + i);
  else
    static_cast<U*>(p)[i] = v;
}

__device__ __forceinline__ float lo16(uint32_t w) { return mxm_u2f(w << 16); }
__device__ __forceinline__ float hi16(uint32_t w) { return mxm_u2f(w & 0xffff0000u); }
__device__ __forceinline__ float grad_at(const void* g, bool bf16, int i) {
  return bf16 ? mxm_bf2f(static_cast<const uint16_t*>(g)[i]) : static_cast<const float*>(g)[i];
}

// Elements before `p`'s next boundary of V elements of `size` bytes.
__device__ __forceinline__ int head_of(const void* p, int size, int V) {
  const int at = (int)(reinterpret_cast<uintptr_t>(p) & (uintptr_t)(V * size - 1)) / size;
  return at ? V - at : 0;
}
// Whether `p` is at such a boundary `head` elements on.
__device__ __forceinline__ bool meets(const void* p, int size, int V, int head) {
  return ((reinterpret_cast<uintptr_t>(p) + (uintptr_t)(head * size)) & (uintptr_t)(V * size - 1)) == 0;
}

// f(i) for vectors i of [0, n), up to UNROLL at a time: load(i, slot) of all of
// them before use(i, slot) of the first.
template <class Load, class Use>
__device__ __forceinline__ void each_vector(int n, Load load, Use use) {
  int i = threadIdx.x;
  for (; i + (UNROLL - 1) * THREADS < n; i += UNROLL * THREADS) {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) load(i + k * THREADS, k);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) use(i + k * THREADS, k);
  }
  for (; i < n; i += THREADS) {
    load(i, 0);
    use(i, 0);
  }
}
// f(i) for the elements outside the vectors: [0, head) and [tail, count).
template <class F>
__device__ __forceinline__ void each_rest(int head, int tail, int count, F f) {
  for (int i = threadIdx.x; i < head; i += THREADS) f(i);
  for (int i = tail + (int)threadIdx.x; i < count; i += THREADS) f(i);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = mxm_xor_lane((uint32_t)u, s), hi = mxm_xor_lane((uint32_t)(u >> 32), s);
    v = v + __builtin_bit_cast(double, lo | hi << 32);
  }
  return v;
}

// Sum over the workgroup, in thread 0.
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += red[w];
  __syncthreads();
  return s;
}

__device__ __forceinline__ void finish_norm(const GradArgs& a, double total) {
  // (a captured step may be replayed after a bind without params: it updates nothing)
  const bool bound = !a.adamw || a.n_chunks == 0 || a.chunks[0].p != nullptr;
  const double norm = sqrt(total);
  const float shown = (float)norm;
  const bool finite = shown <= 3.40282347e38f;  // (what *norm says; false for NaN too)
  if (a.norm) *a.norm = shown;
  double coef = 1.0;
  if (finite && a.max_norm > 0.0) {
    coef = a.max_norm / (norm + 1e-6);
    if (coef > 1.0) coef = 1.0;
  }
  GradScalars r;
  r.coef = (float)coef;
  r.skip = !finite || !bound;
  r.step_size = r.root2 = 0.0f;
  if (a.adamw) {
    if (a.skipped) *a.skipped = r.skip;
    if (!r.skip) {
      const int64_t done = *a.step, t = (done > 0 ? done : 0) + 1;
      *a.step = t;
      r.step_size = (float)(a.lr / (1.0 - pow(a.beta1, (double)t)));
      r.root2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
    }
  }
  *a.scalars = r;
}

// s and the squares of a chunk; ONCE: it is not read again soon.
template <bool ONCE>
__device__ __forceinline__ double add_squares(const GradChunk& k, double s) {
  auto add = [&](float v) { s = __builtin_fma((double)v, (double)v, s); };
  auto read = [](const auto* p) {
    if constexpr (ONCE)
      return __builtin_nontemporal_load(p);
    else
      return *p;
  };
  const bool bf = k.bf16 != 0;
  const int V = bf ? 8 : 4;  // elements of 16 bytes
  const int head = min(head_of(k.g, bf ? 2 : 4, V), k.count);
  const int n = (k.count - head) / V;
  if (bf) {
    const u4* g = reinterpret_cast<const u4*>(static_cast<const uint16_t*>(k.g) + head);
    u4 w[UNROLL];
    each_vector(n, [&](int i, int j) { w[j] = read(g + i); },
                [&](int, int j) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    add(lo16(w[j][e]));
                    add(hi16(w[j][e]));
                  }
                });
  } else {
    const f4* g = reinterpret_cast<const f4*>(static_cast<const float*>(k.g) + head);
    f4 w[UNROLL];
    each_vector(n, [&](int i, int j) { w[j] = read(g + i); },
                [&](int, int j) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) add(w[j][e]);
                });
  }
  each_rest(head, head + n * V, k.count, [&](int i) { add(grad_at(k.g, bf, i)); });
  return s;
}

// The squares of whole chunks per workgroup, one sum each.  Up to TICKET_BLOCKS
// workgroups the last one to finish adds them; past that a second launch does:
// every ticket costs about 45 ns (its release writes an L2 back), one after the
// other.  Ticket / second launch at 32 workgroups 3.9 / 5.4 us, at 64 6.5 /
// 6.7, at 256 8.1 / 5.3, and for 805 MB (2048 / 1024 workgroups) 213 / 119 us,
// which is 6.8 TB/s.
constexpr int TICKET_BLOCKS = 32, MOST_BLOCKS = 1024;

__global__ __launch_bounds__(THREADS) void grad_norm_kernel(GradArgs a) {
  __shared__ double red[THREADS / 64];
  __shared__ int s_last;
  double s = 0.0;
  for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const GradChunk k = a.chunks[c];
    if (c < a.keep_from)
      s = add_squares<true>(k, s);
    else
      s = add_squares<false>(k, s);
  }
  s = block_sum(s, red);
  if (gridDim.x > TICKET_BLOCKS) {
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
    return;
  }
  // One thread stores the sum and takes the ticket, so the ticket's release
  // covers its store; the last workgroup's acquire covers everybody's.
  if (threadIdx.x == 0) {
    __hip_atomic_store(a.partial + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  s = 0.0;
  if (threadIdx.x < gridDim.x)
    s = __hip_atomic_load(a.partial + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s = block_sum(s, red);
  if (threadIdx.x == 0) {
    finish_norm(a, s);
    __hip_atomic_store(a.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// Adds the workgroups' sums, one a thread.
__global__ __launch_bounds__(MOST_BLOCKS) void grad_norm_finish_kernel(GradArgs a, int blocks) {
  __shared__ double red[MOST_BLOCKS / 64];
  const double s = block_sum((int)threadIdx.x < blocks ? a.partial[threadIdx.x] : 0.0, red);
  if (threadIdx.x == 0) finish_norm(a, s);
}

// Clip and AdamW run one vector a thread and no loop: every workgroup takes one
// slice of THREADS vectors of a chunk, the last slices first (what the norm
// read last is what the last-level cache still holds).  Streams of such short
// workgroups in address order, past the caches' usual replacement, reach 6.1
// (AdamW) and 6.6 TB/s (one tensor in, one out) over 1 GiB tensors; workgroups
// that stay and loop over chunks 5.1-5.4 and 5.3-5.7.
struct Slice {
  int head, n, at;  // scalar elements in front, vectors, this thread's vector
};
__device__ __forceinline__ Slice slice_of(int head, int count, int V, int sub) {
  return {head, (count - head) / V, sub * THREADS + (int)threadIdx.x};
}
// f(i) for the elements outside the chunk's vectors, spread over its slices.
template <class F>
__device__ __forceinline__ void each_other(const Slice& s, int V, int count, int slices, F f) {
  for (int i = s.at; i < s.head; i += slices * THREADS) f(i);
  for (int i = s.head + s.n * V + s.at; i < count; i += slices * THREADS) f(i);
}

template <bool EVEN>
__device__ __forceinline__ void clip_vector(const void* g, void* out, bool bf, int i, float coef) {
  if (bf) {
    const u4 w = get<EVEN, u4, u4u>(g, i);
    u4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = mxm_pack_bf2_fast(lo16(w[e]) * coef, hi16(w[e]) * coef);
    put<EVEN, u4, u4u>(out, i, r);
  } else {
    put<EVEN, f4, f4u>(out, i, get<EVEN, f4, f4u>(g, i) * coef);
  }
}

__global__ __launch_bounds__(THREADS) void grad_clip_kernel(GradArgs a) {
  const int b = a.first_slice - (int)blockIdx.x;
  const GradChunk k = a.chunks[b / a.slices];
  const float coef = a.scalars->coef;
  if (coef == 1.0f && k.clipped == k.g) return;  // (in place, and nothing to clip)
  const bool bf = k.bf16 != 0;
  const int V = bf ? 8 : 4, size = bf ? 2 : 4;
  // (tensors out of step with each other: vectors at any address, from the start on)
  int head = min(head_of(k.g, size, V), k.count);
  const bool even = meets(k.clipped, size, V, head);
  if (!even) head = 0;
  const Slice s = slice_of(head, k.count, V, b % a.slices);
  const char* g = static_cast<const char*>(k.g) + head * size;
  char* out = static_cast<char*>(k.clipped) + head * size;
  if (s.at < s.n) {
    if (even)
      clip_vector<true>(g, out, bf, s.at, coef);
    else
      clip_vector<false>(g, out, bf, s.at, coef);
  }
  each_other(s, V, k.count, a.slices, [&](int i) {
    const float g = grad_at(k.g, bf, i) * coef;
    if (bf)
      static_cast<uint16_t*>(k.clipped)[i] = mxm_f2bf(g);
    else
      static_cast<float*>(k.clipped)[i] = g;
  });
}

struct AdamScalars {
  float coef, step_size, root2, b1, c1, b2, c2, eps, decay;
};
__device__ __forceinline__ void adamw_one(const AdamScalars& r, float g, float& p, float& m,
                                          float& v) {
  g = g * r.coef;
  m = __builtin_fmaf(r.b1, m, r.c1 * g);
  v = __builtin_fmaf(r.b2, v, (r.c2 * g) * g);
  const float u = (r.step_size * m) / (__builtin_sqrtf(v) * r.root2 + r.eps);
  p = p - __builtin_fmaf(r.decay, p, u);
}

template <bool EVEN>
__device__ __forceinline__ void adamw_vector(const GradChunk& k, const AdamScalars& r, int head,
                                             int i) {
  f4 g;
  if (k.bf16) {
    const u2 w = get<EVEN, u2, u2u>(static_cast<const uint16_t*>(k.g) + head, i);
    g = f4{lo16(w[0]), hi16(w[0]), lo16(w[1]), hi16(w[1])};
  } else {
    g = get<EVEN, f4, f4u>(static_cast<const float*>(k.g) + head, i);
  }
  f4 m = get<EVEN, f4, f4u>(k.m + head, i), v = get<EVEN, f4, f4u>(k.v + head, i),
     p = get<EVEN, f4, f4u>(k.p + head, i);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float pe = p[e], me = m[e], ve = v[e];
    adamw_one(r, g[e], pe, me, ve);
    p[e] = pe;
    m[e] = me;
    v[e] = ve;
  }
  put<EVEN, f4, f4u>(k.m + head, i, m);
  put<EVEN, f4, f4u>(k.v + head, i, v);
  put<EVEN, f4, f4u>(k.p + head, i, p);
  if (k.p16)
    put<EVEN, u2, u2u>(k.p16 + head, i,
                       u2{mxm_pack_bf2_fast(p[0], p[1]), mxm_pack_bf2_fast(p[2], p[3])});
}

__global__ __launch_bounds__(THREADS) void grad_adamw_kernel(GradArgs a) {
  const int b = a.first_slice - (int)blockIdx.x;
  const GradChunk k = a.chunks[b / a.slices];
  const GradScalars sc = *a.scalars;
  if (sc.skip) return;
  const bool bf = k.bf16 != 0;
  int head = min(head_of(k.p, 4, 4), k.count);
  const bool even = meets(k.m, 4, 4, head) && meets(k.v, 4, 4, head) &&
                    meets(k.g, bf ? 2 : 4, 4, head) && (!k.p16 || meets(k.p16, 2, 4, head));
  if (!even) head = 0;
  const Slice s = slice_of(head, k.count, 4, b % a.slices);
  AdamScalars r;
  r.coef = sc.coef;
  r.step_size = sc.step_size;
  r.root2 = sc.root2;
  r.b1 = a.b1;
  r.c1 = a.c1;
  r.b2 = a.b2;
  r.c2 = a.c2;
  r.eps = a.eps32;
  r.decay = a.lr_decay * k.decay;
  if (s.at < s.n) {
    if (even)
      adamw_vector<true>(k, r, head, s.at);
    else
      adamw_vector<false>(k, r, head, s.at);
  }
  each_other(s, 4, k.count, a.slices, [&](int i) {
    float p = k.p[i], m = k.m[i], v = k.v[i];
    adamw_one(r, grad_at(k.g, bf, i), p, m, v);
    k.m[i] = m;
    k.v[i] = v;
    k.p[i] = p;
    if (k.p16) k.p16[i] = mxm_f2bf(p);
  });
}

}  // namespace

// Pieces that still make eight workgroups a CU for the norm, and at most 64 KB of
// fp32.
int mxm_grad_chunk_elems(int64_t total, int n_cu) {
  int64_t per = 4096;
  while (per < 16384 && total / (per * 2) >= 8 * (int64_t)n_cu) per *= 2;
  return (int)per;
}

// Of gradients that clip or AdamW reads next, the norm reads the last ones, about
// as much as the last-level cache holds, with plain loads and the rest with
// nontemporal ones.  None / 64 / 128 / 192 / 256 MB / all with plain loads (one
// sweep; runs of the last case differ by up to 1.7 %, so 192 MB to all are not told
// apart there): clipping 134 M bf16 130.6 / 130.4 / 128.8 / 126.9 / 125.9 /
// 125.2 us, AdamW over 16.8 M 95.7 / 88.1 / 88.0 / 88.0 / 88.0 / 88.1, over 403 M
// 2298 / 2287 / 2280 / 2266 / 2244 / 2272; a norm alone, of 201 M fp32,
// 119.6 with none, 133 with all.
constexpr int64_t KEPT_BYTES = 256ll << 20;

int mxm_grad_norm_blocks(int n_chunks) { return std::max(1, std::min(n_chunks, MOST_BLOCKS)); }

void mxm_launch_grad_norm(const GradArgs& args, bool again, hipStream_t s) {
  GradArgs a = args;
  a.keep_from = again ? (int)std::max<int64_t>(
                            a.n_chunks - KEPT_BYTES / ((int64_t)a.chunk_elems * (a.all_bf16 ? 2 : 4)), 0)
                      : a.n_chunks;
  const int blocks = mxm_grad_norm_blocks(a.n_chunks);
  hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(THREADS), 0, s, a);
  if (blocks > TICKET_BLOCKS)
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3((blocks + 63) / 64 * 64), 0, s, a, blocks);
}
// f(a, workgroups) for all of a's slices, the last first, in launches whose threads
// are counted in 32 bits.
template <class F>
void each_launch(GradArgs a, F f) {
  constexpr int MOST = 1 << 23;
  for (int64_t left = (int64_t)a.n_chunks * a.slices; left > 0; left -= MOST) {
    a.first_slice = (int)(left - 1);
    f(a, (unsigned)std::min<int64_t>(left, MOST));
  }
}
void mxm_launch_grad_clip(const GradArgs& args, hipStream_t s) {
  GradArgs a = args;
  a.slices = a.chunk_elems / (THREADS * (a.all_bf16 ? 8 : 4));
  each_launch(a, [&](const GradArgs& l, unsigned blocks) {
    hipLaunchKernelGGL(grad_clip_kernel, dim3(blocks), dim3(THREADS), 0, s, l);
  });
}
void mxm_launch_grad_adamw(const GradArgs& args, hipStream_t s) {
  GradArgs a = args;
  a.slices = a.chunk_elems / (THREADS * 4);
  a.b1 = (float)a.beta1;
  a.c1 = (float)(1.0 - a.beta1);
  a.b2 = (float)a.beta2;
  a.c2 = (float)(1.0 - a.beta2);
  a.eps32 = (float)a.eps;
  a.lr_decay = (float)(a.lr * a.weight_decay);
  each_launch(a, [&](const GradArgs& l, unsigned blocks) {
    hipLaunchKernelGGL(grad_adamw_kernel, dim3(blocks), dim3(THREADS), 0, s, l);
  });
}
