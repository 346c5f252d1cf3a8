// A set of gradients: their global norm, clipping by it, and the AdamW step
// with that clipping in it.
//
//   norm = sqrt(sum g^2)                                   in 64 bits
//   coef = min(1, max_norm / (norm + 1e-6))                (1 where the norm is not finite)
//   g' = coef g
//   m = beta1 m + (1 - beta1) g',  v = beta2 v + (1 - beta2) g'^2
//   p = p - lr decay p - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)
// A norm that is not finite leaves p, m, v and the step count as they were.
#include <algorithm>

#include "mxm_kernels.h"
#include "mxm_train.h"

namespace {

constexpr int THREADS = 256;

constexpr int UNROLL = 4;  // vectors in flight per thread and tensor

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

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
  const double norm = sqrt(total);
  const bool finite = total <= 1.7976931348623157e308;  // false for NaN too
  if (a.norm) *a.norm = (float)norm;
  double coef = 1.0;
  if (finite && a.max_norm > 0.0) {
    coef = a.max_norm / (norm + 1e-6);
    if (coef > 1.0) coef = 1.0;
  }
  GradScalars r;
  r.coef = (float)coef;
  r.skip = !finite;
  r.step_size = r.root2 = 0.0f;
  if (a.adamw) {
    if (a.skipped) *a.skipped = !finite;
    if (finite) {
      const int64_t t = *a.step + 1;
      *a.step = t;
      r.step_size = (float)(a.lr / (1.0 - pow(a.beta1, (double)t)));
      r.root2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
    }
  }
  *a.scalars = r;
}

// The squares of whole chunks per workgroup; the last workgroup to finish adds
// the workgroups' sums in their order.
__global__ __launch_bounds__(THREADS) void grad_norm_kernel(GradArgs a) {
  __shared__ double red[THREADS / 64];
  __shared__ int s_last;
  double s = 0.0;
  auto add = [&](float v) { s = __builtin_fma((double)v, (double)v, s); };
  for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const GradChunk k = a.chunks[c];
    const bool bf = k.bf16 != 0;
    const int V = bf ? 8 : 4;  // elements of 16 bytes
    const int head = min(head_of(k.g, bf ? 2 : 4, V), k.count);
    const int n = (k.count - head) / V;
    if (bf) {
      const u4* g = reinterpret_cast<const u4*>(static_cast<const uint16_t*>(k.g) + head);
      u4 w[UNROLL];
      each_vector(n, [&](int i, int j) { w[j] = g[i]; },
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
      each_vector(n, [&](int i, int j) { w[j] = g[i]; },
                  [&](int, int j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) add(w[j][e]);
                  });
    }
    each_rest(head, head + n * V, k.count, [&](int i) { add(grad_at(k.g, bf, i)); });
  }
  s = block_sum(s, red);
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
  for (int b = threadIdx.x; b < (int)gridDim.x; b += THREADS)
    s += __hip_atomic_load(a.partial + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s = block_sum(s, red);
  if (threadIdx.x == 0) {
    finish_norm(a, s);
    __hip_atomic_store(a.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// (Clip and AdamW walk the chunks backwards: what the norm read last is what the
// last-level cache still holds.)
__global__ __launch_bounds__(THREADS) void grad_clip_kernel(GradArgs a) {
  const float coef = a.scalars->coef;
  for (int c = a.n_chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const GradChunk k = a.chunks[c];
    const bool bf = k.bf16 != 0;
    const int V = bf ? 8 : 4, size = bf ? 2 : 4;
    int head = min(head_of(k.g, size, V), k.count);
    if (!meets(k.clipped, size, V, head)) head = k.count;
    const int n = (k.count - head) / V;
    if (bf) {
      const u4* g = reinterpret_cast<const u4*>(static_cast<const uint16_t*>(k.g) + head);
      u4* out = reinterpret_cast<u4*>(static_cast<uint16_t*>(k.clipped) + head);
      u4 w[UNROLL];
      each_vector(n, [&](int i, int j) { w[j] = g[i]; },
                  [&](int i, int j) {
                    u4 r;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      r[e] = (uint32_t)mxm_f2bf(lo16(w[j][e]) * coef) |
                             (uint32_t)mxm_f2bf(hi16(w[j][e]) * coef) << 16;
                    out[i] = r;
                  });
    } else {
      const f4* g = reinterpret_cast<const f4*>(static_cast<const float*>(k.g) + head);
      f4* out = reinterpret_cast<f4*>(static_cast<float*>(k.clipped) + head);
      f4 w[UNROLL];
      each_vector(n, [&](int i, int j) { w[j] = g[i]; }, [&](int i, int j) { out[i] = w[j] * coef; });
    }
    each_rest(head, head + n * V, k.count, [&](int i) {
      const float g = grad_at(k.g, bf, i) * coef;
      if (bf)
        static_cast<uint16_t*>(k.clipped)[i] = mxm_f2bf(g);
      else
        static_cast<float*>(k.clipped)[i] = g;
    });
  }
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

template <bool BF>
__device__ __forceinline__ void adamw_chunk(const GradChunk& k, const AdamScalars& r) {
  int head = min(head_of(k.p, 4, 4), k.count);
  if (!meets(k.m, 4, 4, head) || !meets(k.v, 4, 4, head) || !meets(k.g, BF ? 2 : 4, 4, head) ||
      (k.p16 && !meets(k.p16, 2, 4, head)))
    head = k.count;
  const int n = (k.count - head) / 4;
  f4 *p = reinterpret_cast<f4*>(k.p + head), *m = reinterpret_cast<f4*>(k.m + head),
     *v = reinterpret_cast<f4*>(k.v + head);
  u2* p16 = k.p16 ? reinterpret_cast<u2*>(k.p16 + head) : nullptr;
  const f4* g32 = reinterpret_cast<const f4*>(static_cast<const float*>(k.g) + head);
  const u2* g16 = reinterpret_cast<const u2*>(static_cast<const uint16_t*>(k.g) + head);
  f4 wp[UNROLL], wm[UNROLL], wv[UNROLL], wg[UNROLL];
  u2 wh[UNROLL];
  each_vector(n,
              [&](int i, int j) {
                if (BF)
                  wh[j] = g16[i];
                else
                  wg[j] = g32[i];
                wm[j] = m[i];
                wv[j] = v[i];
                wp[j] = p[i];
              },
              [&](int i, int j) {
                f4 g = wg[j];
                if (BF) g = f4{lo16(wh[j][0]), hi16(wh[j][0]), lo16(wh[j][1]), hi16(wh[j][1])};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float pe = wp[j][e], me = wm[j][e], ve = wv[j][e];
                  adamw_one(r, g[e], pe, me, ve);
                  wp[j][e] = pe;
                  wm[j][e] = me;
                  wv[j][e] = ve;
                }
                m[i] = wm[j];
                v[i] = wv[j];
                p[i] = wp[j];
                if (p16)
                  p16[i] = u2{mxm_pack_bf2_fast(wp[j][0], wp[j][1]),
                              mxm_pack_bf2_fast(wp[j][2], wp[j][3])};
              });
  each_rest(head, head + n * 4, k.count, [&](int i) {
    float p = k.p[i], m = k.m[i], v = k.v[i];
    adamw_one(r, grad_at(k.g, BF, i), p, m, v);
    k.m[i] = m;
    k.v[i] = v;
    k.p[i] = p;
    if (k.p16) k.p16[i] = mxm_f2bf(p);
  });
}

__global__ __launch_bounds__(THREADS) void grad_adamw_kernel(GradArgs a) {
  const GradScalars s = *a.scalars;
  if (s.skip) return;
  AdamScalars r;
  r.coef = s.coef;
  r.step_size = s.step_size;
  r.root2 = s.root2;
  r.b1 = (float)a.beta1;
  r.c1 = (float)(1.0 - a.beta1);
  r.b2 = (float)a.beta2;
  r.c2 = (float)(1.0 - a.beta2);
  r.eps = (float)a.eps;
  for (int c = a.n_chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const GradChunk k = a.chunks[c];
    r.decay = (float)(a.lr * a.weight_decay * (double)k.decay);
    if (k.bf16)
      adamw_chunk<true>(k, r);
    else
      adamw_chunk<false>(k, r);
  }
}

}  // namespace

// Pieces of about an eighth of a CU's share, in whole rounds of the workgroups'
// vectors.
int mxm_grad_chunk_elems(int64_t total, int n_cu) {
  constexpr int64_t round = THREADS * 4 * UNROLL;
  const int64_t share = total / (8 * (int64_t)n_cu);
  const int64_t rounds = (share + round - 1) / round;
  return (int)(round * std::max<int64_t>(1, std::min<int64_t>(rounds, 8)));
}

int mxm_grad_norm_blocks(int n_chunks) { return std::max(1, std::min(n_chunks, 2048)); }

void mxm_launch_grad_norm(const GradArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(grad_norm_kernel, dim3(mxm_grad_norm_blocks(a.n_chunks)), dim3(THREADS), 0, s, a);
}
void mxm_launch_grad_clip(const GradArgs& a, hipStream_t s) {
  if (a.n_chunks > 0)
    hipLaunchKernelGGL(grad_clip_kernel, dim3(std::min(a.n_chunks, 2048)), dim3(THREADS), 0, s, a);
}
void mxm_launch_grad_adamw(const GradArgs& a, hipStream_t s) {
  if (a.n_chunks > 0)
    hipLaunchKernelGGL(grad_adamw_kernel, dim3(std::min(a.n_chunks, 2048)), dim3(THREADS), 0, s, a);
}
