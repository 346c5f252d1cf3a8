// A set of gradients: their global norm, clipping by it, and the AdamW step
// with that clipping in it.
//
//   norm = sqrt(sum g^2)                                   in 64 bits
//   coef = min(1, max_norm / (norm + 1e-6))                (1 where the norm is not finite)
//   g' = coef g
//   m = beta1 m + (1 - beta1) g',  v = beta2 v + (1 - beta2) g'^2
//   p = p - lr decay p - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)
// A norm that is not finite leaves p, m, v and the step count as they were.
#include "mxm_kernels.h"
#include "mxm_train.h"

namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ float grad_at(const GradTensor& t, int64_t i) {
  return t.bf16 ? mxm_bf2f(static_cast<const uint16_t*>(t.g)[i])
                : static_cast<const float*>(t.g)[i];
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
  for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const GradChunk k = a.chunks[c];
    const GradTensor t = a.tensors[k.tensor];
    for (int i = threadIdx.x; i < k.count; i += THREADS) {
      const double g = (double)grad_at(t, k.start + i);
      s = __builtin_fma(g, g, s);
    }
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

__global__ __launch_bounds__(THREADS) void grad_clip_kernel(GradArgs a) {
  const float coef = a.scalars->coef;
  for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const GradChunk k = a.chunks[c];
    const GradTensor t = a.tensors[k.tensor];
    for (int i = threadIdx.x; i < k.count; i += THREADS) {
      const float g = grad_at(t, k.start + i) * coef;
      if (t.bf16)
        static_cast<uint16_t*>(t.clipped)[k.start + i] = mxm_f2bf(g);
      else
        static_cast<float*>(t.clipped)[k.start + i] = g;
    }
  }
}

__global__ __launch_bounds__(THREADS) void grad_adamw_kernel(GradArgs a) {
  const GradScalars r = *a.scalars;
  if (r.skip) return;
  for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const GradChunk k = a.chunks[c];
    const GradTensor t = a.tensors[k.tensor];
    const float decay = (float)(a.lr * a.weight_decay * (double)t.decay);
    const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1);
    const float b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2), eps = (float)a.eps;
    for (int i = threadIdx.x; i < k.count; i += THREADS) {
      const int64_t at = k.start + i;
      const float g = grad_at(t, at) * r.coef;
      const float m = __builtin_fmaf(b1, t.m[at], c1 * g);
      const float v = __builtin_fmaf(b2, t.v[at], c2 * g * g);
      const float p = t.p[at];
      const float u = r.step_size * m / (__builtin_sqrtf(v) * r.root2 + eps);
      const float q = p - __builtin_fmaf(decay, p, u);
      t.m[at] = m;
      t.v[at] = v;
      t.p[at] = q;
      if (t.p16) t.p16[at] = mxm_f2bf(q);
    }
  }
}

}  // namespace

int mxm_grad_chunk_elems(int64_t total, int n_cu) {
  (void)total;
  (void)n_cu;
  return 16384;
}

int mxm_grad_norm_blocks(int n_chunks) { return n_chunks < 1 ? 1 : n_chunks < 2048 ? n_chunks : 2048; }

void mxm_launch_grad_norm(const GradArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(grad_norm_kernel, dim3(mxm_grad_norm_blocks(a.n_chunks)), dim3(THREADS), 0, s, a);
}
void mxm_launch_grad_clip(const GradArgs& a, hipStream_t s) {
  if (a.n_chunks > 0)
    hipLaunchKernelGGL(grad_clip_kernel, dim3(a.n_chunks), dim3(THREADS), 0, s, a);
}
void mxm_launch_grad_adamw(const GradArgs& a, hipStream_t s) {
  if (a.n_chunks > 0)
    hipLaunchKernelGGL(grad_adamw_kernel, dim3(a.n_chunks), dim3(THREADS), 0, s, a);
}
