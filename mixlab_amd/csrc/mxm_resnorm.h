// Shared by the residual norm's two directions: how a row lies in threads, typed
// loads and stores, sums over a row.
//
// A row is held in registers from its one load to its last use, and the next
// row's loads are on their way meanwhile.  V consecutive elements (16 bytes of
// fp32) lie in a thread, NV such vectors a thread; LPR threads of a wave hold a
// row (rows side by side in the wave), or, with LPR 0, a workgroup of a row's
// length does (LPR -1: one of over 512 threads, whose registers do not hold a
// second row).  V = 4 needs D % 4 == 0 and aligned tensors; V = 1 takes any.
#pragma once

#include <type_traits>

#include "mxm_kernels.h"
#include "mxm_train.h"

namespace resnorm {

constexpr int THREADS = 256;  // of a workgroup that holds several rows

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

enum Kind { F32 = 0, BF16 = 1, ANY = 2 };  // ANY: `bf` says

// V elements as they come from memory.
template <int K, int V>
using Raw = std::conditional_t<V == 4, std::conditional_t<K == BF16, u2, f4>, float>;

template <int K, int V>
__device__ __forceinline__ Raw<K, V> load(const void* p, bool bf, size_t i) {
  if constexpr (V == 4 && K == BF16)
    return __builtin_nontemporal_load(
        reinterpret_cast<const u2*>(static_cast<const uint16_t*>(p) + i));
  else if constexpr (V == 4)
    return __builtin_nontemporal_load(
        reinterpret_cast<const f4*>(static_cast<const float*>(p) + i));
  else
    return bf ? mxm_bf2f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}
template <int K, int V>
__device__ __forceinline__ void unpack(const Raw<K, V>& w, float* out) {
  if constexpr (V == 4 && K == BF16) {
    out[0] = mxm_u2f(w[0] << 16);
    out[1] = mxm_u2f(w[0] & 0xffff0000u);
    out[2] = mxm_u2f(w[1] << 16);
    out[3] = mxm_u2f(w[1] & 0xffff0000u);
  } else if constexpr (V == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = w[j];
  } else {
    out[0] = w;
  }
}

// Rounds v to the type it is kept in; v holds the kept values afterwards.
template <int K, int V>
__device__ __forceinline__ void store(void* p, bool bf, size_t i, float* v) {
  if constexpr (V == 4) {
    if (K == BF16) {
      const u2 w = {mxm_pack_bf2_fast(v[0], v[1]), mxm_pack_bf2_fast(v[2], v[3])};
      __builtin_nontemporal_store(w, reinterpret_cast<u2*>(static_cast<uint16_t*>(p) + i));
      v[0] = mxm_u2f(w[0] << 16);
      v[1] = mxm_u2f(w[0] & 0xffff0000u);
      v[2] = mxm_u2f(w[1] << 16);
      v[3] = mxm_u2f(w[1] & 0xffff0000u);
    } else {
      __builtin_nontemporal_store(f4{v[0], v[1], v[2], v[3]},
                                  reinterpret_cast<f4*>(static_cast<float*>(p) + i));
    }
  } else {
    if (bf) {
      const uint16_t b = mxm_f2bf(v[0]);
      static_cast<uint16_t*>(p)[i] = b;
      v[0] = mxm_bf2f(b);
    } else {
      static_cast<float*>(p)[i] = v[0];
    }
  }
}

// V values of a scale or a gate, which many rows read; null: ones.
template <int V>
__device__ __forceinline__ void load_scale(const void* p, bool bf, size_t i, float* out) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = 1.0f;
    return;
  }
  if constexpr (V == 4) {  // (whole vectors where the tensor starts at one's boundary)
    if (!bf && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      unpack<F32, 4>(*reinterpret_cast<const f4*>(static_cast<const float*>(p) + i), out);
      return;
    }
    if (bf && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
      unpack<BF16, 4>(*reinterpret_cast<const u2*>(static_cast<const uint16_t*>(p) + i), out);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    out[j] = bf ? mxm_bf2f(static_cast<const uint16_t*>(p)[i + j])
                : static_cast<const float*>(p)[i + j];
}

__device__ __forceinline__ float gate_of(const ResNormArgs& a, float g) {
  return a.sigmoid ? mxm_sigmoid(g) : g;
}

// Sums of K values over a row's threads, in each of them.  LPR <= 0: `red` holds
// K floats a wave and is not written again before another barrier of the
// workgroup (callers alternate buffers).
template <int LPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* red) {
#pragma unroll
  for (int s = (LPR > 0 ? LPR : 64) / 2; s >= 1; s >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = v[k] + mxm_xor_lane_f(v[k], s);
  if constexpr (LPR <= 0) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = 0.0f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += red[w * K + k];
  }
}

// The index of the row, among those that the workgroup holds, that this thread is
// part of; a scalar where a wave or a workgroup holds one.
template <int LPR>
__device__ __forceinline__ int row_slot() {
  if constexpr (LPR == 64) return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
  if constexpr (LPR > 0) return (int)threadIdx.x / LPR;
  return 0;
}

// How rows of D elements lie in threads.
struct Shape {
  int V, NV, lpr, threads;
  int rows() const { return lpr > 0 ? threads / lpr : 1; }  // rows a workgroup holds at once
};
inline Shape shape_of(int D, bool vectors, bool backward) {
  auto workgroup = [&](int V, int nv) {
    const int per = V * nv * 64;
    const int threads = (D + per - 1) / per * 64;
    return Shape{V, nv, threads > 512 ? -1 : 0, threads};
  };
  if (vectors) {
    if (D <= 64) return {4, 1, 16, THREADS};
    if (D <= 128) return {4, 1, 32, THREADS};
    if (D <= 1024) return {4, (D + 255) / 256, 64, THREADS};
    return workgroup(4, D <= (backward ? 8192 : 4096) ? 2 : 4);
  }
  if (D <= 256) return {1, 4, 64, THREADS};
  return workgroup(1, D <= 2048 ? 4 : D <= 4096 ? 8 : 16);
}
constexpr int most_threads(int lpr) { return lpr > 0 ? THREADS : lpr == 0 ? 512 : 1024; }

inline bool aligned(const void* p, bool bf16) {
  return reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16) == 0;
}

// f(NV, LPR) of a shape with vectors of 4, or of one without (std::integral_constants).
template <class F>
void with_shape4(const Shape& sh, F f) {
  using std::integral_constant;
#define MXM_CASE(nv, l) return f(integral_constant<int, nv>(), integral_constant<int, l>())
  if (sh.lpr == 16) MXM_CASE(1, 16);
  if (sh.lpr == 32) MXM_CASE(1, 32);
  if (sh.lpr == 64) {
    if (sh.NV == 1) MXM_CASE(1, 64);
    if (sh.NV == 2) MXM_CASE(2, 64);
    if (sh.NV == 3) MXM_CASE(3, 64);
    MXM_CASE(4, 64);
  }
  if (sh.NV == 2 && sh.lpr == 0) MXM_CASE(2, 0);
  if (sh.NV == 2) MXM_CASE(2, -1);
  if (sh.lpr == 0) MXM_CASE(4, 0);
  MXM_CASE(4, -1);
}
template <class F>
void with_shape1(const Shape& sh, F f) {
  using std::integral_constant;
  if (sh.lpr == 64) MXM_CASE(4, 64);
  if (sh.NV == 4) MXM_CASE(4, 0);
  if (sh.NV == 8) MXM_CASE(8, 0);
  if (sh.lpr == 0) MXM_CASE(16, 0);
  MXM_CASE(16, -1);
#undef MXM_CASE
}
// f(K0, K1, K2) of three types.
template <class F>
void with_types(bool bf0, bool bf1, bool bf2, F f) {
  using std::integral_constant;
  auto k = [](auto bf) { return integral_constant<int, decltype(bf)::value ? BF16 : F32>(); };
  auto third = [&](auto a, auto b) { bf2 ? f(a, b, k(std::true_type())) : f(a, b, k(std::false_type())); };
  auto second = [&](auto a) { bf1 ? third(a, k(std::true_type())) : third(a, k(std::false_type())); };
  bf0 ? second(k(std::true_type())) : second(k(std::false_type()));
}

}  // namespace resnorm
