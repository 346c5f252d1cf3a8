// Shared by the residual norm's two directions: how a row lies in threads, typed
// loads and stores, sums over a row.
//
// A row is held in registers from its one load to its last use, and the next
// row's loads are on their way meanwhile.  V = 4 consecutive elements (16 bytes
// of fp32) lie in a thread, NV such vectors a thread; LPR threads of a wave hold
// a row (rows side by side in the wave), or, with LPR 0, a workgroup of a row's
// length does (LPR -1: one of over 512 threads, whose registers do not hold a
// second row).
//
// Kernels with ODD 0 need D % 4 == 0 and tensors aligned to their vectors; the
// others take the rest: the part's vector loads and stores need no more than an
// element's alignment, and a row's last vector may be short.  134 M elements of
// 1024 / 1030 / 1023 channels take 312 / 458 / 384 us forwards and 571 / 658 /
// 645 backwards in fp32, 180 / 290 / 227 and 265 / 459 / 342 in bf16; such rows
// share cache lines, so their loads stay in the caches' usual replacement.  Just
// past a shape's widths lanes idle as well: 65 channels 410 and 651 us in fp32,
// 312 and 523 in bf16, 2049 channels 552 and 640, 332 and 590.
#pragma once

#include <type_traits>

#include "mxm_kernels.h"
#include "mxm_train.h"

namespace resnorm {

constexpr int THREADS = 256;  // of a workgroup that holds several rows

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// The same at any element's address.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2u __attribute__((ext_vector_type(2), aligned(2)));

enum Kind { F32 = 0, BF16 = 1 };

constexpr int V = 4;

// V elements as they come from memory.
template <int K>
using Raw = std::conditional_t<K == BF16, u2, f4>;
template <int K>
using Element = std::conditional_t<K == BF16, uint16_t, float>;

__device__ __forceinline__ void widen(u2 w, float* out) {
  out[0] = mxm_u2f(w[0] << 16);
  out[1] = mxm_u2f(w[0] & 0xffff0000u);
  out[2] = mxm_u2f(w[1] << 16);
  out[3] = mxm_u2f(w[1] & 0xffff0000u);
}

// Elements [at, at + V) of a row of D that starts at p[row].  Of a row's short last
// vector (ODD) these are the row's last V, which unpack moves down; a row
// shorter than that (ODD 2: possible) is read by elements.
template <int K, int ODD>
__device__ __forceinline__ Raw<K> load(const void* p, size_t row, int at, int D) {
  const Element<K>* q = static_cast<const Element<K>*>(p) + row;
  if constexpr (!ODD) {
    return __builtin_nontemporal_load(reinterpret_cast<const Raw<K>*>(q + at));
  } else {
    if (ODD == 2 && D < V) {  // (at is 0)
      Raw<K> r = {};
      if constexpr (K == BF16) {
        r[0] = q[0] | (D > 1 ? (uint32_t)q[1] << 16 : 0u);
        if (D > 2) r[1] = q[2];
      } else {
        r[0] = q[0];
        if (D > 1) r[1] = q[1];
        if (D > 2) r[2] = q[2];
      }
      return r;
    }
    using Any = std::conditional_t<K == BF16, u2u, f4u>;
    return *reinterpret_cast<const Any*>(q + min(at, D - V));
  }
}
// Their values, zeros behind the row.
template <int K, int ODD>
__device__ __forceinline__ void unpack(Raw<K> w, int at, int D, float* out) {
  const int over = !ODD || (ODD == 2 && D < V) ? 0 : max(at + V - D, 0) & 3;  // (past the row all is 0)
  if constexpr (K == BF16) {
    if (ODD) {
      const uint64_t u = ((uint64_t)w[1] << 32 | w[0]) >> (16 * over);
      w = u2{(uint32_t)u, (uint32_t)(u >> 32)};
    }
    widen(w, out);
  } else {
    if (ODD) {
      if (over & 1) w = f4{w[1], w[2], w[3], 0.0f};
      if (over & 2) w = f4{w[2], w[3], 0.0f, 0.0f};
    }
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = w[j];
  }
}

// Rounds v to the type it is kept in and stores what of it lies in the row; v holds
// the kept values afterwards.
template <int K, int ODD>
__device__ __forceinline__ void store(void* p, size_t row, int at, int D, float* v) {
  Element<K>* q = static_cast<Element<K>*>(p) + row + at;
  Raw<K> w;
  if constexpr (K == BF16) {
    w = u2{mxm_pack_bf2_fast(v[0], v[1]), mxm_pack_bf2_fast(v[2], v[3])};
    widen(w, v);
  } else {
    w = f4{v[0], v[1], v[2], v[3]};
  }
  if constexpr (!ODD) {
    __builtin_nontemporal_store(w, reinterpret_cast<Raw<K>*>(q));
  } else if (at + V <= D) {
    using Any = std::conditional_t<K == BF16, u2u, f4u>;
    *reinterpret_cast<Any*>(q) = w;
  } else {
#pragma unroll
    for (int j = 0; j < V - 1; ++j) {
      if (at + j >= D) continue;
      if constexpr (K == BF16)
        q[j] = (uint16_t)(mxm_f2u(v[j]) >> 16);
      else
        q[j] = v[j];
    }
  }
}

__device__ __forceinline__ float load_one(const void* p, bool bf, size_t i) {
  return bf ? mxm_bf2f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}
// Values [at, at + V) of a scale, or of a gate's row, of D channels, which many rows
// read; zeros behind them; null: ones.
template <int ODD>
__device__ __forceinline__ void load_scale(const void* p, bool bf, size_t row, int at, int D,
                                           float* out) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = !ODD || at + j < D ? 1.0f : 0.0f;
  } else if constexpr (ODD) {
    if (bf)
      unpack<BF16, ODD>(load<BF16, ODD>(p, row, at, D), at, D, out);
    else
      unpack<F32, ODD>(load<F32, ODD>(p, row, at, D), at, D, out);
  } else if (bf) {
    widen(*reinterpret_cast<const u2u*>(static_cast<const uint16_t*>(p) + row + at), out);
  } else {
    const f4u w = *reinterpret_cast<const f4u*>(static_cast<const float*>(p) + row + at);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = w[j];
  }
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
  int NV, lpr, threads;
  int rows() const { return lpr > 0 ? threads / lpr : 1; }  // rows a workgroup holds at once
};
// Rows so few that the time is one row's chain of steps: rows of over 512 channels
// then lie in a workgroup's threads, which hold fewer elements each.  256 / 1024
// / 2048 rows of 1024 channels, fp32, backwards: 7.6 / 9.7 / 14.5 us, a wave a row
// 12.2 / 12.0 / 14.8; 4096 rows 24.2 against 19.4.  (512 channels: 8.1 against 8.0
// at 1024 rows.)
constexpr int FEW_ROWS = 1024;
inline Shape shape_of(int D, bool backward, int64_t N) {
  if (D <= 64) return {1, 16, THREADS};
  if (D <= 128) return {1, 32, THREADS};
  if (D <= 512 || (D <= 1024 && N > FEW_ROWS)) return {(D + 255) / 256, 64, THREADS};
  const int nv = D <= (backward ? 8192 : 4096) ? 2 : 4, per = V * nv * 64;
  const int threads = (D + per - 1) / per * 64;
  return {nv, threads > 512 ? -1 : 0, threads};
}
constexpr int most_threads(int lpr) { return lpr > 0 ? THREADS : lpr == 0 ? 512 : 1024; }

inline bool aligned(const void* p, bool bf16) {
  return reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16) == 0;
}

// f(NV, LPR) of a shape_of(D, BACKWARD) (std::integral_constants).
template <bool BACKWARD, class F>
void with_shape(const Shape& sh, F f) {
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
  if constexpr (BACKWARD) {
    if (sh.NV == 2) MXM_CASE(2, -1);
  } else {
    if (sh.lpr == 0) MXM_CASE(4, 0);
  }
  MXM_CASE(4, -1);
#undef MXM_CASE
}
// f(K0, K1, K2, ODD) of three types.
template <class F>
void with_types(bool bf0, bool bf1, bool bf2, bool odd, F f) {
  auto as = [](bool on, auto g) { on ? g(std::true_type()) : g(std::false_type()); };
  auto k = [](auto bf) { return std::integral_constant<int, decltype(bf)::value ? BF16 : F32>(); };
  as(bf0, [&](auto a) {
    as(bf1, [&](auto b) {
      as(bf2, [&](auto c) { as(odd, [&](auto o) { f(k(a), k(b), k(c), o); }); });
    });
  });
}

}  // namespace resnorm
