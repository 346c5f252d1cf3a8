// The token loss's three products on MFMA (gfx950, v_mfma_f32_32x32x16_bf16, or _f16 for
// fp32 operands).
//
//   C[m][n] = sum over pairs of planes and k of A(m, k) B(n, k)
//   logits:  m a vocabulary entry, n a row;  A = weight,        B = x
//   dx:      m a channel,          n a row;  A = weight (k out), B = dz
//   dw:      m a channel, n an entry;        A = x (k out),      B = dz (k out)
// An operand is either k-inner (a row holds consecutive k of one m or n) or k-out
// (a row holds one k, consecutive m or n); dz and weight are read both ways, so
// nothing is stored transposed.  Register r of lane l holds C[(r / 4) * 8 + (l / 32)
// * 4 + r % 4][l % 32] of a 32 x 32 MFMA tile.  With the vocabulary along m a lane
// owns one row's logits: the softmax's sums over a block of the vocabulary stay in
// its registers but for one exchange between the wave's halves.  With the channels
// along m a lane owns consecutive channels of one output row and stores them as
// vectors.
//
// Tiles move global -> LDS with global_load_lds_dwordx4 into a ring of NS stages of
// 64 k.  k-inner tiles come out by ds_read_b128 (16-byte chunks swizzled by the row),
// k-out ones by the transposing ds_read_b64_tr_b16: within 16 lanes, lane 4r + q
// supplies the address of row r, columns 4q..4q+3 of a 4 x 16 block and lane i
// receives column i (chunks swizzled by 4 * (k % 4)).  The fragments of the next
// 16-wide k step are read between the MFMAs of the current one; the next stage's
// loads all go out before the first (over the first two k steps a step of 16384 rows of
// D 2048 and 50257 entries took 9.70 ms, so 9.37).
//
// fp32 operands are two fp16 planes with exponents of their rows (mxm_vocab.h); of the
// four products of planes lo lo is left out, the small ones are summed first.  (As three
// bf16 planes, of whose nine products six matter, the products took twice the time: a
// step of 2048 rows, D 512 and 32768 entries 1.27 ms, 0.88 so.)
//
// The grid is persistent; each XCD (workgroup L runs on XCD L % 8) takes an eighth of
// the tile list, in groups of GN n-tiles by all m-tiles.  Products with few tiles and
// a long sum are split along k; the splits' tiles go to scratch in fp32 and are added
// in order by a second launch.
#include <algorithm>
#include <type_traits>

#include "mxm_lanes.h"
#include "mxm_vocab.h"

namespace {

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4_t* lds_bf16x4_p;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BK = 64;  // k per stage
constexpr int GN = 4;   // n-tiles per scheduling group (8: 9.37 ms for that step, 4: 9.23)

// global_load_lds_dwordx4: lane l's 16 bytes land at LDS `lds` + 16 l.  Inline asm,
// so that the compiler's tracking of LDS DMA does not drain the ring; the waits are
// explicit.  M0 holds the LDS base.
__device__ __forceinline__ void dma16(const void* g, const void* lds) {
  const unsigned base = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(g), "s"(base)
               : "memory", "m0");
}
// From a uniform 64-bit base plus the lane's 32-bit byte offset.
__device__ __forceinline__ void dma16s(const void* base, unsigned off_bytes, const void* lds) {
  const unsigned lb = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off_bytes), "s"(base), "s"(lb)
               : "memory", "m0");
}
// At most N of this thread's loads in flight, its LDS reads done, then the barrier.
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// The barrier alone, this wave's LDS accesses done.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// BM x BN per workgroup of WM x WN waves, each (BM / WM) x (BN / WN).
template <int BM_, int BN_, int WM_, int WN_, int NS_, int WPS_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, WPS = WPS_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, BUF = A_BYTES + B_BYTES;
};
using Big = Tile<256, 256, 2, 4, 2, 2>;     // one workgroup per CU, 128 KB of LDS
using Small = Tile<128, 128, 2, 2, 2, 2>;   // two per CU, 64 KB each
using Thin = Tile<192, 256, 2, 4, 2, 2>;    // gradients of widths that 256 divides badly, 112 KB
using Few = Tile<128, 32, 4, 1, 4, 2>;      // few rows: a stream of the table, 80 KB

// One operand: `rows` of m (n) that exist, `k` of its reduction; beyond them k-inner
// rows repeat the last one (for outputs that are not stored), k beyond come from zeros.
struct Operand {
  const uint16_t* p;
  int64_t plane;  // elements between planes
  int ld;         // elements between rows
  int rows, k;
};
struct Product {
  Operand a, b;
  int nk;          // stages of 64 k
  int pairs;       // pairs of planes
  uint32_t amap, bmap;  // their planes, a bit each
  const uint16_t* zeros;
};

// A k-out tile's 16-byte chunk c of row k lies at c ^ swizzle: a read phase (4 rows of
// 4 chunks) has to hit 16 distinct chunks of the 64 banks.  Rows of 256 or 128 elements
// start at the same bank; of 192, every other one half the banks on.
template <int W>
__device__ __forceinline__ int out_swizzle(int k) {
  return W == 192 ? (k & 2) << 1 : (k & 3) << 2;
}

// The loads of one operand's W x 64 (k-inner) or 64 x W (k-out) tile by NW waves; a
// wave-load is 1 KB, 64 chunks of the tile as it lies in LDS.
template <int W, int NW, bool INNER>
struct Loads {
  static constexpr int CR = INNER ? 8 : W / 8;          // chunks per tile row
  static constexpr int Q = W / 8 / NW;
  static_assert(Q >= 1 && Q * NW * 8 == W, "whole wave-loads");
  static_assert(!INNER || (NW * 8) % 16 == 0, "swizzle phase is the same for every load");
  // a k-out operand's rows of its loads, from the first one's: a whole number of rows, or
  // (192 elements, 8 waves) 21 rows and a third
  static constexpr bool EVEN = INNER || (NW * 64) % CR == 0;
  unsigned off[Q];       // bytes from the stage's base
  int k[EVEN ? 1 : Q];   // the lane's k in the stage: of load 0, or of each
  const uint16_t* base;  // of the next stage to load
  // row: the one that the lane loads of (k-inner, one load), or -1
  __device__ __forceinline__ void init(const Operand& o, int x0, int wave, int lane, int row) {
    if constexpr (INNER) {
      const int r0 = wave * 8 + lane / 8, chunk = ((lane % 8) ^ ((r0 / 2) % 8)) * 8;
      k[0] = chunk;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int r = row >= 0 ? row : min(r0 + q * NW * 8, o.rows - 1 - x0);
        off[q] = 2u * ((unsigned)r * (unsigned)o.ld + (unsigned)chunk);
      }
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int at = (wave + NW * q) * 64 + lane, r = at / CR;
        const int col = min(x0 + ((at % CR) ^ out_swizzle<W>(r)) * 8, o.rows - 8);
        off[q] = 2u * ((unsigned)r * (unsigned)o.ld + (unsigned)col);
        if (q == 0 || !EVEN) k[EVEN ? 0 : q] = r;
      }
    }
  }
  __device__ __forceinline__ void seek(const Operand& o, int x0, int plane, int k0) {
    base = o.p + plane * o.plane + (INNER ? (int64_t)x0 * o.ld + k0 : (int64_t)k0 * o.ld);
  }
  __device__ __forceinline__ void step(const Operand& o) { base += INNER ? BK : (int64_t)BK * o.ld; }
  // load q of the stage into `lds` (the operand's part of a stage)
  __device__ __forceinline__ void load(int q, int wave, unsigned char* lds) const {
    dma16s(base, off[q], lds + (wave + NW * q) * 1024);
  }
  // of a stage of which only `left` k exist: zeros behind them
  __device__ __forceinline__ void load_part(int left, const uint16_t* zeros, int q, int wave,
                                            unsigned char* lds) const {
    const int kq = INNER ? k[0] : EVEN ? k[0] + q * (NW * 64 / CR) : k[EVEN ? 0 : q];
    const char* from = reinterpret_cast<const char*>(base) + off[q];
    dma16(kq < left ? from : reinterpret_cast<const char*>(zeros), lds + (wave + NW * q) * 1024);
  }
};

// The MFMA fragment of k step ks of tile rows (columns) col .. col + 31: lane l has
// m (n) = col + l % 32, k = 16 ks + 8 (l / 32) .. + 7.
template <int W, bool INNER>
__device__ __forceinline__ u32x4_t fragment(const unsigned char* t, int ks, int col, int lane) {
  if constexpr (INNER) {
    const int row = col + (lane & 31), kc = ks * 2 + (lane >> 5);
    return *reinterpret_cast<const u32x4_t*>(t + (row * 8 + (kc ^ ((row / 2) % 8))) * 16);
  } else {
    const int li = lane & 15, lg = lane >> 4;
    u32x2_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = ks * 16 + 8 * (lg >> 1) + 4 * h + (li >> 2);
      const int c = col + 16 * (lg & 1) + 4 * (li & 3);
      const unsigned char* p = t + r * (W * 2) + ((c >> 3) ^ out_swizzle<W>(r)) * 16 + (c & 7) * 2;
      v[h] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_p)(p)));
    }
    return u32x4_t{v[0].x, v[0].y, v[1].x, v[1].y};
  }
}

template <bool F16>
__device__ __forceinline__ f32x16_t mfma(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
}

// Stages s_lo .. s_hi - 1 (of pairs * nk) of the tile at (m0, n0) into acc.
template <class TL, bool AIN, bool BIN, bool F16>
__device__ __forceinline__ void product_tile(const Product& p, unsigned char* lds, int m0, int n0,
                                             int s_lo, int s_hi, f32x16_t (&acc)[TL::TM][TL::TN],
                                             int row_b = -1) {
  constexpr int TM = TL::TM, TN = TL::TN, NW = TL::NW, NS = TL::NS, KS = BK / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  using LA = Loads<TL::BM, NW, AIN>;
  using LB = Loads<TL::BN, NW, BIN>;
  constexpr int LDPS = LA::Q + LB::Q;
  static_assert((NS - 1) * LDPS <= 63, "vmcnt counts");
  LA la;
  LB lb;
  la.init(p.a, m0, wave, lane, -1);
  lb.init(p.b, n0, wave, lane, row_b);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // the next stage to load: pair of planes and stage within it
  int dp = s_lo / max(p.nk, 1), dk = s_lo - dp * p.nk;
  auto seek = [&] {
    la.seek(p.a, m0, (p.amap >> dp) & 1, dk * BK);
    lb.seek(p.b, n0, (p.bmap >> dp) & 1, dk * BK);
  };
  auto next = [&] {
    la.step(p.a);
    lb.step(p.b);
    if (++dk == p.nk) {
      dk = 0;
      ++dp;
      seek();
    }
  };
  const bool partial = min(p.a.k, p.b.k) < p.nk * BK;
  auto load = [&](int slot, int from, int to) {
    unsigned char* st = lds + slot * TL::BUF;
    if (!partial || dk + 1 < p.nk) {
#pragma unroll
      for (int q = 0; q < LDPS; ++q) {
        if (q < from || q >= to) continue;
        if (q < LA::Q)
          la.load(q, wave, st);
        else
          lb.load(q - LA::Q, wave, st + TL::A_BYTES);
      }
    } else {
#pragma unroll
      for (int q = 0; q < LDPS; ++q) {
        if (q < from || q >= to) continue;
        if (q < LA::Q)
          la.load_part(p.a.k - dk * BK, p.zeros, q, wave, st);
        else
          lb.load_part(p.b.k - dk * BK, p.zeros, q - LA::Q, wave, st + TL::A_BYTES);
      }
    }
  };
  seek();
  const int n = s_hi - s_lo;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < n) {
      load(s, 0, LDPS);
      next();
    }
  u32x4_t af[2][TM], bf[2][TN];
  auto frags = [&](const unsigned char* st, int set, int ks) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      bf[set][j] = fragment<TL::BN, BIN>(st + TL::A_BYTES, ks, (wn * TN + j) * 32, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i) af[set][i] = fragment<TL::BM, AIN>(st, ks, (wm * TM + i) * 32, lane);
  };
  constexpr int READS = TM * (AIN ? 1 : 2) + TN * (BIN ? 1 : 2);
  int slot = 0;
  for (int kt = 0; kt < n; ++kt) {
    // stage kt has landed (at most NS - 2 later ones in flight) and the stage read at
    // kt - 1 is free: it receives stage kt + NS - 1
    const int ahead = min(NS - 2, n - 1 - kt);
    if (NS >= 4 && ahead >= 2) stage_barrier<2 * LDPS>();
    else if (NS >= 3 && ahead >= 1) stage_barrier<LDPS>();
    else stage_barrier<0>();
    const unsigned char* st = lds + slot * TL::BUF;
    const bool more = kt + NS - 1 < n;
    const int free = slot == 0 ? NS - 1 : slot - 1;
    if (more) {
      load(free, 0, LDPS);
      next();
    }
    frags(st, 0, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) frags(st, (ks + 1) & 1, ks + 1);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = mfma<F16>(af[ks & 1][i], bf[ks & 1][j], acc[i][j]);
      if (ks + 1 < KS) {
        if (ks == 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int q = 0; q < TM * TN; ++q) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          const int nr = READS * (q + 1) / (TM * TN) - READS * q / (TM * TN);
          if (nr == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          else if (nr == 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          else if (nr == 3) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
          else if (nr >= 4) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        }
      }
    }
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  stage_barrier<0>();  // every wave is done reading before the next tile's loads
}

// How a product's tiles are worked off: `whole` of them (whole rounds of the CUs) in one
// piece, each of the others, the last round's, split along the sum so that they fill
// the CUs too.
struct Split {
  int whole, tail, splits;
  int cost;  // of all tiles, in stages of a tile
};
// Costs in stages: a tile's start and end, a split's way through scratch, and the
// second launch's addition per split.
constexpr int TILE_COST = 3, SPLIT_COST = 6, MIN_STAGES = 4;
__host__ __device__ inline Split split_of(int tiles, int stages, int slots, int scratch_tiles) {
  Split p{tiles / slots * slots, 0, 1, tiles / slots * (stages + TILE_COST)};
  p.tail = tiles - p.whole;
  if (p.tail == 0) return p;
  int least = stages + TILE_COST;
  for (int rounds = 1; rounds <= 2; ++rounds) {
    int n = rounds * slots / p.tail;
    if (n > stages / MIN_STAGES) n = stages / MIN_STAGES;
    if (n * p.tail > scratch_tiles) n = scratch_tiles / p.tail;
    if (n < 2) continue;
    const int need = (n * p.tail + slots - 1) / slots;
    const int cost = need * ((stages + n - 1) / n + TILE_COST) + SPLIT_COST + n / 8;
    if (cost < least) least = cost, p.splits = n;
  }
  p.cost += least;
  return p;
}

// Tile `t` of mt x nt tiles, in groups of GN n-tiles by all m-tiles.
__device__ __forceinline__ void tile_at(int t, int mt, int nt, int& m, int& n) {
  const int g = t / (GN * mt), left = t - g * GN * mt, width = min(GN, nt - g * GN);
  m = left / width;
  n = g * GN + left - m * width;
}
// This workgroup's items of `items`: first, first + step, ... below end.
struct Items {
  int first, step, end;
  // behind: another list's items per XCD that start at the first workgroups
  __device__ __forceinline__ explicit Items(int items, int behind = 0) {
    const int xcd = blockIdx.x % 8, per = (items + 7) / 8;
    step = gridDim.x / 8;
    int at = blockIdx.x / 8;
    if (behind != 0) at = (at + step - behind % step) % step;
    first = xcd * per + at;
    end = min((xcd + 1) * per, items);
  }
};

// A wave's block of 32 n by M = 32 TM m, from the accumulators' layout to whole rows:
// through LDS of the wave's own (16-byte chunks swizzled by the row), then 16 bytes a
// lane with M / 8 (of 16 bits) or M / 4 (of 32) lanes to a row.  Stored as they lie in
// the accumulators, a store instruction covers 32 bytes of 32 rows: at D 544 and 32768
// entries the logits' tiles took 34 us with such stores.
template <int TM, int BITS>
struct Rows {
  static constexpr int CR = TM * (BITS == 16 ? 4 : 8);  // chunks per row
  static constexpr int BYTES = 32 * CR * 16;
  unsigned char* st;
  int lane;
  __device__ __forceinline__ void put(int chunk, u32x4_t v) const {
    const int n = lane & 31;
    *reinterpret_cast<u32x4_t*>(st + (n * CR + (chunk ^ (n % CR))) * 16) = v;
  }
  // f(row, chunk, 16 bytes) for all of the block
  template <class F>
  __device__ __forceinline__ void get(F f) const {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int it = 0; it < CR / 2; ++it) {
      const int row = it * (64 / CR) + lane / CR, c = lane % CR;
      f(row, c, *reinterpret_cast<const u32x4_t*>(st + (row * CR + (c ^ (row % CR))) * 16));
    }
    // (read before the next block is put)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  // The MFMA tile i's values as fp16: quads q and q + 1 of the two half-waves exchanged,
  // 8 consecutive m a lane
  __device__ __forceinline__ void put16(int i, const f32x16_t& c) const {
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f16x2_t v = {(_Float16)c[(q + k) * 4 + 2 * h], (_Float16)c[(q + k) * 4 + 2 * h + 1]};
          w[k][h] = __builtin_bit_cast(uint32_t, v);
        }
      const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      put(i * 4 + q + (lane >> 5), u32x4_t{x[0], y[0], x[1], y[1]});
    }
  }
  __device__ __forceinline__ void put32(int i, const f32x16_t& c) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4_t v = {c[q * 4], c[q * 4 + 1], c[q * 4 + 2], c[q * 4 + 3]};
      put(i * 8 + q * 2 + (lane >> 5), __builtin_bit_cast(u32x4_t, v));
    }
  }
};

// ---- logits ----

// What bounds the epilogue is its transcendentals, one per logit and three with a
// softcap, at a quarter of the other instructions' rate: about 4 us of a 256 x 256 tile
// without and 8 with it, next to 1.5 us per stage of the sum.  Under a softcap the
// entries that do not count are put at a tanh far below any other, after it, where the
// few blocks that have some do it: a comparison of every logit took 465 us of 16384 x
// 50257 at D 64, 433 so.
// (What the kernels take, and no more: every argument is a scalar register that the sum's
// loop has to keep, and some forty more of them had it reading them back from vector
// registers: 2720 us of 16384 x 50257 logits at D 2048 became 2940.)
struct LogitsArgs {
  const XentScalars* scalars;
  int64_t r0, piece_rows;  // the piece; arrays of rows start at its first row
  int V, Vp;
  float k2, cap2;          // 2 log2 e / softcap, softcap log2 e
  const int32_t *target, *x_exp, *w_exp;
  float* at_target;
  const int32_t* low;      // L that the table's planes were taken down to, or null
  float2* stat;
  int32_t* stat_exp;
  int64_t stat_ld;
  void* summands;
};
// The rows as a forward of few gets them (GATHER).
struct GatherArgs {
  const int32_t* targets;
  const float* row_weights;
  int rows;
  XentScalars* scalars;
  int32_t *map, *target;
  float *loss, *lse;
};
struct GradArgs {
  const XentScalars* scalars;
  int64_t r0, piece_rows;
  int V, D;
  float* partial;
  int slots, scratch_tiles;
};
template <class A>
__device__ __forceinline__ int rows_of(const A& a) {
  const int64_t left = a.scalars->rows - a.r0;
  return left <= 0 ? 0 : (int)(left < a.piece_rows ? left : a.piece_rows);
}

// What the packing's launch does for more rows (the plan, in order; zeros for the rows
// that take no part), by every workgroup for itself and by the first for the join.
struct Gathered {
  int at[XENT_GATHER], target[XENT_GATHER], rows;
};
__device__ __forceinline__ void gather_rows(const GatherArgs& g, int V, Gathered& lds) {
  if (threadIdx.x < 64) {
    const int n = threadIdx.x;
    int t = -1;
    float w = 0.0f;
    const bool in = n < g.rows && mxm_xent_takes_part(g.targets, g.row_weights, V, n, t, w);
    const unsigned long long m = __ballot(in);
    const int to = __popcll(m & ((1ull << n) - 1));
    if (in) lds.at[to] = n, lds.target[to] = t;
    if (n == 0) lds.rows = __popcll(m);
    if (blockIdx.x == 0) {
      double sum = in ? (double)w : 0.0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      if (n == 0) g.scalars->rows = __popcll(m), g.scalars->weight_sum = sum;
      if (in) {
        g.map[to] = n;
        g.target[to] = t;
      } else if (n < g.rows) {
        if (g.loss) g.loss[n] = 0.0f;
        if (g.lse) g.lse[n] = 0.0f;
      }
    }
  }
  __syncthreads();
}

// (four stages of 20 KB and the exponents under fp32: one workgroup per CU)
template <class TL, bool STORE, bool F16, bool CAP, bool GATHER = false>
__global__ __launch_bounds__(TL::NT, F16 && TL::NS == 4 ? 1 : TL::WPS) void xent_logits_kernel(LogitsArgs a, Product p, GatherArgs g) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::NS * TL::BUF];
  __shared__ __attribute__((aligned(16))) int w_exp[F16 ? TL::BM : 4];
  constexpr int TM = TL::TM, TN = TL::TN;
  int rows, row_b = -1, own_target = -1;
  if constexpr (GATHER) {
    static_assert(TN == 1 && TL::WN == 1 && TL::BN / 8 == TL::NW, "a row's loads by one lane each");
    Gathered& own = *reinterpret_cast<Gathered*>(lds);
    gather_rows(g, a.V, own);
    rows = __builtin_amdgcn_readfirstlane(own.rows);
    row_b = own.at[max(min((int)threadIdx.x / 8, rows - 1), 0)];
    if ((int)(threadIdx.x & 31) < rows) own_target = own.target[threadIdx.x & 31];
    __syncthreads();
  } else {
    rows = rows_of(a);
  }
  p.b.rows = rows;
  const int mt = (a.V + TL::BM - 1) / TL::BM, nt = (rows + TL::BN - 1) / TL::BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  const float k2 = a.k2, cap2 = a.cap2;  // (CAP)
  const Items items(mt * nt);
  for (int item = items.first; item < items.end; item += items.step) {
    int tm, tn;
    tile_at(item, mt, nt, tm, tn);
    const int m0 = tm * TL::BM, n0 = tn * TL::BN;
    int targets[TN], x_exps[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + (wn * TN + j) * 32 + (lane & 31);
      targets[j] = n < rows ? (GATHER ? own_target : a.target[n]) : -1;
      if constexpr (F16) x_exps[j] = n < rows ? a.x_exp[n] : 0;
    }
    // (the sum's barriers stand between this and the epilogue)
    if constexpr (F16)
      for (int i = threadIdx.x; i < TL::BM; i += TL::NT) {
        const int e = a.w_exp[m0 + i];
        w_exp[i] = a.low ? max(e, *a.low) : e;
      }
    f32x16_t acc[TM][TN];
    product_tile<TL, true, true, F16>(p, lds, m0, n0, 0, p.nk * p.pairs, acc, row_b);
    const int mw = m0 + wm * TM * 32;  // the wave's block of the vocabulary
    const int first = mw + (lane >> 5) * 4;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (mw >= a.V && !STORE) continue;
      const int nw = n0 + (wn * TN + j) * 32, n = nw + (lane & 31);
      const int target = targets[j];
      if constexpr (F16) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const i32x4_t we = *reinterpret_cast<const i32x4_t*>(w_exp + first - m0 + i * 32 + q * 8);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][j][q * 4 + k] = ldexpf(acc[i][j][q * 4 + k], we[k] + x_exps[j]);
          }
      }
      // entries behind the vocabulary, and the target (whose logit is kept apart), get one
      // with an exponential of 0.  Under a softcap that is a tanh so small that no ref brings
      // it back and no slope times 0 leaves 0 (a logit of minus infinity is its lowest
      // there: at the least cap, 1/64, this one is 2^-225), or where the summands are kept
      // too, with their slope, the exp(2 z / cap) of about such a tanh: below zero.
      constexpr bool SLOPE = CAP && STORE;
      constexpr float none = SLOPE ? -0.9998f : CAP ? -1.0e4f : -__builtin_inff();
      const bool here = __ballot(target >= mw && target < mw + TM * 32) != 0;
      const int at = target - first;
      if (here) {
        // (as branches with a softcap, and as selections without, the comparisons take some
        // hundred scalar registers too many)
        if constexpr (CAP) {
          float z = 0.0f;
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = at == i * 32 + (r >> 2) * 8 + (r & 3) ? acc[i][j][r] : z;
          // (of the two half-waves the one that holds it)
          if (at >= 0 && at < TM * 32 && (at & 4) == 0) a.at_target[n] = z;
        } else {
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (at == i * 32 + (r >> 2) * 8 + (r & 3)) {
                a.at_target[n] = acc[i][j][r];
                acc[i][j][r] = none;
              }
        }
      }
      if constexpr (CAP) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            acc[i][j][r] = SLOPE ? __builtin_amdgcn_exp2f(acc[i][j][r] * k2) : mxm_xent_capped(acc[i][j][r], k2);
        if (here) {
          int again = at;
          asm volatile("" : "+v"(again));  // (else the comparisons above are kept, in 128 scalar registers)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              acc[i][j][r] = again == i * 32 + (r >> 2) * 8 + (r & 3) ? none : acc[i][j][r];
        }
      }
      if (mw + TM * 32 > a.V) {
        int end = a.V - first;
        asm volatile("" : "+v"(end));  // (nor move before the branch)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            acc[i][j][r] = i * 32 + (r >> 2) * 8 + (r & 3) >= end ? none : acc[i][j][r];
      }
      float top = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, mxm_xor_lane_f(top, 32));
      const bool any = SLOPE ? top >= 0.0f : CAP ? top >= -2.0f : top > -__builtin_inff();
      // 2^(l log2 e - ref) lies in (0, 2^15], or 2^17 where a quarter of the slope comes to
      // it: fp16 keeps 12 bits of summands down to 2^-29 of the block's largest and 2^-39 of
      // it at all
      constexpr float UP = SLOPE ? 17.0f : 15.0f;
      const float t = SLOPE ? fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(1.0f + top), cap2)
                      : CAP ? cap2 * top
                            : top * LOG2E;
      float ref = any ? ceilf(t) - UP : 0.0f, sub = ref;
      if constexpr (SLOPE) {
        // l log2 e - ref = (cap2 - ref) - 2 cap2 r: ref is what the rounded difference makes it
        sub = cap2 - ref;
        ref = cap2 - sub;
      }
      if constexpr (!CAP) {
        // From 2^22 on ref and the exact product may lie further apart than a summand's
        // range allows (a block of masked entries, say): such logits are taken less their
        // largest first, whose summand is 2^15.  Their ref is finite, and above that of no
        // entry at all.
        const bool far = any && !(__builtin_fabsf(t) < 4194304.0f);
        if (__ballot(far) != 0) {
          const float by = far ? top : 0.0f;
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] -= by;
          if (far) {
            sub = -UP;
            ref = fminf(fmaxf(t - UP, 0.5f * XENT_NO_REF), -XENT_NO_REF);
          }
        }
      }
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = acc[i][j][r];
          if constexpr (SLOPE) {
            const float w = __builtin_amdgcn_rcpf(1.0f + v), e = __builtin_amdgcn_exp2f(fmaf(-2.0f * cap2, w, sub));
            s[r & 1] += e;
            acc[i][j][r] = e * mxm_xent_cap_slope(v, w);
            // (else the product moves to where the summands are stored, and its factors of
            // all logits till there spill 300 registers)
            asm("" : "+v"(acc[i][j][r]));
          } else {
            const float e = __builtin_amdgcn_exp2f(fmaf(v, CAP ? cap2 : LOG2E, -sub));
            s[r & 1] += e;
            acc[i][j][r] = e;
          }
        }
      float sum = s[0] + s[1];
      sum += mxm_xor_lane_f(sum, 32);
      const int64_t at_stat = (int64_t)(mw / (TM * 32)) * a.stat_ld + n;
      if (n < rows && mw < a.V && lane < 32) a.stat[at_stat] = make_float2(sum, any ? ref : XENT_NO_REF);
      if constexpr (F16 && STORE) {
        // (2^(w - 1): none overflows)
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const i32x4_t we = *reinterpret_cast<const i32x4_t*>(w_exp + first - m0 + i * 32 + q * 8);
#pragma unroll
            for (int k = 0; k < 4; ++k) big = fmaxf(big, ldexpf(acc[i][j][q * 4 + k], we[k] - 1));
          }
        big = fmaxf(big, mxm_xor_lane_f(big, 32));
        if (n < rows && mw < a.V && lane < 32)
          a.stat_exp[at_stat] = big > 0.0f ? __builtin_amdgcn_frexp_expf(big) + 1 : XENT_NO_EXP;
      }
      if constexpr (STORE) {
        constexpr int BITS = F16 ? 32 : 16, PER = 128 / BITS;
        using R = Rows<TM, BITS>;
        static_assert(TL::NW * R::BYTES <= TL::NS * TL::BUF, "staging fits the ring");
        const R block{lds + wave * R::BYTES, lane};
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if constexpr (F16)
            block.put32(i, acc[i][j]);
          else
            block.put16(i, acc[i][j]);
        }
        block.get([&](int row, int c, u32x4_t v) {
          const int m = mw + c * PER;
          if (nw + row < rows && m < a.Vp)
            *reinterpret_cast<u32x4_t*>(static_cast<char*>(a.summands) +
                                        ((int64_t)(nw + row) * a.Vp + m) * (BITS / 8)) = v;
        });
      }
    }
    if constexpr (STORE || F16) lds_barrier();  // before the next tile's loads
  }
}

// ---- dx and dw ----

// Where C goes: rows n of M elements.
struct Out {
  void* out;
  const float* add;      // earlier sums of the same elements, or null
  const int32_t* map;    // the row that n is, or null: n
  const int32_t* e_row;  // fp32: the exponents of n's sums: dx's E,
  const int32_t* w_exp;  // or dw's C - max(w, L)
  const int32_t* low;
  const XentScalars* scalars;
  int M;
  bool bf16, vec;        // vec (bf16): rows of whole aligned 16 bytes
};

__device__ __forceinline__ int exp_of(const Out& o, int n) {
  return o.e_row ? o.e_row[n] : o.scalars->dw_exp - max(o.w_exp[n], *o.low);
}

// Four elements at place `at`, of which `left` are the row's, at the elements' alignment
// (a step of 2000 rows of D 1001 and 30000 entries 535 us with element stores, 490 so).
__device__ __forceinline__ void put4(const Out& o, int64_t at, int left, f32x4_t c) {
  typedef float at4_t __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned int at2_t __attribute__((ext_vector_type(2), aligned(2)));
  if (left >= 4) {
    if (o.bf16)
      *reinterpret_cast<at2_t*>(static_cast<uint16_t*>(o.out) + at) =
          u32x2_t{mxm_pack_bf2_fast(c[0], c[1]), mxm_pack_bf2_fast(c[2], c[3])};
    else
      *reinterpret_cast<at4_t*>(static_cast<float*>(o.out) + at) = c;
    return;
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (k < left) {
      if (o.bf16)
        static_cast<uint16_t*>(o.out)[at + k] = mxm_f2bf_fast(c[k]);
      else
        static_cast<float*>(o.out)[at + k] = c[k];
    }
}

// Row n's elements m .. m + 3 of an MFMA tile, as each quad of registers holds them.
template <bool F16>
__device__ __forceinline__ void put_tile(const Out& o, int m_first, int n, bool in, int lane, f32x16_t c) {
  if constexpr (F16) {
    const int e = !in ? 0 : exp_of(o, n);
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = ldexpf(c[r], e);
  }
  const int64_t row = in ? (int64_t)(o.map ? o.map[n] : n) * o.M : 0;
  if (o.add && in) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = m_first + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
      if (m < o.M) c[r] += o.add[row + m];
    }
  }
  if (o.vec) {
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[k][h] = mxm_pack_bf2_fast(c[(q + k) * 4 + 2 * h], c[(q + k) * 4 + 2 * h + 1]);
      const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      const u32x4_t v = {x[0], y[0], x[1], y[1]};
      const int m = m_first + (q + (lane >> 5)) * 8;
      if (in && m < o.M) *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(o.out) + row + m) = v;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = m_first + q * 8 + (lane >> 5) * 4;
      if (!in) continue;
      put4(o, row + m, o.M - m, f32x4_t{c[q * 4], c[q * 4 + 1], c[q * 4 + 2], c[q * 4 + 3]});
    }
  }
}

// Elements m .. m + 3 of row n.
template <bool F16>
__device__ __forceinline__ void put_quad(const Out& o, int m, int n, f32x4_t c) {
  if (m >= o.M) return;
  if constexpr (F16) {
    const int e = exp_of(o, n);
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = ldexpf(c[k], e);
  }
  const int64_t at = (int64_t)(o.map ? o.map[n] : n) * o.M + m;
  if (o.add) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (m + k < o.M) c[k] += o.add[at + k];
  }
  put4(o, at, o.M - m, c);
}

// What a launch needs of the device's count of rows: n of dx, k of dw.
template <bool DW>
__device__ __forceinline__ void fit(const GradArgs& a, Product& p) {
  const int rows = rows_of(a);
  if constexpr (DW) {
    p.a.k = p.b.k = rows;
    p.nk = (rows + BK - 1) / BK;
  } else {
    p.b.rows = rows;
  }
}

// The tiles of dx or dw; returns how many of its last round's items an XCD has.
template <class TL, bool DW, bool F16>
__device__ __forceinline__ int grad_tiles(const GradArgs& a, Product p, const Out& o, unsigned char* lds,
                                          float* partial, int behind) {
  constexpr int TM = TL::TM, TN = TL::TN;
  fit<DW>(a, p);
  const int N = DW ? a.V : p.b.rows;
  const int mt = (a.D + TL::BM - 1) / TL::BM, nt = (N + TL::BN - 1) / TL::BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  const int stages = p.nk * p.pairs;
  const Split plan = split_of(mt * nt, stages, a.slots, a.scratch_tiles);
  auto work = [&](int tile, int split, int splits) {
    int tm, tn;
    tile_at(tile, mt, nt, tm, tn);
    f32x16_t acc[TM][TN];
    product_tile<TL, false, !DW, F16>(p, lds, tm * TL::BM, tn * TL::BN, (int)((int64_t)split * stages / splits),
                                 (int)((int64_t)(split + 1) * stages / splits), acc);
    if (splits > 1) {
      f32x4_t* to = reinterpret_cast<f32x4_t*>(partial) +
                    (int64_t)(split * plan.tail + tile - plan.whole) * (TL::BM * TL::BN / 4) +
                    wave * (TM * TN * 4 * 64) + lane;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4_t v = {acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2],
                               acc[i][j][q * 4 + 3]};
            to[((i * TN + j) * 4 + q) * 64] = v;
          }
      return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = tn * TL::BN + (wn * TN + j) * 32 + (lane & 31);
        put_tile<F16>(o, tm * TL::BM + (wm * TM + i) * 32, n, n < N, lane, acc[i][j]);
      }
  };
  // (one loop over both lists: the tile's code once)
  const Items whole(plan.whole, behind), tail(plan.tail * plan.splits, behind);
  int item = whole.first;
  bool rest = item >= whole.end;
  if (rest) item = tail.first;
  while (!rest || item < tail.end) {
    const int split = rest ? item / plan.tail : 0;
    work(rest ? plan.whole + item - split * plan.tail : item, split, rest ? plan.splits : 1);
    item += whole.step;
    if (!rest && item >= whole.end) {
      rest = true;
      item = tail.first;
    }
  }
  return (plan.tail * plan.splits + 7) / 8;
}

template <class TL, bool DW, bool F16>
__global__ __launch_bounds__(TL::NT, TL::WPS) void xent_grad_kernel(GradArgs a, Product p, Out o) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::NS * TL::BUF];
  (void)grad_tiles<TL, DW, F16>(a, p, o, lds, a.partial, 0);
}
// Both, of small tiles: dw's items start at the workgroups behind dx's last ones.  (A step
// of 512 rows of D 512 and 8192 entries 67.6 us with two launches and their joins', 56.8
// so; larger tiles' launches are long enough: 16384 rows of D 2048 and 50257 entries 8.97
// ms with two, 9.03 with one.)
template <class TL, bool F16>
__global__ __launch_bounds__(TL::NT, TL::WPS) void xent_grads_kernel(GradArgs a, Product px, Out ox, Product pw,
                                                                     Out ow) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::NS * TL::BUF];
  const int behind = grad_tiles<TL, false, F16>(a, px, ox, lds, a.partial, 0);
  (void)grad_tiles<TL, true, F16>(a, pw, ow, lds, a.partial + (int64_t)a.scratch_tiles * (TL::BM * TL::BN), behind);
}

// The splits of the last round's tiles added in order; a workgroup per quad of registers
// of all waves.
template <class TL, bool DW, bool F16>
__device__ __forceinline__ int grad_join(const GradArgs& a, Product p, const Out& o, const float* partial,
                                         int item) {
  constexpr int TM = TL::TM, TN = TL::TN, AHEAD = 16;
  fit<DW>(a, p);
  const int N = DW ? a.V : p.b.rows;
  const int mt = (a.D + TL::BM - 1) / TL::BM, nt = (N + TL::BN - 1) / TL::BN;
  const Split plan = split_of(mt * nt, p.nk * p.pairs, a.slots, a.scratch_tiles);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  if (plan.splits == 1) return item;
  const int64_t step = (int64_t)plan.tail * (TL::BM * TL::BN / 4);
  // a quad of each lane's registers at a time
  for (; item < plan.tail * (TM * TN * 4); item += gridDim.x) {
    const int tile = item / (TM * TN * 4), ijq = item % (TM * TN * 4);
    const int i = ijq / (TN * 4), j = ijq / 4 % TN, q = ijq % 4;
    int tm, tn;
    tile_at(plan.whole + tile, mt, nt, tm, tn);
    f32x4_t c = {0.0f, 0.0f, 0.0f, 0.0f};
    const f32x4_t* from = reinterpret_cast<const f32x4_t*>(partial) + (int64_t)tile * (TL::BM * TL::BN / 4) +
                          wave * (TM * TN * 4 * 64) + ijq * 64 + lane;
    for (int s = 0; s < plan.splits; s += AHEAD) {
      f32x4_t v[AHEAD];
#pragma unroll
      for (int h = 0; h < AHEAD; ++h)
        v[h] = s + h < plan.splits ? from[(s + h) * step] : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < AHEAD; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] += v[h][k];
    }
    const int n = tn * TL::BN + (wn * TN + j) * 32 + (lane & 31);
    if (n < N) put_quad<F16>(o, tm * TL::BM + (wm * TM + i) * 32 + q * 8 + (lane >> 5) * 4, n, c);
  }
  return item - plan.tail * (TM * TN * 4);
}
template <class TL, bool DW, bool F16>
__global__ __launch_bounds__(TL::NT) void xent_grad_join_kernel(GradArgs a, Product p, Out o) {
  (void)grad_join<TL, DW, F16>(a, p, o, a.partial, blockIdx.x);
}
template <class TL, bool F16>
__global__ __launch_bounds__(TL::NT) void xent_grads_join_kernel(GradArgs a, Product px, Out ox, Product pw, Out ow) {
  const int item = grad_join<TL, false, F16>(a, px, ox, a.partial, blockIdx.x);
  (void)grad_join<TL, true, F16>(a, pw, ow, a.partial + (int64_t)a.scratch_tiles * (TL::BM * TL::BN), item);
}

// ---- launches ----

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t tiles_of(int64_t m, int64_t n, int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }
unsigned grid_of(int64_t items, int64_t slots) {
  return (unsigned)((std::min(items, slots) + 7) / 8 * 8);
}
// pairs of planes: (hi, lo), (lo, hi), (hi, hi)
void set_planes(const XentArgs& a, Product& p) {
  p.pairs = a.planes == 1 ? 1 : 3;
  p.amap = a.planes == 1 ? 0 : 0b010;
  p.bmap = a.planes == 1 ? 0 : 0b001;
  p.zeros = a.zeros;
}
// The table, its rows' k or (k-out) its columns.
Operand table(const XentArgs& a, bool inner) {
  Operand o{};
  o.p = a.w_direct ? static_cast<const uint16_t*>(a.weight) : a.w_pack;
  o.ld = a.w_direct ? a.D : a.Dp;
  o.plane = (int64_t)a.V * o.ld;
  o.rows = inner ? a.V : o.ld;
  o.k = inner ? o.ld : a.V;
  return o;
}
Operand hidden(const XentArgs& a, bool inner, int64_t r0) {
  Operand o{};
  o.p = a.x_pack + r0 * a.Dp;
  o.ld = a.Dp;
  o.plane = a.x_rows * a.Dp;
  o.rows = a.Dp;  // (k-out; k-inner: the rows that take part, on the device)
  o.k = inner ? a.Dp : 0;
  return o;
}
Operand grad(const XentArgs& a) {
  Operand o{};
  o.p = a.dz;
  o.ld = a.Vp;
  o.plane = a.piece_rows * a.Vp;
  o.rows = a.Vp;
  o.k = a.Vp;
  return o;
}

enum Shape { FEW, SMALL, BIG };
Shape logits_shape(int64_t rows, int V, int n_cu) {
  if (rows <= 32 || tiles_of(V, rows, Few::BM, Few::BN) <= 2 * n_cu) return FEW;
  return rows <= 128 || tiles_of(V, rows, Big::BM, Big::BN) <= n_cu / 2 ? SMALL : BIG;
}

template <class TL>
void launch_logits(const XentArgs& a, const Product& p, int64_t r0, int64_t rows, const int32_t* low, int per_cu,
                   bool gather, hipStream_t s) {
  const unsigned grid = grid_of(tiles_of(a.V, rows, TL::BM, TL::BN), (int64_t)a.n_cu * per_cu);
  const LogitsArgs l{a.scalars, r0, a.piece_rows, a.V, a.Vp, 2.0f * LOG2E / a.softcap, a.softcap * LOG2E, a.target + r0,
                     a.x_exp ? a.x_exp + r0 : nullptr, a.w_exp, a.at_target + r0, low, a.stat, a.stat_exp,
                     a.stat_ld, a.summands};
  const GatherArgs g{a.targets, a.row_weights, (int)a.rows, a.scalars, a.map, a.target, a.loss, a.lse};
  const auto launch = [&](auto kernel) { kernel<<<grid, TL::NT, 0, s>>>(l, p, g); };
  const auto typed = [&](auto cap) {
    constexpr bool CAP = decltype(cap)::value;
    if constexpr (TL::BN == XENT_GATHER) {
      if (gather) return launch(xent_logits_kernel<TL, false, false, CAP, true>);
    }
    if (a.planes == 1)
      a.backward ? launch(xent_logits_kernel<TL, true, false, CAP>) : launch(xent_logits_kernel<TL, false, false, CAP>);
    else
      a.backward ? launch(xent_logits_kernel<TL, true, true, CAP>) : launch(xent_logits_kernel<TL, false, true, CAP>);
  };
  if (a.softcap > 0.0f)
    typed(std::true_type{});
  else
    typed(std::false_type{});
}

// One product's launch.
struct Grad {
  Product p;
  Out o;
  int64_t N;
};
enum GradShape { G_SMALL, G_THIN, G_BIG };

// The shape whose tiles take the least time by split_of's count of stages, at a stage's
// time (Small: of two on a CU).  Those, measured: dw of D 1536 and 32768 entries, whole
// rounds in every shape, 4 to 192 stages, takes 1.81-2.35 us a stage in tiles of Big,
// 1.39-1.80 in Thin (0.79 of that on average) and 0.96-1.31 in Small (0.55).  What the rule
// chooses between: a step of 4096 rows and 32768 entries at D 544 with dx in Big 508 us, Thin
// 488, Small 496; 8192 and 32768 at D 1024 1256 / 1464 / 1387; dw of 4096 and 8192 at D 1024
// 194 / 193 / 170; of 300 and 50257 at D 1000 155 / 151 / 136; of 1024 and 32768 at D 192 in
// fp32, where it takes Thin, 229 / 219 / 205, its worst of 16 such sizes.
GradShape grad_shape(const XentArgs& a, const Grad& g, int64_t k) {
  const int stages = (int)((k + BK - 1) / BK) * g.p.pairs;
  const auto time = [&](auto tile, int per_cu, double stage) {
    using TL = decltype(tile);
    const int slots = a.n_cu * per_cu / 8 * 8;
    return stage * split_of((int)tiles_of(a.D, g.N, TL::BM, TL::BN), stages, slots,
                            (int)(mxm_xent_partial_bytes(a.n_cu) / (TL::BM * TL::BN * 4)))
                       .cost;
  };
  const double big = time(Big{}, 1, 1.0), thin = time(Thin{}, 1, 0.79), small = time(Small{}, 2, 0.55);
  return small < big && small < thin ? G_SMALL : thin < big ? G_THIN : G_BIG;
}

// The device counts the rows that take part, so it decides how tiles are split: the
// second launch is there wherever it may.  dx, dw or (small tiles) both, null: not.
template <class TL>
void launch_grads(const XentArgs& a, const Grad* dx, const Grad* dw, int64_t r0, int per_cu, hipStream_t s) {
  const int slots = a.n_cu * per_cu / 8 * 8;
  const bool both = dx && dw;
  const int scratch = (int)(mxm_xent_partial_bytes(a.n_cu) / (TL::BM * TL::BN * 4)) / (both ? 2 : 1);
  int64_t joins = 0;
  if (dx) joins += std::min<int64_t>(tiles_of(a.D, dx->N, TL::BM, TL::BN), slots - 1);
  if (dw) joins += tiles_of(a.D, dw->N, TL::BM, TL::BN) % slots;
  joins = std::min<int64_t>(joins * TL::TM * TL::TN * 4, (int64_t)a.n_cu * 8);
  const GradArgs g{a.scalars, r0, a.piece_rows, a.V, a.D, a.partial, slots, scratch};
  const auto typed = [&](auto f16) {
    constexpr bool F16 = decltype(f16)::value;
    if constexpr (std::is_same_v<TL, Small>) {
      if (both) {
        xent_grads_kernel<TL, F16><<<slots, TL::NT, 0, s>>>(g, dx->p, dx->o, dw->p, dw->o);
        if (joins > 0)
          xent_grads_join_kernel<TL, F16><<<(unsigned)joins, TL::NT, 0, s>>>(g, dx->p, dx->o, dw->p, dw->o);
        return;
      }
    }
    if (dx) {
      xent_grad_kernel<TL, false, F16><<<slots, TL::NT, 0, s>>>(g, dx->p, dx->o);
      if (joins > 0) xent_grad_join_kernel<TL, false, F16><<<(unsigned)joins, TL::NT, 0, s>>>(g, dx->p, dx->o);
    } else {
      xent_grad_kernel<TL, true, F16><<<slots, TL::NT, 0, s>>>(g, dw->p, dw->o);
      if (joins > 0) xent_grad_join_kernel<TL, true, F16><<<(unsigned)joins, TL::NT, 0, s>>>(g, dw->p, dw->o);
    }
  };
  if (a.planes == 1)
    typed(std::false_type{});
  else
    typed(std::true_type{});
}
void launch_grads(const XentArgs& a, GradShape shape, const Grad* dx, const Grad* dw, int64_t r0, hipStream_t s) {
  switch (shape) {
    case G_SMALL: return launch_grads<Small>(a, dx, dw, r0, 2, s);
    case G_THIN: return launch_grads<Thin>(a, dx, dw, r0, 1, s);
    default: return launch_grads<Big>(a, dx, dw, r0, 1, s);
  }
}

}  // namespace

int64_t mxm_xent_partial_bytes(int n_cu) { return (int64_t)n_cu * 2 * 256 * 256 * 4; }

int mxm_xent_block(int64_t rows, int V, int n_cu) {
  const Shape s = logits_shape(rows, V, n_cu);
  return s == FEW ? Few::TM * 32 : s == SMALL ? Small::TM * 32 : Big::TM * 32;
}

int64_t mxm_xent_stats(int64_t rows, int V, int n_cu) {
  // the most of any number of rows: 32-wide blocks for up to 32 of them or a round of
  // tiles for few rows, 64-wide ones for up to 128 or half a round of big tiles, 128-wide
  const auto of = [&](int64_t n, int block) { return n * ((V + block - 1) / block); };
  const auto tiled = [&](int64_t tiles, int bm, int bn) { return tiles / ((V + bm - 1) / bm) * bn; };
  const int64_t few = std::max<int64_t>(32, tiled(2 * n_cu, Few::BM, Few::BN));
  const int64_t small = std::max<int64_t>(128, tiled(n_cu / 2, Big::BM, Big::BN));
  return std::max({of(rows, 128), of(std::min(rows, small), 64), of(std::min(rows, few), 32)});
}

void mxm_launch_xent_logits(const XentArgs& a, int64_t r0, int64_t rows, const int32_t* low, bool gather,
                            hipStream_t s) {
  Product p{};
  set_planes(a, p);
  p.a = table(a, true);
  p.b = hidden(a, true, r0);
  if (gather) {
    p.b.p = static_cast<const uint16_t*>(a.x);
    p.b.ld = p.b.k = a.D;
  }
  p.nk = a.Dp / BK;
  switch (logits_shape(rows, a.V, a.n_cu)) {
    case FEW: return launch_logits<Few>(a, p, r0, rows, low, 2, gather, s);
    case SMALL: return launch_logits<Small>(a, p, r0, rows, low, 2, false, s);
    default: return launch_logits<Big>(a, p, r0, rows, low, 1, false, s);
  }
}

void mxm_launch_xent_grads(const XentArgs& a, int64_t r0, int64_t rows, bool last, const int32_t* low,
                           hipStream_t s) {
  Grad dx{}, dw{};
  const bool want_dx = a.dx && rows > 0;
  GradShape shape_dx = G_BIG, shape_dw = G_BIG;
  if (want_dx) {
    Product& p = dx.p;
    Out& o = dx.o;
    set_planes(a, p);
    p.a = table(a, false);
    p.b = grad(a);
    p.nk = (a.V + BK - 1) / BK;
    o.out = a.dx;
    o.map = a.map + r0;
    o.e_row = a.e_row + r0;
    o.M = a.D;
    o.bf16 = a.dx_bf16;
    o.vec = o.bf16 && aligned(a.dx) && a.D % 8 == 0;
    dx.N = rows;
    shape_dx = grad_shape(a, dx, a.V);
  }
  if (a.dw) {
    Product& p = dw.p;
    Out& o = dw.o;
    set_planes(a, p);
    p.a = hidden(a, false, r0);
    p.b = grad(a);
    float* sums = a.dw32 ? a.dw32 : static_cast<float*>(a.dw);
    o.out = last ? a.dw : sums;
    o.bf16 = last && a.dw_bf16;
    o.add = r0 > 0 ? sums : nullptr;
    o.w_exp = a.w_exp;
    o.low = low;
    o.scalars = a.scalars;
    o.M = a.D;
    o.vec = o.bf16 && aligned(o.out) && a.D % 8 == 0;
    dw.N = a.V;
    shape_dw = grad_shape(a, dw, rows);
  }
  if (want_dx && a.dw && shape_dx == G_SMALL && shape_dw == G_SMALL) {
    launch_grads(a, G_SMALL, &dx, &dw, r0, s);
    return;
  }
  if (want_dx) launch_grads(a, shape_dx, &dx, nullptr, r0, s);
  if (a.dw) launch_grads(a, shape_dw, nullptr, &dw, r0, s);
}
