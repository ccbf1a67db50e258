// The tile arithmetic that the attention kernels share.
//
// A wave owns 32 packed query rows (row p is query p / group of kv head
// p % group's group, so the heads of a group share every key and value) and
// works on the transposed products, S^T = K Q^T and O^T = V^T P^T:
//   - lane l's column of S^T is its query row l % 32, so the softmax runs
//     within a lane (and its partner l ^ 32, which holds the other keys);
//   - the accumulator layout of S^T is the operand layout of P^T up to the
//     order of the keys, and a product may take its terms in any order: the
//     weights go from one MFMA into the next without leaving their lane;
//   - V^T fragments come out of row-major LDS rows by the transposing read.
// Keys and values reach LDS by copies that bypass registers.  Their 16-byte
// pieces are placed by an XOR of the row, which the copies' source addresses
// carry, so that neither read has bank conflicts.
//
// A row's reference is only moved when a score exceeds the one that set it by
// kSlack log2 units, to kBase below that score: the accumulators are rescaled
// in a few tiles instead of in most, and the row's largest weight stands
// between 2^kBase and 2^(kBase + kSlack).  Weights are rounded to the inputs'
// type.  bf16 holds them as well as weights up to 1.  fp16 loses relative
// precision below 2^-14: with kBase 7 a key's weight is off by at most
// 2^-25 / 2^7 = 2^-32 of the row's sum where half a step is less than that.
// (With 0, 500 keys around 2^-27 beside one of weight 1 came out a third off,
// and weights below 2^-25 were lost.)  Its kSlack leaves 2^5 to fp16's end for
// the rounding of scores up to 2^26.
#pragma once

#include <math.h>
#include <stdint.h>

#include "dft_device.h"

namespace dft {
namespace attend {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  typedef bf16x8 x8;
  static constexpr uint32_t kExp = 0x7f80, kOne = 0x3f80;
  static constexpr float kBase = 0, kSlack = 8;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
struct F16 {
  typedef f16x8 x8;
  static constexpr uint32_t kExp = 0x7c00, kOne = 0x3c00;
  static constexpr float kBase = 7, kSlack = 4;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kTile = 64;          // keys per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kWaitDma = 0x0f70;   // s_waitcnt vmcnt(0)

#define DFT_LDS __attribute__((address_space(3)))

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const DFT_LDS void*)p;
}

// global -> LDS, N copies of 16 bytes a lane: copy i from base + from[i] bytes
// to lds + i STEP + 16 * lane.
// Issued from inline assembly, which the backend's wait analysis does not see:
// it would wait for the copy ahead of the next LDS read of any tile.  The
// caller waits for vmcnt before the tile is read.  m0 is reserved to the
// backend: its value is kept.  A copy needs a wait state after a write of m0,
// and five after a vector write of its scalar base.
template <int N, int STEP>
__device__ __forceinline__ void dma16(uint64_t base, const uint32_t* from, uint32_t lds) {
  uint32_t keep;
  static_assert(N == 1 || N == 2 || N == 4 || N == 8);
  if constexpr (N == 8) {
    dma16<4, STEP>(base, from, lds);
    dma16<4, STEP>(base, from + 4, lds + 4 * STEP);
  } else if constexpr (N == 4) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %6\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, %5\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %5\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %5\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %5\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 2) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %4\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, %3\n\t"
        "s_add_u32 m0, m0, %5\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %3\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 1) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, %2\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  }
}
// the same from addresses of each lane's own; ONCE: of data read once, which
// then does not displace what the caches hold
template <int N, int STEP, bool ONCE>
__device__ __forceinline__ void dma16_at(const uint64_t* from, uint32_t lds) {
  uint32_t keep;
  static_assert(N == 1 || N == 2 || N == 4 || N == 8);
  if constexpr (N == 8) {
    dma16_at<4, STEP, ONCE>(from, lds);
    dma16_at<4, STEP, ONCE>(from + 4, lds + 4 * STEP);
  } else if constexpr (N == 4 && ONCE) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off nt\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, off nt\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, off nt\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 4) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, off\n\t"
        "s_add_u32 m0, m0, %6\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, off\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 2 && ONCE) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_add_u32 m0, m0, %4\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off nt\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 2) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_add_u32 m0, m0, %4\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "v"(from[1]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 1 && ONCE) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  } else if constexpr (N == 1) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(from[0]), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(STEP)
        : "memory", "scc");
  }
}
// and of 4 bytes a lane
__device__ __forceinline__ void dma4_at(uint64_t at, uint32_t lds) {
  uint32_t keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off\n\t"
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0"
      : "=&s"(keep)
      : "v"(at), "s"(__builtin_amdgcn_readfirstlane(lds))
      : "memory");
}

__device__ __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform64((int64_t)v); }

// Where row `row`'s 16-byte piece c of a key / value tile lies: piece
// c ^ swizzle.  Keys are read by 16 lanes of consecutive rows at one piece,
// values by 8 lanes of 4 consecutive rows each over 4 pieces; the LDS serves
// 256 bytes a cycle, which is one row of 128 elements.
template <int D>
__device__ __forceinline__ int key_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

// Bits [0, n) of a word, none for n <= 0.
__device__ __forceinline__ uint64_t first_bits(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

// a where the bit is set, b elsewhere, without a comparison (whose results
// would wait in scalar registers, a pair for each)
__device__ __forceinline__ uint32_t select(uint32_t a, uint32_t b, uint32_t bits, int bit) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, bit, 1);
  return (a & m) | (b & ~m);
}

// What of a scale goes where: |scale| log2(e) multiplies the scores, its sign
// goes into the queries (a rounding-free change), and a scale of 0 clears them
// (a masked score of -inf times 0 would not be one).
struct Scale {
  float c;
  uint32_t keep, flip;
};
inline Scale split_scale(float scale) {
  if (scale == 0) return {kLog2e, 0, 0};
  return {fabsf(scale) * kLog2e, ~0u, scale < 0 ? 0x80008000u : 0};
}

// 1.0 for an infinity of that sign or a NaN in the low half, 0 otherwise
template <class T>
__device__ __forceinline__ uint32_t infinite(uint32_t w, int sign) {
  const uint32_t e = w & 0x7fffu;
  return e > T::kExp || (e == T::kExp && (w >> 15 & 1) == (uint32_t)sign) ? T::kOne : 0;
}

// N times four outputs in a row: value(i) to o[at + offset(i)].  `vec`: in whole pieces
template <int N, class Value, class Offset>
__device__ __forceinline__ void store_all(void* o, int64_t at, int dtype, bool vec, Value value, Offset offset) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  if (dtype == DFT_F32) {
    float* to = static_cast<float*>(o) + at;
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; ++i) *reinterpret_cast<f32x4*>(to + offset(i)) = value(i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const f32x4 x = value(i);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[offset(i) + e] = x[e];
      }
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(o) + at;
  const bool bf16 = dtype == DFT_BF16;
  auto narrow = [&](int i) {
    const f32x4 x = value(i);
    const u16x4 b = __builtin_bit_cast(u16x4, __builtin_convertvector(x, bf16x4));
    const u16x4 h = __builtin_bit_cast(u16x4, __builtin_convertvector(x, f16x4));
    return bf16 ? b : h;
  };
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u16x4*>(to + offset(i)) = narrow(i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u16x4 y = narrow(i);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[offset(i) + e] = y[e];
    }
  }
}

template <int I>
struct At {
  constexpr operator int() const { return I; }
};

// The state of a wave's 32 rows over KW keys of each tile.
template <int D, int KW, class T>
struct Rows {
  static constexpr int kRow = 2 * D;  // bytes
  static constexpr int DT = D / 32, QK = D / 16, ST = KW / 32, PK = KW / 16;
  typedef typename T::x8 x8;

  x8 q[QK];
  f32x16 o[DT];  // lane: d = 32 t + acc_row(r, lane / 32) of its row
  float top;     // the reference that the weights are taken against, in log2 units (-inf: none yet)
  float sum;     // of the weights of this lane's keys
  float high;    // of the lane's scores of the tile at hand
  bool noted;    // whether `notes` holds infinities that the accumulators lack
  uint32_t notes;  // LDS address of kNotes bytes of the wave's own
  static constexpr int kNotes = 256 * DT;

  __device__ __forceinline__ void clear() {
    noted = false;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    top = -INFINITY;
    sum = 0;
  }

  // row: the lane's query row of this head
  __device__ __forceinline__ void load_q(const uint16_t* row, Scale sc) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int k = 0; k < QK; ++k) {
      u32x4 w = *reinterpret_cast<const u32x4*>(row + 16 * k + 8 * half);
      w = (w & sc.keep) ^ sc.flip;
      q[k] = __builtin_bit_cast(x8, w);
    }
  }

  typedef f32x16 Scores[ST];

  // A tile's scores, from its keys at LDS address k (rows of kRow bytes,
  // kRow-aligned).
  __device__ __forceinline__ void scores(uint32_t k, Scores& s) {
#pragma unroll
    for (int t = 0; t < ST; ++t) s[t] = f32x16{};
#pragma unroll
    for (int j = 0; j < QK; ++j)
#pragma unroll
      for (int t = 0; t < ST; ++t) s[t] = T::mfma(key(key_address(k), j, t), q[j], s[t]);
    high = peak(s);
  }

  // Leaves the lane's visible keys, the bits of vis.
  __device__ __forceinline__ void mask(Scores& s, uint64_t vis) {
    const uint64_t mine = vis >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = __uint_as_float(select(__float_as_uint(s[t][r]), 0xff800000u, (uint32_t)(mine >> (32 * t)), acc_row(r, 0)));
    high = peak(s);
  }

  // Moves the reference of the rows whose scores (high: their maximum so far)
  // exceed it by too much.
  __device__ __forceinline__ void settle(float c) {
    constexpr float kMost = T::kBase + T::kSlack;
    if (!__any(high * c > top + kMost)) return;
    // row by row: what a row gets does not depend on the others of the wave
    const float new_top = fmaxf(high, __shfl_xor(high, 32)) * c;
    const bool move = new_top - top > kMost;
    const float next = move ? new_top - T::kBase : top, by = move ? __builtin_amdgcn_exp2f(top - next) : 1.f;
    top = next;
    sum *= by;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      // With 256 columns the accumulators do not fit beside the rest into the
      // registers that vector instructions read, and outside of this branch
      // only the matrix unit needs them: they come into the branch and leave
      // it in the matrix unit's registers.  Else the compiler moves them over
      // and back for every tile.
      if constexpr (D == 256) asm volatile("" : "+a"(o[t]));
      o[t] *= by;
      if constexpr (D == 256) asm volatile("" : "+a"(o[t]));
    }
  }

  // The rest of a tile whose scores are s, with its values at v: the weights
  // and the second product.  With NEXT also the next tile's scores, from its
  // keys at k: the matrix unit forms them while the weights are taken.  The
  // order is pinned product by product, each with the fragment read ahead by
  // kReach products and its share of the weights: left to itself the compiler
  // reads a fragment right in front of its product and waits for the LDS
  // (reaching 6 or 8 ahead changes nothing).  Waves in the first product go
  // first: the other's second product needs little issue beside it (prompt of
  // 8192: 502 us, 513 without, 545 the other way round).
  static constexpr int kReach = 4;

  // Between the products run the four parts of `copy`, which send for tiles
  // to come: in front of the products each would be waited for.
  template <bool NEXT, class Copy>
  __device__ __forceinline__ void step(uint32_t k, uint32_t v, float c, Scores& s, Copy copy) {
    settle(c);
    const float sub = top == -INFINITY ? 0.f : top;
    const uint32_t ka = key_address(k), va = value_address(v);
    x8 p[PK], ring[kReach];
    float part[2] = {0, 0};
    // weight pair i of the tile: scores 2 i and 2 i + 1 of the lane, rounded
    // to the inputs' type, half a step each, for the second product
    f32x8 e;
    auto weigh = [&](int i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int x = 2 * i + y;
        e[x % 8] = __builtin_amdgcn_exp2f(fmaf(s[x / 16][x % 16], c, -sub));
        part[y] += e[x % 8];
        asm volatile("" : "+v"(part[y]));  // here, not when the tile is done with every weight kept until then
      }
      if (i % 4 == 3) p[i / 4] = __builtin_convertvector(e, x8);
    };
    constexpr int kFirst = NEXT ? ST * QK : 0, kSecond = PK * DT, kPairs = 8 * ST;
    auto fragment = [&](int m) {  // of product m of both lists
      return m < kFirst ? key(ka, m % QK, m / QK) : value(va, (m - kFirst) / DT, (m - kFirst) % DT);
    };
    Scores n;
#pragma unroll
    for (int t = 0; t < ST; ++t) n[t] = f32x16{};
#pragma unroll
    for (int m = 0; m < kReach; ++m) ring[m] = fragment(m);
    if constexpr (!NEXT) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) weigh(i);
    }
    __builtin_amdgcn_sched_barrier(0);
    auto products = [&](auto from, auto to) {
#pragma unroll
      for (int m = from; m < to; ++m) {
        if (NEXT && m == kFirst) __builtin_amdgcn_s_setprio(0);
        const x8 f = ring[m % kReach];
        if (m < kFirst)
          n[m / QK] = T::mfma(f, q[m % QK], n[m / QK]);
        else
          o[(m - kFirst) % DT] = T::mfma(f, p[(m - kFirst) / DT], o[(m - kFirst) % DT]);
        if (m + kReach < kFirst + kSecond) ring[m % kReach] = fragment(m + kReach);
        if (m < kFirst) {
#pragma unroll
          for (int i = m * kPairs / (ST * QK); i < (m + 1) * kPairs / (ST * QK); ++i) weigh(i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    constexpr int kPart = (NEXT ? kFirst : kSecond) / 4;
    products(At<0>(), At<kPart>());
    copy(0);
    products(At<kPart>(), At<2 * kPart>());
    copy(1);
    products(At<2 * kPart>(), At<3 * kPart>());
    copy(2);
    products(At<3 * kPart>(), At<4 * kPart>());
    copy(3);
    products(At<4 * kPart>(), At<kFirst + kSecond>());
    if (NEXT) __builtin_amdgcn_s_setprio(1);
    sum += part[0] + part[1];
    if constexpr (NEXT) {
#pragma unroll
      for (int t = 0; t < ST; ++t) s[t] = n[t];
      high = peak(s);
    }
  }

  static __device__ __forceinline__ float peak(const Scores& s) {
    float m = s[0][0];
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = __builtin_elementwise_maximum(m, s[t][r]);
    return m;
  }
  static __device__ __forceinline__ uint32_t key_address(uint32_t k) {
    const int lane = threadIdx.x & 63, row = lane & 31;
    return k + row * kRow + (((lane >> 5) ^ key_swizzle<D>(row)) << 4);
  }
  // K fragment (16 columns j, 32 keys t)
  static __device__ __forceinline__ x8 key(uint32_t ka, int j, int t) {
    return *(const DFT_LDS x8*)(uintptr_t)((ka ^ (j << 5)) + t * 32 * kRow);
  }
  __device__ __forceinline__ static uint32_t value_address(uint32_t v) {
    const int lane = threadIdx.x & 63, r4 = (lane & 15) >> 2;
    return v + (4 * (lane >> 5) + r4) * kRow +
           (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle<D>(r4)) << 4) + ((lane & 1) << 3);
  }

  // V^T fragment (16 keys j, 32 columns t) in the key order of the weights
  __device__ __forceinline__ x8 value(uint32_t va, int j, int t) {
    const uint32_t at = (va ^ (t << 6)) + j * 16 * kRow;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DFT_LDS s16x4*)(uintptr_t)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DFT_LDS s16x4*)(uintptr_t)(at + 8 * kRow));
    return __builtin_bit_cast(x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // Which of the lane's outputs see a value of this tile that is an infinity
  // or a NaN (which counts as both), by products of 0 / 1 matrices.  Kept in
  // the wave's `notes`, for finish(); the tile's values are then cleared of
  // them.  Rare, so written to need few registers.
  __device__ __forceinline__ void note(uint32_t v, uint64_t vis) {
    const int lane = threadIdx.x & 63;
    DFT_LDS uint32_t* note = (DFT_LDS uint32_t*)(uintptr_t)(notes + 4 * lane);
    if (!noted)
      for (int t = 0; t < DT; ++t) note[64 * t] = 0;
    noted = true;
    const uint32_t va = value_address(v);
    uint64_t mine = vis >> (4 * (lane >> 5));
#pragma unroll 1
    for (int j = 0; j < PK; ++j, mine >>= 16) {
      u32x4 seen;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t bits = (uint32_t)mine >> (8 * (x / 2) + 2 * (x % 2));
        seen[x] = (bits & 1) * T::kOne + (bits >> 1 & 1) * (T::kOne << 16);
      }
#pragma unroll 1
      for (int t = 0; t < DT; ++t) {
        const u32x4 w = __builtin_bit_cast(u32x4, value(va, j, t));
        uint32_t word = 0;
#pragma unroll 1
        for (int sign = 0; sign < 2; ++sign) {  // +inf and NaN, -inf and NaN
          u32x4 flag;
#pragma unroll
          for (int x = 0; x < 4; ++x) flag[x] = infinite<T>(w[x], sign) + (infinite<T>(w[x] >> 16, sign) << 16);
          const f32x16 n = T::mfma(__builtin_bit_cast(x8, flag), __builtin_bit_cast(x8, seen), f32x16{});
#pragma unroll
          for (int r = 0; r < 16; ++r) word |= min(__float_as_uint(n[r]), 1u) << (r + 16 * sign);  // counts
        }
        note[64 * t] |= word;
      }
    }
  }

  // The noted infinities go into the accumulators.
  __device__ __forceinline__ void finish() {
    if (!noted) return;
    const DFT_LDS uint32_t* note = (const DFT_LDS uint32_t*)(uintptr_t)(notes + 4 * (threadIdx.x & 63));
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const uint32_t word = note[64 * t];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[t][r] += __uint_as_float(select(0x7f800000u, 0, word, r));
        o[t][r] += __uint_as_float(select(0xff800000u, 0, word, r + 16));
      }
    }
  }

  __device__ __forceinline__ f32x4 four(int t, int x) const {
    return {o[t][4 * x], o[t][4 * x + 1], o[t][4 * x + 2], o[t][4 * x + 3]};
  }
  // The lane's outputs, scaled, to the row at element `at`
  __device__ __forceinline__ void store(void* out, int64_t at, int dtype, bool vec, float by) const {
    store_all<4 * DT>(out, at + 4 * ((threadIdx.x & 63) >> 5), dtype, vec, [&](int i) { return four(i / 4, i % 4) * by; },
                      [](int i) { return 32 * (i / 4) + 8 * (i % 4); });
  }

  // The whole row's sum, in both of its lanes.
  __device__ __forceinline__ float whole_sum() const { return sum + __shfl_xor(sum, 32); }
};

// An unseen value has weight 0, which keeps a finite one out of a row's sum but
// no other.  Where some row of the workgroup does not see some key of a tile,
// these look at a wave's share of the tile's values (BYTES of them), and
// clear what is not finite.
template <class T, int BYTES>
__device__ __forceinline__ bool finite(uint32_t share) {
  bool bad = false;
#pragma unroll 4
  for (int i = 0; i < BYTES / 1024; ++i) {
    const u32x4 w = *(const DFT_LDS u32x4*)(uintptr_t)(share + 1024 * i + 16 * (threadIdx.x & 63));
#pragma unroll
    for (int x = 0; x < 4; ++x) bad |= (w[x] & T::kExp) == T::kExp || (w[x] >> 16 & T::kExp) == T::kExp;
  }
  return !__any(bad);
}
template <class T, int BYTES>
__device__ __forceinline__ void clear_infinite(uint32_t share) {
#pragma unroll 1
  for (int i = 0; i < BYTES / 1024; ++i) {
    DFT_LDS u32x4* at = (DFT_LDS u32x4*)(uintptr_t)(share + 1024 * i + 16 * (threadIdx.x & 63));
    u32x4 w = *at;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if ((w[x] & T::kExp) == T::kExp) w[x] &= 0xffff0000u;
      if ((w[x] >> 16 & T::kExp) == T::kExp) w[x] &= 0xffffu;
    }
    *at = w;
  }
}

// 1 / sum, 0 where a row saw no key, NaN kept
__device__ __forceinline__ float weight_of(float sum) { return sum > 0 ? 1.f / sum : sum == 0 ? 0.f : sum; }
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0 ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

// Whether store_all may write whole pieces: 8 bytes, 16 of fp32.
template <class Args>
bool vector_out(const Args& a) {
  const uintptr_t piece = a.o_dtype == DFT_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(a.o) % piece == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
}

}  // namespace attend
}  // namespace dft
