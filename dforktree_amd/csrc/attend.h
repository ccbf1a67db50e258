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
// The running maximum is only moved when a row's score exceeds it by 2^8: the
// weights then stay below 2^8 times the number of keys, which fp32 sums and
// bf16 / fp16 weights hold as well as weights up to 1, and the accumulators
// are rescaled in a few tiles instead of in most.
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
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kTile = 64;          // keys per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;      // log2 units a row's score may exceed its reference by
constexpr int kWaitDma = 0x0f70;   // s_waitcnt vmcnt(0)

#define DFT_LDS __attribute__((address_space(3)))

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const DFT_LDS void*)p;
}

// global -> LDS, 16 bytes a lane to lds + 16 * lane, from base + off bytes.
// Issued from inline assembly, which the backend's wait analysis does not see:
// it would wait for the copy ahead of the next LDS read of any tile.  The
// caller waits for vmcnt before the tile is read.  m0 is reserved to the
// backend: its value is kept, with the wait state that a write of m0 needs.
__device__ __forceinline__ void dma16(uint64_t base, uint32_t off, uint32_t lds) {
  uint32_t keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0"
      : "=&s"(keep)
      : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds))
      : "memory");
}
// the same from an address of each lane's own; once: of data read once, which
// then does not displace what the caches hold
template <bool ONCE>
__device__ __forceinline__ void dma16_at(uint64_t at, uint32_t lds) {
  uint32_t keep;
  if constexpr (ONCE)
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off nt\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(at), "s"(__builtin_amdgcn_readfirstlane(lds))
        : "memory");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0"
        : "=&s"(keep)
        : "v"(at), "s"(__builtin_amdgcn_readfirstlane(lds))
        : "memory");
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

  // One tile: keys and values at the LDS addresses k and v (rows of kRow
  // bytes, kRow-aligned).  With `partial`, vis holds the lane's visible keys.
  __device__ __forceinline__ void tile(uint32_t k, uint32_t v, float c, bool partial, uint64_t vis) {
    const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 31;
    const uint32_t ka = k + row * kRow + ((half ^ key_swizzle<D>(row)) << 4);
    f32x16 s[ST];
#pragma unroll
    for (int t = 0; t < ST; ++t) s[t] = f32x16{};
#pragma unroll
    for (int j = 0; j < QK; ++j)
#pragma unroll
      for (int t = 0; t < ST; ++t)
        s[t] = T::mfma(*(const DFT_LDS x8*)(uintptr_t)((ka ^ (j << 5)) + t * 32 * kRow), q[j], s[t]);

    if (partial) {
      const uint64_t mine = vis >> (4 * half);
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[t][r] = __uint_as_float(select(__float_as_uint(s[t][r]), 0xff800000u, (uint32_t)(mine >> (32 * t)), acc_row(r, 0)));
    }

    float high = s[0][0];
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) high = fmaxf(high, s[t][r]);
    if (__any(high * c > top + kSlack)) {
      // row by row: what a row gets does not depend on the others of the wave
      const float new_top = fmaxf(high, __shfl_xor(high, 32)) * c;
      const bool move = new_top > top + kSlack;
      const float next = move ? new_top : top, by = move ? __builtin_amdgcn_exp2f(top - next) : 1.f;
      top = next;
      sum *= by;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] *= by;
    }
    const float sub = top == -INFINITY ? 0.f : top;
    x8 p[PK];
    float part[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < PK; ++j) {
      f32x8 e;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        e[x] = __builtin_amdgcn_exp2f(fmaf(s[j / 2][8 * (j % 2) + x], c, -sub));
        part[x & 1] += e[x];
      }
      // the weights are rounded to the inputs' type, half a step each, for the second product
      p[j] = __builtin_convertvector(e, x8);
    }
    sum += part[0] + part[1];

    const uint32_t va = value_address(v);
#pragma unroll
    for (int j = 0; j < PK; ++j)
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] = T::mfma(value(va, j, t), p[j], o[t]);
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

// Four outputs in a row, x scaled by w.
__device__ __forceinline__ void store4(void* o, int64_t at, int dtype, bool vec, f32x4 x) {
  if (vec && dtype == DFT_BF16) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(o) + at) = __builtin_bit_cast(u32x2, __builtin_convertvector(x, bf16x4));
  } else if (vec && dtype == DFT_F16) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(o) + at) = __builtin_bit_cast(u32x2, __builtin_convertvector(x, f16x4));
  } else if (vec) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(o) + at) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (dtype == DFT_BF16)
        static_cast<__bf16*>(o)[at + e] = (__bf16)x[e];
      else
        st_f(o, at + e, dtype, x[e]);
  }
}

// Whether store4 may write whole pieces: 8 bytes, 16 of fp32.
template <class Args>
bool vector_out(const Args& a) {
  const uintptr_t piece = a.o_dtype == DFT_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(a.o) % piece == 0 && a.o_row_stride % 4 == 0 && a.o_h_stride % 4 == 0;
}

}  // namespace attend
}  // namespace dft
