// How the kernels over packed requests find their rows.
#pragma once

#include "dft_device.h"

namespace dft {
namespace packed {

// A request's rows: r0 .. r0 + n - 1.
struct Span {
  int64_t r0;
  int n, status;
};
__device__ __forceinline__ Span span_of(const int32_t* cu_seqlens, int64_t rows, int limit, int b) {
  Span s;
  s.r0 = cu_seqlens ? cu_seqlens[b] : (int64_t)b * limit;
  const int64_t n = cu_seqlens ? (int64_t)cu_seqlens[b + 1] - s.r0 : limit;
  s.status = n < 0 || n > limit || s.r0 < 0 || s.r0 + n > rows ? DFT_STATUS_SPAN : 0;
  const int64_t there = s.r0 < 0 ? 0 : max(rows - s.r0, (int64_t)0);
  s.n = (int)min(min(max(n, (int64_t)0), (int64_t)limit), there);
  return s;
}
template <class Args>
__device__ __forceinline__ Span span_of(const Args& a, int b) {
  return span_of(a.cu_seqlens, a.rows, a.max_len, b);
}

// A request's tiles of R rows have the numbers first_tile .. in a line that has
// room for rows / R + batch of them: ceil(n / R) rows' worth fits in front of
// the next request's first one, since floor((s + n) / R) + 1 >= floor(s / R) +
// ceil(n / R).  So a tile's place needs no sum over the requests before it.
__device__ __forceinline__ int64_t first_tile(int64_t r0, int b, int R) { return r0 / R + b; }
inline int64_t line_tiles(int64_t rows, int batch, int R) { return rows / R + batch; }

// The request whose tile `x` of the line is, looked for by all NT threads of
// the workgroup; -1: none's.
template <int NT, class Args>
__device__ __forceinline__ int find_tile(const Args& a, int64_t x, int R) {
  __shared__ int at;
  if (threadIdx.x == 0) at = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += NT) {
    const Span s = span_of(a, b);
    if (s.n <= 0) continue;
    const int64_t first = first_tile(s.r0, b, R);
    if (x >= first && x < first + (s.n + R - 1) / R) at = b;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(at);
}

// A request's slot: -1 where it is none of the pool's; `initial`: whether the
// request goes on from what it holds.
struct Slot {
  int64_t at;
  bool initial;
  int status;
};
__device__ __forceinline__ Slot slot_of(const void* indices, int dtype, const uint8_t* initial, int64_t slots, int b) {
  Slot s;
  s.at = indices ? ld_i(indices, b, dtype) : b;
  s.status = s.at >= slots ? DFT_STATUS_SLOT : 0;
  if (s.at >= slots || s.at < 0) s.at = -1;
  s.initial = s.at >= 0 && (!initial || initial[b]);
  return s;
}

// Stores whose conversions keep NaN (st_f takes finite values).
__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ void store(void* p, int64_t i, int dt, float v) {
  switch (dt) {
    case DFT_BF16: ((uint16_t*)p)[i] = bf16_bits(v); break;
    case DFT_F16: ((_Float16*)p)[i] = (_Float16)v; break;
    default: ((float*)p)[i] = v; break;
  }
}

}  // namespace packed
}  // namespace dft
